"""CPU: what a later call says of a status that an earlier kernel left."""
import pytest
import torch

from splitd_flash_attn import interface


@pytest.mark.parametrize("code,text", [
    (101, "ended early"), (104, "incomplete"), (106, "max_seqlen_k"), (107, "does not have"), (108, "longer than its row"), (108, "key_weights"),
])
def test_the_message_names_what_happened(monkeypatch, code, text):
    monkeypatch.setattr(interface, "_status_flags", {0: torch.tensor([code], dtype=torch.int32)})
    with pytest.raises(RuntimeError, match=text) as e:
        interface._raise_if_a_kernel_gave_up(torch.device("cuda", 0))
    assert f"status {code}" in str(e.value)
    if code in (107, 108):
        assert "ended early" not in str(e.value)


def test_nothing_is_said_of_status_0(monkeypatch):
    monkeypatch.setattr(interface, "_status_flags", {0: torch.zeros(1, dtype=torch.int32)})
    interface._raise_if_a_kernel_gave_up(torch.device("cuda", 0))
    interface._raise_if_a_kernel_gave_up(torch.device("cuda", 1))
