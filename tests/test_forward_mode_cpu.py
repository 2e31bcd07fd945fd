"""CPU: the dense attention has no forward-mode derivative; a tangent is refused before any CUDA work, not lost."""
import pytest
import torch
from torch.autograd import forward_ad

from splitd_flash_attn import split_flash_attn_func, split_flash_attn_varlen_func

D = 512


@pytest.mark.parametrize("which", range(3))
def test_dense_attention_refuses_tangents(which):
    qkv = [torch.zeros(1, 4, h, D, dtype=torch.bfloat16) for h in (2, 1, 1)]
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with forward_ad.dual_level():
        qkv[which] = forward_ad.make_dual(qkv[which], torch.ones_like(qkv[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            split_flash_attn_func(*qkv)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            split_flash_attn_varlen_func(*(t[0] for t in qkv), cu, cu, 4, 4)


def test_ordinary_tensors_within_a_dual_level_get_as_far_as_ever():
    q = torch.zeros(1, 4, 1, D, dtype=torch.bfloat16)
    with forward_ad.dual_level(), pytest.raises(Exception) as e:
        split_flash_attn_func(q, q, q)
    assert "forward-mode" not in str(e.value)
