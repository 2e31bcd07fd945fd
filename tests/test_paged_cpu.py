"""CPU: what the operators on a paged cache and the rotary positions refuse before any CUDA work, their parameter
structs, their fake kernels, and the frequencies."""
import ctypes
import math
import os
import re

import pytest
import torch

from splitd_flash_attn import _capi

D = 512
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize(
    "name,cls",
    [("splitd_paged_params", "SplitdPagedParams"), ("splitd_rotary_params", "SplitdRotaryParams"),
     ("splitd_append_params", "SplitdAppendParams"), ("splitd_evict_params", "SplitdEvictParams")],
)
def test_param_structs_match_the_header(name, cls):
    text = open(os.path.join(ROOT, "include", "splitd_attn.h")).read()
    end = text.index("} %s;" % name)
    body = re.sub(r"/\*.*?\*/", "", text[text.rindex("typedef struct {", 0, end) + 16 : end], flags=re.S)
    kinds = {"void": ctypes.c_void_p, "int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float, "size_t": ctypes.c_size_t}
    want = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        words = decl.replace("const ", "").split(None, 1)
        for part in words[1].split(","):
            m = re.match(r"\s*(\*?)\s*([a-z_0-9]+)\s*(?:\[(\d+)\])?$", part)
            star = m.group(1) or words[0].endswith("*")
            t = ctypes.c_void_p if star else kinds[words[0]]
            want.append((m.group(2), t * int(m.group(3)) if m.group(3) else t))
    got = getattr(_capi, cls)._fields_
    assert [g[0] for g in got] == [w[0] for w in want]
    for g, w in zip(got, want):
        assert ctypes.sizeof(g[1]) == ctypes.sizeof(w[1]) and getattr(g[1], "_type_", None) == getattr(w[1], "_type_", None), g[0]


def _paged():
    p = _capi.SplitdPagedParams()
    for n in ("q", "k_pages", "v_pages", "o", "page_table", "seqlens_k", "workspace"):
        setattr(p, n, 1 << 20)
    p.batch, p.seqlen_q, p.heads_q, p.heads_kv, p.head_dim = 2, 1, 8, 2, D
    p.num_pages, p.page_size, p.max_pages = 10, 16, 4
    p.softmax_scale, p.workspace_bytes = 0.1, 1 << 40
    for n in ("q_strides", "o_strides", "k_strides", "v_strides"):
        setattr(p, n, (4096, 512, 512))
    return p


def _refused(fn, p, text, code=-1):
    assert fn(ctypes.byref(p), None) == code
    msg = _capi.load_library().splitd_last_error().decode()
    assert text in msg, msg


def test_attention_entry_point_refuses():
    lib = _capi.load_library()
    fn = lib.splitd_paged_attn
    assert fn(None, None) == -1
    assert lib.splitd_paged_attn_workspace_bytes(None) == 0
    for field, value, text in (
        ("q", None, "NULL"), ("seqlens_k", None, "NULL"), ("head_dim", 256, "head_dim == 512"), ("heads_q", 7, "heads_q"),
        ("heads_kv", 0, "heads_q"), ("dtype", 2, "dtype"), ("batch", 0, "batch"), ("batch", 65536, "batch"), ("page_size", 0, "page_size"),
        ("num_pages", -1, "num_pages"), ("max_pages", -1, "max_pages"), ("seqlen_q", 0, "seqlen_q"), ("seqlen_q", 1 << 22, "2^24"),
        ("softmax_scale", 0.0, "softmax_scale"), ("softmax_scale", float("nan"), "softmax_scale"), ("softcap", -1.0, "softcap"),
        ("softcap", float("nan"), "softcap"), ("q", (1 << 20) + 8, "16-byte"), ("k_strides", (4096, 515, 512), "multiple of 8"),
        ("key_weights", 1 << 20, "key_weights_len"),
    ):
        p = _paged()
        setattr(p, field, value)
        _refused(fn, p, text)
    p = _paged()
    p.local, p.window_left = 1, -2
    _refused(fn, p, "window_left")
    p.window_left, p.causal = 4, 1
    _refused(fn, p, "exclusive")
    p = _paged()
    need = lib.splitd_paged_attn_workspace_bytes(ctypes.byref(p))
    assert need > 0
    p.workspace_bytes = need - 1
    _refused(fn, p, "workspace", -5)
    p.workspace_bytes, p.workspace = need, (1 << 20) + 16
    _refused(fn, p, "workspace", -5)


def test_rotary_entry_point_refuses():
    fn = _capi.load_library().splitd_rotary
    assert fn(None, None) == -1

    def make():
        p = _capi.SplitdRotaryParams()
        for n in ("q", "k", "q_out", "k_out", "positions", "inv_freq"):
            setattr(p, n, 1 << 20)
        p.batch, p.seqlen, p.heads_q, p.heads_kv, p.head_dim, p.rotary_dim = 1, 4, 8, 3, D, 512
        return p

    for field, value, text in (
        ("q_out", None, "output"), ("positions", None, "positions"), ("inv_freq", None, "inv_freq"), ("rotary_dim", 514, "rotary_dim"),
        ("rotary_dim", 5, "rotary_dim"), ("rotary_dim", -2, "rotary_dim"), ("head_dim", 128, "head_dim == 512"), ("seqlen", 0, "seqlen"),
        ("heads_kv", 0, "heads"), ("dtype", 7, "dtype"), ("k_out", (1 << 20) + 2, "16-byte"), ("q_strides", (0, 12, 512), "multiple of 8"),
    ):
        p = make()
        setattr(p, field, value)
        _refused(fn, p, text)
    p = make()
    p.q = p.k = None
    _refused(fn, p, "both")


def test_append_entry_point_refuses():
    fn = _capi.load_library().splitd_paged_append
    assert fn(None, None) == -1

    def make():
        p = _capi.SplitdAppendParams()
        for n in ("q", "k", "v", "q_out", "k_pages", "v_pages", "page_table", "seqlens_k", "inv_freq"):
            setattr(p, n, 1 << 20)
        p.batch, p.seqlen, p.heads_q, p.heads_kv, p.head_dim, p.rotary_dim = 2, 4, 8, 2, D, 512
        p.num_pages, p.page_size, p.max_pages = 10, 16, 4
        return p

    for field, value, text in (
        ("k", None, "NULL"), ("q_out", None, "q_out"), ("heads_q", 5, "heads_q"), ("batch", 0, "batch"), ("seqlen", 0, "new token"),
        ("rotary_dim", 3, "rotary_dim"), ("page_size", -4, "page_size"), ("v_pages", (1 << 20) + 8, "16-byte"),
        ("v_page_strides", (8, 8, 4), "multiple of 8"), ("cu_seqlens", 1 << 20, "new token"),
    ):
        p = make()
        setattr(p, field, value)
        _refused(fn, p, text)


def test_evict_entry_point_refuses():
    fn = _capi.load_library().splitd_paged_evict
    assert fn(None, None) == -1

    def make():
        p = _capi.SplitdEvictParams()
        for n in ("k_pages", "v_pages", "page_table", "new_page_table", "seqlens_k", "key_weights", "new_seqlens", "kept", "new_weights"):
            setattr(p, n, 1 << 20)
        p.batch, p.heads_kv, p.head_dim, p.num_pages, p.page_size, p.max_pages, p.new_max_pages = 2, 2, D, 10, 16, 4, 2
        p.key_weights_len, p.keep = 64, 32
        return p

    for field, value, text in (
        ("kept", None, "NULL"), ("keep", 0, "keep"), ("keep", (1 << 30) + 1, "2^30"), ("keep", 33, "do not hold"), ("keep_first", -1, "keep"), ("keep_recent", 33, "keep"),
        ("new_max_pages", -1, "do not hold"), ("key_weights_len", -1, "key_weights_len"), ("batch", 70000, "batch"),
        ("k_strides", (1, 8, 8), "multiple of 8"),
    ):
        p = make()
        setattr(p, field, value)
        _refused(fn, p, text)


# ---------------------------------------------------------------------------
# Python checks: under FakeTensorMode nothing has memory, so what is not refused ends in a fake kernel
# ---------------------------------------------------------------------------


@pytest.fixture
def fake():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        yield


def _cache(dtype=torch.bfloat16, hkv=2, page=16, pages=10, B=3, width=4):
    k = torch.empty(pages, page, hkv, D, dtype=dtype, device="cuda")
    v = torch.empty(pages, page, hkv, D, dtype=dtype, device="cuda")
    return k, v, torch.empty(B, width, dtype=torch.int32, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")


def test_attention_function_checks(fake):
    from splitd_flash_attn import split_flash_attn_paged_func as fn

    k, v, t, n = _cache()
    q = torch.empty(3, 2, 8, D, dtype=torch.bfloat16, device="cuda")
    w = torch.empty(3, 64, device="cuda")
    out, lse = fn(q, k, v, t, n, causal=True, key_weights=w, return_lse=True)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (3, 8, 2) and lse.dtype == torch.float32
    assert fn(q, k, v, t, n).shape == q.shape
    with pytest.raises(ValueError, match="rank 4"):
        fn(q[0], k, v, t, n)
    with pytest.raises(ValueError, match="head_dim"):
        fn(q[..., :256], k, v, t, n)
    with pytest.raises(TypeError):
        fn(q.half(), k, v, t, n)
    with pytest.raises(TypeError):
        fn(q.float(), k.float(), v.float(), t, n)
    with pytest.raises(ValueError, match="divisible"):
        fn(q[:, :, :7], k, v, t, n)
    with pytest.raises(ValueError, match="v_pages"):
        fn(q, k, v[:5], t, n)
    with pytest.raises(ValueError, match="page_table"):
        fn(q, k, v, t[:2], n)
    with pytest.raises(ValueError, match="seqlens_k"):
        fn(q, k, v, t[:2], n[:2])
    with pytest.raises(TypeError, match="page_table"):
        fn(q, k, v, t.long(), n)
    with pytest.raises(TypeError, match="seqlens_k"):
        fn(q, k, v, t, n.long())
    with pytest.raises(RuntimeError, match="CUDA"):
        fn(q.cpu(), k, v, t, n)
    with pytest.raises(RuntimeError, match="seqlens_k"):
        fn(q, k, v, t, n.cpu())
    with pytest.raises(ValueError, match="stride"):
        fn(q, k.transpose(2, 3).contiguous().transpose(2, 3), v, t, n)
    with pytest.raises(ValueError, match="stride"):
        fn(q, torch.empty(10, 16, 2, D + 4, dtype=torch.bfloat16, device="cuda")[..., :D], v, t, n)
    with pytest.raises(ValueError, match="page_size"):
        fn(q, k[:, :0], v[:, :0], t, n)
    with pytest.raises(ValueError, match="key_weights"):
        fn(q, k, v, t, n, key_weights=w[:2])
    with pytest.raises(TypeError, match="key_weights"):
        fn(q, k, v, t, n, key_weights=w.double())
    with pytest.raises(ValueError, match="key_weights"):
        fn(q, k, v, t, n, key_weights=torch.empty(64, 3, device="cuda").T)
    with pytest.raises(ValueError, match="overlap"):
        fn(q, k, v, t, n, key_weights=w[:1].expand(3, -1))
    with pytest.raises(TypeError, match="tuple"):
        fn(q, k, v, t, n, window_size=[1, 2])
    with pytest.raises(NotImplementedError, match="backward"):
        fn(q.requires_grad_(), k, v, t, n)
    with torch.no_grad():
        fn(q, k, v, t, n)


def test_append_function_checks(fake):
    from splitd_flash_attn import split_paged_append_func as fn

    k_pages, v_pages, t, n = _cache()
    q = torch.empty(3, 2, 8, D, dtype=torch.bfloat16, device="cuda")
    k = torch.empty(3, 2, 2, D, dtype=torch.bfloat16, device="cuda")
    f = torch.empty(256, dtype=torch.float64, device="cuda")
    cu = torch.empty(4, dtype=torch.int32, device="cuda")
    pos = torch.empty(3, 2, dtype=torch.int64, device="cuda")
    assert fn(q, k, k, k_pages, v_pages, t, n, inv_freq=f, positions=pos).shape == q.shape
    assert fn(None, k, k, k_pages, v_pages, t, n) is None
    assert fn(q.flatten(0, 1), k.flatten(0, 1), k.flatten(0, 1), k_pages, v_pages, t, n, cu_seqlens_q=cu).shape == (6, 8, D)
    with pytest.raises(ValueError, match="rank 3"):
        fn(q, k, k, k_pages, v_pages, t, n, cu_seqlens_q=cu)
    with pytest.raises(ValueError, match="cu_seqlens_q"):
        fn(None, k.flatten(0, 1), k.flatten(0, 1), k_pages, v_pages, t, n, cu_seqlens_q=cu[:3])
    with pytest.raises(TypeError, match="cu_seqlens_q"):
        fn(None, k.flatten(0, 1), k.flatten(0, 1), k_pages, v_pages, t, n, cu_seqlens_q=cu.long())
    with pytest.raises(ValueError, match="tokens of k"):
        fn(q[:, :1], k, k, k_pages, v_pages, t, n)
    with pytest.raises(ValueError, match="heads"):
        fn(q, q, q, k_pages, v_pages, t, n)
    with pytest.raises(ValueError, match="divisible"):
        fn(q[:, :, :3], k, k, k_pages, v_pages, t, n)
    with pytest.raises(ValueError, match="v has shape"):
        fn(q, k, k[:, :1], k_pages, v_pages, t, n)
    with pytest.raises(ValueError, match="names 2 sequences"):
        fn(q, k, k, k_pages, v_pages, t[:2], n[:2])
    with pytest.raises(TypeError, match="inv_freq"):
        fn(q, k, k, k_pages, v_pages, t, n, inv_freq=f.float())
    with pytest.raises(ValueError, match="inv_freq"):
        fn(q, k, k, k_pages, v_pages, t, n, inv_freq=torch.empty(257, dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError, match="without inv_freq"):
        fn(q, k, k, k_pages, v_pages, t, n, positions=pos)
    with pytest.raises(ValueError, match="positions"):
        fn(q, k, k, k_pages, v_pages, t, n, inv_freq=f, positions=pos[:2])
    with pytest.raises(TypeError, match="k_pages"):
        fn(q, k, k, k_pages.half(), v_pages.half(), t, n)
    with pytest.raises(ValueError, match="expanded"):
        fn(q, k, k, k_pages, v_pages[:1].expand(10, -1, -1, -1), t, n)
    with pytest.raises(NotImplementedError, match="backward"):
        fn(q, k.requires_grad_(), k, k_pages, v_pages, t, n)


def test_evict_function_checks(fake):
    from splitd_flash_attn import split_paged_evict_func as fn

    k, v, t, n = _cache()
    w = torch.empty(3, 64, device="cuda")
    new = torch.empty(3, 2, dtype=torch.int32, device="cuda")
    a, b, c = fn(k, v, t, n, w, new, 32, 2, 3)
    assert a.shape == (3,) and a.dtype == torch.int32 and b.shape == (3, 32) and b.dtype == torch.int32 and c.dtype == torch.float32
    for keep, first, recent in ((0, 0, 0), (5, 3, 3), (-1, 0, 0), (5, -1, 0), (33, 0, 0)):
        with pytest.raises(ValueError):
            fn(k, v, t, n, w, new, keep, first, recent)
    with pytest.raises(TypeError, match="keep"):
        fn(k, v, t, n, w, new, 4.0)
    with pytest.raises(TypeError, match="keep_first"):
        fn(k, v, t, n, w, new, 4, True)
    with pytest.raises(ValueError, match="new_page_table"):
        fn(k, v, t, n, w, new[:2], 4)
    with pytest.raises(TypeError, match="new_page_table"):
        fn(k, v, t, n, w, new.long(), 4)
    with pytest.raises(ValueError, match="key_weights"):
        fn(k, v, t, n, w[0], new, 4)
    with pytest.raises(ValueError, match=r"2\^30"):
        fn(k, v, t, n, w, new, 2**30 + 1)
    with pytest.raises(ValueError, match="expanded"):
        fn(k[:1].expand(10, -1, -1, -1), v, t, n, w, new, 4)


def test_rotary_function_checks(fake):
    from splitd_flash_attn import split_rotary_func as fn

    q = torch.empty(3, 5, 8, D, dtype=torch.float16, device="cuda", requires_grad=True)
    k = torch.empty(3, 5, 3, D, dtype=torch.float16, device="cuda")
    f = torch.empty(100, dtype=torch.float64, device="cuda")
    pos = torch.empty(3, 5, dtype=torch.int32, device="cuda")
    qo, ko = fn(q, k, pos, f)
    assert qo.shape == q.shape and ko.shape == k.shape and qo.dtype == q.dtype and qo.requires_grad
    assert fn(None, k, pos[0], f, interleaved=True)[0] is None
    assert fn(q[0], None, pos[0], f)[0].shape == q[0].shape
    gq, gk = torch.ops.splitd_flash_attn.rotary(q.detach(), None, pos, f, False, 1.0, True)
    assert gq.shape == q.shape and gk.shape == (0,)
    for bad in (
        lambda: fn(None, None, pos, f), lambda: fn(q[0, 0], None, pos, f), lambda: fn(q, k[:2], pos, f), lambda: fn(q, k, pos[:, :4], f),
        lambda: fn(q[..., :128], None, pos, f), lambda: fn(q, k, pos, torch.empty(300, dtype=torch.float64, device="cuda")),
        lambda: fn(q, k, pos, f[None]), lambda: fn(q, k.flatten(0, 1), pos, f), lambda: fn(q.flatten(0, 1), None, pos, f),
    ):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: fn(q, k.bfloat16(), pos, f), lambda: fn(q.float(), None, pos, f), lambda: fn(q, k, pos.float(), f), lambda: fn(q, k, pos, f.float())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: fn(q.cpu(), None, pos, f), lambda: fn(q, k, pos.cpu(), f), lambda: fn(q, k, pos, f.cpu())):
        with pytest.raises(RuntimeError):
            bad()


def test_frequencies():
    from splitd_flash_attn import split_rotary_frequencies as fn

    f, factor = fn(64, 1e6, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and factor == 1.0
    for i in (0, 1, 31):
        assert math.isclose(float(f[i]), 1e6 ** (-2 * i / 64), rel_tol=1e-13)
    lin, _ = fn(64, 1e6, 8.0, device="cpu")
    assert torch.allclose(lin * 8, f, rtol=1e-15, atol=0)
    base, factor = fn(64, 1e6, 8.0, "base", device="cpu")
    assert factor == 1.0 and base[0] == 1.0 and math.isclose(float(f[-1] / base[-1]), 8.0, rel_tol=1e-12)
    ramp, factor = fn(64, 1e6, 8.0, "ramp", original_length=8192, device="cpu")
    assert math.isclose(factor, 1 + 0.1 * math.log(8.0))
    turns = 8192 * f / (2 * math.pi)
    assert torch.equal(ramp[turns > 32], f[turns > 32]) and torch.allclose(ramp[turns < 1] * 8, f[turns < 1], rtol=1e-14, atol=0)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (ramp[between] < f[between]).all() and (ramp[between] > f[between] / 8).all()
    for bad in (
        lambda: fn(63, device="cpu"), lambda: fn(0, device="cpu"), lambda: fn(514, device="cpu"), lambda: fn(64, scale=0.5, device="cpu"),
        lambda: fn(64, method="other", device="cpu"), lambda: fn(64, method="ramp", scale=2.0, device="cpu"),
        lambda: fn(2, method="base", scale=2.0, device="cpu"),
        lambda: fn(64, method="ramp", scale=2.0, original_length=10, low_turns=3, high_turns=3, device="cpu"),
    ):
        with pytest.raises(ValueError):
            bad()
