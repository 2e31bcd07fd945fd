"""Rotary positions for query and key heads of 512 (no counterpart in the reference: its callers rotate before they
call it). Kernel: ``csrc/rotary_kernel.cu``; C-ABI: ``splitd_rotary``."""

from __future__ import annotations

import ctypes
import itertools
import math
from typing import Optional, Tuple

import torch

from . import _capi
from .interface import SUPPORTED_HEAD_DIM, _dual, _refuse_derivatives, _status_flag

__all__ = ["split_rotary_frequencies", "split_rotary_func"]

_DTYPES = {torch.bfloat16: _capi.SPLITD_DTYPE_BF16, torch.float16: _capi.SPLITD_DTYPE_FP16}


def split_rotary_frequencies(
    rotary_dim: int,
    base: float = 10000.0,
    scale: float = 1.0,
    method: str = "linear",
    original_length: Optional[int] = None,
    low_turns: float = 1.0,
    high_turns: float = 32.0,
    device="cuda",
) -> Tuple[torch.Tensor, float]:
    """Frequencies base^(-2 i / rotary_dim) in 64 bits, stretched for contexts ``scale`` times as long as the model was
    trained on, and the factor that goes with them: ``(inv_freq, factor)`` for ``split_rotary_func`` and
    ``split_paged_append_func``.

    ``method``: ``"linear"`` divides every frequency by ``scale``; ``"base"`` raises the base to base *
    scale^(rotary_dim / (rotary_dim - 2)), so that the lowest frequency is divided by ``scale`` and the highest stays;
    ``"ramp"`` divides those that make less than ``low_turns`` turns within ``original_length`` positions, keeps those
    that make more than ``high_turns``, blends in between, and returns the factor 1 + 0.1 ln(scale) (1 for the others).
    """
    if rotary_dim % 2 != 0 or not 0 < rotary_dim <= SUPPORTED_HEAD_DIM:
        raise ValueError(f"rotary_dim must be even and in 2 .. {SUPPORTED_HEAD_DIM}, got {rotary_dim}")
    if not scale >= 1.0:
        raise ValueError(f"scale must be >= 1, got {scale}")
    if method not in ("linear", "base", "ramp"):
        raise ValueError(f"method must be 'linear', 'base' or 'ramp', got {method!r}")
    if method == "base":
        if rotary_dim == 2:
            raise ValueError("method 'base' needs rotary_dim > 2: its only frequency does not depend on the base")
        base = base * scale ** (rotary_dim / (rotary_dim - 2))
    exponent = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    inv_freq = torch.pow(torch.tensor(float(base), dtype=torch.float64), -exponent)
    factor = 1.0
    if method == "linear":
        inv_freq = inv_freq / scale
    elif method == "ramp":
        if original_length is None:
            raise ValueError("method 'ramp' needs original_length")
        if not high_turns > low_turns:
            raise ValueError("high_turns must be greater than low_turns")
        turns = original_length * inv_freq / (2 * math.pi)
        stays = ((turns - low_turns) / (high_turns - low_turns)).clamp(0.0, 1.0)
        inv_freq = inv_freq * (stays + (1 - stays) / scale)
        factor = 1.0 + 0.1 * math.log(scale)
    return inv_freq.to(device), factor


# ---------------------------------------------------------------------------
# argument checks
# ---------------------------------------------------------------------------


def _check_heads(t: torch.Tensor, name: str, rank: int) -> None:
    if t.ndim != rank:
        raise ValueError(f"{name} must have rank {rank}, got rank {t.ndim}")
    if t.shape[-1] != SUPPORTED_HEAD_DIM:
        raise ValueError(f"{name} has head_dim {t.shape[-1]}, head_dim == {SUPPORTED_HEAD_DIM} is required")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be torch.float16 or torch.bfloat16, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be on a CUDA device, got {t.device}")


def _check_same(t: torch.Tensor, name: str, dtype, device) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")


def _check_inv_freq(inv_freq: torch.Tensor, device) -> None:
    if inv_freq.ndim != 1 or inv_freq.shape[0] > SUPPORTED_HEAD_DIM // 2:
        raise ValueError(
            f"inv_freq must have shape (rotary_dim / 2,) with rotary_dim <= {SUPPORTED_HEAD_DIM}, got {tuple(inv_freq.shape)}"
        )
    _check_same(inv_freq, "inv_freq", torch.float64, device)


def _check_positions(positions: torch.Tensor, lead, device) -> None:
    """``lead``: leading dimensions of the tokens, (B, S) or (T,). (S,) stands for the same positions in every sequence."""
    if tuple(positions.shape) != tuple(lead) and not (len(lead) == 2 and tuple(positions.shape) == (lead[1],)):
        raise ValueError(f"positions has shape {tuple(positions.shape)}, expected {tuple(lead)}" + (f" or ({lead[1]},)" if len(lead) == 2 else ""))
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if positions.device != device:
        raise RuntimeError(f"positions is on {positions.device}, expected {device}")


def _position_strides(positions: torch.Tensor, packed: bool):
    if packed:
        return (0, positions.stride(0))
    if positions.ndim == 1:
        return (0, positions.stride(0))
    return positions.stride()


def _token_strides(t: torch.Tensor):
    """Strides of (batch, token, head); packed tokens have no batch."""
    s = t.stride()
    return s[:3] if t.ndim == 4 else (0, s[0], s[1])


# Dispatch keys that every thread includes; any other belongs to something that wants to see each operator.
_UNUSUAL_KEYS = ~(
    torch._C.DispatchKeySet(torch._C.DispatchKey.BackendSelect) | torch._C.DispatchKeySet(torch._C.DispatchKey.ADInplaceOrView)
).raw_repr()


def _traced(*tensors) -> bool:
    """Whether the call goes through its custom op: under torch.compile, for tensors without memory and other subclasses, and
    where a tracer, a dispatch mode or a function transform is at work. Otherwise the kernel is called without the
    dispatcher, which costs several times what the kernels of a decode step take."""
    if torch.compiler.is_compiling() or torch._C._dispatch_tls_local_include_set().raw_repr() & _UNUSUAL_KEYS:
        return True
    for t in tensors:
        if t is not None and type(t) is not torch.Tensor:
            return True
    return False


# ---------------------------------------------------------------------------
# plans
# ---------------------------------------------------------------------------
# A decode step's kernels take a few microseconds, less than checking a dozen tensors, filling a parameter struct and
# allocating in Python do. So what a call's shapes, strides, types and options decide is worked out once and kept under
# exactly those: that the arguments are fine, the filled struct (as bytes; each call puts its pointers into a copy) and
# models of the outputs. No pointer to and no value of a caller's tensor is part of it, and no device memory. Of more than
# _PLANS_MOST, the one that was not used for the longest time goes: packed prompts bring a new number of tokens with nearly
# every call, and must not push out the decode steps' plans.

_PLANS_MOST = 1024


class _Plans(dict):
    """[plan, time of its last use] under its key. Two threads that look for a plan at once may both make it."""

    def __init__(self):
        super().__init__()
        self.clock = itertools.count()

    def find(self, key):
        entry = self.get(key)
        if entry is None:
            return None
        entry[1] = next(self.clock)
        return entry[0]

    def keep(self, key, plan):
        if len(self) >= _PLANS_MOST:
            oldest = min(list(self.items()), key=lambda item: item[1][1])
            self.pop(oldest[0], None)
        self[key] = [plan, next(self.clock)]
        return plan


def _meta(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _model(shape, dtype, device) -> torch.Tensor:
    """``empty_like`` of it is a contiguous tensor of that shape and costs half of ``empty``; its one element is the status
    word's memory, which is there anyway."""
    return _status_flag(device).view(dtype)[0].expand(shape)


def _rows_fit(t: Optional[torch.Tensor]) -> bool:
    """Head rows are moved in 16-byte pieces: unit stride, the others multiples of 8 elements; other tensors are copied."""
    return t is None or (t.stride(-1) == 1 and all(s % 8 == 0 for s in t.stride()[:-1]))


def _copied(t: torch.Tensor) -> torch.Tensor:
    return t.detach().clone(memory_format=torch.contiguous_format)


def _launch(fn, params, index: int) -> None:
    """On the current stream of device `index`, whichever device is current."""
    stream = torch._C._cuda_getCurrentRawStream(index)  # current_stream(index).cuda_stream without the object
    if index == torch.cuda.current_device():
        code = fn(ctypes.byref(params), stream)
    else:
        with torch.cuda.device(index):
            code = fn(ctypes.byref(params), stream)
    if code:
        _capi.check(code)


# ---------------------------------------------------------------------------
# the operator
# ---------------------------------------------------------------------------


def _check_rotary(q, k, positions, inv_freq) -> None:
    first, name = (q, "q") if q is not None else (k, "k")
    if first is None:
        raise ValueError("q and k must not both be None")
    if first.ndim not in (3, 4):
        raise ValueError(f"{name} must have rank 4, or 3 (packed tokens), got rank {first.ndim}")
    _check_heads(first, name, first.ndim)
    if q is not None and k is not None:
        _check_heads(k, "k", q.ndim)
        if k.shape[:-2] != q.shape[:-2]:
            raise ValueError(f"k has shape {tuple(k.shape)}, expected the tokens of q, {tuple(q.shape)}")
        _check_same(k, "k", q.dtype, q.device)
    _check_inv_freq(inv_freq, first.device)
    _check_positions(positions, first.shape[:-2], first.device)


class _RotaryPlan:
    def __init__(self, q, k, positions, inv_freq, interleaved, factor, backward):
        _check_rotary(q, k, positions, inv_freq)
        first = q if q is not None else k
        self.index = first.get_device()
        self.fits = _rows_fit(q) and _rows_fit(k) and (inv_freq.numel() < 2 or inv_freq.stride(0) == 1)
        self.q_model = None if q is None else _model(q.shape, q.dtype, q.device)
        self.k_model = None if k is None else _model(k.shape, k.dtype, k.device)
        packed = first.ndim == 3
        batch, seqlen = (1, first.shape[0]) if packed else first.shape[:2]
        heads = [0 if t is None else t.shape[-2] for t in (q, k)]
        self.has_q, self.has_k = (batch * seqlen * h > 0 for h in heads)
        self.has_freq = inv_freq.numel() > 0
        p = _capi.SplitdRotaryParams()
        p.batch, p.seqlen, p.head_dim = batch, seqlen, SUPPORTED_HEAD_DIM
        p.heads_q, p.heads_kv = heads
        p.rotary_dim, p.interleaved, p.backward = 2 * inv_freq.numel(), int(interleaved), int(backward)
        p.positions_64bit, p.dtype, p.factor = int(positions.dtype == torch.int64), _DTYPES[first.dtype], factor
        p.position_strides = _position_strides(positions, packed)
        if q is not None:
            p.q_strides, p.q_out_strides = _token_strides(q), _token_strides(torch.empty_like(self.q_model))
        if k is not None:
            p.k_strides, p.k_out_strides = _token_strides(k), _token_strides(torch.empty_like(self.k_model))
        self.params = bytes(p)


_rotary_plans = _Plans()


def _rotary(q, k, positions, inv_freq, interleaved, factor, backward):
    """One launch for both; None stays None."""
    key = (_meta(q), _meta(k), _meta(positions), _meta(inv_freq), interleaved, factor, backward)
    plan = _rotary_plans.find(key)
    if plan is None:
        plan = _rotary_plans.keep(key, _RotaryPlan(q, k, positions, inv_freq, interleaved, factor, backward))
    q_at = q.data_ptr() if plan.has_q else 0
    k_at = k.data_ptr() if plan.has_k else 0
    if not plan.fits or q_at % 16 or k_at % 16:
        q = None if q is None else _copied(q)
        k = None if k is None else _copied(k)
        return _rotary(q, k, positions, inv_freq.contiguous(), interleaved, factor, backward)
    p = _capi.SplitdRotaryParams.from_buffer_copy(plan.params)
    q_out = k_out = None
    if q is not None:
        q_out = torch.empty_like(plan.q_model)
    if k is not None:
        k_out = torch.empty_like(plan.k_model)
    if plan.has_q:
        p.q, p.q_out = q_at, q_out.data_ptr()
    if plan.has_k:
        p.k, p.k_out = k_at, k_out.data_ptr()
    if plan.has_q or plan.has_k:
        p.positions = positions.data_ptr()
        if plan.has_freq:
            p.inv_freq = inv_freq.data_ptr()
        _launch(_capi.load_library().splitd_rotary, p, plan.index)
    return q_out, k_out


class RotaryFunc(torch.autograd.Function):
    """The map is linear in q and k; its gradient is the same map with the angle's sign turned."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, factor, backward):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = interleaved, factor, backward
        ctx.set_materialize_grads(False)
        return _rotary(q, k, positions, inv_freq, interleaved, factor, backward)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        interleaved, factor, backward = ctx.how
        if not ctx.needs_input_grad[0]:
            dq = None
        if not ctx.needs_input_grad[1]:
            dk = None
        if dq is None and dk is None:
            return (None,) * 7
        dq, dk = _turned(dq, dk, positions, inv_freq, interleaved, factor, not backward)
        return dq, dk, None, None, None, None, None


class RotaryDualFunc(RotaryFunc):
    """Of inputs that carry tangents, which go through the map as they do."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, factor, backward):
        ctx.save_for_forward(positions, inv_freq)
        return RotaryFunc.forward(ctx, q, k, positions, inv_freq, interleaved, factor, backward)

    @staticmethod
    def jvp(ctx, tq, tk, *none):
        positions, inv_freq = ctx.saved_tensors
        return _turned(tq, tk, positions, inv_freq, *ctx.how)


@torch.library.custom_op("splitd_flash_attn::rotary", mutates_args=())
def _rotary_custom(
    q: Optional[torch.Tensor],
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    interleaved: bool,
    factor: float,
    backward: bool,
) -> tuple[torch.Tensor, torch.Tensor]:
    """An output for an input that is None is an empty tensor."""
    q_out, k_out = _rotary(q, k, positions, inv_freq, interleaved, factor, backward)
    none = inv_freq.new_empty((0,), dtype=(q if q is not None else k).dtype)
    return (none if q_out is None else q_out), (none.clone() if k_out is None else k_out)


@torch.library.register_fake("splitd_flash_attn::rotary")
def _rotary_fake(q, k, positions, inv_freq, interleaved, factor, backward):
    _check_rotary(q, k, positions, inv_freq)
    first = q if q is not None else k
    return tuple(first.new_empty((0,) if t is None else t.shape) for t in (q, k))


def _rotary_setup_context(ctx, inputs, output) -> None:
    q, k, positions, inv_freq, ctx.interleaved, ctx.factor, ctx.backward_ = inputs
    ctx.has = q is not None, k is not None
    ctx.save_for_backward(positions, inv_freq)
    ctx.set_materialize_grads(False)


def _rotary_backward(ctx, dq, dk):
    positions, inv_freq = ctx.saved_tensors
    dq, dk = (g if has else None for g, has in zip((dq, dk), ctx.has))
    if dq is None and dk is None:
        return (None,) * 7
    gq, gk = torch.ops.splitd_flash_attn.rotary(dq, dk, positions, inv_freq, ctx.interleaved, ctx.factor, not ctx.backward_)
    return (None if dq is None else gq), (None if dk is None else gk), None, None, None, None, None


torch.library.register_autograd("splitd_flash_attn::rotary", _rotary_backward, setup_context=_rotary_setup_context)


def _turned(q, k, positions, inv_freq, interleaved, factor, backward):
    if _dual(q, k):
        return _turned_with_tangents(q, k, positions, inv_freq, interleaved, factor, backward)
    if _traced(q, k):
        _check_rotary(q, k, positions, inv_freq)
        q_out, k_out = torch.ops.splitd_flash_attn.rotary(q, k, positions, inv_freq, interleaved, factor, backward)
        return (None if q is None else q_out), (None if k is None else k_out)
    if torch.is_grad_enabled() and (q is not None and q.requires_grad or k is not None and k.requires_grad):
        return RotaryFunc.apply(q, k, positions, inv_freq, interleaved, factor, backward)
    return _rotary(q, k, positions, inv_freq, interleaved, factor, backward)


def _turned_with_tangents(q, k, *how):
    if _traced(q, k):
        raise NotImplementedError("SplitD rotary positions in forward mode cannot be traced or transformed")
    if q is not None and k is not None and _dual(q) != _dual(k):  # an output without a tangent is a call of its own
        _check_rotary(q, k, *how[:2])
        return _turned(q, None, *how)[0], _turned(None, k, *how)[1]
    return RotaryDualFunc.apply(q, k, *how)


def split_rotary_func(
    q: Optional[torch.Tensor],
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    interleaved: bool = False,
    factor: float = 1.0,
):
    """Rotary positions on the first ``2 * len(inv_freq)`` dimensions of every head of q and k. Returns
    ``(q_out, k_out)``, differentiable in q and k, in forward mode too.

    q (B, S, Hq, 512), k (B, S, Hkv, 512), bf16 or fp16, any strides; or packed, (T, Hq, 512) and (T, Hkv, 512). Either
    may be None, and so is its output then. ``positions``: int32 or int64, (B, S), (S,) for all sequences alike, or
    (T,). ``inv_freq``: float64, radians per position (``split_rotary_frequencies``), without a gradient; angles are formed
    in 64 bits, so far positions lose nothing. A pair is dimensions (i, i + rotary_dim / 2), with ``interleaved`` (2 i,
    2 i + 1). ``factor`` scales what is rotated; the dimensions behind pass through unchanged.
    """
    _refuse_derivatives("rotary positions with respect to inv_freq", inv_freq)
    return _turned(q, k, positions, inv_freq, bool(interleaved), float(factor), False)
