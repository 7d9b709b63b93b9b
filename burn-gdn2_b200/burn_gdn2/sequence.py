"""Sequence operators around a gated recurrence, for training and serving.

  gated_scan        the diagonal gated linear recurrence h_t = e^{g_t} h_{t-1} + s_t x_t
  causal_conv_silu  the 4-tap causal convolution with SiLU in front of it
  group_norm_gate   the norm of each token's channel groups behind it, with an affine map and a SiLU
  reorder_states    forking, compacting and freeing the rows of the state pool of a serving batch, in place
  select_states     the same into a new pool of another size

Every operator takes CUDA tensors on any device and launches on that device's
current stream; it is differentiable where an input requires a gradient, and
deterministic.  Sequences come as a dense batch [B,T,C], or packed: one
buffer [1,R,C] with ``cu_seqlens`` (int32 [N+1], ascending from 0), sequence n
in the rows cu_seqlens[n] .. cu_seqlens[n+1].  A ``cu_seqlens`` on the CPU is
checked and copied to the device; one on the device is taken as it is (the
kernels stay inside the buffers whatever it holds).  Rows behind the last
sequence come out as zero, in outputs and gradients.
"""
from __future__ import annotations

import contextlib
import ctypes
import dataclasses
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import LIB, check
from .ops import SHORT_CONV_CACHE, SHORT_CONV_KERNEL, _DT

SCAN_CARRY = 16  # tokens between the states that gated_scan keeps for its backward

_NOTHING = contextlib.nullcontext()


def _on(device: torch.device):
    """The device as the current one for a launch (free when it is already)."""
    return _NOTHING if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)  # current_stream() builds an object: 2 us a call


def _same_device(what: str, device: torch.device, *tensors):
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: tensors on {device} and {t.device}")


def _check_input(what: str, x: torch.Tensor):
    if not x.is_cuda:
        raise RuntimeError(f"{what} runs on the B200 CUDA kernels only; got a CPU tensor")
    if x.dtype not in _DT:
        raise TypeError(f"{what}: unsupported dtype {x.dtype}; use float32 or bfloat16")


def _cu_seqlens(what: str, cu: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """Packed offsets on x's device, int32; the values are checked where they are on the host."""
    if x.shape[0] != 1:
        raise ValueError(f"{what}: packed sequences come as one buffer [1,R,C], got a batch of {x.shape[0]}")
    if cu.dim() != 1 or cu.numel() < 2 or cu.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: cu_seqlens must be int32 [N+1] with N >= 1, got {cu.dtype} {list(cu.shape)}")
    if not cu.is_cuda:
        steps = cu[1:] - cu[:-1]
        if int(cu[0]) != 0 or int(steps.min()) < 0 or int(cu[-1]) > x.shape[1]:
            raise ValueError(f"{what}: cu_seqlens must ascend from 0 to at most {x.shape[1]} rows, got {cu.tolist()}")
        return cu.to(device=x.device, dtype=torch.int32)
    _same_device(what, x.device, cu)
    if cu.dtype != torch.int32:
        raise ValueError(f"{what}: cu_seqlens on the device must be int32, got {cu.dtype}")
    return cu.contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous channels and no broadcast over them."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _view3(t: Optional[torch.Tensor]) -> _lib.View:
    """[B,T,C] as the library's [B,T,1,C] view."""
    if t is None:
        return _lib.View()
    s = t.stride()
    return _lib.View(t.data_ptr(), s[0], s[1], 0)


def _f32(what: str, name: str, t: Optional[torch.Tensor], shape) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype != torch.float32:
        raise TypeError(f"{what}: {name} must be float32, got {t.dtype}")
    return t.contiguous()


def _written(tensors) -> None:
    """Tells autograd that a kernel has written over these tensors."""
    torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


def _workspace(size: int, near: torch.Tensor):
    return (near.new_empty(size, dtype=torch.uint8) if size else None), size


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# -- gated scan ----------------------------------------------------------------


def _scan_args(x, g, state, cu, complement, carry):
    return _lib.ScanArgs(x.shape[0] if cu is None else cu.numel() - 1, x.shape[1], x.shape[2], _DT[x.dtype],
                         _DT[g.dtype], int(complement), _ptr(cu), _view3(x), _view3(g), _ptr(state), _ptr(carry))


def _scan_forward(x, g, state, cu, complement, state_out, keep):
    B, T, C = x.shape
    h = _like(x)
    carry = x.new_empty((B, -(-T // SCAN_CARRY), C), dtype=torch.float32) if keep else None
    a, out = _scan_args(x, g, state, cu, complement, carry), _view3(h)
    with _on(x.device):
        # up to 64 tokens are one block's and never cut into segments
        ws, size = _workspace(LIB.gdn2_gated_scan_workspace_bytes(ctypes.byref(a), out) if T > 64 else 0, x)
        check(LIB.gdn2_gated_scan(ctypes.byref(a), out, _ptr(state_out), _ptr(ws), size, _stream(x.device)))
    return h, carry


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, state, cu, complement):
        n = x.shape[0] if cu is None else cu.numel() - 1
        last = x.new_empty((n, x.shape[2]), dtype=torch.float32)
        h, carry = _scan_forward(x, g, state, cu, complement, last, True)
        ctx.save_for_backward(x, g, state, cu, carry)
        ctx.complement = complement
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_h, d_last):
        x, g, state, cu, carry = ctx.saved_tensors
        d_h = torch.zeros_like(x) if d_h is None else _rows(d_h)
        d_last = None if d_last is None else d_last.contiguous()
        dx, dg = _like(x), _like(g)
        d_state = torch.empty_like(state) if state is not None and ctx.needs_input_grad[2] else None
        a = _lib.ScanBwdArgs(_scan_args(x, g, state, cu, ctx.complement, carry), _view3(d_h), _ptr(d_last),
                             _view3(dx), _view3(dg), _ptr(d_state))
        with _on(x.device):
            ws, size = _workspace(LIB.gdn2_gated_scan_bwd_workspace_bytes(ctypes.byref(a)), x)
            check(LIB.gdn2_gated_scan_bwd(ctypes.byref(a), _ptr(ws), size, _stream(x.device)))
        return dx, dg, d_state, None, None


def gated_scan(x, g, state=None, *, cu_seqlens=None, complement: bool = False,
               inplace: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """The diagonal gated linear recurrence h_t = e^{g_t} h_{t-1} + s_t x_t.

    x [B,T,C] (f32 or bf16); g [B,T,C], the log decay, f32 or x's dtype;
    state [B,C] f32, the state before the first token (None: zeros).  s_t = 1,
    or 1 - e^{g_t} with ``complement`` (a leaky average of x).  Returns
    (h [B,T,C] in x's dtype, the state after the last token [B,C] f32); the
    arithmetic is f32.  Packed: x, g [1,R,C], state [N,C] (see the module).

    T = 1 is the decode step.  ``inplace`` writes the new state over ``state``
    and returns it (serving; no gradients).  g may be anything whose
    exponential is wanted: -inf cuts off what came before.  Decays of spans
    are joined as products in f32: growth (g > 0) is exact as far as the product
    over a span stays below 3e38; beyond, a state of zero stays zero and any
    other one becomes infinite.  Differentiable in x, g and state, once.
    """
    what = "gated_scan"
    _check_input(what, x)
    if x.dim() != 3 or x.shape != g.shape:
        raise ValueError(f"{what}: x and g must both be [B,T,C], got {list(x.shape)} and {list(g.shape)}")
    if g.dtype != torch.float32 and g.dtype != x.dtype:
        raise TypeError(f"{what}: g must be float32 or x's dtype {x.dtype}, got {g.dtype}")
    _same_device(what, x.device, g, state)
    cu = None if cu_seqlens is None else _cu_seqlens(what, cu_seqlens, x)
    B, T, C = x.shape
    n = B if cu is None else cu.numel() - 1
    given, state = state, _f32(what, "state", state, (n, C))
    x, g = _rows(x), _rows(g)
    grads = torch.is_grad_enabled() and (x.requires_grad or g.requires_grad or (state is not None and state.requires_grad))
    if inplace:
        if given is None:
            raise ValueError(f"{what}: inplace needs a state")
        if grads:
            raise ValueError(f"{what}: inplace does not go with gradients; detach the inputs or use torch.no_grad()")
        if state is not given:
            raise ValueError(f"{what}: inplace needs a contiguous state")
    if n == 0 or C == 0 or (T == 0 and cu is None):  # nothing to launch: no token, or nothing in it
        last = torch.zeros((n, C), dtype=torch.float32, device=x.device) if state is None else state
        return x + g.to(x.dtype), last if inplace else last.clone()
    if grads:
        return _GatedScan.apply(x, g, state, cu, bool(complement))
    last = state if inplace else x.new_empty((n, C), dtype=torch.float32)
    h, _ = _scan_forward(x, g, state, cu, complement, last, False)
    if inplace:
        _written([state])
    return h, last


# -- causal convolution --------------------------------------------------------


def _conv_args(x, weight, cache, cu):
    return _lib.ConvArgs(x.shape[0] if cu is None else cu.numel() - 1, x.shape[1], x.shape[2], _DT[x.dtype], _ptr(cu),
                         _view3(x), weight.data_ptr(), _ptr(cache))


def _conv_forward(x, weight, cache, cu):
    n = x.shape[0] if cu is None else cu.numel() - 1
    y = _like(x)
    new = x.new_empty((n, SHORT_CONV_CACHE, x.shape[2]), dtype=torch.float32)
    a = _conv_args(x, weight, cache, cu)
    with _on(x.device):
        check(LIB.gdn2_causal_conv(ctypes.byref(a), _view3(y), new.data_ptr(), _stream(x.device)))
    return y, new


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, cache, cu):
        ctx.save_for_backward(x, weight, cache, cu)
        ctx.set_materialize_grads(False)
        return _conv_forward(x, weight, cache, cu)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_new):
        x, weight, cache, cu = ctx.saved_tensors
        d_y = torch.zeros_like(x) if d_y is None else _rows(d_y)
        d_new = None if d_new is None else d_new.contiguous()
        dx = _like(x)
        d_weight = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        d_cache = torch.empty_like(cache) if cache is not None and ctx.needs_input_grad[2] else None
        a = _lib.ConvBwdArgs(_conv_args(x, weight, cache, cu), _view3(d_y), _ptr(d_new), _view3(dx), _ptr(d_weight),
                             _ptr(d_cache))
        with _on(x.device):
            ws, size = _workspace(LIB.gdn2_causal_conv_bwd_workspace_bytes(ctypes.byref(a)), x)
            check(LIB.gdn2_causal_conv_bwd(ctypes.byref(a), _ptr(ws), size, _stream(x.device)))
        return dx, d_weight, d_cache, None


def causal_conv_silu(x, weight, cache=None, *, cu_seqlens=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """short_conv_1d with gradients and packed sequences: the causal depthwise
    convolution of 4 taps and its SiLU, y_t = silu(sum_j w[:, j] x_{t-3+j}).

    x [B,T,C] (f32 or bf16); weight [C,4] f32; cache [B,3,C] f32, the three
    values before each sequence, or None: copies of its first token
    (src/short_conv.rs:42-54).  Returns (y [B,T,C], the new cache [B,3,C] f32:
    the last three values).  Packed: x [1,R,C], caches [N,3,C] (see the
    module); an empty sequence keeps its cache (zeros without one).  T = 1 is
    the decode step.  f32 arithmetic; differentiable in x, weight and cache,
    once.
    """
    what = "causal_conv_silu"
    _check_input(what, x)
    if x.dim() != 3:
        raise ValueError(f"{what}: x must be [B,T,C], got {list(x.shape)}")
    _same_device(what, x.device, weight, cache)
    cu = None if cu_seqlens is None else _cu_seqlens(what, cu_seqlens, x)
    B, T, C = x.shape
    n = B if cu is None else cu.numel() - 1
    weight = _f32(what, "weight", weight, (C, SHORT_CONV_KERNEL))
    cache = _f32(what, "cache", cache, (n, SHORT_CONV_CACHE, C))
    x = _rows(x)
    if n == 0 or C == 0 or (T == 0 and cu is None):  # nothing to launch: no token, or nothing in it
        return x * weight[:, 0].to(x.dtype), torch.zeros((n, SHORT_CONV_CACHE, C), device=x.device) if cache is None else cache.clone()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, cache)):
        return _CausalConv.apply(x, weight, cache, cu)
    return _conv_forward(x, weight, cache, cu)


# -- group norm ----------------------------------------------------------------


def _norm_args(x, gate, weight, bias, groups, eps, center):
    rows, chan = x.shape
    shared = weight is not None and weight.numel() != chan
    return _lib.GroupNormArgs(rows, groups, chan // groups, _DT[x.dtype], int(center), int(shared), eps, x.data_ptr(),
                              x.stride(0), _ptr(gate), 0 if gate is None else gate.stride(0), _ptr(weight), _ptr(bias))


def _norm_rows(t: Optional[torch.Tensor], chan: int) -> Optional[torch.Tensor]:
    """[..., C] as rows; a copy where the rows are not evenly spaced or their channels not contiguous."""
    if t is None:
        return None
    return _rows(t if t.dim() == 2 else t.reshape(-1, chan))


def _norm_forward(x, gate, weight, bias, groups, eps, center):
    y = _like(x)
    if x.shape[0]:
        a = _norm_args(x, gate, weight, bias, groups, eps, center)
        with _on(x.device):
            check(LIB.gdn2_group_norm_gate(ctypes.byref(a), y.data_ptr(), _stream(x.device)))
    return y


class _GroupNormGate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, weight, bias, groups, eps, center):
        rows, gate_rows = _norm_rows(x, x.shape[-1]), _norm_rows(gate, x.shape[-1])
        ctx.save_for_backward(rows, gate_rows, weight, bias)
        ctx.rest = (groups, eps, center)
        ctx.shape = x.shape
        y = _norm_forward(rows, gate_rows, weight, bias, groups, eps, center)
        return y if x.dim() == 2 else y.view(x.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y):
        x, gate, weight, bias = ctx.saved_tensors
        d_y = _norm_rows(d_y, x.shape[1])
        need = ctx.needs_input_grad
        dx, d_gate, d_weight, d_bias = (_like(t) if need[k] else None for k, t in enumerate((x, gate, weight, bias)))
        if x.shape[0]:
            a = _lib.GroupNormBwdArgs(_norm_args(x, gate, weight, bias, *ctx.rest), d_y.data_ptr(), d_y.stride(0),
                                      _ptr(dx), _ptr(d_gate), _ptr(d_weight), _ptr(d_bias))
            with _on(x.device):
                ws, size = _workspace(LIB.gdn2_group_norm_gate_bwd_workspace_bytes(ctypes.byref(a)), x)
                check(LIB.gdn2_group_norm_gate_bwd(ctypes.byref(a), _ptr(ws), size, _stream(x.device)))
        else:
            d_weight, d_bias = (None if t is None else t.zero_() for t in (d_weight, d_bias))
        if len(ctx.shape) != 2:
            dx, d_gate = (None if t is None else t.view(ctx.shape) for t in (dx, d_gate))
        return dx, d_gate, d_weight, d_bias, None, None, None


def group_norm_gate(x, gate=None, weight=None, bias=None, *, num_groups: int, eps: float = 1e-5, center: bool = True):
    """Norm of each token's channel groups, an affine map and a SiLU.

    x [..., C] (f32 or bf16, channels last): each token's C channels are
    num_groups groups of C / num_groups, each brought to mean 0 and variance 1
    (``center=False``: to root mean square 1), z = n weight + bias, and
    y = z silu(gate), or silu(z) without a gate.  gate: x's shape and dtype.
    weight, bias: f32 [C], or [C / num_groups] for all groups alike, or None.
    With ``center=False``, a gate and a weight per head this is
    rms_norm_gate_per_head on [..., HV*V], with gradients.  f32 arithmetic;
    differentiable in x, gate, weight and bias, once.
    """
    what = "group_norm_gate"
    _check_input(what, x)
    if x.dim() < 1 or num_groups < 1 or x.shape[-1] == 0 or x.shape[-1] % num_groups:
        raise ValueError(f"{what}: the {x.shape[-1] if x.dim() else 0} channels do not split into {num_groups} groups")
    if not eps > 0:
        raise ValueError(f"{what}: eps must be > 0, got {eps}")
    _same_device(what, x.device, gate, weight, bias)
    if gate is not None and (gate.shape != x.shape or gate.dtype != x.dtype):
        raise ValueError(f"{what}: gate must be {list(x.shape)} {x.dtype}, got {list(gate.shape)} {gate.dtype}")
    shape, chan = x.shape, x.shape[-1]
    width = chan // num_groups
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dim() != 1 or t.numel() not in (chan, width)):
            raise ValueError(f"{what}: {name} must be [{chan}] or [{width}], got {list(t.shape)}")
        if t is not None and t.dtype != torch.float32:
            raise TypeError(f"{what}: {name} must be float32, got {t.dtype}")
    if bias is not None and (weight is None or weight.shape != bias.shape):
        raise ValueError(f"{what}: a bias goes with a weight of its shape")
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    rest = (weight, bias, int(num_groups), float(eps), bool(center))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, gate, weight, bias)):
        return _GroupNormGate.apply(x, gate, *rest)
    y = _norm_forward(_norm_rows(x, chan), _norm_rows(gate, chan), *rest)
    return y if x.dim() == 2 else y.view(shape)


# -- state pools ---------------------------------------------------------------


def _pool_tensors(what: str, states) -> list:
    """The tensors of a tensor, a state (its fields), or a sequence of either."""
    if isinstance(states, torch.Tensor):
        return [states]
    if dataclasses.is_dataclass(states):
        return [getattr(states, f.name) for f in dataclasses.fields(states)]
    if isinstance(states, (list, tuple)):
        return [t for s in states for t in _pool_tensors(what, s)]
    raise TypeError(f"{what}: a pool is tensors, states or sequences of them, got {type(states).__name__}")


def _pool_like(states, new):
    """The structure of states, filled from the iterator new."""
    if isinstance(states, torch.Tensor):
        return next(new)
    if dataclasses.is_dataclass(states):
        return dataclasses.replace(states, **{f.name: next(new) for f in dataclasses.fields(states)})
    items = [_pool_like(s, new) for s in states]
    return type(states)(*items) if hasattr(states, "_fields") else type(states)(items)


def _checked_pool(what: str, states):
    tensors = _pool_tensors(what, states)
    if not tensors:
        return tensors
    if not all(t.is_cuda for t in tensors):
        raise RuntimeError(f"{what} runs on the B200 CUDA kernels only; got a CPU tensor")
    if not all(t.dim() for t in tensors) or len({t.shape[0] for t in tensors}) > 1:
        raise ValueError(f"{what}: every tensor of a pool has its rows first and as many, got {[list(t.shape) for t in tensors]}")
    if not all(t.is_contiguous() for t in tensors):
        raise ValueError(f"{what}: the tensors of a pool must be contiguous")
    if any(t.requires_grad for t in tensors):
        raise ValueError(f"{what}: the rows of a pool move without gradients; detach its tensors")
    _same_device(what, tensors[0].device, *tensors)
    if tensors[0].shape[0] > _lib.GDN2_MAX_STATE_ROWS:
        raise ValueError(f"{what}: {tensors[0].shape[0]} rows, at most {_lib.GDN2_MAX_STATE_ROWS}")
    return tensors


def _pool_index(what: str, index, rows: int, device) -> torch.Tensor:
    """Row numbers on the device, int32; checked where they come from the host."""
    if not isinstance(index, torch.Tensor):
        index = torch.tensor(index, dtype=torch.int64)
    if index.dim() != 1 or index.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: index must be a vector of int32 or int64, got {index.dtype} {list(index.shape)}")
    if index.shape[0] > _lib.GDN2_MAX_STATE_ROWS:
        raise ValueError(f"{what}: {index.shape[0]} rows, at most {_lib.GDN2_MAX_STATE_ROWS}")
    if not index.is_cuda:
        if index.numel() and (int(index.min()) < -1 or int(index.max()) >= rows):
            raise ValueError(f"{what}: row numbers must be -1 to {rows - 1}, got {index.tolist()}")
        return index.to(device=device, dtype=torch.int32)
    _same_device(what, device, index)
    if index.dtype == torch.int64:  # as far as 32 bits tell a number inside the pool from one outside
        index = index.clamp(-2, rows).int()
    return index.contiguous()


def _move_rows(sources, targets, index, src_rows):
    device, n = index.device, index.shape[0]
    rows = [(s.data_ptr(), t.data_ptr(), t.nbytes // n) for s, t in zip(sources, targets) if t.nbytes]
    if rows:
        with _on(device):
            check(LIB.gdn2_move_state_rows((_lib.StateRows * len(rows))(*rows), len(rows), index.data_ptr(), src_rows, n,
                                           _stream(device)))


def reorder_states(states, index) -> None:
    """Move the rows of a state pool, in place and in one launch: in every
    tensor row d becomes what row index[d] was, -1 a row of zeros (a freed or
    a fresh sequence); a row's own number leaves it alone.  All rows at once:
    a fork names one source several times, a compaction moves the last live
    rows into the holes, swaps need no third row.

    states: a Gdn2State, a tensor (a scan's state, a convolution's cache), or a
    sequence of them (the layers of a model); rows come first, contiguous, at
    most 4096.  index: one number a row, on the host (checked) or on the device
    (int32 or int64; read by the kernel, so a captured call follows it).  On
    the device a number outside the pool leaves its row as it was and sets bit
    1 of ``read_device_errors()``.
    """
    what = "reorder_states"
    tensors = _checked_pool(what, states)
    if not tensors:
        return
    rows = tensors[0].shape[0]
    spans = sorted([(t.data_ptr(), t.nbytes) for t in tensors])
    if any(a + n > b for (a, n), (b, _) in zip(spans, spans[1:])):
        raise ValueError(f"{what}: a tensor (or a part of one) comes twice")
    index = _pool_index(what, index, rows, tensors[0].device)
    if index.shape[0] != rows:
        raise ValueError(f"{what}: {index.shape[0]} row numbers for {rows} rows")
    _move_rows(tensors, tensors, index, rows)
    _written(tensors)


def select_states(states, index):
    """A new pool of len(index) rows, row d a copy of row index[d] of states
    (-1: zeros): a batch that grows, or is split for another device step.  The
    result has the structure of ``states``; numbers as in reorder_states, but a
    row whose number on the device is outside the pool is zeros."""
    what = "select_states"
    tensors = _checked_pool(what, states)
    if not tensors:
        return _pool_like(states, iter(()))
    rows = tensors[0].shape[0]
    index = _pool_index(what, index, rows, tensors[0].device)
    new = [t.new_empty((index.shape[0], *t.shape[1:])) for t in tensors]
    _move_rows(tensors, new, index, rows)
    return _pool_like(states, iter(new))
