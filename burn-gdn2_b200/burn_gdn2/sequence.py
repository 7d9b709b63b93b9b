"""Sequence operators around a gated recurrence, for training and serving.

  gated_scan        the diagonal gated linear recurrence h_t = e^{g_t} h_{t-1} + s_t x_t
  causal_conv_silu  the 4-tap causal convolution with SiLU in front of it
  group_norm_gate   the norm of each token's channel groups behind it, with an affine map and a SiLU
  reorder_states    forking, compacting and freeing the rows of the state pool of a serving batch, in place
  select_states     the same into a new pool of another size

Every operator takes CUDA tensors on any device and launches on that device's
current stream; it is differentiable where an input requires a gradient (in
reverse mode; a tangent of forward mode is refused), and deterministic.
Sequences come as a dense batch [B,T,C], or packed: one buffer [1,R,C] with
``cu_seqlens`` (int32 [N+1], ascending from 0), sequence n in the rows
cu_seqlens[n] .. cu_seqlens[n+1].  A ``cu_seqlens`` on the CPU is checked and
copied to the device; one on the device is taken as it is (the kernels stay
inside the buffers whatever it holds).  Offsets and row numbers from the host
are copied from pageable memory, for which the call waits on its stream: a
serving loop and a capture pass them on the device.  Rows behind the last
sequence come out as zero, in outputs and gradients.

A backward captured into a CUDA graph wants no eager graph of the same leaves
alive: torch would wait on the eager graph's stream in the middle of the
capture.
"""
from __future__ import annotations

import dataclasses
import re
from typing import Tuple

import torch

from . import _lib  # loads the library that the calls below are linked to
from .ops import _DT


class _NotBuilt:
    """Stands for the extension where it cannot be loaded: the rest of the package needs no torch extension."""

    def __init__(self, error):
        self._error = error

    def __getattr__(self, name):
        raise ImportError("_torch_calls.so not built for this torch: run `python burn-gdn2_b200/build.py`") from self._error


def _release(version: str) -> str:
    """The numbers of a torch version: what its headers give, without a pre-release's or a build's name."""
    return re.match(r"\d+(\.\d+)*", version).group()


try:
    from . import _torch_calls as _calls

    if _calls.torch_version != _release(torch.__version__):
        raise ImportError(f"_torch_calls.so is built for torch {_calls.torch_version}, this is {torch.__version__}")
    _calls.set_error_class(_lib.Gdn2Error)
except ImportError as e:
    _calls = _NotBuilt(e)


def available() -> bool:
    """Whether the extension that the operators run on is there."""
    return not isinstance(_calls, _NotBuilt)


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
        steps = cu.long().diff()
        if int(cu[0]) != 0 or int(steps.min()) < 0 or int(cu[-1]) > x.shape[1]:
            raise ValueError(f"{what}: cu_seqlens must ascend from 0 to at most {x.shape[1]} rows, got {cu.tolist()}")
        return cu.to(device=x.device, dtype=torch.int32)
    if cu.device != x.device:
        raise ValueError(f"{what}: tensors on {x.device} and {cu.device}")
    if cu.dtype != torch.int32:
        raise ValueError(f"{what}: cu_seqlens on the device must be int32, got {cu.dtype}")
    return cu.contiguous()


def _packed(what: str, cu, x: torch.Tensor):
    if cu is None:
        return None
    _check_input(what, x)
    if x.dim() != 3:
        raise ValueError(f"{what}: x must be [B,T,C], got {list(x.shape)}")
    return _cu_seqlens(what, cu, x)


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
    are joined as products in f32: growth (g > 0) is exact as far as the products
    over spans of the sequence stay inside f32 (1e-38 to 3e38); beyond, a state
    of zero stays zero, also one that a reset has cut off in the same span, and
    any other one need not stay finite (or come back).
    Differentiable in x, g and state, once.
    """
    return _calls.gated_scan(x, g, state, _packed("gated_scan", cu_seqlens, x), complement, inplace)


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
    return _calls.causal_conv_silu(x, weight, cache, _packed("causal_conv_silu", cu_seqlens, x))


def group_norm_gate(x, gate=None, weight=None, bias=None, *, num_groups: int, eps: float = 1e-5, center: bool = True):
    """Norm of each token's channel groups, an affine map and a SiLU.

    x [..., C] (f32 or bf16, channels last): each token's C channels are
    num_groups groups of C / num_groups, each brought to mean 0 and variance 1
    (``center=False``: to root mean square 1), z = n weight + bias, and
    y = z silu(gate), or silu(z) without a gate.  gate: x's shape and dtype.
    weight, bias: f32 [C], or [C / num_groups] for all groups alike, or None.
    With ``center=False``, a gate and a weight per head this is
    rms_norm_gate_per_head on [..., HV*V], with gradients.  f32 arithmetic;
    eps must be above 0 in f32; differentiable in x, gate, weight and bias,
    once.
    """
    return _calls.group_norm_gate(x, gate, weight, bias, num_groups, eps, center, False)


def group_norm_gate_again(x, gate, weight, *, num_groups: int, eps: float, center: bool):
    """group_norm_gate for a graph that may be differentiated more often: a
    backward with create_graph runs the formula in torch operations."""
    return _calls.group_norm_gate(x, gate, weight, None, num_groups, eps, center, True)


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


def _index(what: str, index) -> torch.Tensor:
    """index as a tensor; numbers given as a sequence must be whole ones (a mask or a fraction would pass for some)."""
    if isinstance(index, torch.Tensor):
        return index
    t = torch.tensor(index)
    if t.numel() and (t.dtype == torch.bool or t.is_floating_point() or t.is_complex()):
        raise ValueError(f"{what}: index must be whole numbers, got {index!r}")
    return t.to(torch.int64)


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
    tensors = _pool_tensors("reorder_states", states)
    if tensors:
        _calls.reorder_states(tensors, _index("reorder_states", index))


def select_states(states, index):
    """A new pool of len(index) rows, row d a copy of row index[d] of states
    (-1: zeros): a batch that grows, or is split for another device step.  The
    result has the structure of ``states``; numbers as in reorder_states, but a
    row whose number on the device is outside the pool is zeros."""
    tensors = _pool_tensors("select_states", states)
    return _pool_like(states, iter(_calls.select_states(tensors, _index("select_states", index)) if tensors else ()))
