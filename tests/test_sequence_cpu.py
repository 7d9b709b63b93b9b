"""CPU: what the sequence operators refuse, before any launch, and their C
entries' argument errors."""
import collections
import ctypes

import pytest
import torch


def _fake(*shape, dtype=torch.float32):
    """A tensor that says it is on a device: shapes and types without a GPU."""
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_refuses_cpu_tensors():
    import burn_gdn2 as bg

    x = torch.zeros(1, 4, 8)
    with pytest.raises(RuntimeError, match="CPU tensor"):
        bg.gated_scan(x, x)


def test_packed_offsets_are_checked_on_the_host():
    from burn_gdn2 import sequence

    x = _fake(1, 10, 4)
    for bad in ([1, 5], [0, 7, 3], [0, 11], [0, 4, 3, 9], [0, 2147483647, -2, 1]):
        with pytest.raises(ValueError, match="ascend"):
            sequence._cu_seqlens("op", torch.tensor(bad, dtype=torch.int32), x)
    for bad in (torch.tensor([0], dtype=torch.int32), torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([0.0, 1.0])):
        with pytest.raises(ValueError, match="int32"):
            sequence._cu_seqlens("op", bad, x)
    with pytest.raises(ValueError, match="one buffer"):
        sequence._cu_seqlens("op", torch.tensor([0, 3], dtype=torch.int32), _fake(2, 10, 4))


def _scan_args(**over):
    from burn_gdn2 import _lib

    fake = 1 << 20  # never dereferenced: validation fails first
    v = _lib.View(fake, 64, 8, 0)
    a = _lib.ScanArgs(2, 8, 8, 0, 0, 0, None, v, v, None, None)
    for k, val in over.items():
        setattr(a, k, val)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(batch=0), 1), (dict(seq_len=-1), 1), (dict(seq_len=0), 1), (dict(channels=0), 1), (dict(dtype=7), 1),
    (dict(g_dtype=-1), 1), (dict(g_dtype=1), 2), (dict(seq_len=(1 << 30) + 1), 2),
])
def test_scan_argument_errors(over, status):
    from burn_gdn2 import LIB, _lib

    out = _lib.View(1 << 20, 64, 8, 0)
    a = _scan_args(**over)
    assert LIB.gdn2_gated_scan(ctypes.byref(a), out, None, None, 0, None) == status
    assert LIB.gdn2_last_error().decode().startswith("gdn2_gated_scan:")
    b = _lib.ScanBwdArgs(a, out, None, out, out, None)
    assert LIB.gdn2_gated_scan_bwd(ctypes.byref(b), None, 0, None) == status


def test_scan_null_pointers():
    from burn_gdn2 import LIB, _lib

    out, none = _lib.View(1 << 20, 64, 8, 0), _lib.View()
    assert LIB.gdn2_gated_scan(None, out, None, None, 0, None) == _lib.GDN2_EINVAL
    assert LIB.gdn2_gated_scan_bwd(None, None, 0, None) == _lib.GDN2_EINVAL
    a = _scan_args()
    assert LIB.gdn2_gated_scan(ctypes.byref(a), none, None, None, 0, None) == _lib.GDN2_EINVAL
    assert LIB.gdn2_gated_scan(ctypes.byref(_scan_args(x=none)), out, None, None, 0, None) == _lib.GDN2_EINVAL
    for args in ((a, none, out, out), (a, out, none, out), (a, out, out, none), (a, out, out, out)):  # the last: no carry
        b = _lib.ScanBwdArgs(args[0], args[1], None, args[2], args[3], None)
        assert LIB.gdn2_gated_scan_bwd(ctypes.byref(b), None, 0, None) == _lib.GDN2_EINVAL


def test_scan_workspace():
    """Few chains over a long axis need one, many do not; too small a one is refused."""
    from burn_gdn2 import LIB, _lib

    out = _lib.View(1 << 20, 1 << 20, 8, 0)
    long = _scan_args(batch=1, seq_len=4096)
    need = LIB.gdn2_gated_scan_workspace_bytes(ctypes.byref(long), out)
    assert need > 0
    assert LIB.gdn2_gated_scan(ctypes.byref(long), out, None, None, 0, None) == _lib.GDN2_EWORKSPACE
    assert LIB.gdn2_gated_scan(ctypes.byref(long), out, None, 1 << 20, need - 1, None) == _lib.GDN2_EWORKSPACE
    assert LIB.gdn2_gated_scan(ctypes.byref(long), out, None, (1 << 20) + 4, need, None) == _lib.GDN2_EINVAL
    long.carry = 1 << 20
    b = _lib.ScanBwdArgs(long, out, None, out, out, None)
    need = LIB.gdn2_gated_scan_bwd_workspace_bytes(ctypes.byref(b))
    assert need > 0
    assert LIB.gdn2_gated_scan_bwd(ctypes.byref(b), 1 << 20, need - 1, None) == _lib.GDN2_EWORKSPACE
    assert LIB.gdn2_gated_scan_workspace_bytes(ctypes.byref(_scan_args(batch=512, seq_len=4096)), out) == 0
    assert LIB.gdn2_gated_scan_workspace_bytes(ctypes.byref(_scan_args(seq_len=0)), out) == 0
    assert LIB.gdn2_gated_scan_workspace_bytes(None, out) == 0


def test_struct_layouts_match_header(tmp_path):
    import os
    import subprocess

    from burn_gdn2 import _lib

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"gdn2_scan_args": _lib.ScanArgs, "gdn2_scan_bwd_args": _lib.ScanBwdArgs,
             "gdn2_group_norm_args": _lib.GroupNormArgs, "gdn2_group_norm_bwd_args": _lib.GroupNormBwdArgs,
             "gdn2_conv_args": _lib.ConvArgs, "gdn2_conv_bwd_args": _lib.ConvBwdArgs, "gdn2_state_rows": _lib.StateRows}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "gdn2.h"', "int main() {"]
    for c, s in names.items():
        lines.append(f'printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in s._fields_]
    src, exe = tmp_path / "p.c", tmp_path / "p"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        c, f, v = line.split()
        assert int(v) == (ctypes.sizeof(names[c]) if f == "size" else getattr(names[c], f).offset), (c, f)


def _norm_args(**over):
    from burn_gdn2 import _lib

    fake = 1 << 20
    a = _lib.GroupNormArgs(4, 2, 16, 0, 1, 0, 1e-5, fake, 32, fake, 32, fake, fake)
    for k, val in over.items():
        setattr(a, k, val)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(rows=0), 1), (dict(groups=0), 1), (dict(width=-4), 1), (dict(dtype=2), 1), (dict(eps=0.0), 1),
    (dict(eps=float("nan")), 1), (dict(x=None), 1), (dict(groups=1 << 20, width=1 << 12), 2),
])
def test_group_norm_argument_errors(over, status):
    from burn_gdn2 import LIB, _lib

    fake = 1 << 20
    a = _norm_args(**over)
    assert LIB.gdn2_group_norm_gate(ctypes.byref(a), fake, None) == status
    assert LIB.gdn2_last_error().decode().startswith("gdn2_group_norm_gate:")
    b = _lib.GroupNormBwdArgs(a, fake, 32, fake, fake, fake, fake)
    assert LIB.gdn2_group_norm_gate_bwd(ctypes.byref(b), fake, 1 << 30, None) == status
    assert LIB.gdn2_group_norm_gate_bwd_workspace_bytes(ctypes.byref(b)) == 0


def test_group_norm_null_pointers_and_workspace():
    from burn_gdn2 import LIB, _lib

    fake = 1 << 20
    assert LIB.gdn2_group_norm_gate(None, fake, None) == _lib.GDN2_EINVAL
    assert LIB.gdn2_group_norm_gate(ctypes.byref(_norm_args()), None, None) == _lib.GDN2_EINVAL
    bwd = lambda a, *rest: _lib.GroupNormBwdArgs(a, *rest)
    call = lambda b, ws=None, n=0: LIB.gdn2_group_norm_gate_bwd(ctypes.byref(b), ws, n, None)
    assert LIB.gdn2_group_norm_gate_bwd(None, None, 0, None) == _lib.GDN2_EINVAL
    assert call(bwd(_norm_args(), None, 32, fake, fake, None, None)) == _lib.GDN2_EINVAL
    for absent, rest in ((dict(gate=None), (fake, fake, None, None)), (dict(weight=None), (fake, None, fake, None)),
                         (dict(bias=None), (fake, None, None, fake))):
        assert call(bwd(_norm_args(**absent), fake, 32, *rest)) == _lib.GDN2_EINVAL
    b = bwd(_norm_args(), fake, 32, fake, fake, fake, fake)
    need = LIB.gdn2_group_norm_gate_bwd_workspace_bytes(ctypes.byref(b))
    assert need > 0 and need % (2 * 32 * 4) == 0
    assert call(b, fake, need - 1) == _lib.GDN2_EWORKSPACE
    assert call(b) == _lib.GDN2_EWORKSPACE
    assert LIB.gdn2_group_norm_gate_bwd_workspace_bytes(ctypes.byref(bwd(_norm_args(), fake, 32, fake, fake, None, None))) == 0


def _conv_args(**over):
    from burn_gdn2 import _lib

    fake = 1 << 20
    a = _lib.ConvArgs(2, 40, 8, 0, None, _lib.View(fake, 320, 8, 0), fake, None)
    for k, val in over.items():
        setattr(a, k, val)
    return a


@pytest.mark.parametrize("over,status", [
    (dict(batch=0), 1), (dict(seq_len=0), 1), (dict(seq_len=-2), 1), (dict(channels=0), 1), (dict(dtype=3), 1),
    (dict(weight=None), 1), (dict(seq_len=(1 << 30) + 1), 2),
])
def test_conv_argument_errors(over, status):
    from burn_gdn2 import LIB, _lib

    out = _lib.View(1 << 20, 320, 8, 0)
    a = _conv_args(**over)
    assert LIB.gdn2_causal_conv(ctypes.byref(a), out, None, None) == status
    assert LIB.gdn2_last_error().decode().startswith("gdn2_causal_conv:")
    b = _lib.ConvBwdArgs(a, out, None, out, 1 << 20, None)
    assert LIB.gdn2_causal_conv_bwd(ctypes.byref(b), 1 << 20, 1 << 30, None) == status
    assert LIB.gdn2_causal_conv_bwd_workspace_bytes(ctypes.byref(b)) == 0


def test_conv_null_pointers_and_workspace():
    from burn_gdn2 import LIB, _lib

    fake = 1 << 20
    out, none = _lib.View(fake, 320, 8, 0), _lib.View()
    assert LIB.gdn2_causal_conv(None, out, None, None) == _lib.GDN2_EINVAL
    assert LIB.gdn2_causal_conv(ctypes.byref(_conv_args()), none, None, None) == _lib.GDN2_EINVAL
    assert LIB.gdn2_causal_conv(ctypes.byref(_conv_args(x=none)), out, None, None) == _lib.GDN2_EINVAL
    call = lambda *rest, ws=None, n=0: LIB.gdn2_causal_conv_bwd(ctypes.byref(_lib.ConvBwdArgs(_conv_args(), *rest)), ws, n, None)
    assert LIB.gdn2_causal_conv_bwd(None, None, 0, None) == _lib.GDN2_EINVAL
    assert call(none, None, out, None, None) == _lib.GDN2_EINVAL
    assert call(out, None, none, None, None) == _lib.GDN2_EINVAL
    assert call(out, None, out, None, fake) == _lib.GDN2_EINVAL  # d_cache_in without a cache
    b = _lib.ConvBwdArgs(_conv_args(), out, None, out, fake, None)
    need = LIB.gdn2_causal_conv_bwd_workspace_bytes(ctypes.byref(b))
    assert need > 0 and need % (8 * 4 * 4) == 0
    assert call(out, None, out, fake, None, ws=fake, n=need - 1) == _lib.GDN2_EWORKSPACE
    assert call(out, None, out, fake, None) == _lib.GDN2_EWORKSPACE


def test_state_rows_argument_errors():
    from burn_gdn2 import LIB, _lib

    fake = 1 << 20
    idx = ctypes.c_void_p(fake)

    def call(pairs, index=idx, src=4, dst=4, count=None):
        t = (_lib.StateRows * max(1, len(pairs)))(*pairs)
        return LIB.gdn2_move_state_rows(t, len(pairs) if count is None else count, index, src, dst, None)

    good = (fake, fake, 64)
    assert call([good], count=-1) == _lib.GDN2_EINVAL
    assert call([good], src=-1) == _lib.GDN2_EINVAL and call([good], dst=-1) == _lib.GDN2_EINVAL
    assert call([], count=0) == _lib.GDN2_OK and call([good], dst=0, src=0) == _lib.GDN2_OK  # nothing to do
    assert call([good], index=None) == _lib.GDN2_EINVAL
    assert LIB.gdn2_move_state_rows(None, 1, idx, 4, 4, None) == _lib.GDN2_EINVAL
    for bad in ((None, fake, 64), (fake, None, 64), (fake, fake, 0), (fake, fake, -16)):
        assert call([bad]) == _lib.GDN2_EINVAL
    assert call([good], src=4097, dst=4097) == _lib.GDN2_EUNSUPPORTED
    assert call([good], src=5, dst=4) == _lib.GDN2_EINVAL  # in place, rows differ
    assert call([good, (fake, fake + (1 << 16), 64)]) == _lib.GDN2_EINVAL  # in place and not
    assert call([(fake, fake + 3 * 64, 64)]) == _lib.GDN2_EINVAL  # overlap
    assert call([(fake + 3 * 64, fake, 64)]) == _lib.GDN2_EINVAL
    assert LIB.gdn2_last_error().decode().startswith("gdn2_move_state_rows:")


def test_pool_structures():
    import burn_gdn2 as bg
    from burn_gdn2 import sequence

    t = [torch.zeros(2, k + 1) for k in range(6)]
    state = bg.Gdn2State(*t[:4])
    nested = [state, (t[4], [t[5]])]
    flat = sequence._pool_tensors("op", nested)
    assert [a is b for a, b in zip(flat, t)] == [True] * 6 and len(flat) == 6
    again = sequence._pool_like(nested, iter(flat))
    assert isinstance(again[0], bg.Gdn2State) and again[0].conv_v is t[3] and again[1][1][0] is t[5]
    pair = collections.namedtuple("Pair", "cache state")(t[0], t[1])
    again = sequence._pool_like(pair, iter(sequence._pool_tensors("op", pair)))
    assert type(again) is type(pair) and again.cache is t[0] and again.state is t[1]
    with pytest.raises(TypeError):
        sequence._pool_tensors("op", {"a": 1})
    with pytest.raises(RuntimeError, match="CPU tensor"):
        bg.reorder_states(state, [0, 1])
