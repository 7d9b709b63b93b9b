"""CPU: the Rust dispatch (rust/src/kernel/gdn2_dispatch.rs, not compiled here) tells the device error bits apart: a wait
that gave up stops the core call after which it is read, a row number outside a state pool is kept for its own caller."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _text(*path):
    return open(os.path.join(ROOT, *path)).read()


def test_the_bits_are_the_kernels():
    enum = re.search(r"enum : unsigned \{(.*?)\};", _text("burn-gdn2_b200", "csrc", "ptx.cuh"), re.S).group(1)
    bits = {n: int(v) for n, v in re.findall(r"(DEVERR_\w+) = (\d+)u", enum)}
    rust = _text("rust", "src", "kernel", "gdn2_b200.rs")
    header = _text("include", "gdn2.h")
    for name, kernel in (("GDN2_DEVERR_WAIT", "DEVERR_MBAR_TIMEOUT"), ("GDN2_DEVERR_STATE_INDEX", "DEVERR_STATE_INDEX")):
        assert f"pub const {name}: u32 = {bits[kernel]};" in rust
        assert re.search(rf"#define {name} {bits[kernel]}u\b", header)


def _body(src, start):
    body = src[src.index(start):]
    return body[:body.index("\n}")]


def test_a_core_call_does_not_trip_over_a_pool_s_bit():
    src = _text("rust", "src", "kernel", "gdn2_dispatch.rs")
    assert "assert!(flags & GDN2_DEVERR_WAIT == 0," in _body(src, "fn stop_on_wait") and "flags == 0" not in src
    for name in ("fn run_on_device", "pub fn take_state_index_error"):  # whoever reads the word loses neither bit
        body = _body(src, name)
        assert "gdn2_read_device_errors(&mut flags)" in body and "stop_on_wait(flags)" in body
    assert "POOL_ERRORS.fetch_or(flags & GDN2_DEVERR_STATE_INDEX" in _body(src, "fn run_on_device")
    take = _body(src, "pub fn take_state_index_error")
    assert "POOL_ERRORS.swap(0" in take and "(flags | kept) & GDN2_DEVERR_STATE_INDEX != 0" in take
    assert take.index("POOL_ERRORS.swap") > take.index("gdn2_read_device_errors")
