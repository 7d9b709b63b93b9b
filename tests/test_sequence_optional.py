"""CPU: without the torch extension of the sequence operators (not built, or built for another torch) the package is
there all the same; the operators say what is missing, the training layer warns."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _python(code):
    path = os.pathsep.join([os.path.join(ROOT, "burn-gdn2_b200"), os.path.join(ROOT, "tests")])
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": path}, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def test_the_package_imports_without_the_extension():
    out = _python("""
import sys
sys.modules["burn_gdn2._torch_calls"] = None  # as if it were not there
import torch, warnings
import burn_gdn2 as bg
from burn_gdn2 import sequence, training
x = torch.zeros(1, 4, 8)
state = bg.Gdn2State(*(torch.zeros(2, 3) for _ in range(4)))
calls = [lambda: bg.gated_scan(x, x), lambda: bg.causal_conv_silu(x, torch.zeros(8, 4)),
         lambda: bg.group_norm_gate(x, num_groups=2), lambda: bg.reorder_states(x, [0]), lambda: state.select([0, 1])]
for call in calls:
    try:
        call()
    except ImportError as e:
        assert "build.py" in str(e), e
    else:
        raise AssertionError("no ImportError")
assert not sequence.available()
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter("always")
    assert not training.on_operators()
assert len(seen) == 1 and "build.py" in str(seen[0].message)
print(bg.Gdn2Config.__name__)
""")
    assert out.strip() == "Gdn2Config"


def test_with_the_extension():
    from burn_gdn2 import sequence, training

    assert sequence.available() and training.on_operators()


def test_an_extension_of_another_torch_is_not_used():
    out = _python("""
import sys, types
other = types.ModuleType("burn_gdn2._torch_calls")
other.torch_version = "1.0.0"
sys.modules["burn_gdn2._torch_calls"] = other
import torch
import burn_gdn2 as bg
try:
    bg.gated_scan(torch.zeros(1, 4, 8), torch.zeros(1, 4, 8))
except ImportError as e:
    print("1.0.0" in str(e.__cause__))
""")
    assert out.strip() == "True"


def test_release_numbers():
    from burn_gdn2 import sequence

    for version, want in (("2.11.0+cu128", "2.11.0"), ("2.12.0a0+gitabc", "2.12.0"), ("2.12.0.dev20260101", "2.12.0"), ("2.11.1", "2.11.1")):
        assert sequence._release(version) == want
