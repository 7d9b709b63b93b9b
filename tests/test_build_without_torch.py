"""CPU: build.py on a machine without torch builds the C ABI library and says that the torch extension is left out."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import sys
sys.path.insert(0, {path!r})
if {blocked!r}:
    sys.modules["torch"] = None  # as where it is not installed
import build
calls = []
class Ran:
    returncode, stdout, stderr = 0, "", ""
build.subprocess.run = lambda cmd, **kw: calls.append(cmd) or Ran()
build.LIB, build.CALLS = {tmp!r} + "/lib.so", {tmp!r} + "/_torch_calls.so"
build.BUILD = {tmp!r}
assert build.build() == build.LIB
print("nvcc", sum("nvcc" in c[0] for c in calls) > 1, "g++", sum(c[0] == "g++" for c in calls))
"""


def _build(tmp, blocked):
    code = CODE.format(path=os.path.join(ROOT, "burn-gdn2_b200"), tmp=str(tmp), blocked=blocked)
    code = code.replace("import build\n", "import build\nbuild._digest = lambda paths, extra: '0'\n")  # no objects are made
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)


def test_without_torch(tmp_path):
    r = _build(tmp_path, True)
    assert r.returncode == 0, r.stderr
    assert "nvcc True g++ 0" in r.stdout and "torch is not installed" in r.stdout


def test_with_torch(tmp_path):
    r = _build(tmp_path, False)
    assert r.returncode == 0, r.stderr
    assert "nvcc True g++ 1" in r.stdout and "not installed" not in r.stdout
