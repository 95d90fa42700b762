"""The bindings depend on the torch and the Python that they were built for; the
library, and the dense operators with it, do not.  CPU only."""
import os
import subprocess
import sys

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "iris-kernel_b200")


def _python(code):
    return subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {PKG!r})\n{code}"], text=True,
                          capture_output=True)


def test_dense_operators_without_the_bindings():
    """A bindings file that cannot be loaded stops the calls that need it, with
    its own message, and nothing else."""
    r = _python("""
sys.modules["iris_kernel._ops"] = None  # an import of it fails
import torch
import iris_kernel, iris_kernel.step
from iris_kernel import _lib, fused_attention, fused_kv, sparse_attention
assert _lib.lib.iris_b200_version() > 0
fused_kv.fused_rope_int4_paged_append, fused_attention.fused_int4_paged_decode_attention
x, one = torch.zeros(1, 1, 64, dtype=torch.float16), torch.ones(1, dtype=torch.int32)
try:
    sparse_attention.fused_page_select(x, x, x, x, one, max_pages=2)
except ImportError:
    print("refused")
""")
    assert r.returncode == 0 and r.stdout.strip() == "refused", r.stderr


def test_bindings_of_another_torch_are_not_loaded(tmp_path):
    path = tmp_path / "_ops.stamp"
    path.write_text("torch 1.0.0, cpython-38-x86_64-linux-gnu\n")
    r = _python(f"""
from iris_kernel import _runtime, _stamp
real = _stamp.built
_stamp.built = lambda: real({str(path)!r})
try:
    _runtime.ops()
except ImportError as e:
    assert "build.py" in str(e) and "iris_kernel._ops" not in sys.modules
    print("refused")
_stamp.built = real
print(_runtime.ops().__name__)
""")
    assert r.returncode == 0 and r.stdout.split() == ["refused", "iris_kernel._ops"], r.stderr


def test_build_is_stale_where_torch_or_python_is_another_one():
    r = _python("""
import build
real = build._stamp
for other in ("torch 1.0.0, cpython-38-x86_64-linux-gnu", None):
    def changed():
        m = real()
        m.built = lambda: other
        return m
    build._stamp = changed
    assert build._stale()
""")
    assert r.returncode == 0, r.stderr
