"""A kernel library made before whole rows of candidates (include/gvk.h gvk_block_* ... gvk_distill_grad) loads and trains as it did; what it
lacks it names when it is called.  The host build of the engine (tests/hostdev) is such a library."""
import os
import subprocess
import sys

import pytest

from graphvite_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOST_LIBRARY = os.path.join(ROOT, "tests", "hostdev", "build", "libgvk_host.so")
WHOLE_ROWS = ("gvk_block_quantize", "gvk_block_dequantize", "gvk_block_logits_workspace", "gvk_block_logits", "gvk_top_logits_workspace",
              "gvk_top_logits", "gvk_distill_workspace", "gvk_distill", "gvk_distill_grad_workspace", "gvk_distill_grad")

EARLIER = """
import ctypes
from graphvite_amd import _lib
names = %r
plain = ctypes.CDLL(_lib.LIB_PATH)
assert not any(hasattr(plain, name) for name in names), "the host build has whole rows: no earlier library"
lib = _lib.lib()
assert lib.gvk_version() and lib.gvk_train.argtypes
for name in names:
    try:
        getattr(lib, name)(1, 2, 3)
    except _lib.NativeLibraryError as e:
        assert name in str(e) and _lib.LIB_PATH in str(e), e
    else:
        raise AssertionError(name)
print("loaded")
""" % (WHOLE_ROWS,)


def test_an_earlier_library_loads_and_names_what_it_lacks():
    subprocess.check_call(["make", "-s", "-C", os.path.join(ROOT, "oracle"), os.path.join(ROOT, "oracle", "liboracle.so")])
    subprocess.check_call(["make", "-s", "-C", os.path.join(ROOT, "tests", "hostdev")])
    env = dict(os.environ, GVK_LIBRARY=HOST_LIBRARY, GVK_ALLOW_TEST_LIBRARY="1", PYTHONPATH=ROOT)
    run = subprocess.run([sys.executable, "-c", EARLIER], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "loaded" in run.stdout, run.stdout + run.stderr


@pytest.mark.parametrize("name", WHOLE_ROWS)
def test_the_product_has_them_all(name):
    function = getattr(_lib.lib(), name)
    assert function.argtypes and function.restype is not None
