"""What rope, qk_norm_rope, linear_xent and their neighbours refuse at their borders, before any HIP
call (no GPU needed)."""
import ctypes
import os

import pytest

gn = pytest.importorskip("gn_bwd")
if not os.path.exists(gn.LIB_PATH):
    pytest.skip("libgn_bwd.so not built", allow_module_level=True)

BASE = 1 << 30  # addresses that are never read: the checks come first
MB = 1 << 20


def p(off=0):
    return ctypes.c_void_p(BASE + off)


def refused(rc, text, code=-1):
    assert rc == code and text in gn.last_error(), (rc, gn.last_error())


@pytest.mark.parametrize("T,d,V", [(1 << 23, 8, 1 << 20), (1 << 27, 8, 1 << 16), (1 << 22, 1 << 20, 1 << 20)])
def test_more_tiles_than_a_product_counts(T, d, V):
    lib = gn.lib()
    refused(lib.gn_linear_xent_fwd(p(), p(), p(), p(), None, T, d, V, 4, p(), 1, None), "2^43")
    refused(lib.gn_linear_xent_bwd(p(), p(), p(), p(), None, None, 1.0, p(), p(), 0, T, d, V, 4, 0, p(), 1, None), "2^43")
