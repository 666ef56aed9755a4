"""Refusals of the experts' call with shared outputs that need no GPU."""
import ctypes

from agillm41_b200 import _lib

FAKE = ctypes.c_void_p(4096)   # never read: the checks come first
ODD = ctypes.c_void_p(4096 + 8)


def test_shared_arguments():
    lib = _lib.load()

    def call(shared, n_shared, d=128):
        return lib.agm_moe_experts_fp8_shared(FAKE, _lib.AGM_BF16, 64, d, 14, 2, 256, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE,
                                              FAKE, None, shared, n_shared, FAKE, FAKE, 1 << 40, None)

    assert call(FAKE, -1) == -1 and "n_shared" in lib.agm_last_error().decode()
    assert call(None, 2) == -1
    assert call(ODD, 2) == -1 and "aligned" in lib.agm_last_error().decode()
    assert call(None, 0, d=24) == -2
