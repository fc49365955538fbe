"""The argument arrays of launch_device, without a GPU: addresses and sizes as ctypes takes them."""
import ctypes

import numpy as np
import pytest

from ascend_mlir_b200 import descriptors
from ascend_mlir_b200.runtime import ExecutorError
from ascend_mlir_b200.runtime.executor import CudaRuntime, _packed


def words(values, kind):
    return bytes((kind * len(values))(*values))


@pytest.mark.parametrize("address", [0, None, 4096, 2 ** 64 - 1, -1, np.int64(4096), np.uint64(2 ** 63), ctypes.c_void_p(4096), ctypes.c_void_p(None)],
                         ids=repr)
@pytest.mark.parametrize("size", [0, 1, 2 ** 64 - 1, -1, np.int64(12)], ids=repr)
def test_words(address, size):
    pairs = [(8192, 16), (address, size), (12288, 32)]
    try:
        want = words([p for p, _ in pairs], ctypes.c_void_p), words([n for _, n in pairs], ctypes.c_size_t)
    except TypeError:
        pytest.skip("ctypes takes no such value")
    assert _packed(pairs) == want


def test_no_arguments():
    assert _packed([]) == (b"", b"") and _packed(()) == (b"", b"")


def test_a_launch_with_address_objects():
    """Addresses as ctypes pointers reach the launch (and fail there where there is no GPU, or as null ones)."""
    rt = CudaRuntime()
    rt.set_device(0)
    spec = descriptors.add_mul("f32")
    null = (ctypes.c_void_p(None), 16)
    with pytest.raises(ExecutorError, match="null"):
        rt.launch_device(spec.binary, spec.name, [null] * 2, [null], spec.pack({"M": 1, "N": 4}))
