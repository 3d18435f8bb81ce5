"""What the Python calls of attention over a paged cache refuse before they hand out an address (CPU: nothing is launched)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tie_b200 import moe  # noqa: E402

CPU = -1  # torch's number of "no device": what a tensor here and a context there are compared by


def refused(call, *a, **k):
    with pytest.raises(moe.TieCudaError) as e:
        call(*a, **k)
    assert e.value.code == moe.EINVAL
    return str(e.value)


def rows(a, width, n):
    p, stride = moe._rows_ptr(a, width, n, CPU, "call", "q")
    assert p == a.data_ptr()
    return stride


def test_rows_of_a_tensor_are_where_its_first_dimension_puts_them():
    assert rows(torch.zeros(7, 5120), 4096, 7) == 5120  # a fused array handed over whole
    assert rows(torch.zeros(7, 5120), 4096, 5) == 5120
    assert rows(torch.zeros(7, 40, 128), 4096, 7) == 5120
    assert rows(torch.zeros(7, 4096), 4096, 7) == 4096
    assert rows(torch.zeros(7, 32, 128), 4096, 7) == 4096
    both = torch.zeros(7, 5120)
    assert rows(both[:, :4096], 4096, 7) == 5120 and rows(both[:, 4096:4608], 512, 7) == 5120
    assert rows(both[:1, :4096], 4096, 1) >= 4096
    assert rows(both[::2], 4096, 4) == 10240
    # rows one behind the other, whatever is in front
    assert rows(torch.zeros(7 * 4096), 4096, 7) == 4096
    assert rows(torch.zeros(7 * 32, 128), 4096, 7) == 4096
    assert rows(torch.zeros(1, 7, 4096), 4096, 7) == 4096
    assert rows(torch.zeros(1, 7, 32, 128), 4096, 7) == 4096
    assert rows(torch.zeros(0, 4096), 4096, 0) == 4096 and rows(torch.zeros(0), 64, 0) == 64
    assert moe._rows_ptr(4096, 64, 3, CPU, "call", "q") == (4096, 64)


@pytest.mark.parametrize("a, width, n", [
    (torch.zeros(7, 2048), 4096, 7), (torch.zeros(6, 4096), 4096, 7), (torch.zeros(1, 7, 5120), 4096, 7), (torch.zeros(7 * 4096 - 1), 4096, 7),
    (torch.zeros(7, 5120)[:, :4000], 4096, 7), (torch.zeros(6, 5120)[:, :4096], 4096, 7), (torch.zeros(7, 4096, dtype=torch.float16), 4096, 7),
    (torch.zeros(7, 4096, dtype=torch.int32), 4096, 7), (np.zeros((7, 4096), np.float32), 4096, 7), (torch.zeros(10, 3000), 4096, 7),
])
def test_rows_that_are_not_there_are_refused(a, width, n):
    refused(moe._rows_ptr, a, width, n, CPU, "call", "q")


def test_values_that_are_not_there_are_refused():
    assert moe._values_ptr(None, 5, CPU, "call", "x") is None and moe._values_ptr(64, 5, CPU, "call", "x") == 64
    x = torch.zeros(3, 4)
    assert moe._values_ptr(x, 12, CPU, "call", "x") == x.data_ptr()
    for a in (torch.zeros(11), x.half(), x.double(), x.int(), torch.zeros(4, 4)[:, :3], np.zeros(12, np.float32)):
        refused(moe._values_ptr, a, 12, CPU, "call", "x")
    assert "device" in refused(moe._values_ptr, x, 12, 0, "call", "x")  # a host tensor and a context on device 0
    assert "device" in refused(moe._rows_ptr, x, 4, 3, 0, "call", "x")


def cache(kind, dtype, scale=None):
    k, v = (torch.zeros(2, 1, 16, 64, dtype=dtype) for _ in range(2))
    s = (torch.zeros(2, 1, 16, dtype=scale) for _ in range(2)) if scale else (None, None)
    return moe.KvCache(kind, k, v, *s)


@pytest.mark.parametrize("kind, dtype, scale", [
    (moe.KV_F16, torch.bfloat16, None), (moe.KV_F16, torch.float32, None), (moe.KV_BF16, torch.float16, None), (moe.KV_BF16, torch.int8, None),
    (moe.KV_Q8, torch.float16, torch.float32), (moe.KV_Q8, torch.int32, torch.float32),
])
def test_caches_of_another_type_are_refused(kind, dtype, scale):
    assert "is not on" not in refused(cache, kind, dtype, scale)


def test_factors_of_another_type_are_refused_and_what_fits_must_be_on_the_device():
    for kind, dtype, scale in ((moe.KV_F16, torch.float16, None), (moe.KV_BF16, torch.int16, None), (moe.KV_Q8, torch.int8, torch.float16)):
        assert "k is not on the device" in refused(cache, kind, dtype, scale)

    class OnDevice:  # (a tensor on no device that says it is on one)
        is_cuda, dtype, shape = True, torch.int8, (2, 1, 16, 64)

        def __init__(self, dtype=torch.int8, shape=(2, 1, 16, 64)):
            self.dtype, self.shape = dtype, shape

        def is_contiguous(self):
            return True

        def data_ptr(self):
            return 4096

    factors = OnDevice(torch.float32, (2, 1, 16))
    assert moe.KvCache(moe.KV_Q8, OnDevice(), OnDevice(), factors, factors).n_pages == 2
    half = OnDevice(torch.float16, (2, 1, 16))
    assert "k_scale" in refused(moe.KvCache, moe.KV_Q8, OnDevice(), OnDevice(), half, factors)
    assert "v_scale" in refused(moe.KvCache, moe.KV_Q8, OnDevice(), OnDevice(), factors, half)
    # a step's arrays: 64-bit numbers are what torch makes by default
    i32 = lambda *shape: OnDevice(torch.int32, shape)  # noqa: E731
    i64 = lambda *shape: OnDevice(torch.int64, shape)  # noqa: E731
    assert moe.KvStep(i32(3), i32(2), i32(2, 4), 5, tree=i64(5), pos=i32(5)).max_pages == 4
    for name, a in (("tok_start", (i64(3), i32(2), i32(2, 4))), ("kv_len", (i32(3), i64(2), i32(2, 4))), ("page_table", (i32(3), i32(2), i64(2, 4)))):
        assert name in refused(moe.KvStep, *a, 5)
    assert "tree" in refused(moe.KvStep, i32(3), i32(2), i32(2, 4), 5, tree=i32(5))
    assert "pos" in refused(moe.KvStep, i32(3), i32(2), i32(2, 4), 5, pos=i64(5))
    host = torch.zeros(3, dtype=torch.int32)
    assert "device" in refused(moe.KvStep, host, i32(2), i32(2, 4), 5)


def test_the_packed_description_is_the_structures():
    values = (32, 1 << 40, 2, 3, -4, 5, 6, 7, 8, 1e-6, 1e6, 1, 1 << 41)
    s = moe.AttnQkv(*values)
    assert moe._QKV.pack(*values) == bytes(s)
