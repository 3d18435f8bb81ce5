"""How many parts of an operand the attention kernels need, on the CPU: their operands alone, rounded as they round them, sums in 64 bits.

The bound that test_gpu_attn_precision.py holds them to, 2^-19 of the outputs' rms over a launch, is above what all parts leave and below
what is left where any one of them is missing - but for the third bf16 part of p where parts are rounded: without it 2^-17 / (sqrt 12 * 1.5), 2^-19.4, are
left, about as much as fp32 sums leave, so that no bound on the outputs tells it from them."""
import numpy as np
import pytest

BOUND = 2.0 ** -19


def bf16(x, cut):
    b = x.astype(np.float32).view(np.uint32)
    b = b & 0xffff0000 if cut else (b + 0x7fff + (b >> 16 & 1)) & 0xffff0000
    return b.astype(np.uint32).view(np.float32)


def parts(x, kind, n, cut=False):
    """The first n parts of fp32 values, added up."""
    x = x.astype(np.float32)
    total = np.zeros(x.shape)
    for _ in range(n):
        p = bf16(x, cut) if kind == "bf16" else x.astype(np.float16).astype(np.float32)
        total += p
        x = x - p
    return total


def held_rows(q, kind, n, way):
    """Rows of queries as the kernels hold them: `way` "parts" (fp16 ones after the row is brought to 1 .. 2), or "bytes" of Q8's few rows."""
    if way == "bytes":
        unit = np.abs(q).max(-1, keepdims=True) / (127 * 65536)
        w = np.rint(q / unit)
        return unit * (w if n == 3 else np.rint(w / 256) * 256)
    scale = 1.0 if kind == "bf16" else 2.0 ** np.floor(np.log2(np.abs(q).max(-1, keepdims=True)))
    return parts(q / scale, kind, n, way == "cut") * scale


def error(kind, way, keys, q_parts, p_parts):
    rng = np.random.default_rng(keys)
    q = (rng.standard_normal((64, 128)) * 2).astype(np.float32)
    k, v = rng.standard_normal((keys, 128)), rng.standard_normal((keys, 128))

    def attend(x, hold):
        s = x @ k.T / np.sqrt(128)
        p = np.exp(s - s.max(-1, keepdims=True))
        return hold(p) @ v / p.sum(-1, keepdims=True)

    shift = 2.0 ** (-15 if kind == "bf16" else 14)
    want = attend(q.astype(np.float64), lambda p: p)
    got = attend(held_rows(q.astype(np.float64), kind, q_parts, way), lambda p: parts(p * shift, kind, p_parts, way == "cut") / shift)
    return np.sqrt(((got - want) ** 2).mean() / (want ** 2).mean())


WAYS = [("f16", "parts", 2, 2), ("q8", "bytes", 3, 2), ("q8", "parts", 2, 2), ("bf16", "parts", 3, 3), ("bf16", "cut", 3, 3)]


@pytest.mark.parametrize("keys", [128, 640, 9001])
@pytest.mark.parametrize("kind, way, nq, np_", WAYS)
def test_each_part_counts(kind, way, nq, np_, keys):
    assert error(kind, way, keys, nq, np_) < BOUND / 4
    assert error(kind, way, keys, nq - 1, np_) > BOUND
    assert error(kind, way, keys, nq, np_ - 1) > (BOUND * 0.7 if (kind, way) == ("bf16", "parts") else BOUND)
