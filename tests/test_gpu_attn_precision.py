"""Errors of attention over the paged cache as a whole: their rms over a launch relative to the outputs', where test_gpu_attn.py bounds
each output's by the worst case.

Bound 2^-19, from the arithmetic for these inputs (queries of 2, keys and values of 1, normal: scores of 2.9 rms in powers of two, up to 16;
an error d of an exponent is one of 0.69 d in p, and errors of p that differ from key to key are the outputs' relative error):
* 8 sums of a score are cut off at 24 bits of a partial sum (2^-22 for 2 to 4): half of that each, 8 * 2^-23 * 0.69 = 2^-20.5;
* four roundings of numbers of up to 16 (sum of parts, factor, base, difference), rms 2^-21 / sqrt 3 each: 2 * 2^-21.8 * 0.69 = 2^-21.3;
* parts of q 2^-23 of each product, rms 2^-23 * 2.9 = 2^-21.5; parts of p and exp2, 2^-22 each; sums of p v, 2^-22.
Together 2^-19.6 as roots of squares, 2^-19 with half a bit to spare.  test_attn_parts.py: what a missing part would leave."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attn import KINDS, World, trees  # noqa: E402


@pytest.fixture(scope="module")
def be():
    from tie_b200 import moe
    b = moe.MoeBackend(hidden=256, n_expert=16, top_k=1, ffn_dim=256, max_tokens=64)
    yield b
    b.close()


def rms_error(w, q, out, scale):
    off = size = 0.0
    row, g = 0, w.heads // w.kv_heads
    for s, t in enumerate(w.toks):
        k, v, m = (torch.tensor(x).cuda() for x in (w.sequence("k", s), w.sequence("v", s), w.sees(s, row)))
        for h in range(w.heads):
            want = torch.softmax((q[row:row + t, h].double() @ k[:, h // g].T * scale).masked_fill(~m, -float("inf")), 1) @ v[:, h // g]
            off += float(((out[row:row + t, h].double() - want) ** 2).sum())
            size += float((want ** 2).sum())
        row += t
    return (off / size) ** 0.5


# Few rows: one token, up to 16 rows; tiles: trees and prompt pieces.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("toks, lens, drafted", [
    ([1], [127], False), ([1, 1, 1], [639, 200, 300], False), ([1], [9000], False), ([1, 1], [40000, 100], False), ([4], [2000], True),
    ([64], [128], True), ([13], [9001], True), ([64, 30], [3500, 1000], True), ([200], [440], False), ([300, 100], [0, 9000], False),
])
def test_errors_are_those_of_fp32(be, kind, dim, toks, lens, drafted):
    w = World(80, kind, toks, lens, 32, 8, dim, 64, tree=trees(np.random.default_rng(6), toks) if drafted else None, far=True)
    q, out, scale = w.attn(be, scale=dim ** -0.5)
    err = rms_error(w, q, out, scale)
    print(f"{kind} {dim} {toks} {lens}: {err:.2e}")
    assert err <= 2.0 ** -19
