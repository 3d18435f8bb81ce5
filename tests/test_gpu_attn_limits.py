"""Attention over the paged cache where values, their factors or their probabilities lie far apart: against plain arithmetic in 64
bits, with the bounds of test_gpu_attn.py (its head derives them), each row's relative to the largest value that this row sees.
Kernels: `far` False, few rows or short caches; True, tiles of 128 rows."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attn import World, trees  # noqa: E402


@pytest.fixture(scope="module")
def be():
    from tie_b200 import moe
    b = moe.MoeBackend(hidden=256, n_expert=16, top_k=1, ffn_dim=256, max_tokens=64)
    yield b
    b.close()


def factor_at(w, s, slot, up):
    pg, pl = w.slots(s, slot, slot + 1)
    w.v_scale[int(pg[0]), :, int(pl[0])] *= up


# Up to 16 rows, more of them in tiles of 16 and of 128; a tree, tokens one behind the other, enough of these for a warp to have groups of
# keys behind the one with the large factor.
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("up", [200.0, 2.0 ** 13, 1e6, 1e12, 1e37])
@pytest.mark.parametrize("toks, lens, heads, kv_heads, drafted", [
    ([3, 2], [37, 200], 8, 2, True), ([12, 5], [37, 3], 8, 2, True), ([64], [100], 4, 2, True), ([9, 30], [40, 15], 8, 2, False), ([300], [0], 2, 2, False),
])
def test_a_large_factor_that_a_row_does_not_see_is_nothing_to_it(be, far, dim, up, toks, lens, heads, kv_heads, drafted):
    w = World(60, "q8", toks, lens, heads, kv_heads, dim, 16, tree=trees(np.random.default_rng(2), toks) if drafted else None, far=far)
    for s, t in enumerate(toks):
        factor_at(w, s, lens[s] + t // 2, up)
    q, out, scale = w.attn(be)
    w.check_attn(q, out, scale)


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("up", [1e6, 1e12])
def test_factors_that_grow_from_token_to_token(be, far, up):
    """Token i sees factors up to its own alone; and the same the other way round, where the largest comes first."""
    for order in (1, -1):
        w = World(61, "q8", [40], [60], 8, 2, 128, 16, far=far)
        for i in range(40):
            factor_at(w, 0, 60 + i, up ** ((i if order > 0 else 39 - i) / 39))
        q, out, scale = w.attn(be)
        w.check_attn(q, out, scale)


# Values of up to 2^126 and down to 2^-100 in one CTA's keys, in keys of several CTAs that are joined, and in items of their own.
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("power", [122, -100])
@pytest.mark.parametrize("toks, lens, drafted", [([1], [300], False), ([1, 2], [5000, 40], False), ([20, 3], [700, 9], True), ([600], [64], False)])
def test_q8_values_of_any_size(be, far, power, toks, lens, drafted):
    w = World(62, "q8", toks, lens, 16, 2, 128, 32, tree=trees(np.random.default_rng(3), toks) if drafted else None, far=far)
    w.v_scale *= 2.0 ** power
    q, out, scale = w.attn(be)
    assert out.isfinite().all()
    w.check_attn(q, out, scale)


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("power", [124, -80])
@pytest.mark.parametrize("toks, lens, drafted", [([1], [300], False), ([1, 2], [5000, 40], False), ([20, 3], [700, 9], True), ([600], [64], False)])
def test_bf16_values_of_any_size(be, far, power, toks, lens, drafted):
    w = World(63, "bf16", toks, lens, 16, 2, 64, 32, tree=trees(np.random.default_rng(3), toks) if drafted else None, far=far)
    w.v = (w.v.float() * 2.0 ** power).bfloat16()
    assert w.v.isfinite().all()
    w.describe()
    q, out, scale = w.attn(be)
    assert out.isfinite().all()
    w.check_attn(q, out, scale)


# A key with a value that is no number, of a score so low that its p is 0: in front of the step (another warp's or CTA's keys than those that
# count), among the step's own tokens (of which not every row sees all).
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("toks, lens, drafted, slot", [
    ([1], [300], False, 7), ([1], [5000], False, 4800), ([30], [100], False, 110), ([30], [100], False, 3), ([30], [40], True, 45), ([64], [2000], True, 1000), ([200], [900], False, 1000),
])
def test_a_value_that_is_no_number_is_seen_where_its_probability_is_nothing(be, far, kind, bad, toks, lens, drafted, slot):
    w = World(64, kind, toks, lens, 8, 1, 64, 16, tree=trees(np.random.default_rng(4), toks) if drafted else None, far=far)
    q = torch.tensor(w.rng.standard_normal((w.rows, 8, 64)), dtype=torch.float32).cuda() + 1.0
    # every query is about 1 in each dim: this key's scores are about -64 * 4 * scale below the others'
    pg, pl = (int(x[0]) for x in w.slots(0, slot, slot + 1))
    w.k[pg, :, pl] = -120 if kind == "q8" else -40
    if kind == "q8":
        w.k_scale[pg, :, pl] = 1.0 / 3
    _, clean, scale = w.attn(be, q, 1.0)
    sees = torch.tensor(w.sees(0, 0)[:, slot]).cuda()
    assert sees.any() and clean.isfinite().all()
    if kind == "q8":
        w.v_scale[pg, :, pl] = bad
    else:
        w.v[pg, :, pl, 5] = bad
    _, out, _ = w.attn(be, q, 1.0)
    hit = out[sees] if kind == "q8" else out[sees][..., 5:6]
    assert not hit.isfinite().any()
    rest = out.clone()
    if kind == "q8":
        rest[sees] = clean[sees]
    else:
        rest[sees, :, 5] = clean[sees, :, 5]
    # the others' products may be made one by one: another order of the same sums
    assert (rest - clean).abs().max() <= 2.0 ** -17 * w.v_scale[w.v_scale.isfinite()].abs().max() * 127 if kind == "q8" else \
        (rest - clean).abs().max() <= 2.0 ** -17 * 8
