"""Steps that are wrong in one sequence: the call says so, the other sequences' rows and slots are right, and nothing else is written.
Bounds as in test_gpu_attn.py."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attn import KINDS, World, plain_write, trees  # noqa: E402

MARK = 7.25


@pytest.fixture(scope="module")
def be():
    from tie_b200 import moe
    b = moe.MoeBackend(hidden=256, n_expert=16, top_k=1, ffn_dim=256, max_tokens=64)
    yield b
    b.close()


def check_sequence(w, s, q, out, scale, lost=()):
    """Rows of sequence s against 64 bits, `lost` slots seen by nobody."""
    row, g = sum(w.toks[:s]), w.heads // w.kv_heads
    k, v, m = w.sequence("k", s), w.sequence("v", s), w.sees(s, row)
    m[:, list(lost)] = False
    q, out = q.double().cpu().numpy(), out.double().cpu().numpy()
    for i in range(w.toks[s]):
        for h in range(w.heads):
            kk, vv, x = k[m[i], h // g], v[m[i], h // g], q[row + i, h]
            score = scale * (kk @ x)
            p = np.exp(score - score.max())
            tol = (1.0 + abs(scale) * (np.abs(kk) @ np.abs(x)).max()) * 2.0 ** -17 * np.abs(vv).max()
            assert np.abs(out[row + i, h] - p @ vv / p.sum()).max() <= tol, (s, i, h)


HOW = {  # sequences that are right all the same
    "page": [0, 2], "page_high": [0, 2], "len": [0, 2], "len_far": [0, 2], "room": [0, 2], "rows": [0, 1], "start": [1, 2],
}


def spoilt(kind, how, far):
    w = World(70, kind, [2, 3, 2], [70, 33, 20], 32 if far else 8, 2, 64, 16, pad=2, far=far)
    if how == "page":
        w.d_table[1, 0] = -1
    elif how == "page_high":
        w.d_table[1, 2] = w.k.shape[0]
    elif how == "len":
        w.kv_len[1] = -5
    elif how == "len_far":
        w.kv_len[1] = 1 << 30
    elif how == "room":  # a slot for the first token alone
        w.kv_len[1] = w.table.shape[1] * 16 - 1
    elif how == "rows":
        w.tok_start[3] = 99
    else:
        w.tok_start[0] = -3
    bad = {"rows": [2], "start": [0]}.get(how, [1])
    rows = [r for s in bad for r in range(sum(w.toks[:s]), sum(w.toks[:s + 1]))]
    return w, rows[1:] if how == "room" else [] if "page" in how else rows  # rows that have no slot


def refused(call, *a, **k):
    from tie_b200 import moe
    with pytest.raises(moe.TieCudaError) as e:
        call(*a, **k)
    assert e.value.code == moe.EKERNEL and ("page" in str(e.value) or "step" in str(e.value))


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("how", list(HOW))
def test_attention_leaves_out_what_is_wrong_alone(be, far, kind, how):
    w, none = spoilt(kind, how, far)
    q = torch.tensor(w.rng.standard_normal((w.rows, w.heads, 64)) * 2, dtype=torch.float32).cuda()
    out = torch.full_like(q, MARK)
    refused(w.attn, be, q, 0.125, out=out)
    for s in HOW[how]:
        check_sequence(w, s, q, out, 0.125)
    if "page" in how:
        check_sequence(w, 1, q, out, 0.125, lost=range(16) if how == "page" else range(32, 36))
    assert (out[none + [7, 8]] == MARK).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("how", [h for h in HOW if h != "page"])
def test_writing_and_reading_leave_out_what_is_wrong_alone(be, kind, how):
    w, none = spoilt(kind, how, False)
    heads, rng = 8, np.random.default_rng(3)
    q, k, v = (torch.tensor(rng.standard_normal((w.rows, h, 64)), dtype=torch.float32).cuda() for h in (heads, 2, 2))
    names = ["k", "v"] + (["k_scale", "v_scale"] if kind == "q8" else [])
    before = {n: getattr(w, n).clone() for n in names}
    q_out = torch.full_like(q, MARK)
    torch.cuda.synchronize()
    refused(be.qk_norm_rope_ptr, w.cache, w.step, q, k, v, q_out, heads, rope_base=1e4)
    assert (q_out[none + [7, 8]] == MARK).all()
    right = [(s, sum(w.toks[:s]) + i, w.lens[s] + i) for s in HOW[how] for i in range(w.toks[s])]
    want = plain_write(q.double().cpu().numpy()[[r for _, r, _ in right]], None, 0, [x for _, _, x in right], 1e4, False)
    got = q_out.double().cpu().numpy()[[r for _, r, _ in right]]
    assert (np.abs(got - want) <= np.abs(want).max(-1, keepdims=True) * math.sqrt(2) * 2.0 ** -19).all()
    read = [torch.full((w.rows, 2, 64), MARK, device="cuda") for _ in range(2)]
    refused(be.kv_read_ptr, w.cache, w.step, *read)
    lost = none if "page" not in how else [2, 3, 4]
    for x in read:
        assert (x[lost + [7, 8]] == MARK).all()
    for s, row, slot in right:
        pg, pl = (int(x[0]) for x in w.slots(s, slot, slot + 1))
        for n, x in zip("kv", read):
            held = w.held(n)[pg, :, pl]
            assert np.array_equal(x[row].cpu(), torch.tensor(held).float())
            assert not torch.equal(getattr(w, n)[pg, :, pl], before[n][pg, :, pl])
        for n in names:
            getattr(w, n)[pg, :, pl] = before[n][pg, :, pl]
    if how == "room":  # (the one slot of its first token)
        pg, pl = int(w.table[1, -1]), 15
        for n in names:
            getattr(w, n)[pg, :, pl] = before[n][pg, :, pl]
    for n in names:
        assert torch.equal(getattr(w, n), before[n])  # no other slot


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_a_tree_of_too_many_tokens_is_its_own_affair(be, far, kind):
    toks = [3, 70, 5]
    tree = trees(np.random.default_rng(1), [3]) + [1] * 70 + trees(np.random.default_rng(2), [5])
    w = World(71, kind, toks, [40, 33, 7], 8, 2, 64, 16, tree=tree, far=far)
    q = torch.tensor(w.rng.standard_normal((w.rows, 8, 64)) * 2, dtype=torch.float32).cuda()
    out = torch.full_like(q, MARK)
    refused(w.attn, be, q, 0.125, out=out)
    for s in (0, 2):
        check_sequence(w, s, q, out, 0.125)


def test_a_fused_array_may_be_handed_over_whole(be):
    """q's rows are the first values of the rows of a contiguous array that holds k and v behind them."""
    w = World(72, "f16", [2, 5], [3, 30], 8, 2, 64, 16)
    both = torch.tensor(w.rng.standard_normal((7, 12 * 64)), dtype=torch.float32).cuda()
    k, v = both[:, 8 * 64:10 * 64], both[:, 10 * 64:]
    outs = []
    for q in (both[:, :8 * 64].contiguous(), both[:, :8 * 64], both, both.view(7, 12, 64)):
        outs.append(torch.empty(7, 8, 64, device="cuda"))
        torch.cuda.synchronize()
        be.qk_norm_rope_ptr(w.cache, w.step, q, k, v, outs[-1], 8)
    assert all(torch.equal(o, outs[0]) for o in outs[1:])


def test_arrays_that_do_not_fit_are_refused_before_a_kernel_sees_them(be):
    from tie_b200 import moe
    w = World(73, "f16", [2, 5], [3, 30], 8, 2, 64, 16)
    q, kv = torch.zeros(7, 8, 64, device="cuda"), torch.zeros(7, 2, 64, device="cuda")
    before = be.launch_count

    def no(call, *a, **k):
        with pytest.raises(moe.TieCudaError) as e:
            call(*a, **k)
        assert e.value.code == moe.EINVAL

    no(be.attn_ptr, w.cache, w.step, q[:6], q, 8, 0.1)
    no(be.attn_ptr, w.cache, w.step, q, q.half(), 8, 0.1)
    no(be.attn_ptr, w.cache, w.step, q.cpu(), q, 8, 0.1)
    no(be.qk_norm_rope_ptr, w.cache, w.step, q[:, :4].contiguous(), kv, kv, q, 8)
    no(be.qk_norm_rope_ptr, w.cache, w.step, q, kv[:6], kv, q, 8)
    no(be.qk_norm_rope_ptr, w.cache, w.step, q, kv, kv.cpu(), q, 8)
    no(be.qk_norm_rope_ptr, w.cache, w.step, q, kv, kv, q[:6], 8)
    no(be.qk_norm_rope_ptr, w.cache, w.step, q, kv, kv, q, 8, q_norm_w=torch.ones(32, device="cuda"))
    no(be.kv_read_ptr, w.cache, w.step, kv, kv[:6].clone())
    no(be.kv_read_ptr, w.cache, w.step, kv, kv, moe.KV_F16)
    no(be.kv_read_ptr, w.cache, w.step, kv.half(), kv.bfloat16(), moe.KV_F16)
    no(moe.KvStep, w.tok_start.long(), w.kv_len, w.d_table, 7)
    no(moe.KvCache, moe.KV_BF16, w.k, w.v)
    assert be.launch_count == before


def test_a_factor_that_is_no_number_behind_a_bad_page(be):
    """Keys that all rows see, a warp's second ones behind a group with a page missing and factors far apart: a factor that is no number
    is seen although its key's probability is nothing."""
    w = World(74, "q8", [1] * 40, [2000] * 40, 8, 1, 64, 16)
    q = torch.tensor(w.rng.standard_normal((40, 8, 64)), dtype=torch.float32).cuda() + 1.0
    for s in range(40):
        pg, pl = (int(x[0]) for x in w.slots(s, 50, 51))
        w.v_scale[pg, :, pl] *= 1e6
        pg, pl = (int(x[0]) for x in w.slots(s, 300, 301))
        w.k[pg, :, pl], w.k_scale[pg, :, pl], w.v_scale[pg, :, pl] = -120, 1.0 / 3, float("nan")
    w.d_table[:, 2] = -1
    out = torch.zeros_like(q)
    refused(w.attn, be, q, 1.0, out=out)
    assert out.isnan().all()
