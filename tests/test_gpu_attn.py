"""Attention over the paged cache through the C ABI: what is written, what is read back, and attention of single tokens, trees and
prompt pieces, against plain arithmetic in 64 bits.

Tolerances, from the arithmetic alone:
* norm and rotation, fp32: a sum of D squares in a tree (7 + 2 roundings), square root, division, two products, then
  two products and a sum: below 16 half-steps of 2^-24 of the row's largest value times its weight -> 2^-20 of the row's largest
  output-side magnitude; the angle's cosine and sine are off by 2^-22 at most (a turn's fraction rounded to 24 bits).  Together 2^-19.
* a cache element: half a step of its type on top (F16 2^-11, BF16 2^-8 of the value; Q8 half of s, plus s's own 2^-23 times 127).
* attention: with A = |scale| * sum_i |q_i k_i| (natural units), a score is off by at most 14 * 2^-23 A (8 cut-off sums, the
  parts' 2^-22, sums of parts, the factors) + 2^-23 A (log2 e, the subtraction); exp2 2^-22; the parts of p 2^-22; sums over
  keys 2^-19 (16 sequential, then warps and CTAs).  p and the sum each carry it: 2 (A 2^-19 + 2^-18) max|v| < (1 + A) 2^-17 max|v|.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

KINDS = ["f16", "bf16", "q8"]
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "q8": torch.int8}


@pytest.fixture(scope="module")
def be():
    from tie_b200 import moe
    b = moe.MoeBackend(hidden=256, n_expert=16, top_k=1, ffn_dim=256, max_tokens=64)
    yield b
    b.close()


class World:
    """A cache and a step, on the device for the library and in 64 bits on the host for the check."""

    def __init__(self, seed, kind, toks, lens, heads=8, kv_heads=2, dim=128, page=16, pad=0, tree=None, pos=None, spare_pages=2, far=False):
        from tie_b200 import moe
        self.kind, self.toks, self.lens, self.heads, self.kv_heads, self.dim, self.page = kind, toks, lens, heads, kv_heads, dim, page
        self.rng = np.random.default_rng(seed)
        self.n = sum(toks)
        self.rows = self.n + pad
        need = [-(-(a + t) // page) for a, t in zip(lens, toks)]
        # (far: room for more slots than the kernels for few rows are chosen with)
        max_pages = max(1, max(need)) + (32768 // page if far else 0)
        n_pages = sum(need) + spare_pages
        order = self.rng.permutation(n_pages)
        table, at = np.full((len(toks), max_pages), order[-1], np.int32), 0
        for s, u in enumerate(need):
            table[s, :u] = order[at:at + u]
            at += u
        self.table = table
        shape = (n_pages, kv_heads, page, dim)
        k, v = self.rng.standard_normal(shape), self.rng.standard_normal(shape)
        self.k_scale = self.v_scale = None
        if kind == "q8":
            (k, ks), (v, vs) = self.q8(k), self.q8(v)
            self.k_scale, self.v_scale = (torch.tensor(x, dtype=torch.float32).cuda() for x in (ks, vs))
        self.k, self.v = (torch.tensor(x).to(TORCH[kind]).cuda() for x in (k, v))
        self.tree = tree
        dev = lambda x, t: torch.tensor(np.asarray(x), dtype=t).cuda()  # noqa: E731
        self.tok_start = dev(np.concatenate([[0], np.cumsum(toks)]), torch.int32)
        self.kv_len, self.d_table = dev(lens, torch.int32), dev(table, torch.int32)
        self.d_tree = None if tree is None else dev(np.array([m - (1 << 64) if m >> 63 else m for m in tree] + [-1] * pad, dtype=np.int64), torch.int64)
        self.pos = pos
        self.d_pos = None if pos is None else dev(list(pos) + [0] * pad, torch.int32)
        self.moe_kind = {"f16": moe.KV_F16, "bf16": moe.KV_BF16, "q8": moe.KV_Q8}[kind]
        self.describe()

    def describe(self):
        from tie_b200 import moe
        self.cache = moe.KvCache(self.moe_kind, self.k, self.v, self.k_scale, self.v_scale)
        self.step = moe.KvStep(self.tok_start, self.kv_len, self.d_table, self.rows, tree=self.d_tree, pos=self.d_pos)

    @staticmethod
    def q8(x):
        s = np.float32(np.abs(x).max(-1)) / np.float32(127)
        return np.rint(x / s[..., None]).clip(-127, 127), s

    def held(self, which):
        """The whole cache in 64 bits: [page][kv head][place][dim]."""
        x = getattr(self, which).double().cpu().numpy()
        return x if self.kind != "q8" else x * getattr(self, which + "_scale").double().cpu().numpy()[..., None]

    def slots(self, s, lo, hi):
        j = np.arange(lo, hi)
        return self.table[s, j // self.page], j % self.page

    def sequence(self, which, s):
        pg, pl = self.slots(s, 0, self.lens[s] + self.toks[s])
        return self.held(which)[pg, :, pl]  # [slot][kv head][dim]

    def sees(self, s, row):
        """[token][slot] of sequence s, whose first row is `row`."""
        t, a = self.toks[s], self.lens[s]
        m = np.ones((t, a + t), bool)
        m[:, a:] = np.tril(np.ones((t, t), bool)) if self.tree is None else \
            [[bool(self.tree[row + i] >> j & 1) for j in range(t)] for i in range(t)]
        return m

    def check_attn(self, q, out, scale):
        q, out = q.double().cpu().numpy(), out.double().cpu().numpy()
        row, g = 0, self.heads // self.kv_heads
        for s, t in enumerate(self.toks):
            k, v, m = self.sequence("k", s), self.sequence("v", s), self.sees(s, row)
            for h in range(self.heads):
                for i in range(t):
                    see = m[i]
                    got = out[row + i, h]
                    if not see.any():
                        assert (got == 0).all(), (s, i, h)
                        continue
                    kk, vv, x = k[see, h // g], v[see, h // g], q[row + i, h]
                    score = scale * (kk @ x)
                    p = np.exp(score - score.max())
                    want = p @ vv / p.sum()
                    big = 1.0 + abs(scale) * (np.abs(kk) @ np.abs(x)).max()
                    if not np.isfinite(want).all():
                        assert np.array_equal(np.isnan(want), np.isnan(got)) and np.array_equal(np.isposinf(want), np.isposinf(got)), (s, i, h)
                        continue
                    tol = big * 2.0 ** -17 * np.abs(vv).max()
                    assert np.abs(got - want).max() <= tol, (s, i, h, np.abs(got - want).max(), tol)
            row += t

    def attn(self, be, q=None, scale=None, flags=None, out=None):
        from tie_b200 import moe
        scale = 1.0 / math.sqrt(self.dim) if scale is None else scale
        if q is None:
            q = torch.tensor(self.rng.standard_normal((self.rows, self.heads, self.dim)) * 2, dtype=torch.float32).cuda()
        if out is None:
            out = torch.full((self.rows, self.heads, self.dim), 7.25, device="cuda")
        torch.cuda.synchronize()
        be.attn_ptr(self.cache, self.step, q, out, self.heads, scale, flags=moe.DEVICE if flags is None else flags)
        return q, out, scale


def trees(rng, toks, empty=False):
    masks = []
    for t in toks:
        mine = []
        for i in range(t):
            parent = int(rng.integers(-1, i)) if i else -1
            m = (mine[parent] if parent >= 0 else 0) | 1 << i
            mine.append(m)
        if empty:
            mine = [0 if rng.random() < 0.4 else m for m in mine]
        masks += mine
    return masks


# ---- writing and reading back ----


def plain_write(x, w, eps, pos, base, interleaved, rotate=True):
    x = np.asarray(x, np.float64)
    d = x.shape[-1]
    if w is not None:
        x = x * w / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if not rotate:
        return x
    ang = np.asarray(pos, np.float64)[:, None] * float(base) ** (-2.0 * np.arange(d // 2) / d)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y = np.empty_like(x)
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :d // 2], x[..., d // 2:])
    ya, yb = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0::2], y[..., 1::2] = ya, yb
    else:
        y[..., :d // 2], y[..., d // 2:] = ya, yb
    return y


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim, heads, kv_heads, toks, lens, interleaved, norm, pos, fused", [
    (128, 32, 4, [1], [0], False, True, False, False),
    (128, 32, 4, [1], [1000], False, True, False, True),
    (64, 24, 8, [5, 0, 17, 1], [3, 9, 0, 130], False, True, True, False),
    (64, 8, 1, [3, 40], [15, 16], True, False, False, True),
    (128, 7, 7, [33], [31], True, True, True, True),
    (128, 16, 2, [1] * 45, list(range(45)), False, True, False, False),
])
def test_written_rows(be, kind, dim, heads, kv_heads, toks, lens, interleaved, norm, pos, fused):
    from tie_b200 import moe
    rng = np.random.default_rng(5)
    positions = rng.integers(0, 200000, sum(toks)).tolist() if pos else None
    w = World(1, kind, toks, lens, heads, kv_heads, dim, page=16, pad=3, pos=positions)
    n, width = w.rows, (heads + 2 * kv_heads) * dim
    both = torch.tensor(rng.standard_normal((n, width + 8)) * 1.7, dtype=torch.float32).cuda()
    q, k, v = both[:, :heads * dim], both[:, heads * dim:(heads + kv_heads) * dim], both[:, (heads + kv_heads) * dim:width]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    qw, kw = (torch.tensor(1 + 0.3 * rng.standard_normal(dim), dtype=torch.float32).cuda() if norm else None for _ in range(2))
    q_out = torch.full((n, heads, dim), 7.25, device="cuda")
    before = {x: w.held(x) for x in ("k", "v")}
    torch.cuda.synchronize()
    be.qk_norm_rope_ptr(w.cache, w.step, q, k, v, q_out, heads, q_norm_w=qw, k_norm_w=kw, norm_eps=1e-5, rope_base=1e6, rope_interleaved=interleaved)
    at = positions if pos else [a + i for a, t in zip(lens, toks) for i in range(t)]
    host = lambda x: None if x is None else x.double().cpu().numpy()  # noqa: E731
    want = {"q": plain_write(host(q)[:w.n].reshape(w.n, heads, dim), host(qw), 1e-5, at, 1e6, interleaved),
            "k": plain_write(host(k)[:w.n].reshape(w.n, kv_heads, dim), host(kw), 1e-5, at, 1e6, interleaved),
            "v": host(v)[:w.n].reshape(w.n, kv_heads, dim)}
    got_q = host(q_out)
    assert (got_q[w.n:] == 7.25).all()  # rows that no sequence has
    top = np.abs(want["q"]).max(-1, keepdims=True) * math.sqrt(2)
    assert (np.abs(got_q[:w.n] - want["q"]) <= top * 2.0 ** -19).all()
    out = {x: torch.full((n, kv_heads, dim), 7.25, device="cuda") for x in "kv"}
    torch.cuda.synchronize()
    be.kv_read_ptr(w.cache, w.step, out["k"], out["v"], moe.KV_F32)
    for x in "kv":
        after, row = w.held(x), 0
        for s, t in enumerate(toks):
            pg, pl = w.slots(s, lens[s], lens[s] + t)
            mine = after[pg, :, pl]
            exact = want[x][row:row + t]
            top = np.abs(exact).max(-1, keepdims=True)
            slack = (0.0 if x == "v" else 1.0) * top * math.sqrt(2) * 2.0 ** -19
            half = top / 254 * (1 + 2.0 ** -15) if kind == "q8" else np.abs(exact) * HALF[kind] + 2.0 ** -25
            assert (np.abs(mine - exact) <= half + slack * 1.01).all(), x
            if kind != "q8" and x == "v":  # rounded to nearest, to the bit
                assert np.array_equal(mine, torch.tensor(exact).float().to(TORCH[kind]).double().numpy())
            # fp32 holds a value of F16 and BF16, and Q8's product rounded once
            back = out[x][row:row + t].double().cpu().numpy()
            assert (np.abs(back - mine) <= (np.abs(mine) * 2.0 ** -24 if kind == "q8" else 0.0)).all()
            after[pg, :, pl] = before[x][pg, :, pl]
            row += t
        assert np.array_equal(after, before[x])  # and no other slot
        assert (out[x][w.n:] == 7.25).all()


def test_far_positions_keep_their_angle(be):
    """At position 2^20 an angle formed in 32 bits is off by 2^-4 of a radian."""
    w = World(2, "f16", [2], [0], 2, 1, 128, pos=[1 << 20, 131071])
    rng = np.random.default_rng(3)
    q, k, v = (torch.tensor(rng.standard_normal((2, h, 128)), dtype=torch.float32).cuda() for h in (2, 1, 1))
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    be.qk_norm_rope_ptr(w.cache, w.step, q, k, v, out, 2, rope_base=10000.0)
    want = plain_write(q.double().cpu().numpy(), None, 0, [1 << 20, 131071], 10000.0, False)
    assert np.abs(out.double().cpu().numpy() - want).max() <= np.abs(want).max() * math.sqrt(2) * 2.0 ** -19


def test_no_rotation_and_in_place(be):
    w = World(2, "bf16", [3], [4], 4, 2, 64)
    q, k, v = (torch.randn(3, h, 64, device="cuda") for h in (4, 2, 2))
    before = q.clone()
    torch.cuda.synchronize()
    be.qk_norm_rope_ptr(w.cache, w.step, q, k, v, q, 4, rope_base=0.0)
    assert torch.equal(q, before)
    pg, pl = w.slots(0, 4, 7)
    assert np.array_equal(w.held("k")[pg, :, pl], k.bfloat16().double().cpu().numpy())


def test_q8_rows_of_zeros_of_tiny_and_of_no_numbers(be):
    from tie_b200 import moe
    w = World(3, "q8", [5], [0], 1, 1, 64)
    rows = torch.zeros(5, 1, 64, device="cuda")
    rows[1] = 1e-39
    rows[2, 0, 5] = float("inf")
    rows[3, 0, 6] = float("nan")
    rows[4] = torch.linspace(-1, 1, 64) * 3e38  # (linspace of -3e38 .. 3e38 itself overflows)
    q = torch.zeros(5, 1, 64, device="cuda")
    k_out, v_out = (torch.empty(5, 1, 64, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    be.qk_norm_rope_ptr(w.cache, w.step, q, rows, rows, torch.empty_like(q), 1, rope_base=0.0)
    be.kv_read_ptr(w.cache, w.step, k_out, v_out, moe.KV_F32)
    for out in (k_out, v_out):
        assert (out[:2] == 0).all() and out[2:4].isnan().all()
        assert (out[4] - rows[4]).abs().max() <= 3e38 / 254 * 1.0001


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("toks, dim, kv_heads", [([1], 128, 4), ([70, 0, 129], 64, 3), ([1] * 100, 128, 1)])
def test_read_back(be, kind, out, toks, dim, kv_heads):
    from tie_b200 import moe
    w = World(4, kind, toks, [0] * len(toks), kv_heads, kv_heads, dim, page=32, pad=5)
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[out]
    k_out, v_out = (torch.full((w.rows, kv_heads, dim), 7.25, device="cuda", dtype=t) for _ in range(2))
    torch.cuda.synchronize()
    be.kv_read_ptr(w.cache, w.step, k_out, v_out, {"f32": moe.KV_F32, "f16": moe.KV_F16, "bf16": moe.KV_BF16}[out])
    for which, got in (("k", k_out), ("v", v_out)):
        want = np.concatenate([w.held(which)[w.slots(s, 0, n)[0], :, w.slots(s, 0, n)[1]] for s, n in enumerate(toks)])
        # once to fp32 (Q8), once to the type asked for
        assert torch.equal(got[:w.n].cpu(), torch.tensor(want).float().to(t))
        assert (got[w.n:] == 7.25).all()


# ---- attention ----


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim, heads, kv_heads, page", [(128, 32, 4, 16), (64, 24, 8, 64), (128, 4, 4, 128), (64, 10, 2, 32), (128, 32, 1, 16)])
@pytest.mark.parametrize("toks, lens", [
    ([1], [0]), ([1], [1]), ([1], [127]), ([1], [640]), ([1, 1, 1], [5, 0, 300]), ([3, 0, 1], [12, 7, 129]), ([20], [0]), ([9, 30], [200, 15]),
])
def test_attention_of_tokens_that_see_what_is_in_front(be, far, kind, dim, heads, kv_heads, page, toks, lens):
    w = World(11, kind, toks, lens, heads, kv_heads, dim, page, pad=2, far=far)
    q, out, scale = w.attn(be)
    w.check_attn(q, out, scale)
    assert (out[w.n:] == 7.25).all()


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim, heads, kv_heads", [(128, 32, 4), (64, 6, 2)])
@pytest.mark.parametrize("toks, lens, empty", [
    ([2], [40], False), ([13], [255], False), ([64], [100], False), ([64, 1, 33], [0, 500, 31], False), ([7, 64], [0, 0], True), ([40], [33], True),
])
def test_attention_of_trees(be, far, kind, dim, heads, kv_heads, toks, lens, empty):
    tree = trees(np.random.default_rng(8), toks, empty)
    w = World(12, kind, toks, lens, heads, kv_heads, dim, 16, tree=tree, pad=1, far=far)
    q, out, scale = w.attn(be)
    w.check_attn(q, out, scale)
    assert (out[w.n:] == 7.25).all()


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("toks, lens", [([200], [0]), ([130], [77]), ([65, 300], [40, 0])])
def test_attention_of_prompt_pieces(be, far, kind, toks, lens):
    w = World(13, kind, toks, lens, 16, 2, 128, 32, far=far)
    q, out, scale = w.attn(be)
    w.check_attn(q, out, scale)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim, heads, kv_heads, toks, lens, drafted", [
    (128, 32, 4, [512], [1500], False), (128, 16, 4, [2100], [100], False), (64, 32, 8, [2000], [0], False), (128, 32, 4, [13], [9001], True),
    (128, 32, 4, [64, 40, 0, 64], [3500, 700, 5, 1201], True), (64, 24, 8, [64, 64], [128, 4000], True), (128, 24, 2, [700, 300], [64, 900], False),
])
def test_long_caches_and_many_rows(be, kind, dim, heads, kv_heads, toks, lens, drafted):
    """Many tiles of keys a row and many tiles of rows a CTA, a head at a time on the device in 64 bits."""
    tree = trees(np.random.default_rng(9), toks) if drafted else None
    w = World(30, kind, toks, lens, heads, kv_heads, dim, 64, tree=tree)
    q, out, scale = w.attn(be)
    row = 0
    for s, t in enumerate(toks):
        if t == 0:
            continue
        k, v, m = (torch.tensor(x).cuda() for x in (w.sequence("k", s), w.sequence("v", s), w.sees(s, row)))
        for h in range(heads):
            x, kk, vv = q[row:row + t, h].double(), k[:, h // (heads // kv_heads)], v[:, h // (heads // kv_heads)]
            want = torch.softmax((x @ kk.T * scale).masked_fill(~m, -math.inf), 1) @ vv
            big = 1.0 + scale * (x.abs() @ kk.abs().T).max(1, keepdim=True).values
            off = (out[row:row + t, h].double() - want).abs()
            assert (off <= big * 2.0 ** -17 * vv.abs().max()).all(), (s, h, off.max())
        row += t


@pytest.mark.parametrize("far", [False, True])
def test_many_sequences_of_all_lengths(be, far):
    rng = np.random.default_rng(1)
    toks = rng.integers(0, 3, 333).tolist()
    w = World(14, "f16", toks, rng.integers(0, 200, 333).tolist(), 4, 2, 64, 16, far=far)
    q, out, scale = w.attn(be)
    w.check_attn(q, out, scale)


@pytest.mark.parametrize("kind", KINDS)
def test_as_many_sequences_as_a_step_has(be, kind):
    """1024 of them, some empty, more query rows on average than the kernel for few rows takes."""
    rng = np.random.default_rng(5)
    toks = rng.integers(0, 6, 1024).tolist()
    w = World(49, kind, toks, rng.integers(0, 60, 1024).tolist(), 8, 1, 64, 16, far=True)
    k, v = w.held("k"), w.held("v")
    w.held = {"k": k, "v": v}.__getitem__
    q, out, scale = w.attn(be)
    w.check_attn(q, out, scale)


@pytest.mark.parametrize("kind", KINDS)
def test_long_cache_is_split_and_joined_the_same_every_time(be, kind):
    w = World(15, kind, [1, 2], [20011, 9000], 8, 1, 128, 64)
    q, out, scale = w.attn(be)
    w.check_attn(q, out, scale)
    first = out.clone()
    for _ in range(20):
        out.fill_(0)
        w.attn(be, q, scale, out=out)
        assert torch.equal(first, out)


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads", [8, 32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_token_does_not_see_is_nothing_to_it(be, far, kind, bad, heads):
    """Stale slots behind the last token and drafted tokens on other branches hold anything."""
    toks, lens = [12, 5], [37, 3]
    tree = trees(np.random.default_rng(2), toks)
    w = World(16, kind, toks, lens, heads, 2, 128, 16, tree=tree, far=far)
    q, clean, scale = w.attn(be)
    used = np.zeros(w.k.shape[0] * 16, bool)
    for s in range(2):
        pg, pl = w.slots(s, 0, lens[s] + toks[s])
        used[pg * 16 + pl] = True
    stale = torch.tensor(~used.reshape(-1, 16)).cuda()[:, None, :, None]
    w.k.masked_fill_(stale, bad)
    w.v.masked_fill_(stale, bad)
    _, out, _ = w.attn(be, q, scale)
    assert torch.equal(out, clean)
    # a drafted token's value row holds it: rows that see the token get it, the others what they had
    for s, j in ((0, 4), (1, 2)):
        pg, pl = w.slots(s, lens[s] + j, lens[s] + j + 1)
        w.v[int(pg[0]), :, int(pl[0]), 3] = bad
    _, out, _ = w.attn(be, q, scale)
    row = 0
    for s, j in ((0, 4), (1, 2)):
        for i in range(toks[s]):
            mine = out[row + i].clone()
            if tree[row + i] >> j & 1:
                want = torch.full_like(mine[:, 3], bad)
                assert torch.equal(mine[:, 3].isnan(), want.isnan()) and (want.isnan() | (mine[:, 3] == want)).all()
                mine[:, 3] = clean[row + i][:, 3]
            assert (mine - clean[row + i]).abs().max() <= 2.0 ** -17 * 4 * 16
        row += toks[s]


@pytest.mark.parametrize("far", [False, True])
def test_q8_factors_that_are_no_numbers_stay_where_they_are_seen(be, far):
    toks, lens = [6], [20]
    tree = [1, 3, 5, 9, 17, 33]
    w = World(17, "q8", toks, lens, 8, 2, 64, 16, tree=tree, far=far)
    q, clean, scale = w.attn(be)
    for j, bad in ((2, float("nan")), (4, float("inf"))):
        pg, pl = w.slots(0, 20 + j, 21 + j)
        w.v_scale[int(pg[0]), :, int(pl[0])] = bad
        w.k_scale[int(pg[0]), :, int(pl[0])] = float("nan")
    _, out, _ = w.attn(be, q, scale)
    for i in range(6):
        assert out[i].isnan().all() if i in (2, 4) else torch.equal(out[i], clean[i])


def test_rows_of_any_size(be):
    """Queries far from 1 keep their precision, scores far apart do not overflow."""
    w = World(18, "f16", [4], [90], 2, 1, 64)
    q = torch.randn(4, 2, 64, device="cuda")
    q *= torch.tensor([1e-30, 1e-3, 1e4, 1e18], device="cuda")[:, None, None]
    for scale in (0.125, 0.0, -2.0):
        _, out, _ = w.attn(be, q[:3].repeat(2, 1, 1)[:4].contiguous(), scale)
        w.check_attn(q[:3].repeat(2, 1, 1)[:4], out, scale)
    _, out, _ = w.attn(be, q, 0.125)  # the last row's scores are 1e19 apart: one key is left
    k, v = w.sequence("k", 0), w.sequence("v", 0)
    for h in range(2):
        j = int(np.argmax(k[:, 0] @ q[3, h].double().cpu().numpy()))
        assert np.abs(out[3, h].double().cpu().numpy() - v[j, 0]).max() <= 2.0 ** -20 * 4


def test_far_pages(be):
    """Offsets of rows pass 32 bits: the step's pages lie at the end of a cache of 4.5 GB a side."""
    from tie_b200 import moe
    page, kv_heads, dim = 1024, 4, 128
    n_pages = 4500
    free, _ = torch.cuda.mem_get_info()
    if free < 12 << 30:
        pytest.skip("less than 12 GB free")
    w = World(19, "f16", [3], [2000], 8, kv_heads, dim, page=page, spare_pages=0)
    k, v = (torch.zeros(n_pages, kv_heads, page, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    far = n_pages - w.k.shape[0]
    k[far:], v[far:] = w.k, w.v
    small = w.attn(be)
    w.d_table += far
    torch.cuda.synchronize()
    cache = moe.KvCache(moe.KV_F16, k, v)
    out = torch.empty_like(small[1])
    be.attn_ptr(cache, w.step, small[0], out, 8, small[2])
    assert torch.equal(out, small[1])
    q_in, kv_in = torch.randn(3, 8, dim, device="cuda"), torch.randn(3, kv_heads, dim, device="cuda")
    torch.cuda.synchronize()
    be.qk_norm_rope_ptr(cache, w.step, q_in, kv_in, kv_in, torch.empty_like(q_in), 8, rope_base=0.0)
    got = [torch.empty(3, kv_heads, dim, device="cuda") for _ in range(2)]
    be.kv_read_ptr(cache, w.step, *got)
    for g in got:
        assert torch.equal(g, kv_in.half().float())


# ---- together, and as a program uses them ----


@pytest.mark.parametrize("kind", KINDS)
def test_a_conversation_step_by_step(be, kind):
    """A prompt, single tokens, a tree of drafted tokens: written, attended to, read back; the cache's lengths move on."""
    from tie_b200 import moe
    heads, kv_heads, dim, page = 8, 2, 64, 16
    w = World(20, kind, [0, 0], [0, 0], heads, kv_heads, dim, page, spare_pages=16)
    w.table = np.arange(16, dtype=np.int32)[::-1].reshape(2, 8).copy()
    w.d_table = torch.tensor(w.table).cuda()
    rng = np.random.default_rng(4)
    lens = [0, 0]
    for toks, tree in (([30, 7], None), ([1, 1], None), ([1, 0], None), ([9, 12], True), ([2, 5], None)):
        w.toks, w.lens, w.n, w.rows = toks, list(lens), sum(toks), sum(toks)
        w.tree = trees(rng, toks) if tree else None
        w.d_tree = torch.tensor(np.array(w.tree, dtype=np.int64)).cuda() if tree else None
        depth = [bin(m).count("1") - 1 for m in w.tree] if tree else None
        row0 = [0, toks[0]]
        pos = [lens[s] + depth[row0[s] + i] for s in range(2) for i in range(toks[s])] if tree else None
        w.d_pos = torch.tensor(pos, dtype=torch.int32).cuda() if tree else None
        w.tok_start = torch.tensor([0, toks[0], sum(toks)], dtype=torch.int32).cuda()
        w.kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
        w.describe()
        q, k, v = (torch.tensor(rng.standard_normal((w.n, h, dim)), dtype=torch.float32).cuda() for h in (heads, kv_heads, kv_heads))
        wn = torch.ones(dim, device="cuda")
        q_out, out = torch.empty_like(q), torch.empty_like(q)
        torch.cuda.synchronize()
        be.qk_norm_rope_ptr(w.cache, w.step, q, k, v, q_out, heads, q_norm_w=wn, k_norm_w=wn, flags=moe.DEVICE | moe.NO_SYNC)
        be.attn_ptr(w.cache, w.step, q_out, out, heads, 0.125)
        w.check_attn(q_out, out, 0.125)
        lens = [a + t for a, t in zip(lens, toks)]


def test_captured_steps_follow_their_arrays(be):
    """A caller's graph of writing and attention, replayed while the lengths on the device move on; another stream than the context's own."""
    from tie_b200 import moe
    w = World(21, "q8", [1, 1], [300, 40], 8, 2, 128, 16, spare_pages=40)
    w.table = np.concatenate([w.table, np.zeros((2, 2), np.int32)], 1)
    used = set(w.table[:, :19].ravel().tolist())
    rest = [p for p in range(w.k.shape[0]) if p not in used]
    w.table = np.stack([np.array([w.table[s, i] if i * 16 < w.lens[s] + 1 else rest.pop() for i in range(21)], np.int32) for s in range(2)])
    w.d_table = torch.tensor(w.table).cuda()
    w.describe()
    q, k, v = (torch.empty(2, h, 128, device="cuda") for h in (8, 2, 2))
    q_out, out = torch.empty_like(q), torch.empty_like(q)
    flags = moe.DEVICE | moe.NO_SYNC

    def step():
        be.qk_norm_rope_ptr(w.cache, w.step, q, k, v, q_out, 8, flags=flags)
        be.attn_ptr(w.cache, w.step, q_out, out, 8, 0.09, flags=flags)

    side = torch.cuda.Stream()
    try:
        be.set_stream(side.cuda_stream)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            step()
        for i in range(20):
            with torch.cuda.stream(side):
                for x in (q, k, v):
                    x.normal_()
                w.kv_len.copy_(torch.tensor(w.lens, dtype=torch.int32))
                g.replay()
                side.synchronize()
            w.check_attn(q_out, out, 0.09)
            w.lens = [a + 1 for a in w.lens]
    finally:
        be.set_stream(None)
    be.synchronize()


def test_empty_steps_launch_nothing(be):
    w = World(22, "f16", [0], [5], 4, 2, 64)
    before = be.launch_count
    one = torch.zeros(1, 4, 64, device="cuda")
    be.attn_ptr(w.cache, w.step, one, one, 4, 1.0)
    assert be.launch_count == before


# One of each way that work is shared out: few rows; parts of items; items in equal shares of keys; whole items.
SHARES = [([1, 2], [700, 9001], None), ([90, 40], [300, 2000], None), ([700, 300], [64, 900], None), ([64, 3], [1000, 8], True), ([2200], [50], None)]


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("toks, lens, drafted", SHARES)
def test_out_may_be_q(be, far, kind, toks, lens, drafted):
    w = World(40, kind, toks, lens, 32, 4, 128, 32, pad=3, tree=trees(np.random.default_rng(3), toks) if drafted else None, far=far)
    q, out, scale = w.attn(be)
    both = q.clone()
    w.attn(be, both, scale, out=both)
    assert torch.equal(both[:w.n], out[:w.n]) and torch.equal(both[w.n:], q[w.n:])


@pytest.mark.parametrize("kind", KINDS)
def test_two_contexts_at_once(kind):
    """Launches of two contexts overlap on their streams; each has the result that it has alone."""
    from tie_b200 import moe
    two = [moe.MoeBackend(hidden=256, n_expert=16, top_k=1, ffn_dim=256, max_tokens=64) for _ in range(2)]
    try:
        ws = [World(41 + i, kind, toks, lens, 32, 4, 128, 64) for i, (toks, lens) in enumerate([([1] * 5, [4000] * 5), ([150], [1000])])]
        alone = [w.attn(b) for w, b in zip(ws, two)]
        outs = [torch.zeros_like(a[1]) for a in alone]
        torch.cuda.synchronize()
        for _ in range(30):
            for b, w, a, o in zip(two, ws, alone, outs):
                b.attn_ptr(w.cache, w.step, a[0], o, 32, a[2], flags=moe.DEVICE | moe.NO_SYNC)
        for b in two:
            b.synchronize()
        for a, o in zip(alone, outs):
            assert torch.equal(a[1], o)
    finally:
        for b in two:
            b.close()


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_a_captured_prompt_step_follows_its_arrays(be, far, kind):
    """One graph for steps of up to 600 rows: few rows and many, rows in front of the first sequence and behind the last, none at all."""
    from tie_b200 import moe
    w = World(43, kind, [300, 300], [400, 400], 16, 2, 64, 32, far=far)
    q, _, scale = w.attn(be)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    try:
        be.set_stream(side.cuda_stream)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            be.attn_ptr(w.cache, w.step, q, out, 16, scale, flags=moe.DEVICE | moe.NO_SYNC)
        for first, toks, lens in ((0, [300, 300], [400, 400]), (0, [1, 1], [600, 2]), (5, [100, 0], [17, 300]), (0, [0, 0], [5, 5]), (600, [0, 0], [0, 0]), (0, [300, 300], [0, 0])):
            with torch.cuda.stream(side):
                w.tok_start.copy_(torch.tensor([first, first + toks[0], first + sum(toks)], dtype=torch.int32))
                w.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
                out.fill_(7.25)
                g.replay()
                side.synchronize()
            w.toks, w.lens = toks, lens
            end = first + sum(toks)
            assert (out[:first] == 7.25).all() and (out[end:] == 7.25).all()
            if end > first:
                w.check_attn(q[first:end], out[first:end], scale)
    finally:
        be.set_stream(None)
    be.synchronize()


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("toks, lens, drafted", SHARES[:2] + SHARES[3:4])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_no_number_is_its_own_affair(be, far, kind, toks, lens, drafted, bad):
    w = World(44, kind, toks, lens, 16, 2, 64, 32, tree=trees(np.random.default_rng(3), toks) if drafted else None, far=far)
    q, clean, scale = w.attn(be)
    for t, h in ((0, 3), (w.n - 1, 15)):
        q[t, h, 17] = bad
    _, out, _ = w.attn(be, q, scale)
    for t, h in ((0, 3), (w.n - 1, 15)):
        assert not out[t, h].isfinite().any()
        out[t, h] = clean[t, h]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_sequences_may_share_pages(be, far, kind):
    w = World(45, kind, [1, 40, 2], [200, 160, 170], 8, 2, 128, 16, far=far)
    w.table[1:, :10] = w.table[0, :10]  # a prefix of 160 slots
    w.d_table = torch.tensor(w.table).cuda()
    w.describe()
    q, out, scale = w.attn(be)
    w.check_attn(q, out, scale)


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads, kv_heads, toks, lens", [(256, 1, [3], [200]), (1024, 1, [1, 2], [77, 0]), (256, 256, [2, 17], [33, 0]), (1, 1, [150], [9])])
def test_head_layouts_at_their_ends(be, far, kind, heads, kv_heads, toks, lens):
    w = World(46, kind, toks, lens, heads, kv_heads, 64, 16, far=far)
    q, out, scale = w.attn(be)
    w.check_attn(q, out, scale)


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [0.0, -1.5])
def test_scales_of_prompt_pieces(be, far, kind, scale):
    w = World(47, kind, [70], [100], 8, 2, 64, 16, far=far)
    q = torch.randn(70, 8, 64, device="cuda") * torch.logspace(-20, 1, 70, device="cuda")[:, None, None]
    _, out, _ = w.attn(be, q, scale)
    w.check_attn(q, out, scale)


@pytest.mark.parametrize("kind", KINDS)
def test_a_page_may_be_a_whole_cache(be, kind):
    w = World(48, kind, [1, 20], [1000, 3], 8, 2, 64, 65536, spare_pages=0)
    q, out, scale = w.attn(be)
    w.check_attn(q, out, scale)


# ---- refusals and steps that are wrong ----


def test_refusals(be):
    from tie_b200 import moe
    w = World(23, "f16", [2], [5], 4, 2, 64)
    q, kv = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda")

    def refused(code, call, *a, **k):
        with pytest.raises(moe.TieCudaError) as e:
            call(*a, **k)
        assert e.value.code == code

    refused(moe.EINVAL, be.attn_ptr, w.cache, w.step, q, q, 5, 1.0)  # heads
    refused(moe.EINVAL, be.attn_ptr, w.cache, w.step, q, q, 0, 1.0)
    refused(moe.EINVAL, be.attn_ptr, w.cache, w.step, q, q, 4, float("nan"))
    refused(moe.EINVAL, be.attn_ptr, w.cache, w.step, q, q, 4, 1.0, flags=moe.HOST)
    refused(moe.EINVAL, be.attn_ptr, w.cache, w.step, q.data_ptr() + 4, q, 4, 1.0)
    refused(moe.ENOTSUP, be.kv_read_ptr, w.cache, w.step, kv, kv, moe.KV_Q8)
    refused(moe.EINVAL, be.qk_norm_rope_ptr, w.cache, w.step, q, kv, kv, q, 4, norm_eps=float("nan"))
    refused(moe.EINVAL, be.qk_norm_rope_ptr, w.cache, w.step, q, kv, kv, q, 4, rope_base=-1.0)
    wide = torch.zeros(2, 5, 64, device="cuda")
    refused(moe.EINVAL, be.qk_norm_rope_ptr, w.cache, w.step, wide[:, :4], kv, kv, wide, 4)  # in place, rows further apart than q_out's
    odd = torch.zeros(2, 4 * 64 + 2, device="cuda")
    refused(moe.EINVAL, be.qk_norm_rope_ptr, w.cache, w.step, odd[:, :256], kv, kv, q, 4)


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("how", ["page", "page_high", "len", "len_far", "rows", "start", "tree"])
def test_wrong_steps_are_reported_and_the_rest_is_right(be, far, kind, how):
    from tie_b200 import moe
    toks, lens, heads = [2, 3], [70, 33], 32 if far else 8
    w = World(24, kind, toks, lens, heads, 2, 64, 16, far=far)
    q, clean, scale = w.attn(be)
    if how == "page":
        w.d_table[1, 0] = -1
    elif how == "page_high":
        w.d_table[1, 2] = w.k.shape[0]
    elif how == "len":
        w.kv_len[1] = -5
    elif how == "len_far":
        w.kv_len[1] = 1 << 30
    elif how == "rows":
        w.tok_start[2] = 99
    elif how == "start":
        w.tok_start[0] = -3
    else:
        w = World(24, kind, [70, 3], lens, heads, 2, 64, 16, tree=[1] * 73, far=far)
        q, clean, scale = None, None, 0.125
    for call in ("attn", "write", "read"):
        if how in ("tree", "page") and call != "attn":  # (slots 33 .. 35 lie in the third page)
            continue
        with pytest.raises(moe.TieCudaError) as e:
            if call == "attn":
                _, out, _ = w.attn(be, q, scale)
            elif call == "write":
                qi, ki = torch.zeros(5, 8, 64, device="cuda"), torch.zeros(5, 2, 64, device="cuda")
                be.qk_norm_rope_ptr(w.cache, w.step, qi, ki, ki, torch.empty_like(qi), 8)
            else:
                o = torch.empty(5, 2, 64, device="cuda")
                be.kv_read_ptr(w.cache, w.step, o, o.clone())
        assert e.value.code == moe.EKERNEL
        assert "page" in str(e.value) or "step" in str(e.value)
    # the context goes on
    w = World(24, kind, toks, lens, heads, 2, 64, 16, far=far)
    if q is not None:
        _, out, _ = w.attn(be, q, scale)
        assert torch.equal(out, clean)
