"""The attention half of a layer on registered projections (tie_cuda_attn_block_inplace), against the restatement's mat-vecs and
plain arithmetic in 64 bits, and as the half of a layer beside tie_cuda_moe_block_inplace.  Bound: the library's parity bound,
1e-3 of a row's rms (the projections are within 1.2e-5 of it, which scores of up to 30 carry into p)."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV_HEADS, DIM, PAGE, EPS = 512, 8, 2, 64, 16, 1e-5


class Layer:
    def __init__(self, be, seed, types):
        from tie_b200 import moe, synth
        rng = np.random.default_rng(seed)
        self.shapes = {"q": (HIDDEN, HEADS * DIM), "k": (HIDDEN, KV_HEADS * DIM), "v": (HIDDEN, KV_HEADS * DIM), "o": (HEADS * DIM, HIDDEN)}
        self.types = dict(zip("qkvo", types))
        self.w = {}
        for i, n in enumerate("qkvo"):
            k, rows = self.shapes[n]
            make = synth.q4k_blocks if self.types[n] == 12 else synth.q6k_blocks
            self.w[n] = np.ascontiguousarray(make(100 + seed, i, rows * (k // 256)))
            be.register_tensor(self.w[n], self.types[n], k)
        # (the projections' outputs are large: the norms of q and k bring these to 1, wo's input is averages of v)
        self.norm, self.qn, self.kn = (1 + 0.2 * rng.standard_normal(n) for n in (HIDDEN, DIM, DIM))
        dev = lambda x: torch.tensor(x, dtype=torch.float32).cuda()  # noqa: E731
        self.handle = moe.AttnWeights(HEADS, self.w["q"], self.w["k"], self.w["v"], self.w["o"], dev(self.norm), dev(self.qn), dev(self.kn), rope_base=1e4)

    def project(self, port, n, x):
        k, rows = self.shapes[n]
        return np.stack([port.mat_vec(np.ascontiguousarray(r, dtype=np.float32), self.w[n], self.types[n], k, rows) for r in x]).astype(np.float64)

    def norm_of(self, x, w):
        return x * w.astype(np.float32) / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)

    def rotate(self, x, pos):
        ang = np.asarray(pos, np.float64)[:, None] * 1e4 ** (-2.0 * np.arange(DIM // 2) / DIM)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        a, b = x[..., :DIM // 2], x[..., DIM // 2:]
        return np.concatenate([a * c - b * s, b * c + a * s], -1)


@pytest.fixture(scope="module")
def be():
    from tie_b200 import moe
    b = moe.MoeBackend(hidden=HIDDEN, n_expert=32, top_k=4, ffn_dim=256, n_layers=1, max_tokens=128, norm_eps=EPS)
    yield b
    b.close()


def cache_of(pages=24):
    from tie_b200 import moe
    k, v = (torch.full((pages, KV_HEADS, PAGE, DIM), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    return moe.KvCache(moe.KV_BF16, k, v)


def step_of(toks, lens, table, pad=0, tree=None, pos=None):
    from tie_b200 import moe
    dev = lambda x, t=torch.int32: torch.tensor(x, dtype=t).cuda()  # noqa: E731
    return moe.KvStep(dev(np.concatenate([[0], np.cumsum(toks)]).tolist()), dev(lens), dev(table), sum(toks) + pad,
                      tree=None if tree is None else dev(tree, torch.int64), pos=None if pos is None else dev(pos))


@pytest.mark.parametrize("types", [(12, 12, 14, 12), (14, 14, 14, 14), (12, 14, 12, 14)])
def test_prompt_tokens_and_a_tree_through_the_block(be, port_lib, types):
    layer = Layer(be, sum(types), types)
    rng = np.random.default_rng(6)
    cache = cache_of()
    table = [list(range(0, 8)), list(range(20, 12, -1))]
    seen = [{"k": np.zeros((0, KV_HEADS, DIM)), "v": np.zeros((0, KV_HEADS, DIM))} for _ in range(2)]
    lens = [0, 0]
    for toks, tree in (([40, 3], None), ([1, 1], None), ([5, 2], [1, 3, 5, 3 | 8, 16, 1, 2])):
        n, pad = sum(toks), 2
        hidden = rng.standard_normal((n + pad, HIDDEN)).astype(np.float32)
        where = [(s, i) for s in range(2) for i in range(toks[s])]
        depth = [bin(m).count("1") - 1 for m in tree] if tree else [i for _, i in where]
        pos = [lens[s] + d for (s, _), d in zip(where, depth)]
        x = layer.norm_of(hidden[:n].astype(np.float64), layer.norm)
        q, k, v = (layer.project(port_lib, p, x).reshape(n, -1, DIM) for p in "qkv")
        q, k = layer.rotate(layer.norm_of(q, layer.qn), pos), layer.rotate(layer.norm_of(k, layer.kn), pos)
        round16 = lambda a: torch.tensor(a).float().bfloat16().double().numpy()  # noqa: E731
        att = np.zeros((n, HEADS, DIM))
        row = 0
        for s in range(2):
            t = toks[s]
            kk = np.concatenate([seen[s]["k"], round16(k[row:row + t])])
            vv = np.concatenate([seen[s]["v"], round16(v[row:row + t])])
            for i in range(t):
                m = np.ones(lens[s] + t, bool)
                m[lens[s]:] = [bool(tree[row + i] >> j & 1) if tree else j <= i for j in range(t)]
                for h in range(HEADS):
                    sc = kk[m, h // 4] @ q[row + i, h] / math.sqrt(DIM)
                    p = np.exp(sc - sc.max())
                    att[row + i, h] = p @ vv[m, h // 4] / p.sum()
            if not tree:
                seen[s] = {"k": kk, "v": vv}
            row += t
        update = layer.project(port_lib, "o", att.reshape(n, -1))
        got = torch.tensor(hidden).cuda()
        torch.cuda.synchronize()
        be.attn_block_inplace_ptr(layer.handle, cache, step_of(toks, lens, table, pad, tree, pos), got)
        got = got.cpu().numpy()
        assert np.array_equal(got[n:], hidden[n:])  # rows that no sequence has
        diff = np.abs((got[:n] - hidden[:n].astype(np.float64)) - update).max(-1)
        # (a key's or value's rounding to 16 bits may fall to the other side: one step of 2^-8 of a value among those of the row)
        rms = np.sqrt((update ** 2).mean(-1))
        assert (diff <= 1e-3 * rms + 2.0 ** -24 * np.abs(hidden[:n]).max()).mean() > 0.9 and (diff <= 1e-2 * rms).all(), diff / rms
        if not tree:
            lens = [a + t for a, t in zip(lens, toks)]


def test_a_layer_is_its_two_halves_in_a_graph(be, port_lib):
    """Attention half and feed-forward half of a layer, single tokens, captured by the caller and replayed while the lengths move on:
    the bits of the calls made one by one."""
    from tie_b200 import moe, synth
    layer = Layer(be, 77, (12, 12, 14, 12))
    shape = synth.MoeShape(hidden=HIDDEN, n_expert=32, top_k=4, ffn_dim=256)
    be.upload_layer(0, synth.make_layer(5, shape), ffn_norm_w=np.ones(HIDDEN, np.float32))
    table = [[0, 1, 2], [5, 4, 3]]
    caches = [cache_of(8), cache_of(8)]
    start = torch.randn(2, HIDDEN, generator=torch.Generator().manual_seed(1))
    outs = []
    for cache, graphed in zip(caches, (False, True)):
        step = step_of([1, 1], [0, 0], table)
        hidden = start.cuda()
        kv_len = step.keep[1]
        flags = moe.DEVICE | moe.NO_SYNC

        def layer_step():
            be.attn_block_inplace_ptr(layer.handle, cache, step, hidden, flags=flags)
            be.moe_block_inplace_ptr(0, hidden, 2, flags)

        side = torch.cuda.Stream()
        be.set_stream(side.cuda_stream)
        torch.cuda.synchronize()
        try:
            if graphed:
                layer_step()  # (first uses outside of the capture)
                side.synchronize()
                hidden.copy_(start)
                g = torch.cuda.CUDAGraph()
                torch.cuda.synchronize()
                with torch.cuda.graph(g, stream=side):
                    layer_step()
            for i in range(20):
                torch.cuda.synchronize()
                if graphed:
                    with torch.cuda.stream(side):
                        g.replay()
                else:
                    layer_step()
                side.synchronize()
                kv_len += 1
                hidden /= hidden.abs().max()
            outs.append(hidden.clone())
            be.synchronize()
        finally:
            be.set_stream(None)
    assert torch.equal(outs[0], outs[1]) and outs[0].isfinite().all()


def test_refusals_of_the_block(be):
    from tie_b200 import moe
    layer = Layer(be, 5, (12, 12, 12, 12))
    cache, step = cache_of(), step_of([2], [0], [[0, 1]])
    hidden = torch.zeros(2, HIDDEN, device="cuda")

    def refused(code, *a, **k):
        with pytest.raises(moe.TieCudaError) as e:
            be.attn_block_inplace_ptr(*a, **k)
        assert e.value.code == code

    refused(moe.EINVAL, layer.handle, cache, step, hidden, flags=moe.HOST)
    other = moe.AttnWeights(HEADS, layer.w["q"].copy(), layer.w["k"], layer.w["v"], layer.w["o"])
    refused(moe.EINVAL, other, cache, step, hidden)  # not registered
    refused(moe.EINVAL, moe.AttnWeights(4, layer.w["q"], layer.w["k"], layer.w["v"], layer.w["o"]), cache, step, hidden)  # heads
    refused(moe.EINVAL, moe.AttnWeights(HEADS, layer.w["q"], layer.w["k"], None, layer.w["o"]), cache, step, hidden)
    big = step_of([64, 65], [0, 0], [[0, 1, 2, 3, 4], [5, 6, 7, 8, 9]])  # 129 tokens, max_tokens 128
    refused(moe.EINVAL, layer.handle, cache, big, torch.zeros(129, HIDDEN, device="cuda"))
