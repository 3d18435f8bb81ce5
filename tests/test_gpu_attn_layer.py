"""The attention half of a layer (tie_cuda_attn_block_inplace) at heads of 128, with each cache type, both kinds of rotation and the model's
own size, against the restatement's mat-vecs and plain arithmetic in 64 bits.

What it writes is compared with the projections (half a step of the cache's type, and 1e-4 of a row's rms for projections that are
within 1.2e-5 of it and norms and rotations of them); its output with attention over keys and values as they lie in the cache, so that no
rounding of these can fall to another side: the library's parity bound, 1e-3 of a row's rms, for every row."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attn import HALF, TORCH, plain_write  # noqa: E402
from test_gpu_attn_block import step_of  # noqa: E402

DIM, EPS, BASE = 128, 1e-5, 1e4


class Half:
    def __init__(self, be, hidden, heads, kv_heads, types, interleaved, seed):
        from tie_b200 import moe, synth
        self.hidden, self.heads, self.kv_heads, self.interleaved = hidden, heads, kv_heads, interleaved
        rng = np.random.default_rng(seed)
        self.shapes = {"q": (hidden, heads * DIM), "k": (hidden, kv_heads * DIM), "v": (hidden, kv_heads * DIM), "o": (heads * DIM, hidden)}
        self.types, self.w = dict(zip("qkvo", types)), {}
        for i, n in enumerate("qkvo"):
            k, rows = self.shapes[n]
            make = synth.q4k_blocks if self.types[n] == 12 else synth.q6k_blocks
            self.w[n] = np.ascontiguousarray(make(300 + seed, i, rows * (k // 256)))
            be.register_tensor(self.w[n], self.types[n], k)
        self.norm, self.qn, self.kn = (1 + 0.2 * rng.standard_normal(n) for n in (hidden, DIM, DIM))
        dev = lambda x: torch.tensor(x, dtype=torch.float32).cuda()  # noqa: E731
        self.handle = moe.AttnWeights(heads, *(self.w[n] for n in "qkvo"), dev(self.norm), dev(self.qn), dev(self.kn), rope_base=BASE, rope_interleaved=interleaved)

    def project(self, port, n, x):
        k, rows = self.shapes[n]
        return np.stack([port.mat_vec(np.ascontiguousarray(r, dtype=np.float32), self.w[n], self.types[n], k, rows) for r in x]).astype(np.float64)


@pytest.mark.parametrize("hidden, heads, kv_heads, steps", [
    (512, 8, 2, [([40, 3], None), ([1, 1], None), ([5, 2], [1, 3, 5, 3 | 8, 16, 1, 2]), ([1, 30], None)]),
    (2048, 32, 4, [([9, 2], None), ([1, 1], None)]),
])
@pytest.mark.parametrize("kind, types, interleaved", [
    ("f16", (12, 12, 14, 12), False), ("bf16", (14, 14, 14, 14), True), ("q8", (12, 14, 12, 14), False), ("q8", (12, 12, 14, 12), True),
])
def test_the_half_of_a_layer(port_lib, kind, types, interleaved, hidden, heads, kv_heads, steps):
    from tie_b200 import moe
    be = moe.MoeBackend(hidden=hidden, n_expert=32, top_k=4, ffn_dim=256, n_layers=1, max_tokens=128, norm_eps=EPS)
    try:
        run(be, port_lib, Half(be, hidden, heads, kv_heads, types, interleaved, 7), kind, steps)
    finally:
        be.close()


def run(be, port, half, kind, steps):
    from tie_b200 import moe
    rng = np.random.default_rng(6)
    page, g = 16, half.heads // half.kv_heads
    shape = (24, half.kv_heads, page, DIM)
    k, v = (torch.zeros(shape, dtype=TORCH[kind], device="cuda") for _ in range(2))
    scales = [torch.zeros(shape[:3], device="cuda") if kind == "q8" else None for _ in range(2)]
    cache = moe.KvCache({"f16": moe.KV_F16, "bf16": moe.KV_BF16, "q8": moe.KV_Q8}[kind], k, v, *scales)
    table, lens = [list(range(8)), list(range(20, 12, -1))], [0, 0]

    def held(x, scale, s, lo, hi):
        j = np.arange(lo, hi)
        pg, pl = np.array(table[s])[j // page], j % page
        y = x.double().cpu().numpy()[pg, :, pl]
        return y if scale is None else y * scale.double().cpu().numpy()[pg, :, pl][..., None]

    for toks, tree in steps:
        n, pad = sum(toks), 2
        hidden = rng.standard_normal((n + pad, half.hidden)).astype(np.float32)
        where = [(s, i) for s in range(2) for i in range(toks[s])]
        depth = [bin(m).count("1") - 1 for m in tree] if tree else [i for _, i in where]
        pos = [lens[s] + d for (s, _), d in zip(where, depth)]
        x = hidden[:n].astype(np.float64)
        x = x * half.norm.astype(np.float32) / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
        qkv = {p: half.project(port, p, x).reshape(n, -1, DIM) for p in "qkv"}
        q = plain_write(qkv["q"], half.qn.astype(np.float32), EPS, pos, BASE, half.interleaved)
        want = {"k": plain_write(qkv["k"], half.kn.astype(np.float32), EPS, pos, BASE, half.interleaved), "v": qkv["v"]}
        got = torch.tensor(hidden).cuda()
        torch.cuda.synchronize()
        be.attn_block_inplace_ptr(half.handle, cache, step_of(toks, lens, table, pad, tree, pos), got)
        got = got.cpu().numpy()
        assert np.array_equal(got[n:], hidden[n:])  # rows that no sequence has
        att, row = np.zeros((n, half.heads, DIM)), 0
        for s in range(2):
            t = toks[s]
            kk, vv = held(k, scales[0], s, 0, lens[s] + t), held(v, scales[1], s, 0, lens[s] + t)
            for name, lies in (("k", kk), ("v", vv)):
                exact = want[name][row:row + t]
                half_step = np.abs(exact).max(-1, keepdims=True) / 254 if kind == "q8" else np.abs(exact) * HALF[kind]
                slack = 1e-4 * np.sqrt((exact ** 2).mean(-1, keepdims=True))
                assert (np.abs(lies[lens[s]:] - exact) <= half_step * (1 + 2.0 ** -10) + slack).all(), name
            for i in range(t):
                m = np.ones(lens[s] + t, bool)
                m[lens[s]:] = [bool(tree[row + i] >> j & 1) if tree else j <= i for j in range(t)]
                for h in range(half.heads):
                    sc = kk[m, h // g] @ q[row + i, h] / math.sqrt(DIM)
                    p = np.exp(sc - sc.max())
                    att[row + i, h] = p @ vv[m, h // g] / p.sum()
            row += t
        update = half.project(port, "o", att.reshape(n, -1))
        rms = np.sqrt((update ** 2).mean(-1))
        diff = np.abs((got[:n] - hidden[:n].astype(np.float64)) - update).max(-1)
        assert (diff <= 1e-3 * rms + 2.0 ** -24 * np.abs(got[:n]).max()).all(), diff / rms
        if not tree:
            lens = [a + t for a, t in zip(lens, toks)]
