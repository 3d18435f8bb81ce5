"""Attention over a paged cache, as it stands between the projections and the output projection of a layer whose
feed-forward half is the MoE block: what is written into the cache (norms of queries and keys for each head, rotation,
rounding to the cache's type), what is read back out of it, and the attention of a step's tokens over it — single
tokens, trees of drafted tokens, and pieces of prompts.

`run` has two forms: plain torch operations in 32 bits (`own` false), and the calls a program makes of
tie_b200.moe (`own` true).  Sizes are those of the Qwen3-30B-A3B-shaped layer of this repository's workloads (32 query
heads, 4 key/value heads of 128) and of its LFM2-shaped one (heads of 64).
"""
import math

import torch

own = False

DEV = "cuda"
ROPE_BASE, NORM_EPS = 1e6, 1e-6


def listed():
    qwen = {"heads": 32, "kv_heads": 4, "dim": 128}
    return [
        # one token late in a long conversation: its row of q, k and v before the attention of a layer
        {"name": "write_1_f16", "op": "write", "type": "f16", "seqs": 1, "tokens": 1, "length": 100003, "page": 64, **qwen},
        # a serving batch of single tokens with an 8-bit cache, read back as it is handed to a 16-bit copy
        {"name": "write_read_61_q8", "op": "write", "type": "q8", "seqs": 61, "tokens": 1, "length": 2111, "page": 16, **qwen},
        # the largest prompt batch, from an empty cache
        {"name": "write_4096_bf16", "op": "write", "type": "bf16", "seqs": 1, "tokens": 4096, "length": 0, "page": 128, **qwen},
        # a short conversation taken out of the cache
        {"name": "read_777_q8", "op": "read", "type": "q8", "out": "f16", "seqs": 1, "tokens": 777, "length": 0, "page": 32, **qwen},
        # a long conversation taken out, as 32-bit rows
        {"name": "read_120000_q8", "op": "read", "type": "q8", "out": "f32", "seqs": 1, "tokens": 120000, "length": 0, "page": 256, **qwen},
        # one token of a short conversation: latency
        {"name": "decode_1_500_f16", "op": "attn", "type": "f16", "seqs": 1, "tokens": 1, "length": 500, "page": 64, "tree": False, **qwen},
        # one token of a very long conversation, 8-bit cache
        {"name": "decode_1_100003_q8", "op": "attn", "type": "q8", "seqs": 1, "tokens": 1, "length": 100003, "page": 64, "tree": False, **qwen},
        # a decode batch of ragged lengths
        {"name": "decode_48_5000_f16", "op": "attn", "type": "f16", "seqs": 48, "tokens": 1, "length": 5000, "page": 64, "tree": False, **qwen},
        # a small tree of drafted tokens over one conversation, the reference's cache type
        {"name": "tree_13_9001_bf16", "op": "attn", "type": "bf16", "seqs": 1, "tokens": 13, "length": 9001, "page": 32, "tree": True, **qwen},
        # large trees for several conversations at once, 8-bit cache
        {"name": "tree_8x64_3500_q8", "op": "attn", "type": "q8", "seqs": 8, "tokens": 64, "length": 3500, "page": 64, "tree": True, **qwen},
        # a piece of a prompt behind what is in the cache already
        {"name": "prompt_512_1500_f16", "op": "attn", "type": "f16", "seqs": 1, "tokens": 512, "length": 1500, "page": 64, "tree": False, **qwen},
        # the largest prompt batch, heads of 64
        {"name": "prompt_4096_d64_bf16", "op": "attn", "type": "bf16", "seqs": 1, "tokens": 4096, "length": 0, "page": 128, "tree": False,
         "heads": 32, "kv_heads": 8, "dim": 64},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over the logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    heads, kv_heads, dim = rng.choice([(32, 4, 128), (32, 4, 128), (32, 8, 64), (16, 16, 128), (24, 8, 64), (12, 2, 128)])
    wide = max(1, kv_heads * dim // 512)
    c = {"type": rng.choice(["f16", "bf16", "q8"]), "page": rng.choice([16, 32, 64, 128, 256]), "heads": heads, "kv_heads": kv_heads, "dim": dim}
    kind = rng.choice(["write", "read", "decode", "tree", "prompt"])
    if kind == "write":
        seqs = _spread(rng, 1, 128)
        tokens = _spread(rng, 1, 4096 // seqs)
        return {"op": "write", "seqs": seqs, "tokens": tokens, "length": rng.randrange(0, 4000), **c}
    if kind == "read":
        seqs = _spread(rng, 1, 8)
        return {"op": "read", "out": rng.choice(["f16", "f32"]), "seqs": seqs, "tokens": _spread(rng, 100, 100000 // wide // seqs), "length": 0, **c}
    if kind == "decode":
        seqs = _spread(rng, 1, 64)
        return {"op": "attn", "seqs": seqs, "tokens": 1, "length": _spread(rng, 60, 150000 // wide // seqs), "tree": False, **c}
    if kind == "tree":
        seqs = _spread(rng, 1, 8)
        return {"op": "attn", "seqs": seqs, "tokens": rng.randrange(2, 65), "length": _spread(rng, 100, 28000 // seqs), "tree": True, **c}
    seqs = rng.choice([1, 1, 2])
    tokens = _spread(rng, 65, 1400 // seqs)
    return {"op": "attn", "seqs": seqs, "tokens": tokens, "length": rng.choice([0, rng.randrange(1, 2000)]), "tree": False, **c}


def _sizes(case):
    """Per sequence: slots in front of the step's tokens, and tokens of the step.  Ragged where there are several."""
    n = case["seqs"]
    lens = [case["length"] - (s * 7919 % 16) * case["length"] // 32 for s in range(n)]
    toks = [max(1, case["tokens"] - (s * 5 % 4) * case["tokens"] // 8) for s in range(n)]
    return lens, toks


KINDS = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _quantise(x):
    """Rows of the last axis as whole numbers of -127..127 and one factor each."""
    scale = x.abs().amax(-1) / 127
    q = torch.round(x / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]).clamp(-127, 127)
    return q.to(torch.int8), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    lens, toks = _sizes(case)
    n_seq, P, H, KV, D = case["seqs"], case["page"], case["heads"], case["kv_heads"], case["dim"]
    n = sum(toks)
    # a write needs the slots of its own tokens alone: the pages in front of them are another sequence's, or gone
    first = [(a // P if case["op"] == "write" else 0) for a in lens]
    used = [(a + t + P - 1) // P - f for a, t, f in zip(lens, toks, first)]
    max_pages = max(u + f for u, f in zip(used, first))
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=gen, device=DEV).tolist()
    table, at = [], 0
    for u, f in zip(used, first):
        table.append([order[0]] * f + order[at:at + u] + [order[0]] * (max_pages - u - f))
        at += u
    s = {"case": dict(case), "n": n, "max_tokens": max(toks), "max_length": max(a + t for a, t in zip(lens, toks)),
         "tok_start": torch.tensor([sum(toks[:i]) for i in range(n_seq + 1)], dtype=torch.int32, device=DEV),
         "kv_len": torch.tensor(lens, dtype=torch.int32, device=DEV),
         "page_table": torch.tensor(table, dtype=torch.int32, device=DEV), "tree": None}
    # what is in the cache: keys as they leave norm and rotation, values as they leave their projection
    k, v = normal(pages, KV, P, D), normal(pages, KV, P, D) * 0.7
    if case["type"] == "q8":
        (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = _quantise(k), _quantise(v)
    else:
        s["k"], s["v"], s["k_scale"], s["v_scale"] = k.to(KINDS[case["type"]]), v.to(KINDS[case["type"]]), None, None
    del k, v
    if case["op"] == "write":
        s["q_in"], s["k_in"], s["v_in"] = normal(n, H, D) * 2.0, normal(n, KV, D) * 1.5, normal(n, KV, D) * 0.7
        s["q_norm"], s["k_norm"] = 1.0 + 0.2 * normal(D), 1.0 + 0.2 * normal(D)
        s["q_out"] = torch.empty(n, H, D, device=DEV)
    if case["op"] == "write" and case["type"] == "q8":
        s["k_out"], s["v_out"] = (torch.empty(n, KV, D, dtype=torch.float16, device=DEV) for _ in range(2))
    if case["op"] == "read":
        s["k_out"], s["v_out"] = (torch.empty(n, KV, D, dtype=KINDS[case["out"]], device=DEV) for _ in range(2))
    if case["op"] == "attn":
        s["q"], s["out"] = normal(n, H, D) * 2.0, torch.empty(n, H, D, device=DEV)
        if case["tree"]:  # each node hangs below an earlier one or begins a branch of its own; bit j: node j is seen
            up = torch.rand(n, generator=gen, device=DEV).tolist()
            masks, at = [], 0
            for t in toks:
                mine = []
                for i in range(t):
                    parent = max(-1, i - 1 - int(6 * up[at + i] ** 2))
                    mine.append((mine[parent] if parent >= 0 else 0) | (1 << i))
                masks += mine
                at += t
            s["tree"] = torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device=DEV)
    return s


# ---- the plain forms ----


def _places(s):
    """For each token of the step: its sequence, its number in it, its slot, and the slot's page and place."""
    P, n = s["case"]["page"], s["n"]
    row = torch.arange(n, device=DEV)
    seq = torch.searchsorted(s["tok_start"][1:].long(), row, right=True)
    i = row - s["tok_start"].long()[seq]
    slot = s["kv_len"].long()[seq] + i
    return seq, i, slot, s["page_table"].long()[seq, slot // P], slot % P


def _normed(x, w):
    return x * w * torch.rsqrt((x * x).mean(-1, keepdim=True) + NORM_EPS)


def _rotated(x, pos):
    half = x.shape[-1] // 2
    inv = ROPE_BASE ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    angle = (pos.double()[:, None] * inv)[:, None, :]
    c, sn = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * sn, b * c + a * sn], -1)


def _held(s, name, page, place):
    """What the cache holds in the slots given by page and place (of any shape): [..., kv head, dim]."""
    x = s[name][page, :, place].float()
    return x if s[name + "_scale"] is None else x * s[name + "_scale"][page, :, place][..., None]


def _write(s):
    _, _, slot, page, place = _places(s)
    s["q_out"].copy_(_rotated(_normed(s["q_in"], s["q_norm"]), slot))
    k, v = _rotated(_normed(s["k_in"], s["k_norm"]), slot), s["v_in"]
    if s["case"]["type"] != "q8":
        s["k"][page, :, place] = k.to(s["k"].dtype)
        s["v"][page, :, place] = v.to(s["v"].dtype)
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    s["k"][page, :, place], s["k_scale"][page, :, place] = _quantise(k)
    s["v"][page, :, place], s["v_scale"][page, :, place] = _quantise(v)
    return {"q": s["q_out"], **_read(s)}


def _read(s):
    _, _, _, page, place = _places(s)
    s["k_out"].copy_(_held(s, "k", page, place))
    s["v_out"].copy_(_held(s, "v", page, place))
    return {"k": s["k_out"], "v": s["v_out"]}


def _attn(s):
    c = s["case"]
    n_seq, H, KV, D, T, L = c["seqs"], c["heads"], c["kv_heads"], c["dim"], s["max_tokens"], s["max_length"]
    G = H // KV
    slot = torch.arange(L, device=DEV)
    page = s["page_table"].long()[:, slot // c["page"]]
    place = (slot % c["page"]).expand(n_seq, L)
    k, v = _held(s, "k", page, place), _held(s, "v", page, place)  # [seq, slot, kv head, dim]
    # the step's rows, each sequence's padded to T tokens
    start = s["tok_start"].long()
    i = torch.arange(T, device=DEV)
    row = start[:-1, None] + i
    real = row < start[1:, None]
    row = torch.where(real, row, 0)
    q = s["q"][row].view(n_seq, T, KV, G, D).permute(0, 2, 3, 1, 4).reshape(n_seq, KV, G * T, D)
    own_slot = slot[None, None, :] - s["kv_len"].long()[:, None, None]  # number of the step's token in a slot; below 0: in front of them
    if s["tree"] is None:
        seen = own_slot <= i[None, :, None]
    else:
        bits = (s["tree"][row][:, :, None] >> own_slot.clamp(0, 63)) & 1
        seen = (own_slot < 0) | ((own_slot < (start[1:] - start[:-1])[:, None, None]) & (bits > 0))
    seen = seen[:, None, None]  # [seq, 1, 1, token, slot]
    w = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(D)).view(n_seq, KV, G, T, L)
    w = w.masked_fill_(~seen, -math.inf)
    top = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.view(n_seq, KV, G * T, L), v.permute(0, 2, 1, 3)).view(n_seq, KV, G, T, D)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    s["out"][row[real]] = out.permute(0, 3, 1, 2, 4).reshape(n_seq, T, H, D)[real]
    return {"out": s["out"]}


# ---- the framework's calls ----

_backend = None


def _handles(s):
    """The library's context, one for the process, and the descriptions of a state's cache and step, made once as a program keeps them."""
    global _backend
    from tie_b200 import moe

    if _backend is None:
        _backend = moe.MoeBackend(hidden=256, n_expert=16, top_k=1, ffn_dim=256, max_tokens=64)
    if "handles" not in s:
        kind = {"f16": moe.KV_F16, "bf16": moe.KV_BF16, "q8": moe.KV_Q8}[s["case"]["type"]]
        cache = moe.KvCache(kind, s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["handles"] = (cache, moe.KvStep(s["tok_start"], s["kv_len"], s["page_table"], s["n"], tree=s["tree"]))
    _backend.set_stream(torch.cuda.current_stream().cuda_stream)
    return moe, _backend, *s["handles"]


def _own_run(s):
    moe, be, cache, step = _handles(s)
    c, flags = s["case"], moe.DEVICE | moe.NO_SYNC
    if c["op"] == "attn":
        be.attn_ptr(cache, step, s["q"], s["out"], c["heads"], 1.0 / math.sqrt(c["dim"]), flags=flags)
        return {"out": s["out"]}
    if c["op"] == "write":
        be.qk_norm_rope_ptr(cache, step, s["q_in"], s["k_in"], s["v_in"], s["q_out"], c["heads"], q_norm_w=s["q_norm"], k_norm_w=s["k_norm"],
                            norm_eps=NORM_EPS, rope_base=ROPE_BASE, flags=flags)
        if c["type"] != "q8":
            return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    out_type = {torch.float32: moe.KV_F32, torch.float16: moe.KV_F16}[s["k_out"].dtype]
    be.kv_read_ptr(cache, step, s["k_out"], s["v_out"], out_type, flags=flags)
    return ({"q": s["q_out"]} if c["op"] == "write" else {}) | {"k": s["k_out"], "v": s["v_out"]}


def run(state):
    if own:
        return _own_run(state)
    return {"write": _write, "read": _read, "attn": _attn}[state["case"]["op"]](state)


def work(case):
    lens, toks = _sizes(case)
    n, H, KV, D = sum(toks), case["heads"], case["kv_heads"], case["dim"]
    slot = 2 * KV * (D + 4 if case["type"] == "q8" else 2 * D)  # bytes of a slot of the cache
    if case["op"] == "write":
        b = n * (2 * H * D * 4 + 2 * KV * D * 4 + slot)
        return {"bytes": b + (n * (slot + 2 * KV * D * 2) if case["type"] == "q8" else 0), "flops": n * (H + 2 * KV) * D * 10}
    if case["op"] == "read":
        return {"bytes": n * (slot + 2 * KV * D * (4 if case["out"] == "f32" else 2)), "flops": n * 2 * KV * D}
    pairs = sum(t * a + t * (t + 1) // 2 for a, t in zip(lens, toks))
    return {"bytes": 2 * n * H * D * 4 + sum(a + t for a, t in zip(lens, toks)) * slot, "flops": 4 * pairs * H * D}


# ---- the definition, in 64 bits ----


def exact(case, seed):
    s = prepare(case, seed)
    lens, toks = _sizes(case)
    KV, D, P, H = case["kv_heads"], case["dim"], case["page"], case["heads"]
    table = s["page_table"].tolist()
    f64 = torch.float64

    def slots_of(n, lo, hi):
        ids = torch.tensor([table[n][x // P] * P + x % P for x in range(lo, hi)], device=DEV)
        return ids // P, ids % P

    def value(name, pg, pl):  # [slot, kv head, dim]
        x = s[name][pg, :, pl].to(f64)
        return x if case["type"] != "q8" else x * s[name + "_scale"][pg, :, pl].to(f64).unsqueeze(-1)

    if case["op"] == "read":
        got = {"k": [], "v": []}
        for n, (a, t) in enumerate(zip(lens, toks)):
            pg, pl = slots_of(n, a, a + t)
            for name in got:
                got[name].append(value(name, pg, pl))
        return {name: torch.cat(x) for name, x in got.items()}
    if case["op"] == "write":
        pos = torch.tensor([a + i for a, t in zip(lens, toks) for i in range(t)], dtype=f64, device=DEV)
        turn = torch.polar(torch.ones(1, dtype=f64, device=DEV), torch.outer(pos, torch.exp(torch.arange(D // 2, dtype=f64, device=DEV) * (-2.0 * math.log(ROPE_BASE) / D))))

        def head(x, w):
            x = x.to(f64)
            x = x * w.to(f64) / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + NORM_EPS)
            z = torch.complex(x[..., : D // 2], x[..., D // 2:]) * turn[:, None, :]
            return torch.cat([z.real, z.imag], -1)

        q, k, v = head(s["q_in"], s["q_norm"]), head(s["k_in"], s["k_norm"]), s["v_in"].to(f64)
        if case["type"] == "q8":
            def steps(x):
                unit = x.abs().max(-1, keepdim=True).values / 127
                return torch.round(x / unit) * unit
            return {"q": q, "k": steps(k), "v": steps(v)}
        ck, cv, r = s["k"].to(f64), s["v"].to(f64), 0
        for n, (a, t) in enumerate(zip(lens, toks)):
            pg, pl = slots_of(n, a, a + t)
            ck[pg, :, pl], cv[pg, :, pl] = k[r:r + t], v[r:r + t]
            r += t
        return {"q": q, "k": ck, "v": cv}
    out, r = torch.zeros(s["n"], H, D, dtype=f64, device=DEV), 0
    masks = s["tree"].tolist() if s["tree"] is not None else None
    for n, (a, t) in enumerate(zip(lens, toks)):
        pg, pl = slots_of(n, 0, a + t)
        k, v = value("k", pg, pl), value("v", pg, pl)
        hidden = torch.ones(t, t, dtype=torch.bool).triu(1) if masks is None else \
            torch.tensor([[not (masks[r + i] >> j) & 1 for j in range(t)] for i in range(t)])
        hidden = hidden.to(DEV)
        for h in range(H):
            w = s["q"][r:r + t, h].to(f64) @ k[:, h * KV // H].T / math.sqrt(D)
            w[:, a:].masked_fill_(hidden, -math.inf)
            out[r:r + t, h] = torch.softmax(w, -1).nan_to_num(0.0) @ v[:, h * KV // H]
        r += t
    return {"out": out}
