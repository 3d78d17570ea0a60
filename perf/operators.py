"""The operators a speculating, long-running MLA serving process needs beside its decode, measured at
the sizes it meets:

    tree     attention of a tree of drafted tokens over the paged latent cache (`qmla.tree_forward`)
    weights  attention weight that every cached token got in a decode step, added to what it had
             (`qmla.attention_weights`)
    evict    the tokens a request keeps (first, recent and heaviest), their rows moved together into
             other pages (`qmla.evict`)
    rotary   rotary positions of query and key heads, half or interleaved layout, part of the head
             (`qmla.rotary`)

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs on the GPU
    run(state)          one pass; returns its outputs
    work(case)          bytes and flops a pass cannot do without
    exact(case, seed)   the outputs in float64

`own` False computes the plain forms in elementary torch; `own` True calls the package.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

# the cache rows that are deployed: (kv, d_c, rope, heads). bf16 rows hold one bf16 divisor per head,
# fp8 rows one log8 code per head; rows are padded to 16 elements
_ROWS = [("fp8", 512, 64, 24), ("bf16", 512, 64, 24), ("fp8", 768, 232, 24), ("bf16", 256, 116, 12),
         ("fp8", 768, 116, 12), ("bf16", 768, 232, 24)]


def _qmla():
    path = os.path.abspath("qwen-mla-vllm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qmla
    return qmla


def listed():
    return [
        # one user, a small drafted tree on a short chat: latency counts
        dict(name="tree_fp8_b1_t8", kind="tree", kv="fp8", d_c=512, rope=64, heads=24, batch=1, nodes=8, page=64,
             lo=1300, hi=1300, ragged=False),
        # a few requests on a bf16 cache in small pages, trees of different sizes padded to 16
        dict(name="tree_bf16_b4_t16", kind="tree", kv="bf16", d_c=512, rope=64, heads=24, batch=4, nodes=16, page=16,
             lo=500, hi=4096, ragged=True),
        # the deployed FP8 row of rank 768 with its packed rope, large pages, odd sizes
        dict(name="tree_fp8_r768_b7_t25", kind="tree", kv="fp8", d_c=768, rope=232, heads=24, batch=7, nodes=25,
             page=784, lo=300, hi=6000, ragged=False),
        # wide trees over long chats, a full batch
        dict(name="tree_fp8_b16_t64", kind="tree", kv="fp8", d_c=512, rope=64, heads=24, batch=16, nodes=64, page=64,
             lo=2048, hi=8192, ragged=False),
        # the weights of one short request's step
        dict(name="weights_fp8_b1", kind="weights", kv="fp8", d_c=512, rope=64, heads=24, batch=1, qrows=1, page=64,
             lo=1300, hi=1300),
        # a verify step's weights (4 query tokens) on a bf16 cache, ragged lengths
        dict(name="weights_bf16_b9x4", kind="weights", kv="bf16", d_c=512, rope=64, heads=24, batch=9, qrows=4, page=64,
             lo=500, hi=12000),
        # long requests, one step
        dict(name="weights_fp8_b64", kind="weights", kv="fp8", d_c=512, rope=64, heads=24, batch=64, qrows=1, page=64,
             lo=4096, hi=16384),
        # one request gives up half of its tokens
        dict(name="evict_fp8_b1", kind="evict", kv="fp8", d_c=512, rope=64, heads=24, batch=1, page=64, lo=4100,
             hi=4100, keep=2048, sink=4, recent=256),
        # a full batch of long requests is cut to a budget, lengths below it among them
        dict(name="evict_bf16_b40", kind="evict", kv="bf16", d_c=512, rope=64, heads=24, batch=40, page=64, lo=2000,
             hi=32768, keep=6001, sink=4, recent=1000),
        # one decode step of a batch: the rope columns of 576-wide absorbed queries, interleaved pairs
        dict(name="rotary_n33", kind="rotary", n=33, heads=24, kheads=1, dim=576, rot=64, offset=512, dtype="bf16",
             layout="interleaved", scaled=True),
        # a prefill chunk, a quarter of a 256-wide head, half layout
        dict(name="rotary_n12001", kind="rotary", n=12001, heads=24, kheads=4, dim=256, rot=64, offset=0, dtype="bf16",
             layout="half", scaled=False),
        # fp32 heads rotated whole
        dict(name="rotary_f32_n2048", kind="rotary", n=2048, heads=24, kheads=4, dim=64, rot=64, offset=0, dtype="fp32",
             layout="interleaved", scaled=True),
    ]


_TREE_FLOPS = 2.5e11     # of a drawn tree at most
_CACHE_BYTES = 8.0e8     # cached bytes of a drawn case at most


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "weights", "evict", "rotary"])
    if kind == "rotary":
        layout, dtype = rng.choice(["half", "interleaved"]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
        dim, rot, offset = rng.choice([(576, 64, 512), (256, 64, 0), (64, 64, 0), (128, 64, 64), (256, 58, 0), (80, 32, 16)])
        return dict(kind=kind, n=_log_int(rng, 1, 12000), heads=rng.choice([1, 7, 12, 24]), kheads=rng.choice([1, 2, 4]),
                    dim=dim, rot=rot, offset=offset, dtype=dtype, layout=layout, scaled=rng.random() < 0.5)
    kv, d_c, rope, heads = rng.choice(_ROWS)
    page = rng.choice([16, 64, 64, 128, 784])
    hi = _log_int(rng, 1, 12000)
    lo = max(1, int(hi * rng.choice([1.0, 0.5, 0.1])))
    row = (d_c + rope + heads) * (1 if kv == "fp8" else 2)
    batch = _log_int(rng, 1, 48)
    if kind == "tree":
        nodes = rng.choice([1, 2, 5, 8, 13, 16, 26, 32, 47, 64])
        hi, lo = max(hi, nodes), max(lo, nodes)
        while batch > 1 and 2.0 * nodes * heads * batch * hi * (2 * d_c + rope) > _TREE_FLOPS:
            batch -= 1
        return dict(kind=kind, kv=kv, d_c=d_c, rope=rope, heads=heads, batch=batch, nodes=nodes, page=page, lo=lo, hi=hi,
                    ragged=rng.random() < 0.5)
    if kind == "weights":
        qrows = rng.choice([1, 1, 2, 4])
        hi, lo = max(hi, qrows), max(lo, qrows)
        while batch > 1 and float(batch) * hi * row * qrows > _CACHE_BYTES:
            batch -= 1
        return dict(kind=kind, kv=kv, d_c=d_c, rope=rope, heads=heads, batch=batch, qrows=qrows, page=page, lo=lo, hi=hi)
    while batch > 1 and float(batch) * hi * row > _CACHE_BYTES:
        batch -= 1
    keep = _log_int(rng, 1, max(1, hi))
    sink = rng.randint(0, min(8, keep))
    return dict(kind=kind, kv=kv, d_c=d_c, rope=rope, heads=heads, batch=batch, page=page, lo=lo, hi=hi, keep=keep,
                sink=sink, recent=rng.randint(0, (keep - sink) // 2))


# ---- inputs ----------------------------------------------------------------------------------------
def _lens(case, seed):
    """Context lengths of the batch: log-uniform in [lo, hi], the longest one hi."""
    rs = np.random.RandomState(seed % (1 << 31))
    lens = np.exp(rs.uniform(math.log(case["lo"]), math.log(case["hi"]), case["batch"])).round().astype(np.int64)
    lens[rs.randint(case["batch"])] = case["hi"]
    return lens


def _row_elems(case):
    return -(-(case["d_c"] + case["rope"] + case["heads"]) // 16) * 16


def _cache(case, lens, spare, g, dev):
    """A paged cache of rows [latent | rope | divisors | pad], pages in random order; `spare` pages at
    its end belong to no request. Returns (cache, block table, k_scale or None)."""
    page, d_c, rope, heads = case["page"], case["d_c"], case["rope"], case["heads"]
    per = -(-lens // page)
    total = int(per.sum())
    table = torch.zeros(len(lens), int(per.max()), dtype=torch.int32, device=dev)
    at = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    for b, first in enumerate(np.concatenate([[0], np.cumsum(per)[:-1]])):
        table[b, :per[b]] = at[int(first):int(first) + int(per[b])]
    n, fp8 = total * page, case["kv"] == "fp8"
    cache = torch.zeros(total + spare, page, 1, _row_elems(case), dtype=torch.uint8 if fp8 else torch.bfloat16, device=dev)
    flat = cache.view(-1, cache.shape[-1])
    scale = torch.tensor(5.5 / 448.0, dtype=torch.float32, device=dev) if fp8 else None
    for a in range(0, n, 1 << 19):
        e = min(n, a + (1 << 19))
        x = torch.randn(e - a, d_c + rope, generator=g, device=dev)
        rms = x[:, :d_c].square().mean(-1, keepdim=True).sqrt() * torch.exp(0.3 * torch.randn(e - a, heads, generator=g, device=dev))
        if fp8:
            flat[a:e, :d_c + rope] = (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
            flat[a:e, d_c + rope:d_c + rope + heads] = ((rms.log2() + 3.0) * 42.5).round().clamp(0, 255).to(torch.uint8)
        else:
            flat[a:e, :d_c + rope] = x.to(torch.bfloat16)
            flat[a:e, d_c + rope:d_c + rope + heads] = rms.to(torch.bfloat16)
    return cache, table, scale


def _tree_masks(nodes, counts, rs):
    """Words [batch, nodes]: bit i of word j says that node j sees node i (itself and its ancestors)."""
    words = np.zeros((len(counts), nodes), dtype=np.uint64)
    for b, n in enumerate(counts):
        for j in range(int(n)):
            parent = rs.randint(max(0, j - 6), j) if j else -1
            words[b, j] = (words[b, parent] if j else np.uint64(0)) | (np.uint64(1) << np.uint64(j))
    return words.view(np.int64)


_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MAX_POS = 65536


def _frequencies(rot, scaled):
    """Angular frequency of each pair: 10000^(-2i/rot), with its positions interpolated by 4 for a
    scaled context."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return inv / 4.0 if scaled else inv


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rs = np.random.RandomState((seed + 77) % (1 << 31))
    s = dict(case=dict(case))
    if case["kind"] == "rotary":
        dt = _DT[case["dtype"]]
        # [heads | key heads] of one token beside each other, as a projection leaves them
        both = torch.randn(case["n"], case["heads"] + case["kheads"], case["dim"], generator=g, device=dev).to(dt)
        s["q"], s["k"] = both[:, :case["heads"]], both[:, case["heads"]:]
        start = torch.randint(0, _MAX_POS - case["n"], (1,), generator=g, device=dev)
        s["positions"] = start + torch.arange(case["n"], device=dev)
        angle = torch.outer(torch.arange(_MAX_POS, dtype=torch.float64, device=dev), _frequencies(case["rot"], case["scaled"]).to(dev))
        s["table"] = torch.cat([angle.cos(), angle.sin()], -1).float()
        return s
    lens = _lens(case, seed)
    fresh = case["keep"] if case["kind"] == "evict" else 0
    per_new = -(-fresh // case["page"])
    cache, table, scale = _cache(case, lens, per_new * len(lens), g, dev)
    s.update(cache=cache, scale=scale, lens=torch.from_numpy(lens.astype(np.int32)).to(dev), table=table)
    B, H, d_c, rope = len(lens), case["heads"], case["d_c"], case["rope"]
    s["sm_scale"] = 1.0 / math.sqrt(d_c + rope)
    if case["kind"] == "evict":
        W = int(lens.max())
        # attention weight falls off with a heavy tail, and repeats: many tokens never got any
        w = torch.exp(2.0 * torch.randn(B, W, generator=g, device=dev)) * (torch.rand(B, W, generator=g, device=dev) < 0.8)
        s["weights"] = w
        s["weights_out"] = torch.zeros(B, case["keep"], device=dev)
        pool = torch.randperm(per_new * B, generator=g, device=dev).to(torch.int32) + (cache.shape[0] - per_new * B)
        s["new_table"] = pool.view(B, per_new)
        s["new_pages"] = cache[cache.shape[0] - per_new * B:]
        return s
    T = case["nodes"] if case["kind"] == "tree" else case["qrows"]
    # queries that put most of their weight on a few hundred tokens
    s["q_nope"] = (2.0 * torch.randn(B * T, H, d_c, generator=g, device=dev)).to(torch.bfloat16)
    s["q_pe"] = (2.0 * torch.randn(B * T, H, rope, generator=g, device=dev)).to(torch.bfloat16)
    if case["kind"] == "tree":
        counts = rs.randint(1, T + 1, B) if case["ragged"] else np.full(B, T)
        s["counts"] = torch.from_numpy(counts.astype(np.int32)).to(dev) if case["ragged"] else None
        s["mask"] = torch.from_numpy(_tree_masks(T, counts, rs)).to(dev)
    else:
        # one table row and length per query token; query token j of T sees all but the last T-1-j
        s["row_table"] = table.repeat_interleave(T, 0)
        s["row_lens"] = (s["lens"].repeat_interleave(T) + torch.arange(1 - T, 1, device=dev).repeat(B)).to(torch.int32)
        W = int(lens.max())
        s["weights"] = torch.rand(B, W, generator=g, device=dev)
        s["out"] = torch.zeros(B, W, device=dev)
        sc = _scores(s, T)
        sc = sc.masked_fill(~_chain(s, T, sc.shape[-1]), -math.inf)
        s["lse"] = sc.logsumexp(-1).reshape(B * T, H)
    return s


# ---- plain forms -----------------------------------------------------------------------------------
def _dense(s):
    """The cached rows of every request, padded to the longest: latent and rope columns [B, L, C] in
    fp32 and the divisors [B, L, H]."""
    case, cache, table = s["case"], s["cache"], s["table"]
    C, H, page = case["d_c"] + case["rope"], case["heads"], case["page"]
    t = torch.arange(table.shape[1] * page, device=cache.device)[:int(s["table"].shape[1] * page)]
    slots = table.long()[:, t // page] * page + t % page
    rows = cache.view(-1, cache.shape[-1])[slots]
    if case["kv"] == "fp8":
        x = rows[..., :C].contiguous().view(torch.float8_e4m3fn).float() * s["scale"]
        return x, torch.exp2(rows[..., C:C + H].float() * (6.0 / 255.0) - 3.0)
    rms = rows[..., C:C + H].float()
    return rows[..., :C].float(), torch.where(rms > 0, rms, torch.ones_like(rms))


def _scores(s, T, dense=None):
    """[B, T, H, L] in fp32."""
    x, rms = _dense(s) if dense is None else dense
    B, H = x.shape[0], s["case"]["heads"]
    q = torch.cat([s["q_nope"], s["q_pe"]], -1).float().view(B, T * H, -1)
    sc = torch.bmm(q, x.transpose(1, 2)).view(B, T, H, -1)
    return sc / rms.transpose(1, 2)[:, None] * s["sm_scale"]


def _chain(s, T, W):
    t = torch.arange(W, device=s["lens"].device)
    seen = s["lens"][:, None] + torch.arange(1 - T, 1, device=t.device)
    return (t < seen[..., None])[:, :, None]


def _plain_tree(s):
    case, T = s["case"], s["case"]["nodes"]
    dense = _dense(s)
    sc = _scores(s, T, dense)
    t = torch.arange(sc.shape[-1], device=sc.device)
    n = s["counts"].long() if s["counts"] is not None else torch.full_like(s["lens"], T).long()
    node = t - (s["lens"].long() - n)[:, None]                      # [B, L]: which drafted node a token is
    bit = (s["mask"][:, :, None] >> node.clamp(0, 63)[:, None]) & 1
    seen = (node < 0)[:, None] | ((bit == 1) & (node < n[:, None])[:, None])
    seen = seen & (torch.arange(T, device=t.device) < n[:, None])[..., None]
    sc = sc.masked_fill(~seen[:, :, None], -math.inf)
    top = sc.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(sc - top)
    total = p.sum(-1, keepdim=True)
    B, H = sc.shape[0], case["heads"]
    o = torch.bmm((p / total.clamp_min(1e-30)).view(B, T * H, -1), dense[0][..., :case["d_c"]].contiguous())
    lse = torch.log(total) + top
    return {"out": o.view(B * T, H, -1).to(torch.bfloat16), "lse": lse.view(B * T, H)}


def _plain_weights(s):
    T = s["case"]["qrows"]
    sc = _scores(s, T)
    B, H = sc.shape[0], s["case"]["heads"]
    p = torch.exp(sc - s["lse"].view(B, T, H, 1)).masked_fill(~_chain(s, T, sc.shape[-1]), 0.0)
    W = s["weights"].shape[1]
    got = s["weights"] + p.sum((1, 2))[:, :W]
    live = torch.arange(W, device=got.device) < s["lens"][:, None]
    s["out"].copy_(torch.where(live, got, s["out"]))
    return s["out"]


def _plain_evict(s):
    case, w, page = s["case"], s["weights"], s["case"]["page"]
    B, W = w.shape
    K, L = case["keep"], s["lens"].long()[:, None]
    t = torch.arange(W, device=w.device).expand(B, W)
    rank = torch.where((t < case["sink"]) | (t >= L - case["recent"]), 0, 1) + torch.where(t >= L, 2, 0)
    order = torch.sort(torch.where(torch.isnan(w), -math.inf, w), dim=1, descending=True, stable=True).indices
    order = order.gather(1, torch.sort(rank.gather(1, order), dim=1, stable=True).indices)
    n = L.clamp_max(K)
    first = torch.nn.functional.pad(order, (0, max(0, K - W)))[:, :K]
    i = torch.arange(K, device=w.device).expand(B, K)
    index = torch.sort(torch.where(i < n, first, 1 << 40), dim=1).values
    index = torch.where(i < n, index, -1)
    live, src = i < n, index.clamp_min(0)
    flat = s["cache"].view(-1, s["cache"].shape[-1])
    from_slot = s["table"].long().gather(1, src // page) * page + src % page
    to_slot = s["new_table"].long().gather(1, i // page) * page + i % page
    flat[to_slot] = torch.where(live[..., None], flat[from_slot], flat[to_slot])
    s["weights_out"].copy_(torch.where(live, w.gather(1, src), s["weights_out"]))
    return {"index": index.to(torch.int32), "counts": n[:, 0].to(torch.int32), "rows": s["new_pages"], "weights": s["weights_out"]}


def _plain_rotary(s):
    case = s["case"]
    half, o = case["rot"] // 2, case["offset"]
    cos, sin = s["table"][s["positions"]][:, None].split(half, -1)
    turn = _turn_half if case["layout"] == "half" else _turn_pairs
    return {"q": turn(s["q"], cos, sin, o, half), "k": turn(s["k"], cos, sin, o, half)}


def _turn_half(x, cos, sin, o, half):
    y = x.clone()
    a, b = x[..., o:o + half].float(), x[..., o + half:o + 2 * half].float()
    y[..., o:o + half] = (a * cos - b * sin).to(x.dtype)
    y[..., o + half:o + 2 * half] = (b * cos + a * sin).to(x.dtype)
    return y


def _turn_pairs(x, cos, sin, o, half):
    y = x.clone()
    a, b = x[..., o:o + 2 * half:2].float(), x[..., o + 1:o + 2 * half:2].float()
    y[..., o:o + 2 * half:2] = (a * cos - b * sin).to(x.dtype)
    y[..., o + 1:o + 2 * half:2] = (b * cos + a * sin).to(x.dtype)
    return y


# ---- the package's calls ---------------------------------------------------------------------------
def _own(s):
    qmla, case = _qmla(), s["case"]
    if case["kind"] == "rotary":
        q, k = qmla.rotary(s["positions"], s["q"], s["k"], s["table"], layout=case["layout"], offset=case["offset"])
        return {"q": q, "k": k}
    if case["kind"] == "evict":
        index, counts = qmla.evict(s["cache"], s["table"], s["lens"], s["weights"], case["keep"], sink=case["sink"],
                                   recent=case["recent"], dst_block_table=s["new_table"], weights_out=s["weights_out"])
        return {"index": index, "counts": counts, "rows": s["new_pages"], "weights": s["weights_out"]}
    row = dict(page_size=case["page"], sm_scale=s["sm_scale"], kv_fp8=case["kv"] == "fp8", k_scale=s["scale"])
    if case["kind"] == "weights":
        return qmla.attention_weights(s["q_nope"], s["q_pe"], s["cache"], s["row_table"], s["row_lens"], s["lse"],
                                      s["weights"], qrows=case["qrows"], out=s["out"], **row)
    out, lse = qmla.tree_forward(s["q_nope"], s["q_pe"], s["cache"], s["table"], s["lens"], s["mask"],
                                 node_counts=s["counts"], **row)
    return {"out": out, "lse": lse}


_PLAIN = {"tree": _plain_tree, "weights": _plain_weights, "evict": _plain_evict, "rotary": _plain_rotary}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


# ---- bounds and definition -------------------------------------------------------------------------
def work(case):
    if case["kind"] == "rotary":
        es = 4 if case["dtype"] == "fp32" else 2
        heads = case["n"] * (case["heads"] + case["kheads"])
        return dict(bytes=heads * case["dim"] * es * 2 + case["n"] * (case["rot"] * 4 + 8), flops=heads * case["rot"] * 3)
    es = 1 if case["kv"] == "fp8" else 2
    B, H, d_c, rope = case["batch"], case["heads"], case["d_c"], case["rope"]
    lens = _lens(case, 1)
    tokens, row = int(lens.sum()), (d_c + rope + H) * es
    if case["kind"] == "evict":
        kept = int(np.minimum(lens, case["keep"]).sum())
        return dict(bytes=tokens * 4 + kept * (2 * _row_elems(case) * es + 2 * 4 + 4), flops=0)
    T = case["nodes"] if case["kind"] == "tree" else case["qrows"]
    q = B * T * H * (d_c + rope) * 2
    if case["kind"] == "weights":
        return dict(bytes=tokens * (row + 8) + q + B * T * H * 4, flops=2 * T * H * tokens * (d_c + rope))
    return dict(bytes=tokens * row + q + B * T * H * (d_c * 2 + 4), flops=2 * T * H * tokens * (2 * d_c + rope))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        angle = s["positions"].double()[:, None] * _frequencies(case["rot"], case["scaled"]).to(s["q"].device)
        z = torch.polar(torch.ones_like(angle), angle)[:, None]
        o, r = case["offset"], case["rot"]
        out = {}
        for name in ("q", "k"):
            y = s[name].double().clone()
            part = y[..., o:o + r]
            pair = part.unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["layout"] == "half" else part.unflatten(-1, (r // 2, 2))
            turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
            y[..., o:o + r] = (turned.transpose(-1, -2) if case["layout"] == "half" else turned).flatten(-2)
            out[name] = y
        return out
    lens, page, H, d_c = s["lens"].tolist(), case["page"], case["heads"], case["d_c"]
    flat = s["cache"].view(-1, s["cache"].shape[-1])
    if case["kind"] == "evict":
        index = np.full((len(lens), case["keep"]), -1, dtype=np.int32)
        w, to = s["weights"].double().cpu().numpy(), s["weights_out"].double()
        for b, L in enumerate(lens):
            keep = np.arange(L)
            if L > case["keep"]:
                middle = np.arange(case["sink"], L - case["recent"])
                best = middle[np.lexsort((middle, -w[b, middle]))][:case["keep"] - case["sink"] - case["recent"]]
                keep = np.sort(np.concatenate([np.arange(case["sink"]), best, np.arange(L - case["recent"], L)]))
            index[b, :len(keep)] = keep
            src, i = torch.from_numpy(keep).to(flat.device), torch.arange(len(keep), device=flat.device)
            flat[s["new_table"][b].long()[i // page] * page + i % page] = flat[s["table"][b].long()[src // page] * page + src % page]
            to[b, :len(keep)] = s["weights"][b, src].double()
        counts = np.minimum(np.array(lens), case["keep"]).astype(np.int32)
        rows = s["new_pages"] if case["kv"] == "fp8" else s["new_pages"].double()
        return {"index": torch.from_numpy(index), "counts": torch.from_numpy(counts), "rows": rows, "weights": to}
    T = case["nodes"] if case["kind"] == "tree" else case["qrows"]
    out, lses = [], []
    total = s["out"].double() if case["kind"] == "weights" else None
    for b, L in enumerate(lens):
        t = torch.arange(L, device=flat.device)
        rows = flat[s["table"][b].long()[t // page] * page + t % page]
        C = d_c + case["rope"]
        if case["kv"] == "fp8":
            x = rows[:, :C].contiguous().view(torch.float8_e4m3fn).double() * s["scale"].double()
            rms = torch.pow(2.0, rows[:, C:C + H].double() * 6.0 / 255.0 - 3.0)
        else:
            x, rms = rows[:, :C].double(), rows[:, C:C + H].double()
            rms = torch.where(rms > 0, rms, torch.ones_like(rms))
        q = torch.cat([s["q_nope"], s["q_pe"]], -1)[b * T:(b + 1) * T].double()
        sc = torch.matmul(q.reshape(T * H, C), x.T.contiguous()).view(T, H, L) / rms.T * s["sm_scale"]
        if case["kind"] == "weights":
            for j in range(T):
                n = L - (T - 1 - j)
                got = torch.exp(sc[j, :, :n] - s["lse"].view(-1, T, H)[b, j].double()[:, None]).sum(0)
                total[b, :n] += got
            total[b, :L] += s["weights"][b, :L].double()
            continue
        n = int(s["counts"][b]) if s["counts"] is not None else T
        for j in range(T):
            sees = [i for i in range(n) if (int(s["mask"][b, j]) >> i) & 1] if j < n else []
            sel = torch.tensor(sees, device=flat.device, dtype=torch.long) + (L - n)
            sel = torch.cat([torch.arange(L - n, device=flat.device), sel]) if j < n else sel
            if sel.numel() == 0:
                out.append(torch.zeros(H, d_c, dtype=torch.float64, device=flat.device))
                lses.append(torch.full((H,), -math.inf, dtype=torch.float64, device=flat.device))
                continue
            z = sc[j][:, sel]
            lses.append(torch.logsumexp(z, -1))
            out.append(torch.matmul(torch.softmax(z, -1), x[sel, :d_c]))
    if case["kind"] == "weights":
        return total
    return {"out": torch.stack(out), "lse": torch.stack(lses)}
