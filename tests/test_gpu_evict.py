"""Eviction: `evict_select` exactly as a sort says, `cache_compact` byte for byte, in place and to other pages,
and the run decode -> weights -> evict -> decode as it would be used."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ref_select(w, lens, keep, sink, recent):
    w = np.where(np.isnan(w), -np.inf, w).astype(np.float64)
    index = np.full((len(lens), keep), -1, np.int32)
    counts = np.zeros(len(lens), np.int32)
    for b, L in enumerate(lens):
        L = max(0, min(int(L), w.shape[1]))
        kept = np.arange(L)
        if L > keep:
            mid = np.arange(sink, L - recent)
            best = mid[np.lexsort((mid, -w[b, mid]))][:keep - sink - recent]
            kept = np.sort(np.concatenate([np.arange(sink), best, np.arange(L - recent, L)]))
        index[b, :len(kept)], counts[b] = kept, len(kept)
    return index, counts


def _weights(kind, B, W, seed):
    r = np.random.RandomState(seed)
    w = np.exp(2 * r.randn(B, W)).astype(np.float32)
    if kind == "ties":
        w = r.randint(0, 3, (B, W)).astype(np.float32)
    elif kind == "equal":
        w[:] = 0.25
    elif kind == "odd":   # signs, zeros of both signs, infinities, NaN, subnormals
        w = r.choice(np.array([0.0, -0.0, -1.5, 3.0, np.inf, -np.inf, np.nan, 1e-42, -1e-42, 1e38], np.float32), (B, W))
    elif kind == "close":  # equal in all but the last bits
        w = (np.float32(1.0) + r.randint(0, 40, (B, W)).astype(np.float32) * np.float32(2.0 ** -23)).astype(np.float32)
    return w


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd", "close"])
@pytest.mark.parametrize("lens,keep,sink,recent", [
    ([0, 1, 5, 64, 65], 8, 2, 3), ([7, 8, 9, 4097], 8, 8, 0), ([1000, 1023, 1025, 3000], 700, 4, 256), ([40000, 20011], 9999, 4, 1000),
    ([50, 60], 0, 0, 0), ([3, 900], 1, 0, 0), ([3, 900], 1, 0, 1), ([-4, 2000], 2000, 0, 5), ([300, 5000], 299, 149, 149)])
def test_select(gpu, kind, lens, keep, sink, recent):
    import qmla
    W = max(max(lens), 1) + 3
    w = _weights(kind, len(lens), W, seed=keep + len(lens))
    wide = torch.zeros(len(lens), W + 5, device=gpu)
    wide[:, :W] = torch.from_numpy(w)
    index, counts = qmla.evict_select(wide[:, :W], torch.tensor(lens, dtype=torch.int32, device=gpu), keep, sink=sink, recent=recent)
    ri, rc = _ref_select(w, lens, keep, sink, recent)
    assert np.array_equal(counts.cpu().numpy(), rc) and np.array_equal(index.cpu().numpy(), ri)


def test_select_width_cuts_lengths(gpu):
    import qmla
    w = _weights("spread", 1, 500, 1)
    index, counts = qmla.evict_select(torch.from_numpy(w).to(gpu), torch.tensor([900], dtype=torch.int32, device=gpu), 100, recent=10)
    ri, rc = _ref_select(w, [500], 100, 0, 10)
    assert np.array_equal(index.cpu().numpy(), ri) and int(counts) == 100


def _cache(gpu, pages, P, row, dtype, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.randint(0, 256, (pages, P, row), dtype=torch.uint8, generator=g, device=gpu)
    return x.view(dtype) if dtype != torch.uint8 else x


def _moved(cache, table, dst, index, counts, first, P):
    """The cache after the copies, from its bytes before them."""
    out = cache.clone()
    flat, old = out.view(-1, cache.shape[-1]), cache.view(-1, cache.shape[-1]).clone()
    for b in range(index.shape[0]):
        for i in range(int(counts[b])):
            t, f = int(index[b, i]), int(first[b]) + i
            flat[int(dst[b, f // P]) * P + f % P] = old[int(table[b, t // P]) * P + t % P]
    return out


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("P,row,dtype,keep", [(64, 608, torch.uint8, 300), (16, 1200, torch.bfloat16, 37), (100, 613, torch.uint8, 200),
                                              (1, 36, torch.uint8, 90), (784, 1048, torch.bfloat16, 2500), (7, 6, torch.bfloat16, 64)])
def test_compact(gpu, in_place, P, row, dtype, keep):
    import qmla
    B = 3
    lens = [keep + 70, keep, max(1, keep // 2)]
    per = -(-max(lens) // P)
    pages = 2 * B * per + 3
    cache = _cache(gpu, pages, P, row, dtype)
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(5)).to(torch.int32)
    table, other = perm[:B * per].view(B, per).to(gpu), perm[B * per:2 * B * per].view(B, per).to(gpu)
    r = np.random.RandomState(keep)
    index = np.full((B, keep + 4), -1, np.int32)
    counts, first = np.array([keep, keep // 3, 0], np.int32), np.array([0, 2, 1], np.int32)
    for b in range(B):
        if counts[b]:
            index[b, :counts[b]] = np.sort(r.choice(np.arange(first[b], lens[b]), min(counts[b], lens[b] - first[b]), replace=False))
    w = torch.rand(B, max(lens), device=gpu)
    wide = torch.from_numpy(index).to(gpu)
    cnt, fst = torch.from_numpy(counts).to(gpu), torch.from_numpy(first).to(gpu)
    dst = table if in_place else other
    want = _moved(cache.view(torch.uint8), table, dst, index, counts, first, P)
    w_out = w if in_place else torch.full((B, keep + 9), 7.0, device=gpu)
    w_want = w_out.clone()
    for b in range(B):
        n = counts[b]
        w_want[b, first[b]:first[b] + n] = w[b][wide[b, :n].long()]
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    qmla.cache_compact(cache, table, wide, cnt, first=fst, dst_block_table=None if in_place else other, weights=w, weights_out=w_out, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0 and torch.equal(cache.view(torch.uint8), want) and torch.equal(w_out, w_want)


def test_in_place_over_many_steps(gpu):
    """A dense move of one token over more rows than a step holds, and the reverse hazard: rows whose
    source is a few rows ahead of them, whole request."""
    import qmla
    P, row = 64, 608
    for L, drop in ((9000, [0]), (9000, [3, 4, 5, 2047, 2048, 2049, 4096, 8191])):
        pages = -(-L // P)
        cache = _cache(gpu, pages, P, row, torch.uint8, seed=L)
        table = torch.randperm(pages, device=gpu).to(torch.int32)[None]
        keep = np.setdiff1d(np.arange(L), drop).astype(np.int32)
        src = torch.from_numpy(keep).to(gpu).long()
        old = cache.view(-1, row).clone()
        slot = table[0].long()[src // P] * P + src % P
        qmla.cache_compact(cache, table, torch.from_numpy(keep)[None].to(gpu), torch.tensor([len(keep)], dtype=torch.int32, device=gpu))
        i = torch.arange(len(keep), device=gpu)
        assert torch.equal(cache.view(-1, row)[table[0].long()[i // P] * P + i % P], old[slot])


def test_compact_refuses_rows_outside(gpu):
    """Tokens and pages outside the tables or the cache: left out and reported."""
    import qmla
    for in_place in (True, False):
        cache = _cache(gpu, 6, 16, 32, torch.uint8)
        table = torch.tensor([[0, 1], [2, 99]], dtype=torch.int32, device=gpu)
        other = torch.tensor([[3, 4], [5, -1]], dtype=torch.int32, device=gpu)
        index = torch.tensor([[3, 33, 1 << 30], [17, 18, -5]], dtype=torch.int32, device=gpu)
        before = cache.clone()
        status = torch.zeros(1, dtype=torch.int32, device=gpu)
        qmla.cache_compact(cache, table, index, torch.tensor([3, 99], dtype=torch.int32, device=gpu),
                           dst_block_table=None if in_place else other, status=status)
        torch.cuda.synchronize()
        assert int(status) == -8
        page = 0 if in_place else 3
        assert torch.equal(cache[page, 0], before[0, 3])
        cache[page, 0] = before[page, 0]
        assert torch.equal(cache, before)


def test_compact_far_pages(gpu):
    import qmla
    P, row = 64, 608
    far = (1 << 32) // (P * row) + 3
    cache = torch.empty(far + 4, P, row, dtype=torch.uint8, device=gpu)
    cache[far:] = _cache(gpu, 4, P, row, torch.uint8)
    table = torch.tensor([[far, far + 1]], dtype=torch.int32, device=gpu)
    index = torch.arange(1, 128, 2, dtype=torch.int32, device=gpu)[None]
    want = cache[far:far + 2].reshape(-1, row)[1:128:2].clone()
    cnt = torch.tensor([64], dtype=torch.int32, device=gpu)
    qmla.cache_compact(cache, table, index, cnt, dst_block_table=torch.tensor([[far + 2]], dtype=torch.int32, device=gpu))
    assert torch.equal(cache[far + 2], want)
    qmla.cache_compact(cache, table, index, cnt)
    assert torch.equal(cache[far], want)


@pytest.mark.parametrize("in_place", [True, False])
def test_decode_weigh_evict_decode(gpu, in_place):
    """As a server runs it: a decode step, its weights, the cut, and the next decode on what was kept equals a
    decode over those tokens' rows gathered by hand. Graph replays repeat the eager cut."""
    import qmla
    from qmla.synth import make_case
    lens = [900, 130, 4000]
    c = make_case(batch=3, heads=24, d_c=512, rope_w=64, page_size=64, lens=lens, kv="fp8", rms_mode="log8", seed=3, device=gpu, q_amp=3.0,
                  extra_pages=12)
    kw = dict(page_size=64, sm_scale=c.sm_scale, kv_fp8=True, k_scale=c.k_scale)
    w = torch.zeros(3, 4000, device=gpu)
    _, lse = qmla.forward(c.q_nope, c.q_pe, c.cache, c.block_table, c.seq_lens, **kw)
    qmla.attention_weights(c.q_nope, c.q_pe, c.cache, c.block_table, c.seq_lens, lse, w, **kw)
    ri, rc = _ref_select(w.cpu().numpy(), lens, 200, 4, 50)
    used = set(int(x) for b, L in enumerate(lens) for x in c.block_table[b, :-(-L // 64)])
    free = [x for x in range(c.cache.shape[0]) if x not in used][:12]
    new = torch.tensor(free, dtype=torch.int32, device=gpu).view(3, 4)
    before, w0 = c.cache.clone(), w.clone()
    dst = None if in_place else new
    table = c.block_table if in_place else new

    def cut():
        return qmla.evict(c.cache, c.block_table, c.seq_lens, w, 200, sink=4, recent=50, dst_block_table=dst)
    index, counts = cut()
    assert np.array_equal(index.cpu().numpy(), ri) and np.array_equal(counts.cpu().numpy(), rc)
    after, w1 = c.cache.clone(), w.clone()
    if in_place:
        for b in range(3):
            assert torch.equal(w[b, :rc[b]], w0[b][torch.from_numpy(ri[b, :rc[b]]).long().to(gpu)])
    o, lse = qmla.forward(c.q_nope, c.q_pe, c.cache, table, counts, **kw)
    hand = torch.zeros(12, 64, 1, 608, dtype=torch.uint8, device=gpu)
    for b in range(3):
        t = torch.from_numpy(ri[b, :rc[b]]).long()
        slot = c.block_table[b].cpu().long()[t // 64] * 64 + t % 64
        hand.view(3, 256, 608)[b, :rc[b]] = before.view(-1, 608)[slot.to(gpu)]
    ho, hl = qmla.forward(c.q_nope, c.q_pe, hand, torch.arange(12, dtype=torch.int32, device=gpu).view(3, 4), counts, **kw)
    assert torch.equal(o, ho) and torch.equal(lse, hl)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gi, gc = cut()
    for _ in range(3):
        c.cache.copy_(before)
        w.copy_(w0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(gi, index) and torch.equal(gc, counts) and torch.equal(c.cache, after) and torch.equal(w, w1)


def test_tree_accept_then_decode(gpu):
    """A verified tree: the accepted nodes' rows move behind the context in place, and a decode over context
    plus path equals the last accepted node's row of the tree call, to both calls' roundings."""
    import qmla
    from tests.op_cases import ref_tree, row_kw, tree_case
    lens, T = [150, 700], 8
    c, qn, qp, _, _ = tree_case(gpu, kv="bf16", rms_mode="bf16", d_c=512, rope=64, heads=24, page=16, lens=lens, nodes=T, seed=9)
    parents = [[-1, 0, 0, 1, 1, 2, 4, 5], [-1, -1, 1, 1, 3, 2, 4, 6]]
    mask = qmla.tree_mask(parents).to(gpu)
    o, lse = qmla.tree_forward(qn, qp, c.cache, c.block_table, c.seq_lens, mask, **row_kw(c))
    paths = [[0, 1, 4, 6], [1, 3, 4]]
    first = c.seq_lens - T
    index = torch.full((2, 4), -1, dtype=torch.int32)
    for b, path in enumerate(paths):
        index[b, :len(path)] = torch.tensor(path, dtype=torch.int32) + lens[b] - T
    counts = torch.tensor([4, 3], dtype=torch.int32, device=gpu)
    _, _, ob, lb = ref_tree(c, qn, qp, lens, mask.cpu(), None)
    qmla.cache_compact(c.cache, c.block_table, index.to(gpu), counts, first=first)
    last = torch.tensor([paths[0][-1], T + paths[1][-1]], device=gpu)
    fo, fl = qmla.forward(qn[last], qp[last], c.cache, c.block_table, first + counts, **row_kw(c))
    assert (fo.float() - o[last].float()).abs().max() < 2e-2 and (fl - lse[last]).abs().max() < 2e-2
