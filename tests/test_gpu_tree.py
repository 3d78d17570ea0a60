"""`qmla.tree_forward` against float64 at the layouts, lengths and masks where it can go wrong. Bounds are the
ones tests/op_cases.py derives."""
import pytest
import torch

from tests.op_cases import close, fp8_kw, ref_tree, row_kw, tree_case

pytestmark = pytest.mark.gpu

# (kv, rms, d_c, rope, heads, page)
LAYOUTS = [
    ("fp8", "log8", 512, 64, 24, 64), ("bf16", "bf16", 512, 64, 24, 16), ("fp8", "e4m3", 512, 64, 7, 64),
    ("fp8", "bf16_bytes", 512, 64, 24, 100), ("bf16", "none", 512, 0, 3, 64), ("fp8", "none", 512, 40, 1, 1),
    ("fp8", "log8", 768, 232, 24, 784), ("bf16", "bf16", 768, 116, 12, 64), ("fp8", "log8", 256, 116, 12, 32),
    ("bf16", "bf16", 256, 232, 24, 64), ("fp8", "log8", 1792, 232, 24, 64), ("bf16", "bf16", 1792, 64, 24, 1600),
    ("fp8", "log8", 512, 64, 64, 64), ("bf16", "bf16", 256, 256, 24, 64),
]


def _run(c, qn, qp, mask, counts, cap=0.0, **kw):
    import qmla
    o, lse = qmla.tree_forward(qn, qp if c.rope_w else None, c.cache, c.block_table, c.seq_lens, mask, node_counts=counts,
                               **row_kw(c, cap), **kw)
    torch.cuda.synchronize()
    return o, lse


def _check(name, c, qn, qp, mask, counts, o, lse, cap=0.0, lens=None):
    ro, rl, ob, lb = ref_tree(c, qn, qp, c.seq_lens.cpu() if lens is None else lens, mask.cpu(),
                              None if counts is None else counts.cpu(), cap)
    close(f"{name} out", o, ro, ob, o.dtype)
    if lse is not None:
        close(f"{name} lse", lse, rl, lb, lse.dtype)


@pytest.mark.parametrize("nodes", [1, 5, 24])
@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda f: "-".join(map(str, f)))
def test_layouts(gpu, layout, nodes):
    import qmla
    kv, rms, d_c, rope, heads, page = layout
    c, qn, qp, par, counts = tree_case(gpu, kv=kv, rms_mode=rms, d_c=d_c, rope=rope, heads=heads, page=page,
                                       lens=[nodes, 33 + nodes, 500], nodes=nodes, seed=nodes + d_c, ragged=nodes == 24)
    mask = qmla.tree_mask(par).to(gpu)
    counts = None if counts is None else counts.to(gpu)
    o, lse = _run(c, qn, qp, mask, counts)
    _check(f"{layout} nodes {nodes}", c, qn, qp, mask, counts, o, lse)


# lengths of zero, below the node count, on and beside tile and page borders, and one long request
@pytest.mark.parametrize("lens", [[0, 1, 3, 9], [31, 32, 33, 64], [65, 63, 128, 1], [5000, 0, 77, 2], [0, 0]])
@pytest.mark.parametrize("kv", ["fp8", "bf16"])
def test_lengths(gpu, kv, lens):
    import qmla
    c, qn, qp, par, counts = tree_case(gpu, kv=kv, rms_mode={"fp8": "log8", "bf16": "bf16"}[kv], d_c=512, rope=64, heads=24,
                                       page=16, lens=lens, nodes=9, seed=sum(lens), ragged=True)
    c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    mask = qmla.tree_mask(par).to(gpu)
    for cnt in (None, counts.to(gpu)):
        o, lse = _run(c, qn, qp, mask, cnt)
        _check(f"{kv} lens {lens}", c, qn, qp, mask, cnt, o, lse)


def test_full_tree_of_64_nodes_bit_63(gpu):
    """64 nodes: the last node's own bit is the sign bit of its word; a chain sees what `forward`'s rows see."""
    import qmla
    c, qn, qp, _, _ = tree_case(gpu, kv="fp8", rms_mode="log8", d_c=512, rope=64, heads=24, page=64, lens=[300, 64], nodes=64,
                                seed=3)
    chain = torch.arange(-1, 63).repeat(2, 1)
    mask = qmla.tree_mask(chain).to(gpu)
    assert int(mask[0, 63]) == -1
    o, lse = _run(c, qn, qp, mask, None)
    _check("chain of 64", c, qn, qp, mask, None, o, lse)


def test_chain_equals_forward(gpu):
    """A chain of drafted tokens, written by the cache writer, gives what `forward` gives on the same
    cache, to the sum of both calls' roundings."""
    import qmla
    T, lens = 4, [130, 700]
    c, qn, qp, _, _ = tree_case(gpu, kv="fp8", rms_mode="log8", d_c=512, rope=64, heads=24, page=64, lens=lens, nodes=T, seed=11)
    slots = torch.stack([c.block_table[b, t // 64].long() * 64 + t % 64 for b, L in enumerate(lens) for t in range(L - T, L)])
    x = torch.randn(len(slots), 512, device=gpu).to(torch.bfloat16)
    pe = torch.cat([torch.randn(len(slots), 64, device=gpu), 1 + torch.rand(len(slots), 24, device=gpu)], 1).to(torch.bfloat16)
    qmla.cache_write(x, pe, c.cache, slots, rope_w=64, rms_heads=24, kv_fp8=True, rms="log8", k_scale=c.k_scale)
    mask = qmla.tree_mask(torch.arange(-1, T - 1).repeat(2, 1)).to(gpu)
    o, lse = _run(c, qn, qp, mask, None)
    _check("written chain", c, qn, qp, mask, None, o, lse)
    table = c.block_table.repeat_interleave(T, 0)
    sl = (c.seq_lens.repeat_interleave(T) + torch.arange(1 - T, 1, device=gpu).repeat(2)).to(torch.int32)
    fo, fl = qmla.forward(qn, qp, c.cache, table, sl, page_size=64, sm_scale=c.sm_scale, qrows=T, **fp8_kw(c))
    assert (o.float() - fo.float()).abs().max() < 6e-2 and (lse - fl).abs().max() < 2e-2


def test_masks_that_leave_a_row_empty(gpu):
    """Mask word 0 with no context: zeros and -inf; with context: the context alone."""
    c, qn, qp, _, _ = tree_case(gpu, kv="bf16", rms_mode="bf16", d_c=512, rope=64, heads=24, page=16, lens=[6, 40], nodes=6, seed=5)
    mask = torch.zeros(2, 6, dtype=torch.int64, device=gpu)
    mask[0, 2] = 0b000101
    mask[1, 5] = 0b111111
    o, lse = _run(c, qn, qp, mask, None)
    _check("empty rows", c, qn, qp, mask, None, o, lse)
    assert torch.isneginf(lse[0]).all() and (o[0] == 0).all()
    # bits of nodes that are not there change nothing
    o2, lse2 = _run(c, qn, qp, mask | (1 << 6) | (1 << 40), None)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("kv", ["fp8", "bf16"])
@pytest.mark.parametrize("d_c,rope", [(512, 64), (768, 232), (1792, 64)])
def test_bad_elements_reach_the_rows_that_see_them(gpu, kv, d_c, rope):
    """NaN (and bf16 infinities) in a drafted token's latent or rope, in the slots past the length, in another
    head's divisor, and in a query row."""
    import qmla
    T, lens = 8, [40, 100]
    c, qn, qp, par, _ = tree_case(gpu, kv=kv, rms_mode={"fp8": "log8", "bf16": "bf16"}[kv], d_c=d_c, rope=rope, heads=24, page=64,
                                  lens=lens, nodes=T, seed=21)
    mask = qmla.tree_mask(par).to(gpu)
    flat = c.cache.view(-1, c.cache.shape[-1])
    bad = 0x7f if kv == "fp8" else float("nan")

    def slot(b, t):
        return int(c.block_table[b, t // 64]) * 64 + t % 64
    # past the lengths, whole rows
    for b, L in enumerate(lens):
        for t in range(L, (L + 63) // 64 * 64):
            flat[slot(b, t)] = bad
    o, lse = _run(c, qn, qp, mask, None)
    _check("stale rows", c, qn, qp, mask, None, o, lse)
    # drafted node 3 of request 0 in its latent, node 5 of request 1 in its rope
    keep = flat.clone()
    flat[slot(0, lens[0] - T + 3), 77] = bad if kv == "fp8" else float("inf")
    flat[slot(1, lens[1] - T + 5), d_c + 3] = bad
    got, glse = _run(c, qn, qp, mask, None)
    for b, i in ((0, 3), (1, 5)):
        for j in range(T):
            row = b * T + j
            if (int(mask[b, j]) >> i) & 1:
                assert torch.isnan(got[row]).all() and torch.isnan(glse[row]).all(), (b, j)
            else:
                assert torch.equal(got[row], o[row]) and torch.equal(glse[row], lse[row]), (b, j)
    flat.copy_(keep)
    # a query row
    q2 = qn.clone()
    q2[3, 4, 100] = float("nan")
    got, glse = _run(c, q2, qp, mask, None)
    assert torch.isnan(got[3, 4]).all() and torch.isnan(glse[3, 4])
    got[3, 4], glse[3, 4] = o[3, 4], lse[3, 4]
    assert torch.equal(got, o) and torch.equal(glse, lse)
    if kv == "bf16":   # a divisor of head 2 of drafted node 1: infinite, so its score is 0 for that head
        flat[slot(0, lens[0] - T + 1), d_c + rope + 2] = float("inf")
        got, glse = _run(c, qn, qp, mask, None)
        _check("infinite divisor", c, qn, qp, mask, None, got, glse)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
def test_strides_types_cap_and_workspaces(gpu, dt):
    import qmla
    c, qn, qp, par, counts = tree_case(gpu, kv="fp8", rms_mode="log8", d_c=512, rope=64, heads=7, page=64, lens=[400, 90], nodes=11,
                                       seed=31, ragged=True)
    mask = torch.full((2, 20), 7, dtype=torch.int64, device=gpu)[:, :11]
    mask.copy_(qmla.tree_mask(par))
    counts = counts.to(gpu)
    whole = torch.zeros(22, 9, 577, dtype=torch.bfloat16, device=gpu)      # odd strides: element loads
    whole[:, 1:8, :512], whole[:, 1:8, 512:576] = qn, qp
    out = torch.full((22, 8, 520), 5.0, dtype=dt, device=gpu)
    lse = torch.full((22, 9), 5.0, dtype=torch.float32, device=gpu)
    ws = qmla.Workspace()
    o, l = _run(c, whole[:, 1:8, :512], whole[:, 1:8, 512:576], mask, counts, 9.0, out=out[:, :7, :512], lse=lse[:, :7], workspace=ws)
    _check(f"strided {dt}", c, qn, qp, mask, counts, o, l, 9.0)
    assert (out[:, 7] == 5).all() and (out[:, :, 512:] == 5).all() and (lse[:, 7:] == 5).all()
    o2, _ = _run(c, qn, qp, mask, counts, 9.0, out=torch.empty_like(out[:, :7, :512].contiguous()), workspace=ws, return_lse=False)
    assert torch.equal(o2, o)


def test_repeats_bit_for_bit_and_in_a_graph(gpu):
    """Equal inputs give equal bits, eager and replayed; the graph's scratch is its own."""
    import qmla
    c, qn, qp, par, _ = tree_case(gpu, kv="bf16", rms_mode="bf16", d_c=512, rope=64, heads=24, page=16, lens=[2000, 300], nodes=16, seed=41)
    mask = qmla.tree_mask(par).to(gpu)
    first = _run(c, qn, qp, mask, None)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _run(c, qn, qp, mask, None)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = qmla.tree_forward(qn, qp, c.cache, c.block_table, c.seq_lens, mask, **row_kw(c))
    for q in (1.0, 0.5, 1.0):
        qn.mul_(q)
        want = _run(c, qn, qp, mask, None)
        o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    assert torch.equal(first[0], first[0])


def test_pages_outside_the_cache(gpu):
    """An entry outside the cache reads page 0 and says so; the other request is untouched."""
    import qmla
    c, qn, qp, par, _ = tree_case(gpu, kv="fp8", rms_mode="log8", d_c=512, rope=64, heads=24, page=64, lens=[300, 300], nodes=4, seed=51)
    mask = qmla.tree_mask(par).to(gpu)
    want, _ = _run(c, qn, qp, mask, None)
    c.block_table[0, 2] = c.cache.shape[0]
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    got, _ = _run(c, qn, qp, mask, None, status=status)
    assert int(status) == -8 and torch.equal(got[4:], want[4:])


def test_far_pages(gpu):
    """Pages whose offset passes 2^32 bytes."""
    import qmla
    c, qn, qp, par, _ = tree_case(gpu, kv="fp8", rms_mode="log8", d_c=512, rope=64, heads=24, page=64, lens=[200, 64], nodes=4, seed=61)
    mask = qmla.tree_mask(par).to(gpu)
    want, wl = _run(c, qn, qp, mask, None)
    n = c.cache.shape[0]
    far = (1 << 32) // (64 * c.cache.shape[-1]) + 5
    big = torch.empty(far + n, *c.cache.shape[1:], dtype=torch.uint8, device=gpu)
    big[far:] = c.cache
    c.cache, c.block_table = big, c.block_table + far
    o, lse = _run(c, qn, qp, mask, None)
    assert torch.equal(o, want) and torch.equal(lse, wl)


def test_context_larger_than_the_batch_of_rows(gpu):
    """Many workgroups on one row tile, and many row tiles of one workgroup."""
    import qmla
    for lens, nodes, heads in (([6000], 1, 1), ([40] * 150, 6, 24)):
        c, qn, qp, par, counts = tree_case(gpu, kv="fp8", rms_mode="log8", d_c=256, rope=64, heads=heads, page=64, lens=lens, nodes=nodes, seed=71, ragged=True)
        mask = qmla.tree_mask(par).to(gpu)
        counts = counts.clamp_min(1).to(gpu)
        o, lse = _run(c, qn, qp, mask, counts)
        _check(f"{len(lens)} requests", c, qn, qp, mask, counts, o, lse)
