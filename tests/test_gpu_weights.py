"""`qmla.attention_weights` against float64. Bounds: see tests/op_cases.py; a token's sum adds its rows' p, each
off by its score's bound, with one fp32 rounding an addition."""
import pytest
import torch

from qmla.synth import make_case
from tests.op_cases import U32, close, queries, row_kw, rows_of, scores

pytestmark = pytest.mark.gpu

LAYOUTS = [  # (kv, rms, d_c, rope, heads, qrows, groups, page)
    ("fp8", "log8", 512, 64, 24, 1, 1, 64), ("fp8", "log8", 512, 64, 24, 4, 1, 64), ("fp8", "log8", 512, 64, 24, 4, 2, 64),
    ("bf16", "bf16", 512, 64, 24, 3, 1, 16), ("bf16", "bf16", 512, 64, 7, 1, 1, 100), ("fp8", "e4m3", 512, 64, 7, 2, 1, 64),
    ("fp8", "bf16_bytes", 512, 64, 24, 1, 1, 1), ("fp8", "bf16_bytes", 512, 64, 5, 1, 1, 64), ("bf16", "none", 512, 0, 3, 1, 1, 64),
    ("fp8", "none", 512, 40, 1, 1, 1, 64), ("fp8", "log8", 768, 232, 24, 4, 1, 784), ("bf16", "bf16", 256, 116, 12, 4, 1, 64),
    ("bf16", "bf16", 768, 116, 12, 1, 1, 64), ("fp8", "log8", 768, 116, 12, 1, 1, 64), ("fp8", "log8", 1792, 232, 24, 4, 1, 64),
    ("bf16", "bf16", 1792, 64, 24, 2, 1, 1600), ("fp8", "log8", 512, 64, 64, 8, 1, 64), ("bf16", "bf16", 64, 18, 24, 1, 1, 64),
]


def _case(gpu, layout, lens, seed):
    kv, rms, d_c, rope, heads, qrows, groups, page = layout
    return make_case(batch=len(lens), heads=heads, d_c=d_c, rope_w=rope, page_size=page, lens=lens, kv=kv, rms_mode=rms, seed=seed,
                     device=gpu, qrows=qrows, groups=groups, rms="spread", q_amp=2.0)


def _ref(c, lse, before, cap=0.0):
    """(weights, bound) in float64."""
    T, n_req = c.qrows, c.seq_lens.shape[0] // c.qrows
    out, bound = before.cpu().double().clone(), torch.zeros_like(before.cpu().double())
    sl = c.seq_lens.cpu()
    for b in range(n_req):
        L = int(sl[b * T + T - 1])
        if L <= 0:
            continue
        x, _, rms = rows_of(c, b * T + T - 1, L)
        s, d = scores(c, queries(c, c.q_nope, c.q_pe, list(range(b * T, b * T + T))), x, rms, cap)
        l = lse.cpu().double()[b * T:b * T + T]
        n = min(L, before.shape[1])
        for j in range(T):
            seen = max(0, L - (T - 1 - j))
            p = torch.exp(s[j] - l[j][:, None]).masked_fill(torch.isneginf(l[j])[:, None], 0.0)
            far = d[j] + U32 * 8.0 * (l[j].abs()[:, None].nan_to_num(0, 0, 0))
            p[:, seen:], far[:, seen:] = 0, 0
            out[b, :n] += p.sum(0)[:n]
            bound[b, :n] += (p * torch.expm1(far)).sum(0)[:n]
        bound[b, :n] += U32 * (T * c.heads + 2) * out[b, :n].abs()
    return out, bound


def _decode(c, cap=0.0):
    import qmla
    from tests.op_cases import fp8_kw
    return qmla.forward(c.q_nope, c.q_pe if c.rope_w else None, c.cache, c.block_table, c.seq_lens, d_c=c.d_c, rope_w=c.rope_w,
                        rms_offset=c.rms_offset, page_size=c.page_size, sm_scale=c.sm_scale, qrows=c.qrows, groups=c.groups,
                        logit_cap=cap, **fp8_kw(c))


def _lse(c, cap=0.0):
    """What the softmax of every row sums to, in float64, as a decode returns it."""
    T = c.qrows
    out = torch.full((c.seq_lens.shape[0], c.heads), -float("inf"), dtype=torch.float64)
    for b in range(out.shape[0] // T):
        L = int(c.seq_lens[b * T + T - 1])
        if L <= 0:
            continue
        x, _, rms = rows_of(c, b * T + T - 1, L)
        s, _ = scores(c, queries(c, c.q_nope, c.q_pe, list(range(b * T, b * T + T))), x, rms, cap)
        for j in range(T):
            n = L - (T - 1 - j)
            if n > 0:
                out[b * T + j] = torch.logsumexp(s[j][:, :n], -1)
    return out.float().to(c.cache.device)


def _run(c, lse, w, cap=0.0, **kw):
    import qmla
    r = qmla.attention_weights(c.q_nope, c.q_pe if c.rope_w else None, c.cache, c.block_table, c.seq_lens, lse, w, qrows=c.qrows,
                               groups=c.groups, **row_kw(c, cap), **kw)
    torch.cuda.synchronize()
    return r


@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda f: "-".join(map(str, f)))
def test_layouts(gpu, layout):
    lens = [1, 33, 64, 333, 0, 2]
    c = _case(gpu, layout, lens, seed=layout[2] + layout[4])
    lse = _lse(c)
    w = torch.rand(len(lens), 340, device=gpu)
    want, bound = _ref(c, lse, w)
    got = w.clone()
    assert _run(c, lse, got) is got
    close(f"weights {layout}", got, want, bound, torch.float32)
    for b, L in enumerate(lens):   # columns behind the sequence stay as they were
        assert torch.equal(got[b, L:], w[b, L:])
    out = torch.full((len(lens), 400), 3.0, device=gpu)[:, :340]
    _run(c, lse, w, out=out)
    for b, L in enumerate(lens):
        assert torch.equal(out[b, :L], got[b, :L]) and (out[b, L:] == 3).all()


def test_follows_forward(gpu):
    """With the decode's own lse every row's weights sum to one, to the decode's accuracy; a cap and a second step
    accumulate."""
    c = _case(gpu, ("fp8", "log8", 512, 64, 24, 4, 1, 64), [700, 90, 3], seed=7)
    w = torch.zeros(3, 700, device=gpu)
    _, lse = _decode(c, 20.0)
    _run(c, lse, w, 20.0)
    rows = torch.tensor([4, 4, 3]) * 24.0   # the first row of the request of 3 tokens sees none
    assert (w.sum(1).cpu() - rows).abs().max() < 96 * 2e-2
    once = w.clone()
    _run(c, lse, w, 20.0)
    assert torch.allclose(w, 2 * once, rtol=1e-6)


def test_width_and_pages(gpu):
    """Tokens from `width` on are left out; a page outside the cache is reported and read as page 0."""
    c = _case(gpu, ("fp8", "log8", 512, 64, 24, 1, 1, 64), [300, 200], seed=9)
    lse = _lse(c)
    full, part = torch.zeros(2, 300, device=gpu), torch.zeros(2, 300, device=gpu)
    _run(c, lse, full)
    _run(c, lse, part[:, :130])
    assert torch.equal(part[:, :130], full[:, :130]) and (part[:, 130:] == 0).all()
    c.block_table[0, 1] = -7
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    got = _run(c, lse, torch.zeros_like(full), status=status)
    assert int(status) == -8 and torch.equal(got[1], full[1])


@pytest.mark.parametrize("kv", ["fp8", "bf16"])
def test_bad_elements(gpu, kv):
    """A NaN key gives NaN at its token only; slots past the length reach nothing; a NaN query row reaches its
    request's tokens; a row with lse -inf adds nothing whatever its query holds."""
    c = _case(gpu, (kv, {"fp8": "log8", "bf16": "bf16"}[kv], 512, 64, 24, 1, 1, 64), [70, 100], seed=13)
    lse = _lse(c)
    base = _run(c, lse, torch.zeros(2, 100, device=gpu)).clone()
    flat = c.cache.view(-1, c.cache.shape[-1])
    bad = 0x7f if kv == "fp8" else float("nan")
    for b, L in enumerate((70, 100)):
        for t in range(L, 128):
            flat[int(c.block_table[b, t // 64]) * 64 + t % 64] = bad
    assert torch.equal(_run(c, lse, torch.zeros(2, 100, device=gpu)), base)
    flat[int(c.block_table[0, 0]) * 64 + 5, 9] = bad
    got = _run(c, lse, torch.zeros(2, 100, device=gpu))
    assert torch.isnan(got[0, 5])
    got[0, 5] = base[0, 5]
    assert torch.equal(got, base)
    flat[int(c.block_table[0, 0]) * 64 + 5, 9] = 0
    c.q_nope[1, 3] = float("nan")
    got = _run(c, lse, torch.zeros(2, 100, device=gpu))
    assert torch.isnan(got[1]).all() and not torch.isnan(got[0, :70]).any()
    lse[1] = -float("inf")
    assert (_run(c, lse, torch.zeros(2, 100, device=gpu))[1] == 0).all()


def test_same_bits_again_and_in_a_graph(gpu):
    c = _case(gpu, ("bf16", "bf16", 512, 64, 24, 4, 1, 64), [3000, 900, 17], seed=17)
    lse, w = _lse(c), torch.rand(3, 3000, device=gpu)
    out = torch.zeros_like(w)
    _run(c, lse, w, out=out)
    g = torch.cuda.CUDAGraph()
    o2 = torch.zeros_like(w)
    import qmla
    with torch.cuda.graph(g):
        qmla.attention_weights(c.q_nope, c.q_pe, c.cache, c.block_table, c.seq_lens, lse, w, qrows=4, out=o2, **row_kw(c))
    for _ in range(3):
        o2.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o2, out)
        w.add_(0.5)
        _run(c, lse, w, out=out)


def test_far_pages_and_strided_queries(gpu):
    c = _case(gpu, ("fp8", "log8", 512, 64, 24, 1, 1, 64), [200], seed=19)
    lse = _lse(c)
    want = _run(c, lse, torch.zeros(1, 200, device=gpu)).clone()
    n = c.cache.shape[0]
    far = (1 << 32) // (64 * c.cache.shape[-1]) + 5
    big = torch.empty(far + n, *c.cache.shape[1:], dtype=torch.uint8, device=gpu)
    big[far:] = c.cache
    c.cache, c.block_table = big, c.block_table + far
    whole = torch.zeros(1, 26, 577, dtype=torch.bfloat16, device=gpu)
    whole[:, 1:25, :512], whole[:, 1:25, 512:576] = c.q_nope, c.q_pe
    c.q_nope, c.q_pe = whole[:, 1:25, :512], whole[:, 1:25, 512:576]
    assert torch.equal(_run(c, lse, torch.zeros(1, 200, device=gpu)), want)
