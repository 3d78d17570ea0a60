"""`qmla.rotary` against float64 with the same fp32 table: a rotated element is two fp32 products and their
sum (3 roundings of at most |x| + |y|) rounded once to the heads' type."""
import pytest
import torch

from tests.op_cases import U32

pytestmark = pytest.mark.gpu


def _ref(x, table, pos, layout, offset, inverse):
    """(rotated, bound) in float64."""
    rot = table.shape[1]
    x = x.cpu().double()
    ok = (pos >= 0) & (pos < table.shape[0])
    row = table.cpu().double()[pos.clamp(0, table.shape[0] - 1)]
    row[~ok] = float("nan")
    cos, sin = row[:, None, :rot // 2], row[:, None, rot // 2:] * (-1 if inverse else 1)
    y, bound = x.clone(), torch.zeros_like(x)
    ia = torch.arange(rot // 2) if layout == "half" else torch.arange(0, rot, 2)
    ib = ia + (rot // 2 if layout == "half" else 1)
    a, b = x[..., offset + ia], x[..., offset + ib]
    y[..., offset + ia], y[..., offset + ib] = a * cos - b * sin, b * cos + a * sin
    bound[..., offset + ia] = bound[..., offset + ib] = 3 * U32 * (a.abs() + b.abs()) * float(table.abs().max())
    return y, bound


def _close(name, got, want, bound, src, offset, rot):
    from tests.op_cases import close
    close(name, got, want, bound, got.dtype)
    rest = [i for i in range(src.shape[-1]) if not offset <= i < offset + rot]
    assert torch.equal(got[..., rest].cpu(), src[..., rest].cpu())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("n,heads,kheads,dim,rot,offset", [(1, 24, 1, 576, 64, 512), (33, 24, 4, 256, 64, 0), (5, 3, 1, 58, 58, 0),
                                                           (257, 1, 2, 80, 32, 16), (7, 2, 0, 64, 2, 31), (64, 12, 1, 128, 64, 64), (3, 5, 5, 64, 48, 8)])
def test_against_float64(gpu, dtype, layout, n, heads, kheads, dim, rot, offset):
    import qmla
    g = torch.Generator().manual_seed(n + dim)
    both = torch.randn(n, heads + kheads, dim, generator=g).to(dtype).to(gpu)
    q, k = both[:, :heads], both[:, heads:] if kheads else None
    pos = torch.randint(0, 5000, (n,), generator=g)
    pos[0] = 4999
    table = qmla.rotary_table(rot, 5000, scaling="yarn", factor=4.0, original_max_pos=1250, device=gpu)
    for inverse in (False, True):
        qo, ko = qmla.rotary(pos.to(gpu), q, k, table, layout=layout, offset=offset, inverse=inverse)
        torch.cuda.synchronize()
        for name, x, y in (("q", q, qo), ("k", k, ko)):
            if x is not None:
                want, bound = _ref(x, table, pos, layout, offset, inverse)
                _close(f"{name} {layout} {dtype}", y, want, bound, x, offset, rot)
        assert (ko is None) == (k is None)
    # in place gives the same bits and touches nothing else
    keep = qmla.rotary(pos.to(gpu), q, k, table, layout=layout, offset=offset)
    qmla.rotary(pos.to(gpu).to(torch.int32), q, k, table, layout=layout, offset=offset, q_out=q, k_out=k)
    assert torch.equal(q, keep[0]) and (k is None or torch.equal(k, keep[1]))


def test_positions_outside_strides_and_empty(gpu):
    import qmla
    table = qmla.rotary_table(8, 10, device=gpu)
    wide = torch.zeros(10, 16, device=gpu)[:, :8]
    wide.copy_(table)
    pos = torch.tensor([0, 9, 10, -1, 1 << 40, 3], device=gpu)
    x = torch.randn(6, 3, 16, device=gpu)
    y, _ = qmla.rotary(pos, x, None, wide, offset=4)
    want, bound = _ref(x, table, pos.cpu(), "half", 4, False)
    _close("outside", y, want, bound, x, 4, 8)
    # positions and heads with strides, an output with strides of its own
    p2 = torch.stack([pos, pos + 1], 1)[:, 0]
    big = torch.full((6, 5, 33), 9.0, device=gpu)
    xs = torch.zeros(3, 6, 17, device=gpu)[..., :16].transpose(0, 1)
    xs.copy_(x)
    y2, _ = qmla.rotary(p2, xs, None, wide, offset=4, q_out=big[:, 1:4, :16])
    assert torch.equal(y2.nan_to_num(-5), y.nan_to_num(-5)) and (big[:, 0] == 9).all() and (big[..., 16:] == 9).all()
    e = torch.zeros(0, 3, 16, device=gpu)
    assert qmla.rotary(pos[:0], e, e, wide, offset=4)[0].shape == (0, 3, 16)


def test_matches_the_prep_rotation(gpu):
    """Half layout on the prep's own q: the prep rounds each product and sum to bf16 (three roundings of at most
    |x| + |y| plus one of cos and sin each), this one once."""
    import qmla
    n, H, rd, hd, d_c = 9, 24, 64, 256, 512
    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(gpu)  # noqa: E731
    q, table = rnd(n, H, hd), qmla.partial_rope_table(range(32), 64, 10000.0, 100, device=gpu)
    pos = torch.arange(n, device=gpu)
    q_out, _ = qmla.mla_decode_prep(pos, q, rnd(n, d_c), rnd(n, 4 * rd), rnd(H * (hd - rd), d_c), torch.ones(rd, device=gpu), table,
                                    head_offset=0, rope_group=6, rope_first=0, rope_span=4, declared_rope=296, eps=1e-6)
    mine, _ = qmla.rotary(pos, q, None, table)
    for h in range(H):
        s = hd - rd + (h // 6) * rd
        far = (q_out[:, h, s:s + rd].float() - mine[:, h, :rd].float()).abs()
        a, b = q[:, h, :32].float().abs(), q[:, h, 32:64].float().abs()
        assert (far <= 5 * 2.0 ** -8 * torch.cat([a + b, a + b], -1) + 1e-30).all()


def test_graph_and_other_stream(gpu):
    import qmla
    table = qmla.rotary_table(64, 1000, device=gpu)
    pos, x = torch.arange(50, device=gpu), torch.randn(50, 24, 64, device=gpu).to(torch.bfloat16)
    want, _ = qmla.rotary(pos, x, None, table, layout="interleaved")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, _ = qmla.rotary(pos.to(torch.int32), x, None, table, layout="interleaved")
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, _ = qmla.rotary(pos, x, None, table, layout="interleaved")
    for i in range(3):
        x.mul_(0.5)
        want, _ = qmla.rotary(pos, x, None, table, layout="interleaved")
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
