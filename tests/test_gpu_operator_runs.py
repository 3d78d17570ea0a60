"""The tree and weights operators where their work is laid out differently: requests that share workgroups, scores
that climb by more than the softmax reference allows, more heads than one thread row of divisors, two streams at
once. Bounds are the ones tests/op_cases.py and tests/test_gpu_weights.py derive."""
import pytest
import torch

from tests.op_cases import close, ref_tree, row_kw, tree_case
from tests.test_gpu_weights import _case, _lse, _ref
from tests.test_gpu_weights import _run as _weigh

pytestmark = pytest.mark.gpu


def _tree(c, qn, qp, mask, counts=None, **kw):
    import qmla
    return qmla.tree_forward(qn, qp if c.rope_w else None, c.cache, c.block_table, c.seq_lens, mask, node_counts=counts,
                             **row_kw(c), **kw)


def _check(name, c, qn, qp, mask, counts, got):
    torch.cuda.synchronize()
    o, lse, ob, lb = ref_tree(c, qn, qp, c.seq_lens.cpu(), mask.cpu(), None if counts is None else counts.cpu())
    close(f"{name} out", got[0], o, ob, got[0].dtype)
    close(f"{name} lse", got[1], lse, lb, got[1].dtype)


@pytest.mark.parametrize("kv,rms", [("fp8", "log8"), ("bf16", "bf16")])
def test_tree_requests_share_workgroups(gpu, kv, rms):
    """150 row tiles of 13 to 15 token tiles on 256 workgroups: too many for two workgroups each, so a workgroup ends
    one and starts the next; then so few that some workgroups have nothing."""
    import qmla
    for lens in ([416 + 11 * (i % 5) for i in range(150)], [95, 0, 33]):
        c, qn, qp, par, counts = tree_case(gpu, kv=kv, rms_mode=rms, d_c=512, rope=64, heads=1, page=64, lens=lens, nodes=4,
                                           seed=len(lens), ragged=True)
        if len(lens) == 3:
            c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        mask, counts = qmla.tree_mask(par).to(gpu), counts.clamp_min(1).to(gpu)
        _check(f"{kv} {len(lens)} requests", c, qn, qp, mask, counts, _tree(c, qn, qp, mask, counts))


@pytest.mark.parametrize("kv,rms,d_c", [("fp8", "log8", 512), ("bf16", "bf16", 512), ("fp8", "log8", 768), ("fp8", "log8", 1792)])
def test_tree_scores_that_climb(gpu, kv, rms, d_c):
    """Scores with a deviation of some 30: rows' maxima pass the reference by far, again and again."""
    import qmla
    c, qn, qp, par, _ = tree_case(gpu, kv=kv, rms_mode=rms, d_c=d_c, rope=64, heads=5, page=64, lens=[1500, 200], nodes=7, seed=d_c,
                                  q_amp=30.0)
    mask = qmla.tree_mask(par).to(gpu)
    _check(f"{kv} {d_c} climbing", c, qn, qp, mask, None, _tree(c, qn, qp, mask))


@pytest.mark.parametrize("rms,rope", [("e4m3", 64), ("bf16_bytes", 64), ("bf16_bytes", 57), ("log8", 57), ("none", 64)])
@pytest.mark.parametrize("heads", [33, 42])
def test_tree_many_heads_and_odd_divisor_offsets(gpu, rms, rope, heads):
    import qmla
    c, qn, qp, par, _ = tree_case(gpu, kv="fp8", rms_mode=rms, d_c=512, rope=rope, heads=heads, page=48, lens=[150, 34], nodes=3, seed=heads)
    mask = qmla.tree_mask(par).to(gpu)
    _check(f"{rms} {rope} {heads} heads", c, qn, qp, mask, None, _tree(c, qn, qp, mask))


def test_tree_pages_of_one_token(gpu):
    """More pages than a workgroup holds ids of at once."""
    import qmla
    c, qn, qp, par, _ = tree_case(gpu, kv="fp8", rms_mode="log8", d_c=512, rope=64, heads=1, page=1, lens=[600] * 300, nodes=4, seed=5)
    mask = qmla.tree_mask(par).to(gpu)
    _check("pages of one token", c, qn, qp, mask, None, _tree(c, qn, qp, mask))


@pytest.mark.parametrize("kv,rms", [("fp8", "log8"), ("bf16", "bf16")])
def test_tree_two_streams_at_once(gpu, kv, rms):
    """Calls that overlap, each with a workspace of its own, give the bits they give alone."""
    import qmla
    calls = []
    for seed, lens in ((1, [1500, 80]), (2, [40, 900, 333])):
        c, qn, qp, par, _ = tree_case(gpu, kv=kv, rms_mode=rms, d_c=512, rope=64, heads=24, page=64, lens=lens, nodes=9, seed=seed)
        mask = qmla.tree_mask(par).to(gpu)
        calls.append((c, qn, qp, mask, _tree(c, qn, qp, mask), qmla.Workspace(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for c, qn, qp, mask, _, ws, s in calls:
            with torch.cuda.stream(s):
                got.append(_tree(c, qn, qp, mask, workspace=ws))
    torch.cuda.synchronize()
    for i, (o, lse) in enumerate(got):
        assert torch.equal(o, calls[i % 2][4][0]) and torch.equal(lse, calls[i % 2][4][1])


def test_select_counts_in_place_of_lengths(gpu):
    """counts given as the lengths themselves: what a call with its own gives."""
    import qmla
    g = torch.Generator().manual_seed(3)
    w = torch.rand(300, 2500, generator=g).to(gpu)
    lens = torch.randint(0, 2600, (300,), generator=g).to(torch.int32).to(gpu)
    want, counts = qmla.evict_select(w, lens, 700, sink=3, recent=100)
    for _ in range(5):
        own = lens.clone()
        got, n = qmla.evict_select(w, own, 700, sink=3, recent=100, counts=own)
        assert n is own and torch.equal(n, counts) and torch.equal(got, want)


@pytest.mark.parametrize("layout,lens", [
    (("bf16", "bf16", 64, 18, 3, 1, 1, 64), [70 + i % 9 for i in range(900)]),   # more requests than workgroups
    (("fp8", "log8", 256, 64, 12, 2, 1, 32), [20000, 1, 64, 0, 65]),             # one that takes nearly all of them
    (("bf16", "bf16", 64, 18, 24, 4, 1, 16), [0, 127, 128, 129, 700]),
])
def test_weights_pieces(gpu, layout, lens):
    c = _case(gpu, layout, lens, seed=len(lens))
    lse = _lse(c)
    w = torch.rand(len(lens), max(lens), device=gpu)
    want, bound = _ref(c, lse, w)
    close(f"weights {len(lens)} requests", _weigh(c, lse, w.clone()), want, bound, torch.float32)
    out = torch.full_like(w, 3.0)
    _weigh(c, lse, w, out=out)
    for b in (0, len(lens) - 1):
        assert (out[b, lens[b]:] == 3).all()
