"""Refusals and host-side parts of the tree, weights, eviction and rotary operators. CPU only: the library's
checks run before any device work, the wrappers' before the library is called."""
import math
import re

import pytest
import torch

import qmla
from qmla import _lib
from tests.test_abi import HEADER

BASE = 0x10000


@pytest.mark.parametrize("name,mirror", [("qmla_rotary_params", _lib.RotaryParams), ("qmla_evict_params", _lib.EvictParams)])
def test_struct_mirrors_match_header(name, mirror):
    text = HEADER.read_text()
    body = re.sub(r"/\*.*?\*/", "", text[text.index("typedef struct " + name):text.index("} " + name + ";")], flags=re.S)
    fields = []
    for decl in body.split("{", 1)[1].split(";"):
        if decl.strip():
            parts = decl.split(",")
            fields.append(re.findall(r"(\w+)\s*$", parts[0])[0])
            fields.extend(re.sub(r"[\*\s]", "", x) for x in parts[1:])
    assert fields == [f[0] for f in mirror._fields_]


def _rotary(**over):
    p = _lib.RotaryParams()
    p.q, p.q_token_stride, p.q_head_stride = BASE, 24 * 64, 64
    p.q_out, p.q_out_token_stride, p.q_out_head_stride = BASE + 0x100000, 24 * 64, 64
    p.positions, p.pos_stride, p.cos_sin, p.max_pos, p.cos_sin_stride = BASE + 0x200000, 1, BASE + 0x300000, 100, 64
    p.n, p.q_heads, p.head_dim, p.rot, p.dtype = 4, 24, 64, 64, _lib.DT_BF16
    for k, v in over.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,code", [
    (dict(dtype=3), _lib.ERR_MODE), (dict(rot=63), _lib.ERR_SHAPE), (dict(rot=66), _lib.ERR_SHAPE), (dict(offset=2), _lib.ERR_SHAPE),
    (dict(offset=-2), _lib.ERR_SHAPE), (dict(n=-1), _lib.ERR_SHAPE), (dict(max_pos=0), _lib.ERR_SHAPE), (dict(cos_sin_stride=62), _lib.ERR_SHAPE),
    (dict(q=None), _lib.ERR_NULL), (dict(k_heads=1), _lib.ERR_NULL), (dict(positions=None), _lib.ERR_NULL), (dict(cos_sin=None), _lib.ERR_NULL),
    (dict(q=BASE + 1), _lib.ERR_ALIGN), (dict(cos_sin=BASE + 2), _lib.ERR_ALIGN), (dict(positions=BASE + 4), _lib.ERR_ALIGN),
    (dict(n=0), _lib.OK), (dict(q_heads=0), _lib.OK)])
def test_rotary_error_codes(over, code):
    assert _lib.lib().qmla_rotary(_rotary(**over), None) == code


def _evict(**over):
    p = _lib.EvictParams()
    p.weights, p.weights_stride, p.seq_lens, p.index, p.index_stride, p.counts = BASE, 100, BASE, BASE, 10, BASE
    p.requests, p.width, p.keep, p.sink, p.recent = 2, 100, 10, 2, 3
    p.cache, p.page_stride, p.token_stride, p.row_bytes, p.page_size, p.num_pages = BASE, 64 * 608, 608, 608, 64, 9
    p.block_table, p.bt_stride, p.bt_cols = BASE, 4, 4
    for k, v in over.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,code", [
    (dict(requests=-1), _lib.ERR_SHAPE), (dict(requests=70000), _lib.ERR_SHAPE), (dict(sink=8), _lib.ERR_SHAPE), (dict(recent=-1), _lib.ERR_SHAPE),
    (dict(keep=-1), _lib.ERR_SHAPE), (dict(weights=None), _lib.ERR_NULL), (dict(seq_lens=None), _lib.ERR_NULL), (dict(index=None), _lib.ERR_NULL),
    (dict(counts=None), _lib.ERR_NULL), (dict(requests=0), _lib.OK)])
def test_select_error_codes(over, code):
    assert _lib.lib().qmla_evict_select(_evict(**over), None) == code


@pytest.mark.parametrize("over,code", [
    (dict(page_size=0), _lib.ERR_SHAPE), (dict(row_bytes=0), _lib.ERR_SHAPE), (dict(row_bytes=624), _lib.ERR_SHAPE), (dict(bt_cols=-1), _lib.ERR_SHAPE),
    (dict(num_pages=-1), _lib.ERR_SHAPE), (dict(keep=0x7fffffff), _lib.ERR_SHAPE), (dict(cache=None), _lib.ERR_NULL), (dict(index=None), _lib.ERR_NULL),
    (dict(block_table=None), _lib.ERR_NULL), (dict(weights=None, weights_out=BASE), _lib.ERR_NULL), (dict(requests=0), _lib.OK), (dict(keep=0), _lib.OK)])
def test_compact_error_codes(over, code):
    assert _lib.lib().qmla_cache_compact(_evict(**over), None) == code


def _decode(**over):
    p = _lib.DecodeParams()
    p.q_nope, p.q_nope_stride_row, p.q_nope_stride_head = BASE, 24 * 512, 512
    p.q_pe, p.q_pe_stride_row, p.q_pe_stride_head = BASE, 24 * 64, 64
    p.kv_cache, p.page_stride, p.token_stride, p.kv_dtype, p.page_size = BASE, 64 * 608, 608, _lib.KV_FP8, 64
    p.d_c, p.rope_w, p.rms_offset, p.rms_mode, p.sm_scale = 512, 64, 576, _lib.RMS_LOG8, 0.04
    p.block_table, p.bt_stride, p.seq_lens, p.rows, p.heads, p.rms_heads, p.qrows, p.groups = BASE, 4, BASE, 16, 24, 24, 8, 1
    p.out, p.out_stride_row, p.out_stride_head, p.num_pages = BASE, 24 * 512, 512, 9
    p.workspace, p.workspace_bytes = BASE, 1 << 40
    for k, v in over.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,code", [
    (dict(groups=2), _lib.ERR_SHAPE), (dict(qrows=65, rows=65), _lib.ERR_SHAPE), (dict(rows=15), _lib.ERR_SHAPE), (dict(d_c=384, rms_offset=448), _lib.ERR_NOKERNEL),
    (dict(rope_w=72, rms_offset=584, token_stride=624, page_stride=64 * 624), _lib.ERR_NOKERNEL), (dict(token_stride=596, page_stride=64 * 596), _lib.ERR_SHAPE),
    (dict(kv_cache=BASE + 4), _lib.ERR_ALIGN), (dict(workspace=None), _lib.ERR_WORKSPACE), (dict(workspace_bytes=1 << 20), _lib.ERR_WORKSPACE),
    (dict(workspace=BASE + 4), _lib.ERR_ALIGN), (dict(out=None), _lib.ERR_NULL), (dict(seq_lens=None), _lib.ERR_NULL), (dict(kv_dtype=7), _lib.ERR_MODE),
    (dict(rms_mode=_lib.RMS_BF16), _lib.ERR_MODE), (dict(num_workgroups=-1), _lib.ERR_SHAPE), (dict(rows=0), _lib.OK),
    (dict(heads=65, rms_heads=65, token_stride=656, page_stride=64 * 656), _lib.ERR_NOKERNEL)])
def test_tree_error_codes(over, code):
    lib = _lib.lib()
    assert lib.qmla_tree_forward(_decode(**over), BASE, 8, None, None) == code
    if not over.get("rows") == 0:
        assert lib.qmla_tree_forward(_decode(), None, 8, None, None) == _lib.ERR_NULL
        assert lib.qmla_tree_forward(_decode(), BASE + 4, 8, None, None) == _lib.ERR_ALIGN


def test_tree_workspace_covers_every_layout():
    lib = _lib.lib()
    for d_c, rope in ((256, 116), (512, 64), (768, 232), (1792, 232)):
        row = -(-(d_c + rope + 24) // 16) * 16
        p = _decode(d_c=d_c, rope_w=rope, rms_offset=d_c + rope, token_stride=row, page_stride=64 * row, num_workgroups=16)
        assert lib.qmla_tree_workspace_bytes(p) >= 2 * 16 * d_c * 4
    assert lib.qmla_tree_workspace_bytes(_decode(d_c=100)) == 0


@pytest.mark.parametrize("over,width,lse,out,code", [
    ({}, -1, BASE, BASE, _lib.ERR_SHAPE), ({}, 10, None, BASE, _lib.ERR_NULL), ({}, 10, BASE, None, _lib.ERR_NULL), ({}, 0, BASE, BASE, _lib.OK),
    (dict(rows=0), 10, BASE, BASE, _lib.OK), (dict(kv_cache=BASE + 4), 10, BASE, BASE, _lib.ERR_ALIGN), (dict(rms_heads=12), 10, BASE, BASE, _lib.ERR_SHAPE),
    (dict(d_c=5120, rms_offset=5184, token_stride=5216, page_stride=64 * 5216), 10, BASE, BASE, _lib.ERR_NOKERNEL)])
def test_weights_error_codes(over, width, lse, out, code):
    assert _lib.lib().qmla_attention_weights(_decode(**over), lse, 24, None, 0, out, 100, width, None) == code


# ---- the wrappers ------------------------------------------------------------------------------------
def _cpu(**over):
    a = dict(q_nope=torch.zeros(8, 24, 512, dtype=torch.bfloat16), q_rope=torch.zeros(8, 24, 64, dtype=torch.bfloat16),
             kv_cache=torch.zeros(2, 64, 1, 608, dtype=torch.uint8), block_table=torch.zeros(2, 1, dtype=torch.int32),
             seq_lens=torch.ones(2, dtype=torch.int32), tree_mask=torch.zeros(2, 4, dtype=torch.int64))
    a.update(over)
    return a


@pytest.mark.parametrize("over,exc", [
    (dict(tree_mask=torch.zeros(2, 4, dtype=torch.int32)), TypeError), (dict(tree_mask=torch.zeros(2, 65, dtype=torch.int64)), ValueError),
    (dict(tree_mask=torch.zeros(2, 3, dtype=torch.int64)), ValueError), (dict(seq_lens=torch.ones(8, dtype=torch.int32)), ValueError),
    (dict(node_counts=torch.ones(2, dtype=torch.int64)), TypeError), (dict(node_counts=torch.ones(3, dtype=torch.int32)), TypeError), ({}, ValueError)])
def test_tree_refusals(over, exc):
    a = _cpu(**over)
    with pytest.raises(exc):   # the last one: tensors on the CPU
        qmla.tree_forward(a.pop("q_nope"), a.pop("q_rope"), a.pop("kv_cache"), a.pop("block_table"), a.pop("seq_lens"), a.pop("tree_mask"),
                          page_size=64, sm_scale=0.1, kv_fp8=True, **a)


def test_weights_and_eviction_refusals():
    a = _cpu()
    q = (a["q_nope"], a["q_rope"], a["kv_cache"], torch.zeros(8, 1, dtype=torch.int32), torch.ones(8, dtype=torch.int32))
    kw = dict(page_size=64, sm_scale=0.1, kv_fp8=True)
    lse, w = torch.zeros(8, 24), torch.zeros(2, 10)
    for l2, w2, extra, exc in ((lse, w, dict(qrows=3), ValueError), (lse, w, {}, ValueError), (lse.double(), w, dict(qrows=4), TypeError),
                               (lse, w.double(), dict(qrows=4), TypeError), (lse[:, :20], w, dict(qrows=4), TypeError), (lse, w, dict(qrows=4, out=w[:, :5]), ValueError),
                               (lse, w, dict(qrows=4), ValueError)):
        with pytest.raises(exc):
            qmla.attention_weights(*q, l2 if l2.shape[1] == 24 else torch.zeros(8, 48)[:, ::2], w2, **{**kw, **extra})
    lens = torch.ones(2, dtype=torch.int32)
    for args, extra, exc in (((w, lens.long(), 3), {}, TypeError), ((w, lens[:1], 3), {}, ValueError), ((w, lens, 3), dict(sink=2, recent=2), ValueError),
                             ((w, lens, -1), {}, ValueError), ((w, lens, 3), dict(index=torch.zeros(2, 4, dtype=torch.int32)), ValueError), ((w, lens, 3), {}, ValueError)):
        with pytest.raises(exc):
            qmla.evict_select(*args, **extra)
    idx, cnt, bt = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), a["block_table"]
    for args, extra, exc in (((a["kv_cache"], bt, idx.long(), cnt), {}, TypeError), ((a["kv_cache"], bt[:1], idx, cnt), {}, ValueError),
                             ((a["kv_cache"], bt, idx, cnt), dict(weights_out=w), ValueError), ((a["kv_cache"], bt, idx, cnt), dict(first=cnt[:1]), ValueError),
                             ((a["kv_cache"], bt, idx, cnt), dict(weights=w, weights_out=w, dst_block_table=bt), ValueError),
                             ((a["kv_cache"][..., ::2], bt, idx, cnt), {}, ValueError), ((a["kv_cache"], bt, idx, cnt), {}, ValueError)):
        with pytest.raises(exc):
            qmla.cache_compact(*args, **extra)


def test_rotary_refusals():
    pos, q, table = torch.arange(3), torch.zeros(3, 2, 16), qmla.rotary_table(8, 10)
    for args, extra, exc in (((pos.float(), q, None, table), {}, TypeError), ((pos, q, None, table.double()), {}, TypeError), ((pos, q.double(), None, table), {}, TypeError),
                             ((pos, q, q[:2], table), {}, TypeError), ((pos, q, q.half(), table), {}, TypeError), ((pos, q, None, table), dict(offset=9), ValueError),
                             ((pos, q, None, table), dict(layout="neox"), ValueError), ((pos, q[..., ::2], None, table), {}, ValueError),
                             ((pos, q, None, table[:0]), {}, TypeError), ((pos, q, None, table), dict(k_out=q), ValueError), ((pos, q, None, table), {}, ValueError)):
        with pytest.raises(exc):
            qmla.rotary(*args, **extra)
    from qmla.positions import _check_out
    buf = torch.zeros(4, 2, 16)
    _check_out("q", buf[:3], buf[:3])
    with pytest.raises(ValueError):
        _check_out("q", buf[:3], buf[1:])


def test_tree_mask_from_parents():
    m = qmla.tree_mask([[-1, 0, 0, 1, -1], [-1, 0, 1, 2, 3]])
    assert m.tolist() == [[1, 0b11, 0b101, 0b1011, 0b10000], [1, 3, 7, 15, 31]]
    assert int(qmla.tree_mask([list(range(-1, 63))])[0, 63]) == -1
    for bad in ([[0]], [[-1, 1]], [[-2]], [list(range(-1, 64))]):
        with pytest.raises(ValueError):
            qmla.tree_mask(bad)


def test_rotary_tables():
    """Each scaling from its formula at a few entries, in float64."""
    def at(table, pos, i):
        return math.atan2(float(table[pos, 32 + i]), float(table[pos, i])), math.hypot(float(table[pos, 32 + i]), float(table[pos, i]))

    def turn(x):
        return math.remainder(x, 2 * math.pi)
    plain = qmla.rotary_table(64, 5000)
    for pos, i in ((1, 0), (4999, 3), (777, 31)):
        a, r = at(plain, pos, i)
        assert abs(turn(a - pos * 10000.0 ** (-2 * i / 64))) < 1e-6 and abs(r - 1) < 1e-6
    a, _ = at(qmla.rotary_table(64, 5000, scaling="linear", factor=4.0), 4000, 2)
    assert abs(turn(a - 1000 * 10000.0 ** (-4 / 64))) < 1e-6
    ntk = qmla.rotary_table(64, 5000, scaling="ntk", factor=4.0)
    assert abs(turn(at(ntk, 4000, 0)[0] - 4000)) < 1e-6 and abs(turn(at(ntk, 4000, 31)[0] - 1000 * 10000.0 ** (-62 / 64))) < 1e-6
    for kind in ("yarn", "llama3"):
        t = qmla.rotary_table(64, 5000, scaling=kind, factor=8.0, original_max_pos=4096)
        assert abs(turn(at(t, 4000, 0)[0] - 4000)) < 1e-6                               # fast pairs keep their frequency
        assert abs(turn(at(t, 4000, 31)[0] - 500 * 10000.0 ** (-62 / 64))) < 1e-6       # slow ones are interpolated
        assert abs(at(t, 9, 4)[1] - (0.1 * math.log(8.0) + 1.0 if kind == "yarn" else 1.0)) < 1e-6
    assert abs(at(qmla.rotary_table(64, 10, scaling="yarn", factor=8.0, original_max_pos=4096, mscale=1.0), 9, 4)[1] - 1) < 1e-6
    far = qmla.rotary_table(4, 1 << 20)   # angles in float64 at far positions
    assert abs(float(far[(1 << 20) - 1, 0]) - math.cos((1 << 20) - 1)) < 1e-6
    for kw in (dict(rot=7, max_pos=4), dict(rot=8, max_pos=0), dict(rot=8, max_pos=4, theta=1.0), dict(rot=8, max_pos=4, scaling="x"),
               dict(rot=8, max_pos=4, scaling="yarn", factor=2.0), dict(rot=2, max_pos=4, scaling="ntk", factor=2.0), dict(rot=8, max_pos=4, scaling="linear", factor=0.5),
               dict(rot=8, max_pos=4, scaling="llama3", factor=2.0, original_max_pos=100, low_freq_factor=4.0, high_freq_factor=4.0)):
        with pytest.raises(ValueError):
            qmla.rotary_table(**kw)


def test_rows_that_lie_on_other_rows_are_refused():
    """Weights read through one view and written through another that is shifted against it; columns of one buffer
    beside each other are fine (the next refusal is the device's)."""
    buf = torch.zeros(8 * 100 + 100)
    w, lens, q = buf[:800].view(8, 100), torch.zeros(8, dtype=torch.int32), torch.zeros(8, 24, 512, dtype=torch.bfloat16)
    cache, bt = torch.zeros(4, 64, 608, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.int32)
    idx = torch.zeros(8, 4, dtype=torch.int32)

    def weigh(a, b):
        qmla.attention_weights(q, None, cache, bt, lens, torch.zeros(8, 24), a, out=b, page_size=64, sm_scale=1.0)

    def compact(a, b, dst=None):
        qmla.cache_compact(cache, bt, idx, lens, dst_block_table=dst, weights=a, weights_out=b)

    for shift in (1, 50, 100):
        for call in (weigh, compact):
            with pytest.raises(ValueError, match="beside"):
                call(w, buf[shift:shift + 800].view(8, 100))
    with pytest.raises(ValueError, match="beside"):
        weigh(w[:, :60], w[:, 30:90])
    with pytest.raises(ValueError, match="beside"):
        compact(w[:, :60], w[:, 59:90], bt)
    for a, b in ((w, w), (w, w.view(8, 100)), (w[:, :50], w[:, 50:]), (w[:, 50:], w[:, :50]), (w, torch.zeros(8, 100))):
        for call in (weigh, compact):
            with pytest.raises(ValueError, match="GPU"):
                call(a, b)


@pytest.mark.parametrize("kv,d_c,rope,heads,fits", [
    (_lib.KV_BF16, 768, 116, 53, True), (_lib.KV_BF16, 768, 116, 54, False), (_lib.KV_FP8, 768, 232, 53, True),
    (_lib.KV_BF16, 512, 64, 64, True), (_lib.KV_BF16, 1792, 256, 64, True), (_lib.KV_FP8, 1792, 256, 64, True),
    (_lib.KV_FP8, 256, 256, 64, True), (_lib.KV_FP8, 512, 64, 65, False), (_lib.KV_FP8, 512, 65, 24, False)])
def test_tree_layouts_that_fit(kv, d_c, rope, heads, fits):
    p = _lib.DecodeParams()
    p.rows, p.qrows, p.heads, p.d_c, p.rope_w, p.rms_offset, p.kv_dtype = 8, 4, heads, d_c, rope, d_c + rope, kv
    p.rms_mode, p.num_workgroups = (_lib.RMS_LOG8 if kv == _lib.KV_FP8 else _lib.RMS_BF16), 256
    assert (_lib.lib().qmla_tree_workspace_bytes(p) > 0) == fits


def test_outputs_that_lie_on_themselves_are_refused():
    q = torch.zeros(4, 3, 64)
    pos, table = torch.zeros(4, dtype=torch.int64), qmla.rotary_table(64, 8)
    flat = torch.zeros(4 * 3 * 64)
    for out in (torch.zeros(4, 1, 64).expand(4, 3, 64), torch.zeros(1, 3, 64).expand(4, 3, 64),
                torch.as_strided(flat, (4, 3, 64), (64, 64, 1)), torch.as_strided(flat, (4, 3, 64), (100, 32, 1))):
        with pytest.raises(ValueError, match="lie on one another"):
            qmla.rotary(pos, q, None, table, q_out=out)
    e = torch.zeros(4, 1, 64).expand(4, 3, 64)
    with pytest.raises(ValueError, match="lie on one another"):
        qmla.rotary(pos, e, None, table, q_out=e)                      # in place on broadcast heads
    for out in (q, torch.zeros(3, 4, 64).transpose(0, 1), torch.zeros(4, 5, 80)[:, 1:4, 8:72], torch.zeros(8, 3, 64)[::2]):
        with pytest.raises(ValueError, match="GPU"):
            qmla.rotary(pos, q, None, table, q_out=out)
    w, lens = torch.zeros(8, 100), torch.zeros(8, dtype=torch.int32)
    one = torch.zeros(1, 100).expand(8, 100)
    with pytest.raises(ValueError, match="lie on one another"):
        qmla.evict_select(w, lens, 10, index=torch.zeros(1, 10, dtype=torch.int32).expand(8, 10))
    with pytest.raises((ValueError, TypeError)):
        qmla.evict_select(w, lens, 10, counts=torch.zeros(1, dtype=torch.int32).expand(8))
    cache, bt = torch.zeros(4, 64, 608, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="lie on one another"):
        qmla.cache_compact(cache, bt, torch.zeros(8, 4, dtype=torch.int32), lens, dst_block_table=bt, weights=w, weights_out=one)
    with pytest.raises(ValueError, match="lie on one another"):
        qmla.attention_weights(torch.zeros(8, 24, 512, dtype=torch.bfloat16), None, cache, bt, lens, torch.zeros(8, 24), w, out=one,
                               page_size=64, sm_scale=1.0)
