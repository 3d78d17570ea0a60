"""Eviction from the paged cache by accumulated attention weight: the weight every cached token got
(`attention_weights`, after each `forward`), the tokens a request keeps (`evict_select`), their rows moved
together (`cache_compact`), and the last two as one call (`evict`). `cache_compact` also brings the accepted
path of a verified tree behind its context. HIP kernels of libqmla.so; there is no CPU path. The reference has
no counterpart.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .decode import _kv_code, _rms_mode, build_params


def _rows32(fn: str, name: str, t: torch.Tensor, dtype, dim: int) -> None:
    if t.dtype is not dtype or t.dim() != dim or (t.stride(-1) != 1 and t.shape[-1] > 1 and t.numel() > 0):
        raise TypeError(f"{fn}: {name} must be a {dim}-D {dtype} tensor with contiguous rows")


def _written(fn: str, name: str, t: torch.Tensor) -> None:
    """Rows that are written may not lie on one another."""
    if t.shape[0] > 1 and t.stride(0) < (t.shape[1] if t.dim() == 2 else 1):
        raise ValueError(f"{fn}: rows of {name} lie on one another")


def _clash(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Rows of `b` lie on other rows of `a` ([requests, columns], one type): written through one, read through the
    other, what is read would depend on the order."""
    if a is b or a.numel() == 0 or b.numel() == 0:
        return False
    es, pa, pb = a.element_size(), a.data_ptr(), b.data_ptr()
    sa, sb, wa, wb = a.stride(0) * es, b.stride(0) * es, a.shape[1] * es, b.shape[1] * es
    if pa + (a.shape[0] - 1) * sa + wa <= pb or pb + (b.shape[0] - 1) * sb + wb <= pa:
        return False
    if a.shape[0] == 1 and b.shape[0] == 1:
        return pa != pb
    if sa != sb or sa == 0:
        return True
    return pa != pb and not ((pb - pa) % sa >= wa and (pa - pb) % sa >= wb)   # columns of one buffer, beside each other


def attention_weights(q_nope, q_rope, kv_cache, block_table, seq_lens, lse, weights, *, d_c=None, rope_w=None,
                      rms_offset=None, page_size, sm_scale, kv_fp8=None, fp8_rms="log8", k_scale=None, qrows=1, groups=1,
                      rms_heads=None, logit_cap=0.0, out=None, status=None):
    """Add to weights [requests, width] (fp32) what every cached token got in a decode step: out[b, t] =
    weights[b, t] + the sum over request b's qrows query rows and heads of exp(score - lse), for t below the
    request's length; later columns stay as they are, tokens from `width` on are left out. Returns `out`, by
    default `weights` itself; no other row of `out` may lie on a row of `weights`.

    The other arguments are those of the `forward` call that gave `lse` [rows, H] (fp32), block_table and
    seq_lens flattened one row per query token. Rows that saw no token add nothing. The sum's order is fixed."""
    rows, H = q_nope.shape[0], q_nope.shape[1]
    if qrows < 1 or rows % qrows:
        raise ValueError(f"attention_weights: rows {rows} not a multiple of qrows {qrows}")
    n_req = rows // qrows
    out = weights if out is None else out
    _rows32("attention_weights", "weights", weights, torch.float32, 2)
    _rows32("attention_weights", "out", out, torch.float32, 2)
    _rows32("attention_weights", "lse", lse, torch.float32, 2)
    if weights.shape[0] != n_req or out.shape != weights.shape:
        raise ValueError(f"attention_weights: weights and out must be [{n_req}, width]")
    if tuple(lse.shape) != (rows, H) or block_table.shape[0] != rows or seq_lens.shape[0] != rows:
        raise ValueError("attention_weights: lse, block_table and seq_lens need one row per query row")
    _written("attention_weights", "out", out)
    if _clash(weights, out):
        raise ValueError("attention_weights: out must be weights or lie beside it")
    _lib.same_device("attention_weights", "q_nope", q_nope, "q_rope", q_rope, "kv_cache", kv_cache,
                     "block_table", block_table, "seq_lens", seq_lens, "lse", lse, "weights", weights, "out", out,
                     "status", status)
    p = row_params(q_nope, q_rope, kv_cache, block_table, seq_lens, q_nope, None, d_c=d_c, rope_w=rope_w, rms_offset=rms_offset,
                   page_size=page_size, sm_scale=sm_scale, kv_fp8=kv_fp8, fp8_rms=fp8_rms, k_scale=k_scale, groups=groups,
                   rms_heads=rms_heads, logit_cap=logit_cap, status=status)
    p.qrows = qrows
    _lib.check("qmla_attention_weights", _lib.lib().qmla_attention_weights(
        p, lse.data_ptr(), lse.stride(0), weights.data_ptr(), weights.stride(0), out.data_ptr(), out.stride(0),
        weights.shape[1], _lib.stream()))
    return out


def row_params(q_nope, q_rope, kv_cache, block_table, seq_lens, out, lse, *, d_c, rope_w, rms_offset, page_size, sm_scale,
               kv_fp8, fp8_rms, k_scale, groups, rms_heads, logit_cap, status):
    """The parameter block of a call with `forward`'s arguments and defaults."""
    if q_nope.dim() != 3 or (q_rope is not None and (q_rope.dim() != 3 or q_rope.shape[:2] != q_nope.shape[:2])):
        raise ValueError("queries must be [rows, heads, width]")
    if d_c is None:
        d_c = q_nope.shape[-1] * groups
    if rope_w is None:
        rope_w = 0 if q_rope is None else q_rope.shape[-1]
    if q_nope.shape[-1] * groups < d_c or (rope_w > 0 and (q_rope is None or q_rope.shape[-1] < rope_w)):
        raise ValueError(f"queries are narrower than d_c {d_c} and rope_w {rope_w} need")
    if rms_offset is None:
        rms_offset = d_c + rope_w
    kv = _kv_code(kv_cache, kv_fp8)
    if kv_cache.element_size() != (1 if kv == _lib.KV_FP8 else 2):
        raise TypeError(f"cache of {kv_cache.dtype} does not hold {'fp8' if kv == _lib.KV_FP8 else 'bf16'} rows")
    if k_scale is not None and not (torch.is_tensor(k_scale) and k_scale.dtype == torch.float32 and k_scale.device == q_nope.device):
        raise TypeError("k_scale must be a float32 tensor on the query's device")
    return build_params(q_nope=q_nope, q_pe=q_rope, kv_cache=kv_cache, block_table=block_table, seq_lens=seq_lens, out=out,
                        lse=lse, d_c=d_c, rope_w=rope_w, rms_offset=rms_offset,
                        rms_mode=_rms_mode(kv, rms_offset, fp8_rms == "bf16", fp8_rms == "log8"), kv=kv, page_size=page_size,
                        sm_scale=sm_scale, k_scale=k_scale, logit_cap=logit_cap, groups=groups, rms_heads=rms_heads,
                        num_splits=1, status=status)


def _select_params(weights, seq_lens, keep, sink, recent, index, counts):
    _rows32("evict_select", "weights", weights, torch.float32, 2)
    _rows32("evict_select", "seq_lens", seq_lens, torch.int32, 1)
    n = weights.shape[0]
    if seq_lens.shape[0] != n:
        raise ValueError("evict_select: one length per row of weights")
    if keep < 0 or sink < 0 or recent < 0 or sink + recent > keep:
        raise ValueError("evict_select: sink and recent must fit in keep")
    if index is not None:
        _rows32("evict_select", "index", index, torch.int32, 2)
        if tuple(index.shape) != (n, keep):
            raise ValueError(f"evict_select: index must be [{n}, {keep}]")
        _written("evict_select", "index", index)
    if counts is not None:
        _rows32("evict_select", "counts", counts, torch.int32, 1)
        if counts.shape[0] != n:
            raise ValueError(f"evict_select: counts must be [{n}]")
        _written("evict_select", "counts", counts)
    _lib.same_device("evict_select", "weights", weights, "seq_lens", seq_lens, "index", index, "counts", counts)
    if index is None:
        index = torch.empty(n, keep, dtype=torch.int32, device=weights.device)
    if counts is None:
        counts = torch.empty(n, dtype=torch.int32, device=weights.device)
    p = _lib.EvictParams()
    p.weights, p.weights_stride = weights.data_ptr(), weights.stride(0)
    p.seq_lens = seq_lens.data_ptr()
    p.index, p.index_stride, p.counts = index.data_ptr(), index.stride(0), counts.data_ptr()
    p.requests, p.width, p.keep, p.sink, p.recent = n, weights.shape[1], keep, sink, recent
    return p, index, counts


def evict_select(weights, seq_lens, keep: int, *, sink: int = 0, recent: int = 0, index=None, counts=None):
    """The tokens each request keeps: (index [requests, keep] int32, counts [requests] int32).

    A request of at most `keep` tokens keeps them all; a longer one its first `sink`, its last `recent` and
    the heaviest of the others by weights [requests, width] (fp32), ties to the lower token, NaN as -inf.
    index[b, :counts[b]] ascends, the rest of the row is -1. Lengths above `width` count as width. counts may be
    seq_lens itself."""
    p, index, counts = _select_params(weights, seq_lens, keep, sink, recent, index, counts)
    _lib.check("qmla_evict_select", _lib.lib().qmla_evict_select(ctypes.byref(p), _lib.stream()))
    return index, counts


def cache_compact(kv_cache, block_table, index, counts, *, first=None, dst_block_table=None, weights=None, weights_out=None,
                  status=None) -> None:
    """Copy the cached row of token index[b, i] of request b to its token first[b] + i (i without `first`) for
    i < counts[b]; kv_cache [num_pages, page_size, (1,) row], block_table [requests, pages] (int32).

    Without dst_block_table the rows move inside the request's own pages: index[b] must ascend strictly with
    index[b, i] >= first[b] + i, and no two requests may share a page. With it they go to those pages, none of
    which may be a source. weights_out[b, first[b] + i] = weights[b, index[b, i]] (fp32) goes along when given;
    in place weights_out may be weights. Rows outside the tables or the cache are left out, and QMLA_ERR_PAGE is
    stored into `status` (device int32) when given.

    The accepted path of a tree (see `tree_forward`): index = context + the accepted nodes in order, first =
    the context's length."""
    p = _lib.EvictParams()
    _compact_params(p, kv_cache, block_table, index, counts, first, dst_block_table, weights, weights_out, status)
    _lib.check("qmla_cache_compact", _lib.lib().qmla_cache_compact(ctypes.byref(p), _lib.stream()))


def _compact_params(p, kv_cache, block_table, index, counts, first, dst_block_table, weights, weights_out, status) -> None:
    if kv_cache.dim() not in (3, 4) or (kv_cache.dim() == 4 and kv_cache.shape[2] != 1) or kv_cache.stride(-1) != 1:
        raise ValueError("cache_compact: kv_cache must be [num_pages, page_size, (1,) row] with contiguous rows")
    _rows32("cache_compact", "block_table", block_table, torch.int32, 2)
    _rows32("cache_compact", "index", index, torch.int32, 2)
    _rows32("cache_compact", "counts", counts, torch.int32, 1)
    n = index.shape[0]
    if block_table.shape[0] != n or counts.shape[0] != n:
        raise ValueError("cache_compact: block_table, index and counts need one row per request")
    if first is not None:
        _rows32("cache_compact", "first", first, torch.int32, 1)
        if first.shape[0] != n:
            raise ValueError("cache_compact: first needs one entry per request")
    if dst_block_table is not None:
        _rows32("cache_compact", "dst_block_table", dst_block_table, torch.int32, 2)
        if dst_block_table.shape[0] != n:
            raise ValueError("cache_compact: dst_block_table needs one row per request")
    if weights_out is not None:
        if weights is None:
            raise ValueError("cache_compact: weights_out without weights")
        for name, t in (("weights", weights), ("weights_out", weights_out)):
            _rows32("cache_compact", name, t, torch.float32, 2)
            if t.shape[0] != n:
                raise ValueError(f"cache_compact: {name} needs one row per request")
        same = weights_out.data_ptr() == weights.data_ptr()
        if dst_block_table is not None and same:
            raise ValueError("cache_compact: weights_out may be weights in place only")
        _written("cache_compact", "weights_out", weights_out)
        if _clash(weights, weights_out):
            raise ValueError("cache_compact: weights_out must be weights or lie beside it")
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise TypeError("cache_compact: status must be an int32 tensor")
    _lib.same_device("cache_compact", "kv_cache", kv_cache, "block_table", block_table, "index", index,
                     "counts", counts, "first", first, "dst_block_table", dst_block_table, "weights", weights,
                     "weights_out", weights_out, "status", status)
    es = kv_cache.element_size()
    p.index, p.index_stride, p.counts = index.data_ptr(), index.stride(0), counts.data_ptr()
    p.requests, p.keep = n, index.shape[1]
    p.cache = kv_cache.data_ptr()
    p.page_stride, p.token_stride = kv_cache.stride(0) * es, kv_cache.stride(1) * es
    p.row_bytes = kv_cache.shape[-1] * es
    p.page_size, p.num_pages = kv_cache.shape[1], kv_cache.shape[0]
    p.block_table, p.bt_stride, p.bt_cols = block_table.data_ptr(), block_table.stride(0), block_table.shape[1]
    if dst_block_table is not None:
        p.dst_block_table, p.dst_bt_stride = dst_block_table.data_ptr(), dst_block_table.stride(0)
        p.dst_bt_cols = dst_block_table.shape[1]
    p.first = None if first is None else first.data_ptr()
    if weights_out is not None:
        p.weights, p.weights_stride, p.width = weights.data_ptr(), weights.stride(0), weights.shape[1]
        p.weights_out, p.weights_out_stride, p.weights_out_width = weights_out.data_ptr(), weights_out.stride(0), weights_out.shape[1]
    p.status = None if status is None else status.data_ptr()


def evict(kv_cache, block_table, seq_lens, weights, keep: int, *, sink: int = 0, recent: int = 0, dst_block_table=None,
          weights_out=None, index=None, counts=None, status=None):
    """`evict_select` and `cache_compact` in one call: cut every request to at most `keep` tokens. Returns
    (index, counts); counts are the new lengths. Without dst_block_table rows and weights move in place; with
    it the rows go to those pages and the weights to weights_out, when given. Columns of the weights from the new length on
    keep what they held: clear them before later tokens add theirs."""
    if dst_block_table is None and weights_out is None:
        weights_out = weights
    p, index, counts = _select_params(weights, seq_lens, keep, sink, recent, index, counts)
    _compact_params(p, kv_cache, block_table, index, counts, None, dst_block_table, weights, weights_out, status)
    lib, st = _lib.lib(), _lib.stream()
    _lib.check("qmla_evict_select", lib.qmla_evict_select(ctypes.byref(p), st))
    _lib.check("qmla_cache_compact", lib.qmla_cache_compact(ctypes.byref(p), st))
    return index, counts
