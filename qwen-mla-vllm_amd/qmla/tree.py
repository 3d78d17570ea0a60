"""Attention of a tree of drafted tokens over the paged latent cache (libqmla.so, `qmla_tree_forward`).

Beside `forward(qrows=...)`, whose drafted tokens form a chain (qwen_mla/mla_impl.py:628-662): here each
request's last cached tokens are the nodes of a tree, and a node sees the context and its ancestors, as a mask
says. After verification `cache_compact` brings the accepted path together. There is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .decode import Workspace
from .eviction import row_params

MAX_NODES = 64


def tree_mask(parents) -> torch.Tensor:
    """The mask words [requests, nodes] (int64) of trees given by their nodes' parents [requests, nodes] (an
    integer tensor or nested lists; -1: a root, whose parent is the context): bit i of word j is set where i is j or an
    ancestor of j. A node's parent precedes it. Host work."""
    par = torch.as_tensor(parents, device="cpu").to(torch.int64)
    if par.dim() != 2 or par.shape[1] > MAX_NODES:
        raise ValueError(f"tree_mask: parents must be [requests, nodes] with at most {MAX_NODES} nodes")
    if bool(((par >= torch.arange(par.shape[1])) | (par < -1)).any()):
        raise ValueError("tree_mask: a node's parent must be -1 or an earlier node")
    words = torch.zeros_like(par)
    for j in range(par.shape[1]):
        up = par[:, j]
        above = words.gather(1, up.clamp_min(0)[:, None])[:, 0]
        own_bit = 1 << j if j < 63 else -(1 << 63)
        words[:, j] = torch.where(up >= 0, above, torch.zeros_like(above)) | own_bit
    return words


def tree_forward(q_nope, q_rope, kv_cache, block_table, seq_lens, tree_mask, *, node_counts=None, d_c=None, rope_w=None,
                 rms_offset=None, page_size, sm_scale, kv_fp8=None, fp8_rms="log8", k_scale=None, rms_heads=None, logit_cap=0.0,
                 out=None, lse=None, workspace=None, return_lse=True, status=None):
    """Attention of every request's drafted nodes; returns (o, lse).

    q_nope [requests * nodes, H, d_c] and q_rope [requests * nodes, H, rope_w] (bf16); block_table [requests,
    pages] and seq_lens [requests] (int32), one row per request, lengths with the drafted tokens, whose rows are the
    request's last: node i of n is token seq_len - n + i. n = node_counts[b] (int32) or all of `nodes` = 64 at most.
    tree_mask [requests, nodes] int64: bit i of word j lets node j see node i (its own bit among them, see
    `tree_mask`); the context before the nodes is seen by all. Rows from n on, and rows that see no token, come
    back as zeros with lse -inf. d_c 256, 512 (rope up to 64), 768 and 1792 (rope up to 256 elsewhere), bf16 and FP8
    rows with every divisor format, at most 64 heads (53 at d_c 768); other layouts raise NotImplementedError. A non-finite
    element in a drafted token's row makes the rows that see it NaN.

    workspace: a `Workspace` (or a uint8 tensor) reserved for `qmla_tree_workspace_bytes`; without one the call
    takes its scratch from torch's allocator. Calls that may overlap need workspaces of their own."""
    if tree_mask.dtype != torch.int64 or tree_mask.dim() != 2 or (tree_mask.numel() and tree_mask.shape[1] > 1 and tree_mask.stride(1) != 1):
        raise TypeError("tree_forward: tree_mask must be [requests, nodes] int64 with contiguous rows")
    n_req, nodes = tree_mask.shape
    rows, H = q_nope.shape[0], q_nope.shape[1]
    if nodes < 1 or nodes > MAX_NODES:
        raise ValueError(f"tree_forward: 1 to {MAX_NODES} nodes, got {nodes}")
    if rows != n_req * nodes:
        raise ValueError(f"tree_forward: {rows} query rows for {n_req} requests of {nodes} nodes")
    if block_table.shape[0] != n_req or seq_lens.shape[0] != n_req:
        raise ValueError("tree_forward: block_table and seq_lens need one row per request")
    if node_counts is not None and (node_counts.dtype != torch.int32 or node_counts.dim() != 1 or node_counts.shape[0] != n_req
                                    or (n_req > 1 and node_counts.stride(0) != 1)):
        raise TypeError("tree_forward: node_counts must be [requests] int32, contiguous")
    _lib.same_device("tree_forward", "q_nope", q_nope, "q_rope", q_rope, "kv_cache", kv_cache,
                     "block_table", block_table, "seq_lens", seq_lens, "tree_mask", tree_mask,
                     "node_counts", node_counts, "out", out, "lse", lse, "status", status)
    dv = q_nope.shape[-1] if d_c is None else d_c
    if out is None:
        out = torch.empty(rows, H, dv, dtype=torch.bfloat16, device=q_nope.device)
    if lse is None and return_lse:
        lse = torch.empty(rows, H, dtype=torch.float32, device=q_nope.device)
    if tuple(out.shape) != (rows, H, dv) or (lse is not None and tuple(lse.shape) != (rows, H)):
        raise ValueError(f"tree_forward: out must be [{rows}, {H}, {dv}] and lse [{rows}, {H}]")
    p = row_params(q_nope, q_rope, kv_cache, block_table, seq_lens, out, lse, d_c=d_c, rope_w=rope_w, rms_offset=rms_offset,
                   page_size=page_size, sm_scale=sm_scale, kv_fp8=kv_fp8, fp8_rms=fp8_rms, k_scale=k_scale, groups=1,
                   rms_heads=rms_heads, logit_cap=logit_cap, status=status)
    p.qrows = nodes
    lib = _lib.lib()
    if workspace is None or isinstance(workspace, Workspace):
        need = max(int(lib.qmla_tree_workspace_bytes(p)), 256)
        ws = torch.empty(need, dtype=torch.uint8, device=q_nope.device) if workspace is None \
            else workspace.reserve(need, q_nope.device)
    else:
        _lib.same_device("tree_forward", "workspace", workspace)
        ws = workspace
    p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel() * ws.element_size()
    _lib.check("qmla_tree_forward", lib.qmla_tree_forward(p, tree_mask.data_ptr(), tree_mask.stride(0),
                                                          None if node_counts is None else node_counts.data_ptr(), _lib.stream()))
    return out, lse
