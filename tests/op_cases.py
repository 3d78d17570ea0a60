"""Float64 references of the tree, weights, eviction and rotary operators, written from their formulas, and
the error bounds their arithmetic allows. Everything runs on the CPU.

Bounds. Scores are sums of C exact products of bf16 (or e4m3) numbers in fp32: off by at most C 2^-24 of the sum
of the terms' magnitudes, then a few roundings of the divide, scale and exponent (8 counted, each 2^-24 of
|score| + |lse| + 1). With `d` that bound, exp(s) is off by exp(d) - 1 of itself."""
from __future__ import annotations

import math

import torch

from qmla.synth import make_case

F8 = torch.float8_e4m3fn
U32 = 2.0 ** -24


def rows_of(case, b: int, L: int, table=None):
    """Keys [L, C], values [L, d_c] and divisors [L, H] of request b in float64."""
    P, C, H = case.page_size, case.d_c + case.rope_w, case.heads
    table = case.block_table if table is None else table
    flat = case.cache.cpu().reshape(-1, case.cache.shape[-1])
    t = torch.arange(L)
    rows = flat[table[b].cpu().long()[t // P] * P + t % P]
    ks = 1.0 if case.k_scale is None else float(case.k_scale)
    if case.kv == "fp8":
        x = rows[:, :C].contiguous().view(F8).double() * ks
    else:
        x = rows[:, :C].double()
    if case.rms_mode == "none":
        rms = torch.ones(L, H, dtype=torch.float64)
    elif case.rms_mode == "log8":
        rms = torch.exp2(rows[:, C:C + H].double() * 6.0 / 255.0 - 3.0)
    elif case.rms_mode == "bf16":
        rms = rows[:, C:C + H].double()
    elif case.rms_mode == "bf16_bytes":
        rms = rows[:, C:C + 2 * H].contiguous().view(torch.bfloat16).double()
    else:
        rms = rows[:, C:C + H].contiguous().view(F8).double() * ks
    return x, x[:, :case.d_c], torch.where(rms > 0, rms, torch.ones_like(rms))


def scores(case, q, x, rms, cap: float):
    """q [R, H, C] (float64) -> scores [R, H, L] and the bound `d` on their error."""
    s = torch.einsum("rhc,lc->rhl", q, x) / rms.T[None] * case.sm_scale
    mag = torch.einsum("rhc,lc->rhl", q.abs(), x.abs()) / rms.T[None] * case.sm_scale
    d = U32 * (x.shape[1] * mag + 8.0 * (s.abs() + 1.0))
    if cap > 0:
        s = cap * torch.tanh(s / cap)
        d = d + U32 * 16.0 * cap   # 1 - 2 / (e^2x + 1): a few roundings of numbers up to 2
    return s, d


def queries(case, q_nope, q_pe, rows):
    """[len(rows), H, C] in float64; with groups each head's latent part sits in its group's columns."""
    G, H, dg = case.groups, case.heads, case.d_c // case.groups
    qn = q_nope.cpu().double()[rows]
    full = torch.zeros(len(rows), H, case.d_c, dtype=torch.float64)
    for g in range(G):
        hs = slice(g * H // G, (g + 1) * H // G)
        full[:, hs, g * dg:(g + 1) * dg] = qn[:, hs]
    return torch.cat([full, q_pe.cpu().double()[rows]], -1) if case.rope_w else full


def ref_tree(case, q_nope, q_pe, lens, mask, counts, cap=0.0, table=None):
    """(out, lse, out bound, lse bound), rows [B * T]; the bound of out leaves out its own rounding."""
    B, T = mask.shape
    H = case.heads
    o = torch.zeros(B * T, H, case.d_c, dtype=torch.float64)
    lse = torch.full((B * T, H), -math.inf, dtype=torch.float64)
    ob, lb = torch.zeros_like(o), torch.zeros_like(lse)
    for b in range(B):
        L = int(lens[b])
        n = T if counts is None else max(0, min(T, int(counts[b])))
        if L <= 0:
            continue
        x, v, rms = rows_of(case, b, L, table)
        s, d = scores(case, queries(case, q_nope, q_pe, list(range(b * T, b * T + T))), x, rms, cap)
        for j in range(n):
            seen = [t for t in range(L) if t < L - n or (int(mask[b, j]) >> (t - (L - n))) & 1]
            if not seen:
                continue
            z, dz = s[j][:, seen], d[j][:, seen]
            p = torch.softmax(z, -1)
            o[b * T + j] = p @ v[seen]
            lse[b * T + j] = torch.logsumexp(z, -1)
            far = dz.amax(-1, keepdim=True)
            # P rounds to bf16 (2^-8), its sum with it: twice that, and scores shift p by up to e^2d - 1
            ob[b * T + j] = (2.02 * 2.0 ** -8 + 2.0 * torch.expm1(2 * far)) * (p @ v[seen].abs())
            lb[b * T + j] = far[:, 0] + U32 * 8.0 * (lse[b * T + j].abs() + 1.0) + U32 * len(seen)
    return o, lse, ob, lb


def close(name, got, want, bound, dtype):
    """|got - want| <= bound + the rounding to dtype, infinities and NaN alike."""
    got, want = got.detach().cpu().double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"[{name}] NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"[{name}] infinities differ"
    allow = bound.expand_as(want) + torch.finfo(dtype).eps / 2 * (want.abs() + bound) + torch.finfo(dtype).tiny
    over = ((got - want).abs() - allow)[fine]
    worst = float(((got - want).abs() / allow)[fine].max()) if fine.any() else 0.0
    print(f"[{name}] worst error {worst:.3f} of its bound", flush=True)
    assert not (over > 0).any(), f"[{name}] {worst:.2f} times the bound"


def fp8_kw(case):
    return dict(kv_fp8=True, fp8_rms={"bf16_bytes": "bf16"}.get(case.rms_mode, case.rms_mode), k_scale=case.k_scale) \
        if case.kv == "fp8" else {}


def row_kw(case, cap=0.0):
    return dict(d_c=case.d_c, rope_w=case.rope_w, rms_offset=case.rms_offset, page_size=case.page_size,
                sm_scale=case.sm_scale, logit_cap=cap, **fp8_kw(case))


def tree_case(device, *, kv, rms_mode, d_c, rope, heads, page, lens, nodes, seed, amp=1.0, q_amp=2.0, ragged=False):
    """A cache (one table row and length per request), queries of every node, random trees."""
    c = make_case(batch=len(lens), heads=heads, d_c=d_c, rope_w=rope, page_size=page, lens=lens, kv=kv, rms_mode=rms_mode,
                  seed=seed, device=device, rms="spread", amp=amp)
    g = torch.Generator().manual_seed(seed + 5)
    B = len(lens)
    qn = (q_amp * torch.randn(B * nodes, heads, d_c, generator=g)).to(torch.bfloat16).to(device)
    qp = (q_amp * torch.randn(B * nodes, heads, rope, generator=g)).to(torch.bfloat16).to(device)
    parents = torch.tensor([[int(torch.randint(-1, max(j, 0), (1,), generator=g)) if j else -1 for j in range(nodes)]
                            for _ in range(B)])
    counts = torch.randint(0, nodes + 1, (B,), generator=g).to(torch.int32) if ragged else None
    return c, qn, qp, parents, counts
