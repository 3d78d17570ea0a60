// Attention of a tree of drafted tokens over the paged latent cache (qmla_tree_forward). See
// include/qmla.h for what a node sees.
//
// A request's nodes x heads are its query rows (node-major, so a row's head is row % heads), up to
// 64 x heads of them on one latent: a matrix-core problem, not a streaming one like the decode. A
// workgroup of four waves holds ROWS of them and walks the request's tokens in tiles of 32:
//   S^T = K Q^T   v_mfma_f32_32x32x16_bf16, keys from LDS as A, queries in registers as B, so a lane
//                 holds one row's scores of 16 tokens and the softmax needs one exchange with the lane
//                 32 away;
//   O^T = V^T P^T the same product, values by transposed LDS reads as A; P stays in the registers the
//                 scores came in (their token order 8(i/4) + 4(lane/32) + i%4 is the order the two
//                 transposed reads of a fragment fetch).
// With NS = 1 a wave owns 32 rows whole. Wider latents do not fit one wave's registers (32 rows x d_c fp32
// and 32 rows of queries): NS waves share 32 rows, each with 1/NS of the score columns and of the output
// columns, and add their partial scores through LDS in one order, so they hold equal scores.
// FP8 rows become bf16 exactly, beside the products (tree8_kernel) or, where their rows are too wide for that, on their
// way into LDS (tree_kernel, which holds the bf16 rows). P is bf16, the sum that normalizes is of the same rounded P, the lse
// of the unrounded.
//
// Bound by what one wave a SIMD issues: 16 FP8 requests of 64 nodes x 24 heads on 2048 .. 8192 tokens take 336 us, where
// their 213 Gflop alone need 157; the matrix cores are busy 37 % and the vector units 42 % of it.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmla.h"
#include "qmla_common.h"

namespace qmla {
namespace tr {

constexpr int TT = 32, NT = 256;
constexpr int LDS_MAX = 160 * 1024;
constexpr int MAXH = 64;
// log2 units a row's maximum may pass its softmax reference by. Moving the reference multiplies all accumulators, 3500
// cycles of a wave, which one of 32 rows suffices for: at 8 it came every other tile of scores with a deviation of 2
// (nats), 16 requests of 64 nodes 405 us, 338 at 24. P and the sums are floats, as exact at 2^24 as at 1, and leave the
// values 2^80.
constexpr float kMoveAt = 24.f;

struct TrParams {
  KParams k;
  const int64_t* mask;
  int64_t mask_sr;
  const int* counts;
  int rt;              // row tiles of a request
  int rows;            // query rows of a request
  int cols;            // d_c + rope_w
  int nwg, min_chunk;
  int rms_mode, rms_b;
  int64_t* plan;       // [0] chunk, [1 + b] tiles before request b
  float* part_o;
  float* part_lse;
};

__device__ __forceinline__ f32x16 mfma32(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// The score products name VGPRs: the output accumulators take every AGPR, and left to itself the compiler
// accumulates scores there too, spilling what they displace (all 36 query fragments, reloaded each tile). The
// compiler sees no matrix instruction in these statements, so the waits are their own: two states after a vector
// instruction that may have written an operand (a copy the allocator placed; they pass behind the last product),
// and 24 before the result is read, more than the longest 32x32 product needs.
__device__ __forceinline__ void mfma32_v0(f32x16& d, const bf16x8& a, const bf16x8& b) {
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma32_v(f32x16& d, const bf16x8& a, const bf16x8& b) {
  asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma_v_done(f32x16& d) { asm volatile("s_nop 15\n\ts_nop 7" : "+v"(d)); }

__device__ __forceinline__ int node_count(const TrParams& t, int b) {
  const int n = t.counts ? t.counts[b] : t.k.qrows;
  return n < 0 ? 0 : n < t.k.qrows ? n : t.k.qrows;
}
__device__ __forceinline__ int tiles_of(const TrParams& t, int b) {
  const int L = t.k.seq_lens[b];
  return L <= 0 || node_count(t, b) == 0 ? 0 : (L + TT - 1) / TT;
}

// Work units are (row tile, token tile) pairs, requests outermost, tokens innermost. Either workgroup w owns units
// [w * chunk, (w + 1) * chunk), which may be the end of one row tile's and the start of the next's, or each row tile's
// tokens are split evenly over workgroups of their own, at most chunk tiles each. The latter is taken where it
// needs at most SECOND tiles more a workgroup: a second piece costs its start and its end, about as much as
// 5 tiles (1 request of 8 nodes, 41 tiles in two row tiles: 43 us with one workgroup on both, 27 us so).
constexpr int SECOND = 4;
struct Range {
  int64_t lo, hi;
  int b, w;
  int64_t c0;   // units before request b
};
__device__ inline Range unit_range(const TrParams& t) {
  const int lane = threadIdx.x & 63, blk = blockIdx.x;
  auto tiles = [&](int base) { return base + lane < t.k.n_req ? tiles_of(t, base + lane) : 0; };
  int64_t total = 0;
  for (int base = 0; base < t.k.n_req; base += 64) total += lane_value(wave_incl_sum(tiles(base)), 63);
  Range r{};
  const int64_t units = total * t.rt;
  int64_t chunk = (units + t.nwg - 1) / t.nwg;
  if (chunk < t.min_chunk) chunk = t.min_chunk;
  int even = 0;   // tiles of a workgroup where none has two row tiles', 0: some have
  int64_t active = (units + chunk - 1) / chunk;
  if (chunk < (1 << 24))
    for (int c = (int)chunk; !even && c <= (int)chunk + SECOND; c += SECOND / 2) {
      int64_t pieces = 0;
      for (int base = 0; base < t.k.n_req; base += 64) pieces += lane_value(wave_incl_sum((tiles(base) + c - 1) / c), 63);
      if (pieces * t.rt <= t.nwg) {
        even = c;
        active = pieces * t.rt;
      }
    }
  // consecutive workgroups go to consecutive XCDs: give each XCD consecutive ranges, which share tokens
  const int per = (int)((active + 7) / 8);
  r.w = t.nwg % 8 == 0 ? (blk & 7) * per + (blk >> 3) : blk;
  const bool live = r.w < active && (t.nwg % 8 != 0 || (blk >> 3) < per), store = blk == 0;
  if (store && lane == 0) t.plan[0] = even ? -even : chunk;
  if (!live && !store) return r;
  const int64_t start = even ? r.w : r.w * chunk;
  int64_t run = 0, before = 0;
  int nt = 0;
  for (int base = 0; base < t.k.n_req; base += 64) {
    const int b = base + lane, all = tiles(base);
    const int n = even ? (all + even - 1) / even : all;
    const int in = wave_incl_sum(n);
    const int64_t c = run + in - n;
    if (store && b < t.k.n_req) t.plan[1 + b] = c;
    const uint64_t m = __builtin_amdgcn_ballot_w64(b < t.k.n_req && c * t.rt <= start);
    if (m) {
      const int x = 63 - __builtin_clzll(m);
      r.b = base + x;
      before = (run + lane_value(in - n, x)) * t.rt;
      nt = lane_value(all, x);
    }
    run += lane_value(in, 63);
  }
  if (!live) return r;
  if (even) {
    const int k = (nt + even - 1) / even, x = (int)(r.w - before), m = x / k, i = x - m * k;
    r.lo = (int64_t)m * nt + (int64_t)i * nt / k;
    r.hi = (int64_t)m * nt + (int64_t)(i + 1) * nt / k;
  } else {
    r.lo = start;
    r.hi = start + chunk < units ? start + chunk : units;
    r.c0 = before;
  }
  return r;
}

// Staged tile: 32 rows of CP bf16 columns in 16-byte chunks, chunk c of row r at c ^ swz(r) inside its
// aligned group. Over 32 chunks of 16 bytes (128 banks) a row's stride takes `b` of the row's five bits apart;
// the others are spread by the swizzle, low ones first onto the 4-chunk bit: 32 rows' same chunk (score
// reads) and 8 rows' same 4 chunks (value reads) then lie on distinct banks.
template <int RS>
__device__ __forceinline__ int swz(int r) {
  static_assert(RS % 8 == 0);
  constexpr int b = RS % 32 == 0 ? 0 : RS % 32 == 16 ? 1 : 2, n = 5 - b;
  const int x = (r & 31) >> b;
  return ((x & ((1 << (n - 2)) - 1)) << 2) | (x >> (n - 2));
}

__device__ __forceinline__ float inv_divisor(uint32_t raw, int mode, float ks) {
  if (mode == QMLA_RMS_LOG8) return fast_exp2(3.0f - (float)raw * (6.0f / 255.0f));
  if (mode == QMLA_RMS_NONE) return 1.f;
  const float r = mode == QMLA_RMS_E4M3 ? fp8_to_f32(raw) * ks : bf16_bits_to_f32(raw);
  return r > 0.f ? __builtin_amdgcn_rcpf(r) : 1.f;   // within 1 ulp
}

// any element of 16 bytes not finite
template <bool FP8>
__device__ __forceinline__ bool any_odd(const i32x4& v) {
  bool odd = false;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t u = (uint32_t)v[d];
    if constexpr (FP8) {
      const uint32_t x = (u & 0x7f7f7f7fu) + 0x01010101u;   // 0x7f becomes 0x80
      odd = odd || (x & 0x80808080u);
    } else {
      odd = odd || (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
    }
  }
  return odd;
}

template <bool FP8_, int DC_, int CP_, int NS_, int STAGES_, int QL_>
struct Cfg {
  static constexpr bool FP8 = FP8_;
  static constexpr int DC = DC_, CP = CP_, NS = NS_, STAGES = STAGES_;
  static constexpr int QL = QL_;                   // a wave's last query fragments, kept in LDS
  static constexpr int ROWS = 128 / NS;            // query rows of a workgroup
  static constexpr int RS = CP / 8;                // 16-byte chunks of a staged row
  static constexpr int QC = CP / NS, NQ = QC / 16; // score columns of a wave, its products
  static constexpr int OB = DC / NS / 32;          // output column blocks of a wave
  static constexpr int UC = FP8 ? 16 : 8;          // columns of a 16-byte load
  static constexpr int UPR = CP / UC;              // loads of a row
  static constexpr int LOADS = (UPR + 7) / 8;      // loads of a thread
  static constexpr int TILE_B = TT * CP * 2;
  static_assert(DC % (32 * NS) == 0 && CP % (16 * NS) == 0 && CP % 64 == 0);
  static constexpr int out_col(int ob, int i4) { return 32 * ob + 8 * i4; }   // first of accumulators 4 i4 .., h = 0
};

constexpr int KD = 5, VD = 4;   // LDS reads ahead of a score product, fragments ahead of a value product
constexpr int RL = 2;         // dwords of divisors a thread loads ahead
constexpr int IRS = TT + 4;   // floats of a head's divisors in LDS

template <class C>
__host__ __device__ constexpr int lds_bytes(int heads) {
  return C::STAGES * (C::TILE_B + heads * IRS * 4) + (C::NS > 1 ? 4 * 4096 : 0) + 4 * C::QL * 1024 + 4 * TT * 8 + 32;
}

typedef __attribute__((address_space(3))) char lchar;

// ---- what the kernels share: a tile's scores of a lane's row to P, the running sums, a finished piece ------
// divide by the divisors (ir: this row's, from LDS, scaled) and cap: log2-domain scores
__device__ __forceinline__ void finish_scores(const TrParams& t, f32x16& s, const float* ir) {
#pragma unroll
  for (int i4 = 0; i4 < 4; ++i4) {
    const f32x4 iv = *reinterpret_cast<const f32x4*>(ir + 8 * i4);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[4 * i4 + i] *= iv[i];
  }
  const float cap = t.k.logit_cap;
  if (__builtin_expect(cap > 0.f, 0)) {
    const float in = 2.0f * kLog2e / cap, out = cap * kLog2e;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = out - 2.0f * out * __builtin_amdgcn_rcpf(fast_exp2(s[i] * in) + 1.0f);
  }
}
// a tile with drafted tokens: what the row's node does not see, and tokens with a bad element
__device__ __forceinline__ void mask_scores(const TrParams& t, f32x16& s, int j, int b, int base, int nodes, int r0, int me,
                                            uint32_t odd) {
  const int r = r0 + (me & 31), node = r / t.k.heads, h = (me >> 5) & 1, d = j * TT - base;   // -TT < d < nodes <= 64
  uint64_t sees = 0;
  if (r < t.rows && node < nodes) sees = (uint64_t)t.mask[b * t.mask_sr + node] & (~0ull >> (64 - nodes));
  // (used at once on every way through: a load that stays pending here is waited for, and every DMA with it, by the
  // tiles that never come here)
  const uint32_t vis = (d >= 0 ? (uint32_t)(sees >> d) : (uint32_t)(sees << -d) | ((1u << -d) - 1)) >> (4 * h);
  odd >>= 4 * h;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int x = 8 * (i >> 2) + (i & 3);
    const float v = (odd >> x) & 1 ? __uint_as_float(0x7fc00000u) : s[i];
    s[i] = (vis >> x) & 1 ? v : kNegInf;
  }
}

// The softmax of s against a reference that moves when a row's maximum has passed it by kMoveAt (a row's own
// doing: what its neighbours hold does not move it; a NaN maximum moves nothing), in steps 0 .. NSOFT - 1 small
// enough to lie beside one product each.
struct Soft {
  float mx, m_use, m_new, es, ep;
};
constexpr int NSOFT = 24;
__device__ __forceinline__ void soft_step(int i, f32x16& s, bf16x8 (&pn)[2], Soft& sf, float m_ref) {
  if (i == 0) {
    sf.mx = fmaxf(fmaxf(s[0], s[1]), s[2]);
    sf.es = sf.ep = 0.f;
  } else if (i < 6) {
    sf.mx = fmaxf(fmaxf(sf.mx, s[2 * i + 1]), s[2 * i + 2]);
  } else if (i == 6) {
    sf.mx = fmaxf(fmaxf(sf.mx, s[13]), fmaxf(s[14], s[15]));
  } else if (i == 7) {
    const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(sf.mx), __float_as_uint(sf.mx), false, false);
    sf.mx = fmaxf(__uint_as_float(o[0]), __uint_as_float(o[1]));
    sf.m_new = sf.mx > m_ref + kMoveAt ? sf.mx : m_ref;
    sf.m_use = is_neg_inf(sf.m_new) ? 0.f : sf.m_new;
  } else if (i < 16) {
    const int x = 2 * (i - 8);
    s[x] = fast_exp2(s[x] - sf.m_use);
    s[x + 1] = fast_exp2(s[x + 1] - sf.m_use);
  } else if (i < 24) {
    const int x = 2 * (i - 16);
    sf.es += s[x] + s[x + 1];
    const bf16x2 e{(__bf16)s[x], (__bf16)s[x + 1]};
    pn[x >> 3][x & 7] = e[0];
    pn[x >> 3][(x & 7) + 1] = e[1];
    sf.ep = __builtin_amdgcn_fdot2_f32_bf16(e, bf16x2{(__bf16)1.f, (__bf16)1.f}, sf.ep, false);
  }
}
// the accumulators of 16 blocks are in AGPRs, all at once: else the compiler may keep one in VGPRs over the loop and
// copy it there and back each tile (16 requests of 64 nodes 355 us, 338 so)
template <int OB>
__device__ __forceinline__ void in_agprs(f32x16 (&a)[OB]) {
  if constexpr (OB == 16)
    asm volatile("" : "+a"(a[0]), "+a"(a[1]), "+a"(a[2]), "+a"(a[3]), "+a"(a[4]), "+a"(a[5]), "+a"(a[6]), "+a"(a[7]),
                 "+a"(a[8]), "+a"(a[9]), "+a"(a[10]), "+a"(a[11]), "+a"(a[12]), "+a"(a[13]), "+a"(a[14]), "+a"(a[15]));
}
template <int OB>
__device__ __forceinline__ void rescale(const Soft& sf, float& m_ref, float& l_sum, float& l_p, f32x16 (&acc)[OB]) {
  const bool moves = sf.m_new != m_ref;
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(moves) != 0, 0)) {
    const float alpha = moves ? fast_exp2(m_ref - sf.m_new) : 1.f;
    l_sum *= alpha;
    l_p *= alpha;
#pragma unroll
    for (int ob = 0; ob < OB; ++ob) {
      // one block at a time, there and back: left to the compiler all of them pass through VGPRs at once and
      // displace the queries
      asm volatile("" : "+a"(acc[ob]));
      acc[ob] *= alpha;
      asm volatile("" : "+a"(acc[ob]));
      __builtin_amdgcn_sched_barrier(0);
    }
    m_ref = sf.m_new;
  }
  l_sum += sf.es;
  l_p += sf.ep;
}

// The rows of a finished piece: the final output and lse where it held all of the request's tokens, else
// partial slot `slot`. me: the thread.
struct Piece {
  int b, m, nodes, rg, cp;
  int64_t slot;
  bool whole;
};
template <class C>
__device__ __forceinline__ void store_piece(const TrParams& t, const Piece& q, int me, float ks, float m_ref, float l_sum,
                                            float l_p, const f32x16 (&acc)[C::OB]) {
  const KParams& p = t.k;
  const int n = me & 31, h = (me >> 5) & 1;
  const int r = q.m * C::ROWS + q.rg * 32 + n;
  if (r >= t.rows) return;
  const int node = r / p.heads, head = r - node * p.heads;
  {
    const auto o = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_sum), __float_as_uint(l_sum), false, false);
    l_sum = __uint_as_float(o[0]) + __uint_as_float(o[1]);
    const auto o2 = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_p), __float_as_uint(l_p), false, false);
    l_p = __uint_as_float(o2[0]) + __uint_as_float(o2[1]);
  }
  if (node >= q.nodes) l_sum = l_p = 0.f;
  const float inv = empty_sum(l_p) ? 0.f : (q.whole ? ks : 1.f) / l_p;
  const int col = q.cp * (C::DC / C::NS) + 4 * h;
  const int64_t row = (int64_t)q.b * p.qrows + node, prow = q.slot * C::ROWS + q.rg * 32 + n;
  const int dt = p.out_dt;
  char* ob0 = reinterpret_cast<char*>(p.out) + (row * p.o_sr + head * p.o_sh + col) * out_bytes(dt);
  auto store = [&](auto dtc) {
    constexpr int DT = decltype(dtc)::value, ES = DT == QMLA_DT_F32 ? 4 : 2;
#pragma unroll
    for (int ob = 0; ob < C::OB; ++ob)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = empty_sum(l_p) ? 0.f : acc[ob][4 * i4 + i] * inv;
        store_out4<DT>(ob0 + C::out_col(ob, i4) * ES, v);
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  if (!q.whole) {
    // as the accumulators lie: [wave][block][accumulators 4 i4 ..][lane] 16 bytes
    char* at = reinterpret_cast<char*>(t.part_o) + ((q.slot * 4 + q.rg * C::NS + q.cp) * C::OB * 256 + (me & 63)) * 16;
#pragma unroll
    for (int ob = 0; ob < C::OB; ++ob)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = empty_sum(l_p) ? 0.f : acc[ob][4 * i4 + i] * inv;
        *reinterpret_cast<f32x4*>(at + (ob * 4 + i4) * 1024) = v;
        __builtin_amdgcn_sched_barrier(0);
      }
  } else if (dt == QMLA_DT_F32) store(std::integral_constant<int, QMLA_DT_F32>{});
  else if (dt == QMLA_DT_F16) store(std::integral_constant<int, QMLA_DT_F16>{});
  else store(std::integral_constant<int, QMLA_DT_BF16>{});
  if (h == 0 && q.cp == 0) {
    if (!q.whole) t.part_lse[prow] = empty_sum(l_sum) ? kNegInf : m_ref + fast_log2(l_sum);
    else if (p.lse) store_out(p.lse, p.lse_dt, row * p.lse_sr + head, row_lse(m_ref, l_sum));
  }
}

template <class C>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(1, 1))) void tree_kernel(const TrParams t) {
  extern __shared__ __align__(16) char lds[];
  const KParams& p = t.k;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int rg = wave / C::NS, cp = wave % C::NS;
  lchar* const kt = QMLA_LDS(char, lds);
  float* irms = reinterpret_cast<float*>(lds + C::STAGES * C::TILE_B);   // [STAGES][heads][IRS]
  char* part = lds + C::STAGES * (C::TILE_B + p.heads * IRS * 4);        // [4 waves][4][64] 16 bytes
  char* ql = part + (C::NS > 1 ? 4 * 4096 : 0);                          // [4 waves][QL][64] 16 bytes
  int64_t* rowoff = reinterpret_cast<int64_t*>(ql + 4 * C::QL * 1024);   // [4][TT]
  uint32_t* odd = reinterpret_cast<uint32_t*>(rowoff + 4 * TT);          // [4], bit per token
  const Range rng = unit_range(t);
  if (rng.lo >= rng.hi) return;
  const float ks = p.k_scale ? *p.k_scale : 1.f;
  const float fs = p.sm_scale * ks * (p.logit_cap > 0.f ? 1.f : kLog2e);
  int bad = 0;
  // this lane's reads of a staged tile. A tile and its rows lie on multiples of a swizzle group, so the chunk's
  // low bits go onto an address with one exclusive or and the rest into the instruction's offset: score chunk
  // 2f + h of row n, and the value fragment of columns 32 ob .. in rows 16 k2 + 8 x + vr
  constexpr int NSW = C::RS % 32 == 0 ? 5 : C::RS % 32 == 16 ? 4 : 3;   // bits the swizzle flips
  constexpr int GM = (1 << NSW) - 1;
  static_assert((C::QC / 8) % 2 == 0 && (C::DC / C::NS / 8) % 4 == 0);
  const int kc0 = cp * (C::QC / 8), vc0 = cp * (C::DC / C::NS / 8);
  const uint32_t klane = n * (C::CP * 2) + ((swz<C::RS>(n) ^ h) << 4);
  const int vq = lane & 15, vr = 4 * h + (vq >> 2), vc = 2 * ((lane >> 4) & 1) + ((vq & 3) >> 1);
  uint32_t vlane[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) vlane[x] = (8 * x + vr) * (C::CP * 2) + ((swz<C::RS>(8 * x + vr) ^ vc) << 4) + (vq & 1) * 8;
  int64_t u = rng.lo, c0 = rng.c0;
  int b = rng.b;
  while (u < rng.hi) {
    const int nt = tiles_of(t, b);
    if (u >= c0 + (int64_t)nt * t.rt) {
      c0 += (int64_t)nt * t.rt;
      ++b;
      continue;
    }
    const int m = (int)((u - c0) / nt), ta = (int)((u - c0) - (int64_t)m * nt);
    const int te = rng.hi - u < nt - ta ? ta + (int)(rng.hi - u) : nt;
    const int L = p.seq_lens[b], nodes = node_count(t, b), base = L - nodes;
    // ---- this lane's query row
    // Of the thread only what the tile loop uses is kept over it: the rest is worked out again where it is
    // needed (`own` keeps the compiler from doing so ahead). Held, it would push other values into scratch, whose
    // reloads wait for every load in flight.
    auto own = [&]() {
      int x = tid;
      asm volatile("" : "+v"(x));
      return x;
    };
    const int r0 = m * C::ROWS + rg * 32;
    const bool wlive = r0 < t.rows;
    int irms_at;   // this row's head in the divisors
    bf16x8 qf[C::NQ - C::QL];
    char* const qlw = ql + (wave * C::QL * 64 + lane) * 16;
    {
      // rows may be aligned to their elements only
      typedef bf16x8 bf16x8_e __attribute__((aligned(2)));
      const int r = r0 + n < t.rows ? r0 + n : t.rows - 1, node = r / p.heads, head = r - node * p.heads;
      irms_at = head * IRS + 4 * h;
      const int64_t row = (int64_t)b * p.qrows + node;
      const __bf16* qn = p.q_nope + row * p.qn_sr + head * p.qn_sh;
      const __bf16* qp = p.q_pe + row * p.qp_sr + head * p.qp_sh;
      const int whole8 = p.rope_w & ~7;
      bf16x8 tail{};
      for (int i = 0; i < (p.rope_w & 7); ++i) {
        const __bf16 x = qp[whole8 + i];
#pragma unroll
        for (int e = 0; e < 8; ++e) tail[e] = e == i ? x : tail[e];
      }
#pragma unroll
      for (int f = 0; f < C::NQ; ++f) {
        // dead rows keep what they read: their columns of the products go nowhere
        const int c = cp * C::QC + 16 * f + 8 * h, o = c - C::DC;
        if (C::NS == 1 && 16 * f < C::DC) {
          if (f < C::NQ - C::QL) qf[f] = *reinterpret_cast<const bf16x8_e*>(qn + c);
          else *reinterpret_cast<bf16x8*>(qlw + (f - (C::NQ - C::QL)) * 1024) = *reinterpret_cast<const bf16x8_e*>(qn + c);
        } else {
          bf16x8 v = tail;
          if (o < 0) v = *reinterpret_cast<const bf16x8_e*>(qn + c);
          else if (o < whole8) v = *reinterpret_cast<const bf16x8_e*>(qp + o);
          i32x4 x = __builtin_bit_cast(i32x4, v);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = o <= whole8 ? x[e] : 0;
          if (f < C::NQ - C::QL) qf[f] = __builtin_bit_cast(bf16x8, x);
          else *reinterpret_cast<i32x4*>(qlw + (f - (C::NQ - C::QL)) * 1024) = x;
        }
      }
    }
    f32x16 acc[C::OB];
#pragma unroll
    for (int i = 0; i < C::OB; ++i) acc[i] = f32x16{};
    float m_ref = kNegInf, l_sum = 0.f, l_p = 0.f;
    Soft sf;

    // ---- staging
    i32x4 raw[C::LOADS];
    uint32_t rraw[RL];
    const int rd0 = p.rms_off_b >> 2, rskip = p.rms_off_b & 3;           // the divisors' first dword, bytes before them
    const int rdw = t.rms_mode == QMLA_RMS_NONE ? 0 : (rskip + p.heads * t.rms_b + 3) >> 2;
    // byte offsets of tile j's rows, in two steps: a thread's page id, and a step later its row. The id is
    // loaded before the step's rows are, so the wait for the last step's rows covers it.
    int pid = 0;
    auto page_of = [&](int j) {
      const int tok = j * TT + tid;
      if (tid < TT && tok < L) pid = p.bt[b * p.bt_stride + page_div(p, tok)];
    };
    auto rows_of = [&](int j) {
      if (tid < TT) {
        const int tok = j * TT + tid;
        int64_t off = -1;
        if (tok < L) off = checked_page(p, pid, bad) * p.page_stride_b + (int64_t)(tok - page_div(p, tok) * p.page_size) * p.token_stride_b;
        rowoff[(j & 3) * TT + tid] = off;
      }
    };
    // Loads of tile j's rows. Rows past the request read the cache's first row and loads past a row's units its
    // first unit; put() drops both.
    auto fetch = [&](int j) {
      const int me = own(), row = me >> 3, c = me & 7;
      const int64_t off = rowoff[(j & 3) * TT + row];
      const char* src = p.kv + (off >= 0 ? off : 0);
      if (t.cols == C::CP) {
#pragma unroll
        for (int i = 0; i < C::LOADS; ++i) {
          const bool past = C::UPR % 8 != 0 && i + 1 == C::LOADS && c >= C::UPR % 8;
          raw[i] = *reinterpret_cast<const i32x4*>(src + (past ? 0 : 16 * c + 128 * i));
        }
      } else {
        int cols = t.cols;
        asm volatile("" : "+s"(cols));
#pragma unroll
        for (int i = 0; i < C::LOADS; ++i)
          raw[i] = *reinterpret_cast<const i32x4*>(src + ((c + 8 * i) * C::UC < cols ? 16 * c + 128 * i : 0));
      }
      if (rdw > 0) {
        const char* rs = src + 4 * rd0;
#pragma unroll
        for (int i = 0; i < RL; ++i)
          if (8 * i < rdw) rraw[i] = *reinterpret_cast<const uint32_t*>(rs + 4 * (c + 8 * i < rdw ? c + 8 * i : 0));
      }
    };
    // dword d of a row's divisors (heads past the last go into `none`: branches around their stores cost more)
    auto put_rms = [&](float* o, int d, uint32_t v) {
      float* none = reinterpret_cast<float*>(odd + 4);
      auto put1 = [&](int hd, float x) { *((uint32_t)hd < (uint32_t)p.heads ? o + hd * IRS : none) = x; };
      if (__builtin_expect(t.rms_b == 1, C::FP8)) {
        const int hd = 4 * d - rskip;
#pragma unroll
        for (int e = 0; e < 4; ++e) put1(hd + e, fs * inv_divisor((v >> (8 * e)) & 0xff, t.rms_mode, ks));
      } else {
        // an odd byte offset splits a divisor over two dwords: those rows have theirs read by bytes below
        const int hd = 2 * d - (rskip >> 1);
#pragma unroll
        for (int e = 0; e < 2; ++e) put1(hd + e, fs * inv_divisor((v >> (16 * e)) & 0xffff, QMLA_RMS_BF16, ks));
      }
    };
    auto put = [&](int j) {
      const int me = own(), row = me >> 3, sc0 = me & 7;
      const uint32_t slane = (uint32_t)(uintptr_t)(kt + (j % C::STAGES) * C::TILE_B) + row * (C::CP * 2) +
                             (((C::FP8 ? 2 * sc0 : sc0) ^ swz<C::RS>(row)) << 4);
      if (t.cols != C::CP) {   // columns past the row's keys
        int cols = t.cols;
        asm volatile("" : "+s"(cols));
#pragma unroll
        for (int i = 0; i < C::LOADS; ++i) {
          const int left = cols - (sc0 + 8 * i) * C::UC;
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const int bits = left * (C::FP8 ? 8 : 16) - 32 * d;
            raw[i][d] = bits <= 0 ? 0 : bits >= 32 ? raw[i][d] : raw[i][d] & (int)((1u << (bits & 31)) - 1);
          }
        }
      }
      if (__builtin_expect((j + 1) * TT > base, 0)) {   // rows past the request; drafted tokens: what is not finite goes into `odd`
        const int tok = j * TT + row;
        bool any = false;
#pragma unroll
        for (int i = 0; i < C::LOADS; ++i) {
          const bool o = tok >= base && any_odd<C::FP8>(raw[i]);
          const bool past = C::UPR % 8 != 0 && i + 1 == C::LOADS && sc0 >= C::UPR % 8;
          any = any || (o && !past);
          raw[i] = o || tok >= L ? i32x4{} : raw[i];
        }
        if (any && tok < L) atomicOr(&odd[j & 3], 1u << row);
      }
#pragma unroll
      for (int i = 0; i < C::LOADS; ++i) {
        if (C::UPR % 8 == 0 || i + 1 < C::LOADS || sc0 < C::UPR % 8) {
          constexpr int per = C::FP8 ? 16 : 8;   // chunks from load to load
          const uint32_t at = slane ^ (((per * i) & GM) << 4);
          typedef __attribute__((address_space(3))) bf16x8 lvec;
          if constexpr (C::FP8) {
            bf16x8 x, y;
            fp8x16_to_bf16(raw[i], x, y);
            *(lvec*)(uintptr_t)(at + (((per * i) & ~GM) << 4)) = x;
            *(lvec*)(uintptr_t)((at ^ 16) + (((per * i) & ~GM) << 4)) = y;
          } else {
            *(lvec*)(uintptr_t)(at + (((per * i) & ~GM) << 4)) = __builtin_bit_cast(bf16x8, raw[i]);
          }
        }
      }
      float* ir = irms + (j % C::STAGES) * p.heads * IRS + row;
      if (__builtin_expect(t.rms_mode == QMLA_RMS_NONE, 0)) {
        for (int hd = sc0; hd < p.heads; hd += 8) ir[hd * IRS] = fs;
      } else if (__builtin_expect(t.rms_b == 2 && (rskip & 1), 0)) {
        for (int hd = sc0; hd < p.heads; hd += 8) {
          const int64_t off_put = rowoff[(j & 3) * TT + row];
          const uint8_t* at = reinterpret_cast<const uint8_t*>(p.kv + off_put + p.rms_off_b + 2 * hd);
          ir[hd * IRS] = off_put >= 0 ? fs * inv_divisor(at[0] | ((uint32_t)at[1] << 8), t.rms_mode, ks) : 0.f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < RL; ++i)
          if (8 * i < rdw) put_rms(ir, sc0 + 8 * i, rraw[i]);
        // many heads: the rest of the divisors without a step's head start
        for (int d = sc0 + 8 * RL; d < rdw; d += 8) {
          const int64_t off_put = rowoff[(j & 3) * TT + row];
          put_rms(ir, d, off_put >= 0 ? *reinterpret_cast<const uint32_t*>(p.kv + off_put + 4 * (rd0 + d)) : 0);
        }
      }
    };
    // ---- scores of tile j. One wave a SIMD: nothing but this order hides the LDS, so a slot of one product
    // issues the read KD products ahead, and nothing moves between slots
    auto score = [&](int j, f32x16& s) {
      const uint32_t src = (uint32_t)(uintptr_t)(kt + (j % C::STAGES) * C::TILE_B) + klane + (kc0 << 4);
      typedef __attribute__((address_space(3))) const bf16x8 lvec;
      auto read = [&](int f) { return *(lvec*)(uintptr_t)((src ^ (((2 * f) & GM) << 4)) + (((2 * f) & ~GM) << 4)); };
      bf16x8 k[KD], q[C::QL > 0 ? C::QL : 1];
      const uint32_t qsrc = (uint32_t)(uintptr_t)QMLA_LDS(char, qlw);
#pragma unroll
      for (int f = 0; f < KD; ++f) k[f] = read(f);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int f = 0; f < C::NQ; ++f) {
        const bf16x8 a = k[f % KD];
        if (f + KD < C::NQ) k[f % KD] = read(f + KD);
        if (f == 0) mfma32_v0(s, a, qf[f]);
        else if (f < C::NQ - C::QL) mfma32_v(s, a, qf[f]);
        else mfma32_v(s, a, q[f - (C::NQ - C::QL)]);
        constexpr int Q0 = C::NQ - C::QL - KD;   // the queries in LDS as far ahead
        if (f >= Q0 && f < Q0 + C::QL) q[f - Q0] = *(lvec*)(uintptr_t)(qsrc + (f - Q0) * 1024);
        __builtin_amdgcn_sched_barrier(0);
      }
      mfma_v_done(s);
    };
    auto value_read = [&](uint32_t src, int i) {   // fragment i: columns 32 (i / 2) .., tokens 16 (i % 2) ..
      typedef short i16x8 __attribute__((ext_vector_type(8)));
      i16x4 v[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int c = (C::NS > 1 ? vc0 : 0) + 4 * (i >> 1);
        const uint32_t at = ((src + vlane[2 * (i & 1) + x]) ^ ((c & GM) << 4)) + ((c & ~GM) << 4);
        v[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(uintptr_t)at);
      }
      const i16x8 va = {v[0][0], v[0][1], v[0][2], v[0][3], v[1][0], v[1][1], v[1][2], v[1][3]};
      return __builtin_bit_cast(bf16x8, va);
    };
    // values of tile j against P, `beside(i)` in the slot of product i
    auto values = [&](int j, const bf16x8 (&pf)[2], auto&& beside) {
      const uint32_t src = (uint32_t)(uintptr_t)(kt + (j % C::STAGES) * C::TILE_B);
      bf16x8 v[VD];
#pragma unroll
      for (int i = 0; i < VD; ++i) v[i] = value_read(src, i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 2 * C::OB; ++i) {
        const bf16x8 a = v[i % VD];
        if (i + VD < 2 * C::OB) v[i % VD] = value_read(src, i + VD);
        acc[i >> 1] = mfma32(a, pf[i & 1], acc[i >> 1]);
        beside(i);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    __syncthreads();   // the last piece's tiles are read
    if (tid < 4) odd[tid] = 0;
    // (rows past the piece's end but inside the request are looked up and not fetched)
#pragma unroll
    for (int x = 0; x < 3; ++x) {
      page_of(ta + x);
      rows_of(ta + x);
    }
    page_of(ta + 3);
    __syncthreads();
    fetch(ta);
    put(ta);
    if (ta + 1 < te) fetch(ta + 1);

    // step j: tile j's scores and softmax beside tile j-1's values (three stages), or before its own; tile
    // j+1 goes into LDS, j+2's loads start. A wave without rows stages only.
    constexpr bool PIPE = C::STAGES >= 3;
    bf16x8 pf[2] = {};
    for (int j = ta; j < te; ++j) {
      __syncthreads();
      in_agprs(acc);
      odd[(j + 2) & 3] = 0;
      if constexpr (C::STAGES > 1) {
        if (j + 1 < te) put(j + 1);
      }
      rows_of(j + 3);
      page_of(j + 4);
      if constexpr (C::STAGES > 1) {
        if (j + 2 < te) fetch(j + 2);
      }
      f32x16 s{};
      if (__builtin_expect(wlive, 1)) score(j, s);
      if constexpr (C::NS > 1) {
        if (__builtin_expect(wlive, 1)) {
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4)
            *reinterpret_cast<f32x4*>(part + ((wave * 4 + i4) * 64 + lane) * 16) =
                f32x4{s[4 * i4], s[4 * i4 + 1], s[4 * i4 + 2], s[4 * i4 + 3]};
        }
        __syncthreads();
        if (__builtin_expect(wlive, 1)) {
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            f32x4 sum = *reinterpret_cast<const f32x4*>(part + ((rg * C::NS * 4 + i4) * 64 + lane) * 16);
#pragma unroll
            for (int x = 1; x < C::NS; ++x) sum += *reinterpret_cast<const f32x4*>(part + (((rg * C::NS + x) * 4 + i4) * 64 + lane) * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * i4 + i] = sum[i];
          }
        }
      }
      if (__builtin_expect(wlive, 1)) {
        finish_scores(t, s, irms + (j % C::STAGES) * p.heads * IRS + irms_at);
        if (__builtin_expect((j + 1) * TT > base, 0)) mask_scores(t, s, j, b, base, nodes, m * C::ROWS + rg * 32, own(), odd[j & 3]);
        bf16x8 pn[2];
        if constexpr (PIPE) {
          // (a piece's first step has no tile before it: zeros against its own)
          static_assert(2 * C::OB >= NSOFT || 2 * C::OB == 16);
          constexpr int PER = 2 * C::OB >= NSOFT ? 1 : 2;   // softmax steps a slot
          values(j > ta ? j - 1 : j, pf, [&](int i) {
#pragma unroll
            for (int x = 0; x < PER; ++x) soft_step(PER * i + x, s, pn, sf, m_ref);
          });
          rescale(sf, m_ref, l_sum, l_p, acc);
          pf[0] = pn[0];
          pf[1] = pn[1];
        } else {
#pragma unroll
          for (int i = 0; i < NSOFT; ++i) soft_step(i, s, pn, sf, m_ref);
          rescale(sf, m_ref, l_sum, l_p, acc);
          values(j, pn, [](int) {});
        }
      }
      if constexpr (C::STAGES == 1) {
        __syncthreads();
        if (j + 1 < te) put(j + 1);
        if (j + 2 < te) fetch(j + 2);
      }
    }
    if (PIPE && wlive) values(te - 1, pf, [](int) {});

    store_piece<C>(t, Piece{b, m, nodes, rg, cp, 2 * rng.w + (u > rng.lo ? 1 : 0), ta == 0 && te == nt}, own(), ks, m_ref, l_sum, l_p, acc);
    u += te - ta;
  }
  report_pages(p, bad);
}

// ---- FP8 rows as they are --------------------------------------------------------------------------------
// The tiles stay in LDS as the cache holds them, and a wave converts what it multiplies, beside the products. Staged
// to bf16 (tree_kernel) they cost each workgroup the conversion before its first product of a step, and the LDS
// twice the bytes: transposed 16-bit reads run at half the LDS rate, 8-bit ones bring 8 tokens of a column in the
// same time (16 requests of 64 nodes, 2048 .. 8192 tokens: 533 us staged, 337 us so). The rows arrive by LDS-DMA, A tiles ahead, which holds no registers.
// Scores on the FP8 products (the query as two e4m3 parts) would need no conversion, but those sum with less than fp32:
// 1.4e-4 off at scores of 5, 5e-6 of the terms, where the bf16 products give 1e-6.
static_assert(MAXH <= 64);   // divisors: 8 threads a row, 4 heads a thread, twice
template <int DC_, int K_, bool MASKED_, int NS_, int STAGES_, int SR_>
struct Cfg8 {
  static constexpr int DC = DC_, NS = NS_, STAGES = STAGES_;
  static constexpr int SR = SR_;                          // 16-byte chunks of a staged row, odd: 32 rows on distinct banks
  static constexpr bool MASKED = MASKED_;                 // the last blocks hold other columns than keys
  static constexpr int ROWS = 128 / NS;
  static constexpr int NB = 2 * ((DC / 64 + K_ + NS - 1) / NS);   // 32-column score blocks of a wave
  static constexpr int F0 = DC / 32 - (NS - 1) * NB > 0 ? DC / 32 - (NS - 1) * NB : 0;   // from here on columns may not be keys
  static constexpr int OB = DC / NS / 32;
  static constexpr int RSTRIDE = SR * 16, TILE_B = TT * RSTRIDE;
  static constexpr int CHUNKS = TT * SR, DI = (CHUNKS + NT - 1) / NT;   // DMA instructions of a wave for a tile
  static constexpr int A = STAGES > 2 ? STAGES - 2 : 1;   // tiles ahead
  static constexpr bool PIPE = STAGES > 2;
  static constexpr int IRB = PIPE ? 2 : 1;                // tiles of divisors held
  static constexpr int NX = PIPE ? 6 : 2;                 // steps of the work beside the value products
  static constexpr int PITCH = (2 * NB - 2) / DI;         // score products from one DMA to the next
  static constexpr int ROPE_MAX = 64 * K_;
  static_assert(PITCH * (DI - 1) + 2 < 2 * NB);
  static_assert(SR % 2 == 1 && DC % (32 * NS) == 0);
  static constexpr int out_col(int ob, int i4) { return 32 * ob + 8 * i4; }
};
#define QMLA_IN __attribute__((always_inline))   // (calls on unlikely paths are not inlined by themselves)
constexpr int PIDN = 256;   // page ids of a piece held at once
// f(0) .. f(N - 1) with constants: what is laid out by slots must not wait for the unroller
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<N, I + 1>(f);
  }
}
constexpr int KB = 4, VB = 6;   // score blocks, value fragments read ahead

__host__ __device__ constexpr int heads4(int heads) { return (heads + 3) & ~3; }
template <class C>
__host__ __device__ constexpr int lds_bytes8(int heads) {
  return C::STAGES * C::TILE_B + (C::IRB * heads4(heads) + 4) * IRS * 4 + (C::NS > 1 ? 4 * 4096 : 0) + 8 * TT * 8 + PIDN * 4 + 16 + 1024;
}

// 16 bytes a lane of `lanes`, or of none where left <= 0, from memory to LDS at base + 16 lane, unseen by the
// compiler, whose waits for its own loads and LDS reads would drain it: counted by wait_vmcnt below. Called by whole
// waves; the lanes are masked here, as a branch around the load costs more than it (a taken one about 115 cycles of a
// lone wave)
__device__ __forceinline__ void dma_row(const char* src, uint32_t base, uint64_t lanes, int left) {
  asm volatile("s_mov_b32 m0, %1\n\ts_cmp_gt_i32 %3, 0\n\ts_cselect_b64 exec, %2, 0\n\tglobal_load_lds_dwordx4 %0, off\n\ts_mov_b64 exec, -1"
               ::"v"(src), "s"(__builtin_amdgcn_readfirstlane((int)base)), "s"(lanes), "s"(__builtin_amdgcn_readfirstlane(left))
               : "memory", "scc");
}

template <class C>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(1, 1))) void tree8_kernel(const TrParams t) {
  extern __shared__ __align__(16) char lds[];
  typedef __attribute__((address_space(3))) char lchar;
  const KParams& p = t.k;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int rg = wave / C::NS, cp = wave % C::NS;
  const uint32_t kt = (uint32_t)(uintptr_t)QMLA_LDS(char, lds);
  const int h4 = heads4(p.heads);
  float* irms = reinterpret_cast<float*>(lds + C::STAGES * C::TILE_B);   // [IRB][h4][IRS], [4][IRS] for heads past the last
  char* part = lds + C::STAGES * C::TILE_B + (C::IRB * h4 + 4) * IRS * 4; // [4 waves][4][64] 16 bytes
  const char** rowoff = reinterpret_cast<const char**>(part + (C::NS > 1 ? 4 * 4096 : 0));   // [8][TT] where rows lie
  int* pids = reinterpret_cast<int*>(rowoff + 8 * TT);                   // [PIDN]
  uint32_t* odd = reinterpret_cast<uint32_t*>(pids + PIDN);              // [4], bit per token
  float* codes = reinterpret_cast<float*>(odd + 4);                      // [256] what a one-byte divisor multiplies by
  const Range rng = unit_range(t);
  if (rng.lo >= rng.hi) return;
  const float ks = p.k_scale ? *p.k_scale : 1.f;
  const float fs = p.sm_scale * ks * (p.logit_cap > 0.f ? 1.f : kLog2e);
  const int rows_b = (p.rms_off_b + (t.rms_mode == QMLA_RMS_NONE ? 0 : p.heads * t.rms_b) > t.cols
                          ? p.rms_off_b + p.heads * t.rms_b : t.cols);   // bytes of a row that are used
  codes[tid] = fs * inv_divisor(tid, t.rms_mode, ks);
  const int last_n = C::CHUNKS - ((C::DI - 1) * 4 + wave) * 64;         // lanes of this wave's last DMA of a tile
  const uint64_t last_lanes = last_n <= 0 ? 0 : last_n >= 64 ? ~0ull : (1ull << last_n) - 1;
  auto own = [&]() QMLA_IN {
    int x = tid;
    asm volatile("" : "+v"(x));
    return x;
  };
  // chunk `lane` of this wave's DMA i: its row in the tile, and the chunks before it in the row (what lies behind the
  // used bytes: the row's first), 8 bits each, two DMAs a register
  uint32_t place[(C::DI + 1) / 2] = {};
#pragma unroll
  for (int i = 0; i < C::DI; ++i) {
    const int id = (i * 4 + wave) * 64 + lane, row = id / C::SR, c = id - row * C::SR;
    place[i / 2] |= ((row < TT ? row : TT - 1) << 8 | (16 * c < rows_b ? c : 0)) << (16 * (i & 1));
  }
  int64_t u = rng.lo, c0 = rng.c0;
  int b = rng.b;
  while (u < rng.hi) {
    const int nt = tiles_of(t, b);
    if (u >= c0 + (int64_t)nt * t.rt) {
      c0 += (int64_t)nt * t.rt;
      ++b;
      continue;
    }
    const int m = (int)((u - c0) / nt), ta = (int)((u - c0) - (int64_t)m * nt);
    const int te = rng.hi - u < nt - ta ? ta + (int)(rng.hi - u) : nt;
    const int L = p.seq_lens[b], nodes = node_count(t, b), base = L - nodes;
    const int r0 = m * C::ROWS + rg * 32;
    const bool wlive = r0 < t.rows;

    // ---- staging
    // page ids [pw, pw + PIDN) of the request in LDS, checked; refilled when a tile's last page lies behind them
    int pw = 0;
    const int npg = page_div(p, L - 1) + 1;
    auto fill_pages = [&]() QMLA_IN {
      const int x = pw + own();
      if (x < npg) {
        int bad = 0;
        pids[x - pw] = checked_page(p, p.bt[b * p.bt_stride + x], bad);
        report_pages(p, bad);
      }
    };
    int lim = 0;   // tokens whose pages are there
    auto refill = [&](int j) QMLA_IN {   // new page ids where tile j needs them (the same for all threads)
      const int last = (j + 1) * TT < L ? (j + 1) * TT : L;
      if (__builtin_expect(j * TT >= L || last <= lim, 1)) return;
      lds_barrier();
      pw = page_div(p, j * TT);
      const int64_t e = (int64_t)(pw + PIDN) * p.page_size;
      lim = e < L ? (int)e : L;
      fill_pages();
      __syncthreads();
    };
    // where tile j's rows lie (rows past the request: its last), 8 threads a row, in two steps
    auto row_token = [&](int j) {
      const int tok = j * TT + (own() & 31);
      return tok < L ? tok : L - 1;
    };
    auto row_page = [&](int j) { return pids[page_div(p, row_token(j)) - pw]; };
    auto row_put = [&](int j, int id) {
      const uint32_t tok = row_token(j), in = tok - page_div(p, tok) * p.page_size;
      rowoff[(j & 7) * TT + (own() & 31)] = p.kv + ((uint64_t)(uint32_t)id * (uint64_t)p.page_stride_b + (uint64_t)in * (uint32_t)p.token_stride_b);
    };
    // this wave's DMA instruction i of tile j: where its row lies, itself
    const char* nx[C::DI];
    auto placed = [&](int i) {   // (opaque: unpacked ahead of the loop they would take 3 registers a DMA)
      uint32_t x = place[i / 2];
      asm volatile("" : "+v"(x));
      return x >> (16 * (i & 1));
    };
    auto dma_row_of = [&](int j, int i) { nx[i] = rowoff[(j & 7) * TT + (placed(i) >> 8 & 255)]; };
    auto dma = [&](int j, int i) {   // (none from tile te on)
      dma_row(nx[i] + 16 * (placed(i) & 255), kt + (j % C::STAGES) * C::TILE_B + (i * 4 + wave) * 1024, i + 1 < C::DI ? ~0ull : last_lanes, te - j);
    };
    // the DMA of the tiles up to all but the last N issued has landed (DMAs without lanes may not count: waited as if
    // every wave had one less a tile)
    auto wait_left = [&](auto left) { wait_vmcnt<decltype(left)::value * (C::DI - (C::CHUNKS % 256 != 0 ? 1 : 0))>(); };
    // tile j's divisors, 8 threads a row, 4 heads a thread (those of 32 i ..), in two steps
    typedef __attribute__((address_space(3))) const uint64_t lu64_b __attribute__((aligned(1)));
    auto div_read = [&](int j, int i) QMLA_IN -> uint64_t {   // (one-byte codes: the lower half)
      return *(lu64_b*)(uintptr_t)(kt + (j % C::STAGES) * C::TILE_B + (own() >> 3) * C::RSTRIDE + p.rms_off_b +
                                   ((own() & 7) + 8 * i) * 4 * t.rms_b);
    };
    auto div_put = [&](int j, int i, uint64_t v) QMLA_IN {
      const int hd = 4 * (own() & 7) + 32 * i;
      float* ir = irms + (hd < h4 ? (j % C::IRB) * h4 + hd : C::IRB * h4) * IRS + (own() >> 3);
      if (__builtin_expect(t.rms_b == 2, 0)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float r = __uint_as_float((uint32_t)(v >> (16 * e)) << 16);
          ir[e * IRS] = r > 0.f ? fs * __builtin_amdgcn_rcpf(r) : fs;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) ir[e * IRS] = codes[(uint32_t)v >> (8 * e) & 255];
      }
    };
    auto divisors = [&](int j) QMLA_IN {
      div_put(j, 0, div_read(j, 0));
      if (__builtin_expect(p.heads > 32, 0)) div_put(j, 1, div_read(j, 1));
    };
    // the work of step j that lies beside its value products, in steps 0 .. NX - 1: rows of tile j + A + 1, divisors of
    // tile j + 1
    int xp = 0;
    uint64_t xd[2] = {};
    auto extra = [&](int j, auto ic) {
      constexpr int i = decltype(ic)::value;
      if constexpr (i == 0) xp = row_page(j + C::A + 1);
      else if constexpr (i == 1) row_put(j + C::A + 1, xp);
      else if constexpr (i == 2) xd[0] = div_read(j + 1, 0);
      else if constexpr (i == 3) {
        if (__builtin_expect(p.heads > 32, 0)) xd[1] = div_read(j + 1, 1);
      } else if constexpr (i == 4) div_put(j + 1, 0, xd[0]);
      else if (__builtin_expect(p.heads > 32, 0)) div_put(j + 1, 1, xd[1]);
    };
    auto extras = [&](int j, auto slot) {
      constexpr int S = 2 * C::OB, X0 = decltype(slot)::value * C::NX / S, X1 = (decltype(slot)::value + 1) * C::NX / S;
      each<X1 - X0>([&](auto i) { extra(j, std::integral_constant<int, X0 + decltype(i)::value>{}); });
    };
    // what the drafted tokens hold that is not finite, and rows past the request, become zeros, the former flagged
    // in `odd`
    auto mend = [&](int j) QMLA_IN {
      const int me = own(), row = me >> 3, tok = j * TT + row;
      char* src = lds + (j % C::STAGES) * C::TILE_B + row * C::RSTRIDE;
      if (tok < base) return;
      bool any = false;
#pragma unroll
      for (int i = 0; i < (C::DC + C::ROPE_MAX + 127) / 128; ++i) {
        const int c = (me & 7) + 8 * i;
        if (16 * c >= t.cols) continue;
        i32x4 v = *reinterpret_cast<const i32x4*>(src + 16 * c), keys = v;
        const int left = t.cols - 16 * c;   // columns that are keys
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int bits = 8 * left - 32 * d;
          const int mask = bits <= 0 ? 0 : bits >= 32 ? -1 : (int)((1u << (bits & 31)) - 1);
          keys[d] = v[d] & mask;
          v[d] &= ~mask;
        }
        const bool o = any_odd<true>(keys);
        any = any || o;
        if (o || tok >= L) *reinterpret_cast<i32x4*>(src + 16 * c) = v;
      }
      if (any && tok < L) atomicOr(&odd[j & 3], 1u << row);
    };

    lds_barrier();   // the last piece's tiles are read
    if (tid < 4) odd[tid] = 0;
#pragma unroll 1
    for (int x = 0; x <= C::A; ++x) {
      refill(ta + x);
      row_put(ta + x, row_page(ta + x));
    }
    lds_barrier();
#pragma unroll 1
    for (int x = 0; x < C::A; ++x)
      if (ta + x < te) {
#pragma unroll
        for (int i = 0; i < C::DI; ++i) {
          dma_row_of(ta + x, i);
          dma(ta + x, i);
        }
      }

    // ---- this lane's query row
    bf16x8 qf[2 * C::NB];       // products 2 f and 2 f + 1: columns 32 f + 16 h + 0..7 and + 8..15
    int irms_at;                // this row's head in the divisors
    {
      // rows may be aligned to their elements only
      typedef bf16x8 bf16x8_e __attribute__((aligned(2)));
      const int r = r0 + n < t.rows ? r0 + n : t.rows - 1, node = r / p.heads, head = r - node * p.heads;
      irms_at = head * IRS + 4 * h;
      const int64_t row = (int64_t)b * p.qrows + node;
      const __bf16* qn = p.q_nope + row * p.qn_sr + head * p.qn_sh;
      const __bf16* qp = p.q_pe + row * p.qp_sr + head * p.qp_sh;
      const int whole8 = p.rope_w & ~7;
      bf16x8 tail{};
      for (int i = 0; i < (p.rope_w & 7); ++i) {
        const __bf16 x = qp[whole8 + i];
#pragma unroll
        for (int e = 0; e < 8; ++e) tail[e] = e == i ? x : tail[e];
      }
#pragma unroll
      for (int f = 0; f < 2 * C::NB; ++f) {
        // dead rows keep what they read: their columns of the products go nowhere
        const int c = cp * C::NB * 32 + 32 * (f >> 1) + 16 * h + 8 * (f & 1), o = c - C::DC;
        if (C::NS == 1 && 16 * f < C::DC) {
          qf[f] = *reinterpret_cast<const bf16x8_e*>(qn + c);
        } else {
          bf16x8 v = tail;
          if (o < 0) v = *reinterpret_cast<const bf16x8_e*>(qn + c);
          else if (o < whole8) v = *reinterpret_cast<const bf16x8_e*>(qp + o);
          i32x4 x = __builtin_bit_cast(i32x4, v);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = o <= whole8 ? x[e] : 0;
          qf[f] = __builtin_bit_cast(bf16x8, x);
        }
      }
    }
    f32x16 acc[C::OB];
#pragma unroll
    for (int i = 0; i < C::OB; ++i) acc[i] = f32x16{};
    float m_ref = kNegInf, l_sum = 0.f, l_p = 0.f;
    Soft sf;

    // ---- scores of tile j, `beside(slot)` in the slots of its 2 NB products; one wave a SIMD: nothing but this
    // order hides the LDS. A block's keys are converted in the slots of the block before
    auto score = [&](int j, f32x16& s, auto&& beside) {
      // 16 bytes of row n from column 32 block + 16 h
      const int me = own();
      const uint32_t src = kt + (j % C::STAGES) * C::TILE_B + (me & 31) * C::RSTRIDE + ((me & 32) >> 1) + cp * C::NB * 32;
      typedef __attribute__((address_space(3))) const i32x4 lvec;
      auto read = [&](int f) { return *(lvec*)(uintptr_t)(src + 32 * f); };
      auto keys = [&](i32x4 x, int f) {   // bytes past the row's keys go
        if (C::MASKED && f >= C::F0) {
          const int left = t.cols - (cp * C::NB + f) * 32 - ((me & 32) >> 1);
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const int bits = 8 * left - 32 * d;
            x[d] = bits <= 0 ? 0 : bits >= 32 ? x[d] : x[d] & (int)((1u << (bits & 31)) - 1);
          }
        }
        return x;
      };
      i32x4 k[KB];
#pragma unroll
      for (int f = 0; f < KB; ++f) k[f] = read(f);
      __builtin_amdgcn_sched_barrier(0);
      bf16x8 lo, hi;
      fp8x16_to_bf16(keys(k[0], 0), lo, hi);
      __builtin_amdgcn_sched_barrier(0);
      each<C::NB>([&](auto fc) {
        constexpr int f = decltype(fc)::value;
        if constexpr (f + KB < C::NB) k[f % KB] = read(f + KB);
        if constexpr (f == 0) mfma32_v0(s, lo, qf[0]);
        else mfma32_v(s, lo, qf[2 * f]);
        i32x4 x{};
        bf16x8 next;
        if constexpr (f + 1 < C::NB) {
          x = keys(k[(f + 1) % KB], f + 1);
          next = fp8x8_to_bf16(i32x2{x[0], x[1]});
        }
        beside(2 * f);
        __builtin_amdgcn_sched_barrier(0);
        mfma32_v(s, hi, qf[2 * f + 1]);
        if constexpr (f + 1 < C::NB) {
          lo = next;
          hi = fp8x8_to_bf16(i32x2{x[2], x[3]});
        }
        beside(2 * f + 1);
        __builtin_amdgcn_sched_barrier(0);
      });
      mfma_v_done(s);
    };
    // values of tile j against P, `beside(i)` in the slot of product i: columns 32 (i / 2) .., tokens 16 (i % 2) ..
    auto values = [&](int j, const bf16x8 (&pf)[2], auto&& beside) {
      // 8 bytes of tokens 16 k2 + 4 h + {0..3, 8..11}, columns 32 ob + 16 (lane / 16 % 2) + 8 (lane % 2). (Some of these
      // reads meet on banks; columns 64 apart meet on a third as many, in the same time.)
      const int me = own(), q = (me & 15) >> 1;
      const uint32_t src = kt + (j % C::STAGES) * C::TILE_B + ((q < 4 ? q : q + 4) + ((me & 32) >> 3)) * C::RSTRIDE + (me & 16) +
                           8 * (me & 1) + cp * (C::DC / C::NS);
      auto read = [&](int i) {
        return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(uintptr_t)(src + 32 * (i >> 1) + 16 * (i & 1) * C::RSTRIDE));
      };
      i32x2 v[VB];
#pragma unroll
      for (int i = 0; i < VB; ++i) v[i] = read(i);
      __builtin_amdgcn_sched_barrier(0);
      bf16x8 a[2] = {fp8x8_to_bf16(v[0]), fp8x8_to_bf16(v[1])};   // two ahead: a product waits for an operand just written
      __builtin_amdgcn_sched_barrier(0);
      in_agprs(acc);
      each<2 * C::OB>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        acc[i >> 1] = mfma32(a[i & 1], pf[i & 1], acc[i >> 1]);
        if constexpr (i + VB < 2 * C::OB) v[i % VB] = read(i + VB);
        if constexpr (i + 2 < 2 * C::OB) a[i & 1] = fp8x8_to_bf16(v[(i + 2) % VB]);
        beside(ic);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    // tiles ta and (their divisors a step ahead) ta + 1 are there before step ta
    if constexpr (C::PIPE) {
      if (ta + C::A <= te) wait_left(std::integral_constant<int, C::A - 2>{});
      else wait_vmcnt<0>();
    } else {
      if (ta + C::A <= te) wait_left(std::integral_constant<int, C::A - 1>{});
      else wait_vmcnt<0>();
    }
    lds_barrier();
    if constexpr (C::PIPE) divisors(ta);

    bf16x8 pf[2] = {};
    for (int j = ta; j < te; ++j) {
      lds_barrier();
      in_agprs(acc);
      odd[(j + 2) & 3] = 0;   // (all threads: a branch costs more)
      if constexpr (!C::PIPE) divisors(j);
      if (__builtin_expect((j + 1) * TT > base, 0)) {
        if constexpr (!C::PIPE) lds_barrier();   // the divisors lie in chunks that mend() may write
        mend(j);
        lds_barrier();
      }
      refill(j + C::A + 1);
      f32x16 s{};
      const bool more = j + C::A < te;
      auto stage = [&](int slot) {   // a tile's DMA, its rows two slots ahead
        if (slot % C::PITCH == 0 && slot / C::PITCH < C::DI) dma_row_of(j + C::A, slot / C::PITCH);
        if (slot >= 2 && (slot - 2) % C::PITCH == 0 && (slot - 2) / C::PITCH < C::DI) dma(j + C::A, (slot - 2) / C::PITCH);
      };
      auto finish = [&]() {   // scores to P, and the values
        finish_scores(t, s, irms + (j % C::IRB) * h4 * IRS + irms_at);
        if (__builtin_expect((j + 1) * TT > base, 0)) mask_scores(t, s, j, b, base, nodes, r0, own(), odd[j & 3]);
        bf16x8 pn[2];
        if constexpr (C::PIPE) {
          // (a piece's first step has no tile before it: zeros against its own)
          constexpr int PER = 2 * C::OB >= NSOFT ? 1 : 2;   // softmax steps a slot
          static_assert(2 * C::OB * PER >= NSOFT);
          values(j > ta ? j - 1 : j, pf, [&](auto i) {
#pragma unroll
            for (int x = 0; x < PER; ++x) soft_step(PER * i + x, s, pn, sf, m_ref);
            extras(j, i);
          });
          rescale(sf, m_ref, l_sum, l_p, acc);
          pf[0] = pn[0];
          pf[1] = pn[1];
        } else {
#pragma unroll
          for (int i = 0; i < NSOFT; ++i) soft_step(i, s, pn, sf, m_ref);
          rescale(sf, m_ref, l_sum, l_p, acc);
          values(j, pn, [&](auto i) { extras(j, i); });
        }
      };
      auto idle_dma = [&]() {   // a wave without rows
#pragma unroll
        for (int i = 0; i < C::DI; ++i) {
          dma_row_of(j + C::A, i);
          dma(j + C::A, i);
        }
      };
      auto idle_work = [&]() { each<C::NX>([&](auto i) { extra(j, i); }); };
      if constexpr (C::NS == 1) {
        if (__builtin_expect(wlive, 1)) {
          score(j, s, stage);
          finish();
        } else {
          idle_dma();
          idle_work();
        }
      } else {
        if (__builtin_expect(wlive, 1)) {
          score(j, s, stage);
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4)
            *reinterpret_cast<f32x4*>(part + ((wave * 4 + i4) * 64 + lane) * 16) =
                f32x4{s[4 * i4], s[4 * i4 + 1], s[4 * i4 + 2], s[4 * i4 + 3]};
        } else {
          idle_dma();
        }
        lds_barrier();
        if (__builtin_expect(wlive, 1)) {
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            f32x4 sum = *reinterpret_cast<const f32x4*>(part + ((rg * C::NS * 4 + i4) * 64 + lane) * 16);
#pragma unroll
            for (int x = 1; x < C::NS; ++x) sum += *reinterpret_cast<const f32x4*>(part + (((rg * C::NS + x) * 4 + i4) * 64 + lane) * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * i4 + i] = sum[i];
          }
          finish();
        } else {
          idle_work();
        }
      }
      // the next step's tile (and, a step ahead for its divisors, the one behind it) has landed
      if constexpr (C::PIPE) {
        if (__builtin_expect(more, 1)) wait_left(std::integral_constant<int, C::A - 2>{});
        else wait_vmcnt<0>();
      } else {
        if (__builtin_expect(more, 1)) wait_left(std::integral_constant<int, C::A - 1>{});
        else wait_vmcnt<0>();
      }
    }
    if (C::PIPE && wlive) values(te - 1, pf, [](auto) {});
    store_piece<C>(t, Piece{b, m, nodes, rg, cp, 2 * rng.w + (u > rng.lo ? 1 : 0), ta == 0 && te == nt}, own(), ks, m_ref, l_sum, l_p, acc);
    u += te - ta;
  }
}

// Rows whose tokens several workgroups shared, and rows of requests without tokens. A wave joins one block of 32 rows,
// as the accumulators lay: whole 1 KB reads, those of 4 shares under way together (a wave a row, share after share:
// 16 us for 192 rows of 21 shares, 31 us for 1536 rows of 18).
template <class C>
__global__ __launch_bounds__(256) void tree_combine_kernel(const TrParams t) {
  const KParams& p = t.k;
  const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
  const int v = blockIdx.x * 4 + (threadIdx.x >> 6), wave = v / C::OB, ob = v - wave * C::OB, m = blockIdx.y, b = blockIdx.z;
  const int rg = wave / C::NS, cp = wave - rg * C::NS, r = m * C::ROWS + rg * 32 + n;
  if (r >= t.rows) return;
  const int node = r / p.heads, head = r - node * p.heads;
  const int64_t row = (int64_t)b * p.qrows + node;
  const int nt = tiles_of(t, b);
  f32x16 acc{};
  float sum = 0.f, top = kNegInf;
  if (nt > 0) {
    const int64_t chunk = t.plan[0];
    int64_t slot;
    int k, odd;   // shares; the first lies in its workgroup's second slot
    if (chunk < 0) {
      k = (nt - (int)chunk - 1) / -(int)chunk;
      slot = 2 * (t.plan[1 + b] * t.rt + (int64_t)m * k);
      odd = 0;
    } else {
      const int64_t u0 = t.plan[1 + b] * t.rt + (int64_t)m * nt, w0 = u0 / chunk;
      k = (int)((u0 + nt - 1) / chunk - w0) + 1;
      slot = 2 * w0;
      odd = u0 > w0 * chunk ? 1 : 0;
    }
    if (k == 1) return;
    auto at = [&](int i) { return slot + (i < k ? 2 * i + (i == 0 ? odd : 0) : 2 * (k - 1)); };   // (k > 1)
    const float* lse = t.part_lse + rg * 32 + n;
    for (int i = 0; i < k; i += 8) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = lse[at(i + e) * C::ROWS];
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, x[e]);
    }
    const float ref = is_neg_inf(top) ? 0.f : top;
    const f32x4* src = reinterpret_cast<const f32x4*>(t.part_o) + (wave * C::OB + ob) * 256 + lane;
    for (int i = 0; i < k; i += 4) {
      float x[4];
      f32x4 o[4][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = lse[at(i + e) * C::ROWS];
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) o[e][i4] = src[at(i + e) * (4 * C::OB * 256) + i4 * 64];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < k) {
          const float g = fast_exp2(x[e] - ref);   // NaN stays NaN
          sum += g;
#pragma unroll
          for (int c = 0; c < 16; ++c) acc[c] += o[e][c >> 2][c & 3] * g;
        }
    }
  }
  const float ks = p.k_scale ? *p.k_scale : 1.f;
  const float inv = empty_sum(sum) ? 0.f : ks / sum;
  const int64_t o0 = row * p.o_sr + head * p.o_sh + cp * (C::DC / C::NS) + 4 * h;
  auto put = [&](auto dtc) {
    constexpr int DT = decltype(dtc)::value, ES = DT == QMLA_DT_F32 ? 4 : 2;
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4)
      store_out4<DT>(reinterpret_cast<char*>(p.out) + (o0 + C::out_col(ob, i4)) * ES,
                     f32x4{acc[4 * i4] * inv, acc[4 * i4 + 1] * inv, acc[4 * i4 + 2] * inv, acc[4 * i4 + 3] * inv});
  };
  if (p.out_dt == QMLA_DT_F32) put(std::integral_constant<int, QMLA_DT_F32>{});
  else if (p.out_dt == QMLA_DT_F16) put(std::integral_constant<int, QMLA_DT_F16>{});
  else put(std::integral_constant<int, QMLA_DT_BF16>{});
  if (ob == 0 && cp == 0 && h == 0 && p.lse) store_out(p.lse, p.lse_dt, row * p.lse_sr + head, nt > 0 ? row_lse(top, sum) : kNegInf);
}

struct Inst {
  bool fp8;
  int d_c, rope_max, rows;
  const void* fn;
  const void* combine;
  int combine_wgs;  // of a row tile
  int (*lds)(int heads);
  int row_b;        // bytes of a cached row a kernel that stages them as they are has room for (0: any)
  bool exact;       // rope_w == rope_max only
};

#define QMLA_TR(FP8, DC, CP, NS, ST, QL) \
  {FP8, DC, CP - DC, 128 / NS, (const void*)&tree_kernel<Cfg<FP8, DC, CP, NS, ST, QL>>, \
   (const void*)&tree_combine_kernel<Cfg<FP8, DC, CP, NS, ST, QL>>, DC / NS / 32, [](int heads) { return lds_bytes<Cfg<FP8, DC, CP, NS, ST, QL>>(heads); }, 0, false}
#define QMLA_TR8(DC, K, M, NS, ST, SR) \
  {true, DC, 64 * K, 128 / NS, (const void*)&tree8_kernel<Cfg8<DC, K, M, NS, ST, SR>>, \
   (const void*)&tree_combine_kernel<Cfg8<DC, K, M, NS, ST, SR>>, DC / NS / 32, [](int heads) { return lds_bytes8<Cfg8<DC, K, M, NS, ST, SR>>(heads); }, 16 * SR, !M}
// the first that fits: FP8 rows as they are where their divisors leave them room (24 heads of one byte), staged to bf16
// with more
static const Inst kInst[] = {
    QMLA_TR8(512, 1, false, 1, 6, 39), QMLA_TR8(512, 1, true, 1, 6, 39),
    QMLA_TR8(256, 2, true, 1, 6, 27),  QMLA_TR8(256, 4, true, 1, 6, 35),
    QMLA_TR8(768, 2, true, 2, 4, 59),  QMLA_TR8(768, 4, true, 2, 4, 65),
    QMLA_TR8(1792, 4, true, 4, 2, 131),
    QMLA_TR(true, 512, 576, 1, 3, 4),   QMLA_TR(false, 512, 576, 1, 3, 4),
    QMLA_TR(true, 256, 512, 1, 3, 0),   QMLA_TR(false, 256, 512, 1, 3, 0),
    QMLA_TR(true, 768, 1024, 2, 2, 0),  QMLA_TR(false, 768, 1024, 2, 2, 0),
    QMLA_TR(true, 1792, 2048, 4, 1, 0), QMLA_TR(false, 1792, 2048, 4, 1, 0),
};

static const Inst* find(const qmla_decode_params* p) {
  const int div_b = p->rms_mode == QMLA_RMS_BF16 || p->rms_mode == QMLA_RMS_BF16_BYTES ? 2 : 1;
  const int64_t cols = (int64_t)p->d_c + p->rope_w;
  const int64_t end = p->rms_mode == QMLA_RMS_NONE ? cols : (int64_t)p->rms_offset + (int64_t)p->heads * div_b;
  for (const Inst& i : kInst)
    if (i.fp8 == (p->kv_dtype == QMLA_KV_FP8) && i.d_c == p->d_c && (i.exact ? p->rope_w == i.rope_max : p->rope_w <= i.rope_max) &&
        p->heads <= MAXH && i.lds(p->heads) <= LDS_MAX && (i.row_b == 0 || (end <= i.row_b && cols <= i.row_b)))
      return &i;
  return nullptr;
}

struct Layout {
  size_t lse_off, o_off, total;
  int nwg;
};
static Layout layout(const qmla_decode_params* p, const Inst& in) {
  Layout l;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  l.nwg = p->num_workgroups > 0 ? p->num_workgroups : cu_count();
  const int64_t n_req = p->rows / p->qrows;
  l.lse_off = up((size_t)(1 + n_req) * 8);
  l.o_off = l.lse_off + up((size_t)2 * l.nwg * in.rows * 4);
  l.total = l.o_off + (size_t)2 * l.nwg * in.rows * p->d_c * 4;
  return l;
}

}  // namespace tr
}  // namespace qmla

using namespace qmla;

extern "C" {

size_t qmla_tree_workspace_bytes(const qmla_decode_params* p) {
  if (!p || p->rows <= 0 || p->qrows <= 0 || p->rows % p->qrows) return 0;
  const tr::Inst* in = tr::find(p);
  return in ? tr::layout(p, *in).total : 0;
}

int qmla_tree_forward(const qmla_decode_params* p0, const int64_t* tree_mask, int64_t mask_stride, const int32_t* node_counts,
                      void* stream) {
  if (!p0) return QMLA_ERR_NULL;
  qmla_decode_params p = *p0;
  p.num_splits = 1;
  const int rc = validate_params(&p);
  if (rc) return rc;
  if (p.groups != 1 || p.qrows > 64 || p.num_workgroups < 0) return QMLA_ERR_SHAPE;
  if (!rows16(&p)) return QMLA_ERR_ALIGN;
  const int eb = p.kv_dtype == QMLA_KV_FP8 ? 1 : 2;
  // the last load of a row may reach past its columns, never past its 16-byte multiple
  const int64_t div_b = p.rms_mode == QMLA_RMS_NONE ? 0 : p.rms_mode == QMLA_RMS_BF16 || p.rms_mode == QMLA_RMS_BF16_BYTES ? 2 : 1;
  const int64_t keys_end = (int64_t)(p.d_c + p.rope_w) * eb, div_end = div_b ? (int64_t)p.rms_offset * eb + p.heads * div_b : 0;
  if ((p.page_size > 1 ? p.token_stride : p.page_stride) * eb < ((keys_end > div_end ? keys_end : div_end) + 15) / 16 * 16) return QMLA_ERR_SHAPE;
  const tr::Inst* in = tr::find(&p);
  if (!in) return QMLA_ERR_NOKERNEL;
  if (p.rows == 0) return QMLA_OK;
  if (!tree_mask) return QMLA_ERR_NULL;
  if ((uintptr_t)tree_mask % 8) return QMLA_ERR_ALIGN;
  const int64_t n_req = p.rows / p.qrows;
  if (n_req > 65535) return QMLA_ERR_SHAPE;
  const tr::Layout l = tr::layout(&p, *in);
  if (!p.workspace || p.workspace_bytes < l.total) return QMLA_ERR_WORKSPACE;
  if ((uintptr_t)p.workspace % 16) return QMLA_ERR_ALIGN;
  tr::TrParams t{};
  t.k = make_kparams(&p);
  if (p.rms_mode == QMLA_RMS_NONE) t.k.rms_off_b = 0;   // whatever it was: nothing lies there
  t.mask = tree_mask;
  t.mask_sr = mask_stride;
  t.counts = node_counts;
  t.rows = p.qrows * p.heads;
  t.rt = (t.rows + in->rows - 1) / in->rows;
  t.cols = p.d_c + p.rope_w;
  t.nwg = l.nwg;
  t.min_chunk = 2;
  t.rms_mode = p.rms_mode;
  t.rms_b = p.rms_mode == QMLA_RMS_BF16 || p.rms_mode == QMLA_RMS_BF16_BYTES ? 2 : 1;
  char* ws = reinterpret_cast<char*>(p.workspace);
  t.plan = reinterpret_cast<int64_t*>(ws);
  t.part_lse = reinterpret_cast<float*>(ws + l.lse_off);
  t.part_o = reinterpret_cast<float*>(ws + l.o_off);
  const int bytes = in->lds(p.heads);
  if (hipFuncSetAttribute(in->fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return QMLA_ERR_LAUNCH;
  void* args[] = {&t};
  if (hipLaunchKernel(in->fn, dim3(t.nwg), dim3(tr::NT), args, bytes, (hipStream_t)stream) != hipSuccess) return QMLA_ERR_LAUNCH;
  const hipError_t e = hipLaunchKernel(in->combine, dim3(in->combine_wgs, t.rt, (unsigned)n_req), dim3(256), args, 0, (hipStream_t)stream);
  return e == hipSuccess ? QMLA_OK : QMLA_ERR_LAUNCH;
}

}  // extern "C"
