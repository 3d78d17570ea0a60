// Attention weight of every cached token (qmla_attention_weights): a second pass over the keys that sums
// exp(s - lse) over a request's query rows and heads. See include/qmla.h.
//
// S = Q K^T in 16x16 blocks of v_mfma_f32_16x16x32_bf16 with the queries as A, so a lane holds one token's
// scores of 4 rows a block and the sum over rows stays in the lane (and its partners 16, 32 and 48 lanes away). A
// lane loads its token's row straight from memory, 16 bytes a load, the 4 lane groups beside each other: the
// contraction's order is free as long as both operands share it, so lane group g takes columns 16g.. of each 64
// FP8 columns (two products) or 8g.. of each 32 bf16 ones (one), and no key passes through LDS. A group of 9
// loads is in flight at once (a row of 576 FP8 columns): in 32x32 blocks with 6 loads of 32 bytes a row the lines
// left the L1 before their second half was asked for, 64 FP8 requests 96 us. The queries wait in LDS in the order
// of the products, a 1 KB read a product. FP8 keys become bf16 exactly, so scores are exact products summed in
// fp32: the query as e4m3 parts (the decode's scores) would be 5e-6 of the terms off, too much for a
// fp32 result. 64 FP8 requests of 4096 .. 16384 tokens: 83 us, 4.0 TB/s of their 329 MB; few tokens are bound by the
// queries' way into LDS (9 bf16 requests of 96 rows: 27 us).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmla.h"
#include "qmla_common.h"

namespace qmla {
namespace wt {

constexpr int U = 9;             // loads of a group
constexpr int QB = 7;            // query loads of a lane under way together
constexpr int MAXRB = 8;         // row blocks of 16 held at once
constexpr int LDS_MAX = 160 * 1024;

struct WtParams {
  KParams k;
  const float* lse;
  int64_t lse_sr;
  const float* win;
  int64_t win_s;
  float* out;
  int64_t out_s;
  int width;
  int rows;        // query rows of a request (qrows * heads)
  int cols;        // d_c + rope_w
  int d_c, dcg;
  int steps;       // 16-byte loads of a lane for one token, and how many of them hold keys only
  int whole;
  int passes;      // passes over the tokens, NRB row blocks each
  int rms_mode, rms_b;   // divisor bytes of a head
  int rms4;        // 4 heads' divisors load at once
};

// queries may be aligned to their elements only
typedef bf16x8 bf16x8_e __attribute__((aligned(2)));

__device__ __forceinline__ float inv_divisor(uint32_t raw, int mode, float ks) {
  const float r = mode == QMLA_RMS_E4M3 ? fp8_to_f32(raw) * ks : bf16_bits_to_f32(raw);
  return r > 0.f ? __builtin_amdgcn_rcpf(r) : 1.f;   // within 1 ulp
}

// a query row: where it lies, and its head's latent group
struct RowAt {
  const __bf16 *qn, *qp;
};
// where the 8 columns from c0 of a query row lie
struct QueryAt {
  const __bf16* src;
  int o, q;          // the first column's place in the latent part and in the rotary one
  bool whole, part;  // all 8 in one of them; some
};
__device__ __forceinline__ QueryAt query_at(const WtParams& w, const RowAt& row, int group, int c0) {
  QueryAt a;
  a.o = c0 - group * w.dcg;
  a.q = c0 - w.d_c;
  const bool live = group >= 0, latent = a.o >= 0 && a.o + 8 <= w.dcg, rope = !latent && a.q >= 0 && a.q + 8 <= w.k.rope_w;
  a.src = !live ? reinterpret_cast<const __bf16*>(w.k.kv) : latent ? row.qn + a.o : rope ? row.qp + a.q : reinterpret_cast<const __bf16*>(w.k.kv);
  a.whole = live && (latent || rope);
  a.part = live && !latent && !rope && a.o + 8 > 0 && c0 < w.cols && (a.o < w.dcg || a.q + 8 > 0);
  return a;
}

// A workgroup's tokens, in units of T (its waves' tiles): each request's split evenly over workgroups of their own, if
// that takes at most one unit more than an even split of all, which it falls back to. With tokens of two requests
// a workgroup loads and lays out queries twice, as long as one or two units take (9 requests of 96 rows, 500 .. 12000
// tokens: 35 us, 29 us so).
template <int T, class F>
__device__ __forceinline__ void for_each_piece(const KParams& p, F&& f) {
  const int lane = threadIdx.x & 63;
  auto units = [&](int b) { return b < p.n_req ? (req_len(p, b) + T - 1) / T : 0; };
  int64_t total = 0;
  for (int base = 0; base < p.n_req; base += 64) total += lane_value(wave_incl_sum(units(base + lane)), 63);
  const int64_t per = (total + p.nwg - 1) / p.nwg;
  int64_t lo = 0, hi = 0, c0 = 0;   // units [lo, hi), c0 before request b
  int b = 0;
  bool found = false;
  for (int64_t c = per; !found && c > 0 && c <= per + 1 && c < 1 << 24; ++c) {
    int64_t pieces = 0;
    lo = hi = 0;
    for (int base = 0; base < p.n_req; base += 64) {
      const int n = units(base + lane), k = (n + (int)c - 1) / (int)c, in = wave_incl_sum(k);
      const int64_t x = (int64_t)blockIdx.x - pieces;
      const uint64_t m = __builtin_amdgcn_ballot_w64(in - k <= x && x < in);
      if (m) {
        const int l = __builtin_ctzll(m), nl = lane_value(n, l), kl = lane_value(k, l), y = (int)(x - lane_value(in - k, l));
        b = base + l;
        lo = (int64_t)nl * y / kl;
        hi = (int64_t)nl * (y + 1) / kl;
      }
      pieces += lane_value(in, 63);
    }
    found = pieces <= p.nwg;
  }
  if (!found) {
    lo = blockIdx.x * per;
    hi = lo + per < total ? lo + per : total;
    b = 0;
  }
  while (lo < hi) {
    const int L = req_len(p, b);
    const int64_t n = (L + T - 1) / T;
    if (lo >= c0 + n) {
      c0 += n;
      ++b;
      continue;
    }
    const int64_t a = lo - c0, e = hi - c0 < n ? hi - c0 : n;
    f(b, (int)a * T, e * T < L ? (int)e * T : L, L);
    lo += e - a;
  }
}

// Up to two row blocks (32 rows): three workgroups a CU of four waves; more: their queries take the LDS of one
// workgroup of eight.
template <bool FP8, int NRB>
__global__ __launch_bounds__(NRB <= 2 ? 256 : 512, NRB <= 2 ? 3 : 2) void weights_kernel(const WtParams w) {
  extern __shared__ __align__(16) char lds[];
  constexpr int NT = NRB <= 2 ? 256 : 512, NWV = NT / 64;
  const KParams& p = w.k;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, lg = lane >> 4;
  constexpr int PPS = FP8 ? 2 : 1;            // products a step
  const int nm = w.steps * PPS;
  bf16x8* qf = reinterpret_cast<bf16x8*>(lds);                      // [NRB][nm][64]
  float* lse_s = reinterpret_cast<float*>(lds + NRB * nm * 1024);   // [NRB * 16], log2 domain
  int* lim_s = reinterpret_cast<int*>(lse_s + NRB * 16);            // tokens a row sees
  int* div_s = lim_s + NRB * 16;                                    // byte of a row's divisor in the cached row
  int* group_s = div_s + NRB * 16;                                  // its head's latent group, -1: no row
  RowAt* row_s = reinterpret_cast<RowAt*>(group_s + NRB * 16);
  const float ks = p.k_scale ? *p.k_scale : 1.f;
  int bad = 0;
  for_each_piece<16 * NWV>(p, [&](int b, int a, int e, int L) {
    // a request's pages are its last row's, as its length
    const int* bt = p.bt + ((int64_t)b * p.qrows + p.qrows - 1) * p.bt_stride;
    for (int pass = 0; pass < w.passes; ++pass) {
      const int rbase = pass * NRB * 16;
      __syncthreads();
      for (int x = threadIdx.x; x < NRB * 16; x += NT) {
        const int r = rbase + x;
        float l = -kNegInf;   // adds nothing
        int lim = 0, at = p.rms_off_b, group = -1;
        RowAt row{};
        if (r < w.rows) {
          const int j = r / p.heads, hd = r - j * p.heads;
          const int64_t qrow = (int64_t)b * p.qrows + j;
          group = p.heads > p.hpg ? hd / p.hpg : 0;
          row.qn = p.q_nope + qrow * p.qn_sr + hd * p.qn_sh;
          row.qp = p.q_pe + qrow * p.qp_sr + hd * p.qp_sh;
          l = w.lse[qrow * w.lse_sr + hd];
          l = is_neg_inf(l) ? -kNegInf : l * kLog2e;
          lim = L - (p.qrows - 1 - j);
          at += hd * w.rms_b;
        }
        lse_s[x] = l;
        lim_s[x] = lim;
        div_s[x] = at;
        group_s[x] = group;
        row_s[x] = row;
      }
      __syncthreads();
      // 8 columns of a row a lane: QB loads under way together, from the cache's first bytes where there is nothing to
      // load; what straddles an end is put together by elements behind them
      for (int x0 = wave; x0 < NRB * nm; x0 += QB * NWV) {
        bf16x8 v[QB];
        auto at = [&](int x) {
          const int m = x / NRB, rx = 16 * (x - m * NRB) + n;
          return query_at(w, row_s[rx], group_s[rx], FP8 ? 64 * (m >> 1) + 16 * lg + 8 * (m & 1) : 32 * m + 8 * lg);
        };
        uint32_t whole = 0, part = 0;
#pragma unroll
        for (int y = 0; y < QB; ++y) {
          const QueryAt q = at(x0 + y * NWV < NRB * nm ? x0 + y * NWV : x0);
          v[y] = *reinterpret_cast<const bf16x8_e*>(q.src);
          whole |= (uint32_t)q.whole << y;
          part |= (uint32_t)q.part << y;
        }
#pragma unroll
        for (int y = 0; y < QB; ++y) {
          const int x = x0 + y * NWV;
          if (x >= NRB * nm) break;
          i32x4 bits = __builtin_bit_cast(i32x4, v[y]);
#pragma unroll
          for (int k = 0; k < 4; ++k) bits[k] = (whole >> y) & 1 ? bits[k] : 0;
          v[y] = __builtin_bit_cast(bf16x8, bits);
          if (__builtin_expect((part >> y) & 1, 0)) {
            const QueryAt q = at(x);
            const RowAt row = row_s[16 * (x % NRB) + n];
            for (int i = 0; i < 8; ++i) {
              __bf16 e = (__bf16)0.f;
              if (q.o + i >= 0 && q.o + i < w.dcg) e = row.qn[q.o + i];
              else if (q.q + i >= 0 && q.q + i < p.rope_w) e = row.qp[q.q + i];
#pragma unroll
              for (int k = 0; k < 8; ++k) v[y][k] = k == i ? e : v[y][k];
            }
          }
          qf[((x % NRB) * nm + x / NRB) * 64 + lane] = v[y];
        }
      }
      __syncthreads();
      // a tile's page ids are loaded a tile ahead, its divisors and its old weights before its keys
      auto page_of = [&](int t0) { return t0 < e ? bt[page_div(p, t0 + n < e ? t0 + n : e - 1)] : 0; };
      int pid = page_of(a + 16 * wave);
      for (int t0 = a + 16 * wave; t0 < e; t0 += 16 * NWV) {
        const int t = t0 + n;
        const int tc = t < e ? t : e - 1;
        const int id = checked_page(p, pid, bad);
        const char* row = p.kv + id * p.page_stride_b + (int64_t)(tc - page_div(p, tc) * p.page_size) * p.token_stride_b;
        const char* krow = row + 16 * lg;
        pid = page_of(t0 + 16 * NWV);
        i32x2 rraw[NRB];
        if (w.rms4) {
#pragma unroll
          for (int rb = 0; rb < NRB; ++rb) {
            const char* at = row + div_s[rb * 16 + 4 * lg];
            if (w.rms_b == 1) rraw[rb][0] = *reinterpret_cast<const int*>(at);
            else rraw[rb] = *reinterpret_cast<const i32x2*>(at);
          }
        }
        float* o = w.out + b * w.out_s + t;
        float before = 0.f;
        if (lg == 0 && t < e && t < w.width) before = pass > 0 ? *o : w.win ? w.win[b * w.win_s + t] : 0.f;
        f32x4 s[NRB];
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) s[rb] = f32x4{};
        auto load = [&](int st) { return *reinterpret_cast<const i32x4*>(krow + 64 * st); };
        auto use = [&](int st, const i32x4& raw) {
          if constexpr (FP8) {
            bf16x8 k0, k1;
            fp8x16_to_bf16(raw, k0, k1);
#pragma unroll
            for (int rb = 0; rb < NRB; ++rb) {
              s[rb] = mfma16(qf[(rb * nm + 2 * st) * 64 + lane], k0, s[rb]);
              s[rb] = mfma16(qf[(rb * nm + 2 * st + 1) * 64 + lane], k1, s[rb]);
            }
          } else {
            const bf16x8 k0 = __builtin_bit_cast(bf16x8, raw);
#pragma unroll
            for (int rb = 0; rb < NRB; ++rb) s[rb] = mfma16(qf[(rb * nm + st) * 64 + lane], k0, s[rb]);
          }
        };
#pragma unroll 1
        for (int st = 0; st < w.whole; st += U) {
          i32x4 x[U];
          if (st + U <= w.whole) {
#pragma unroll
            for (int i = 0; i < U; ++i) x[i] = load(st + i);
#pragma unroll
            for (int i = 0; i < U; ++i) use(st + i, x[i]);
          } else {
#pragma unroll
            for (int i = 0; i < U - 1; ++i)
              if (st + i < w.whole) x[i] = load(st + i);
#pragma unroll
            for (int i = 0; i < U - 1; ++i)
              if (st + i < w.whole) use(st + i, x[i]);
          }
        }
        for (int st = w.whole; st < w.steps; ++st) {
          // columns past the row's keys read as zeros
          constexpr int PER = FP8 ? 16 : 8, CB = FP8 ? 8 : 16;   // columns of a load, bits of a column
          const int left = w.cols - PER * (4 * st + lg);          // valid columns of this load
          i32x4 v{};
          if (left > 0) v = load(st);
          if (left < PER) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              const int bits = left * CB - 32 * d;
              v[d] = bits <= 0 ? 0 : bits >= 32 ? v[d] : v[d] & (int)((1u << bits) - 1);
            }
          }
          use(st, v);
        }
        const bool edge = t0 + 16 > L - (p.qrows - 1);
        const float f = p.sm_scale * ks;
        float sum = 0.f;
        // inv(r4, rb, i): f over the divisor of row r4 + i; chosen once a tile, a branch a row costs more than the row
        auto add = [&](auto inv) {
#pragma unroll
          for (int rb = 0; rb < NRB; ++rb) {
            const int r4 = rb * 16 + 4 * lg;
            const f32x4 l4 = *reinterpret_cast<const f32x4*>(lse_s + r4);
            const i32x4 lim4 = *reinterpret_cast<const i32x4*>(lim_s + r4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float v = s[rb][i] * inv(r4, rb, i);
              if (__builtin_expect(p.logit_cap > 0.f, 0)) v = p.logit_cap * (1.0f - 2.0f / (fast_exp2(2.0f * kLog2e * (v / p.logit_cap)) + 1.0f));
              const float l = l4[i];
              const bool dead = __float_as_uint(l) == 0x7f800000u || (edge && t >= lim4[i]);
              const float pr = fast_exp2(v * kLog2e - l);
              sum += dead ? 0.f : pr;
            }
          }
        };
        if (w.rms4 && w.rms_mode == QMLA_RMS_LOG8) {
          add([&](int, int rb, int i) { return f * fast_exp2(3.0f - (float)(((uint32_t)rraw[rb][0] >> (8 * i)) & 0xff) * (6.0f / 255.0f)); });
        } else if (w.rms4 && w.rms_b == 2) {
          add([&](int, int rb, int i) { return f * inv_divisor(((uint32_t)rraw[rb][i >> 1] >> (16 * (i & 1))) & 0xffff, QMLA_RMS_BF16, ks); });
        } else {
          add([&](int r4, int, int i) {
            if (w.rms_mode == QMLA_RMS_NONE) return f;
            const uint8_t* at = reinterpret_cast<const uint8_t*>(row + div_s[r4 + i]);
            uint32_t raw = at[0];
            if (w.rms_b == 2) raw |= (uint32_t)at[1] << 8;
            return w.rms_mode == QMLA_RMS_LOG8 ? f * fast_exp2(3.0f - (float)raw * (6.0f / 255.0f)) : f * inv_divisor(raw, w.rms_mode, ks);
          });
        }
        sum = sum_lg(sum);
        if (lg == 0 && t < e && t < w.width) *o = before + sum;
      }
    }
  });
  report_pages(p, bad);
}

static int lds_bytes(int nrb, int nm) { return nrb * (nm * 1024 + 16 * (4 * 4 + 16)); }

template <bool FP8>
static const void* pick(int nrb) {
  switch (nrb) {
    case 1: return (const void*)&weights_kernel<FP8, 1>;
    case 2: return (const void*)&weights_kernel<FP8, 2>;
    case 3: return (const void*)&weights_kernel<FP8, 3>;
    case 4: return (const void*)&weights_kernel<FP8, 4>;
    case 6: return (const void*)&weights_kernel<FP8, 6>;
    default: return (const void*)&weights_kernel<FP8, 8>;
  }
}

}  // namespace wt
}  // namespace qmla

using namespace qmla;

extern "C" int qmla_attention_weights(const qmla_decode_params* p0, const float* lse, int64_t lse_stride, const float* weights,
                                      int64_t weights_stride, float* out, int64_t out_stride, int32_t width, void* stream) {
  if (!p0) return QMLA_ERR_NULL;
  qmla_decode_params p = *p0;
  p.out = out;                  // unused by the checks below but for its presence
  p.out_dtype = QMLA_DT_F32;
  p.lse = nullptr;
  p.num_splits = 1;
  p.workspace = nullptr;
  const int rc = validate_params(&p);
  if (rc) return rc;
  if (width < 0) return QMLA_ERR_SHAPE;
  if (!rows16(&p)) return QMLA_ERR_ALIGN;
  if (p.rows == 0 || width == 0) return QMLA_OK;
  if (!lse || !out) return QMLA_ERR_NULL;
  const bool fp8 = p.kv_dtype == QMLA_KV_FP8;
  wt::WtParams w{};
  w.k = make_kparams(&p);
  w.cols = p.d_c + p.rope_w;
  w.d_c = p.d_c;
  w.dcg = p.d_c / p.groups;
  w.steps = fp8 ? (w.cols + 63) / 64 : (w.cols + 31) / 32;
  w.whole = fp8 ? w.cols / 64 : w.cols / 32;
  const int nm = w.steps * (fp8 ? 2 : 1);
  // the last load of a row may reach past its columns, never past its 16-byte multiple
  const int64_t need = ((int64_t)w.cols * (fp8 ? 1 : 2) + 15) / 16 * 16, ts = (p.page_size > 1 ? p.token_stride : p.page_stride) * (fp8 ? 1 : 2);
  if (ts < need) return QMLA_ERR_SHAPE;
  w.rows = p.qrows * p.heads;
  if ((int64_t)p.qrows * p.heads > 1 << 20) return QMLA_ERR_SHAPE;
  const int blocks = (w.rows + 15) / 16;
  // row blocks at once: all of them, as far as LDS holds their queries and a kernel has them
  int nrb = blocks < wt::MAXRB ? blocks : wt::MAXRB;
  while (nrb > 1 && wt::lds_bytes(nrb, nm) > wt::LDS_MAX) --nrb;
  if (nrb == 5 || nrb == 7) nrb += wt::lds_bytes(nrb + 1, nm) <= wt::LDS_MAX ? 1 : -1;
  const int bytes = wt::lds_bytes(nrb, nm);
  if (bytes > wt::LDS_MAX) return QMLA_ERR_NOKERNEL;
  w.passes = (blocks + nrb - 1) / nrb;
  w.rms_mode = p.rms_mode;
  w.rms_b = p.rms_mode == QMLA_RMS_BF16 || p.rms_mode == QMLA_RMS_BF16_BYTES ? 2 : 1;
  w.rms4 = p.rms_mode != QMLA_RMS_NONE && p.heads % 4 == 0 && w.k.rms_off_b % (4 * w.rms_b) == 0;
  w.lse = lse;
  w.lse_sr = lse_stride;
  w.win = weights;
  w.win_s = weights_stride;
  w.out = out;
  w.out_s = out_stride;
  w.width = width;
  const int occ = wt::LDS_MAX / bytes < 3 ? wt::LDS_MAX / bytes : 3;
  w.k.nwg = cu_count() * occ;
  w.k.num_splits = 0;
  const void* fn = fp8 ? wt::pick<true>(nrb) : wt::pick<false>(nrb);
  if (bytes > 64 * 1024 && hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return QMLA_ERR_LAUNCH;
  void* args[] = {&w};
  const hipError_t e = hipLaunchKernel(fn, dim3(w.k.nwg), dim3(nrb <= 2 ? 256 : 512), args, bytes, (hipStream_t)stream);
  return e == hipSuccess ? QMLA_OK : QMLA_ERR_LAUNCH;
}
