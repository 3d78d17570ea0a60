// Attention weight of every cached token (qmla_attention_weights): a second pass over the keys that sums
// exp(s - lse) over a request's query rows and heads. See include/qmla.h.
//
// S = Q K^T in 32x32 blocks of v_mfma_f32_32x32x16_bf16 with the queries as A, so a lane holds one token's
// scores of 16 rows and the sum over rows stays in the lane (and its partner 32 lanes away). A lane loads
// its token's row straight from memory, 16 bytes a load: the contraction's order is free as long as both
// operands share it, so lane half h takes columns 16h.. of each 32 FP8 columns (two products) or 8h.. of
// each 16 bf16 ones (one), and no key passes through LDS. The queries wait in LDS in the order of the
// products, a 1 KB read a product. FP8 keys become bf16 exactly, so scores are exact products summed in
// fp32: the query as e4m3 parts (the decode's scores) would be 5e-6 of the terms off, too much for a
// fp32 result.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmla.h"
#include "qmla_common.h"

namespace qmla {
namespace wt {

constexpr int NT = 256, NWV = NT / 64;
constexpr int U = 6;             // loads in flight ahead of the products, and as many behind them
constexpr int MAXRB = 4;         // row blocks of 32 held at once
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
  int steps;       // 16-byte loads of a lane for one token
  int nrb;         // row blocks held at once (template), passes over them
  int passes;
  int rms_mode, rms_b;   // divisor bytes of a head
  int rms4;        // 4 heads' divisors load at once
};

__device__ __forceinline__ f32x16 mfma32(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float divisor(uint32_t raw, int mode, float ks) {
  float r;
  if (mode == QMLA_RMS_LOG8) return fast_exp2((float)raw * (6.0f / 255.0f) - 3.0f);
  if (mode == QMLA_RMS_E4M3) r = fp8_to_f32(raw) * ks;
  else r = bf16_bits_to_f32(raw);
  return r > 0.f ? r : 1.f;
}

template <bool FP8, int NRB>
__global__ __launch_bounds__(NT) void weights_kernel(const WtParams w) {
  extern __shared__ __align__(16) char lds[];
  const KParams& p = w.k;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  constexpr int PPS = FP8 ? 2 : 1;            // products a step
  const int nm = w.steps * PPS;
  bf16x8* qf = reinterpret_cast<bf16x8*>(lds);                      // [NRB][nm][64]
  float* lse_s = reinterpret_cast<float*>(lds + NRB * nm * 1024);   // [NRB * 32], log2 domain
  int* lim_s = reinterpret_cast<int*>(lse_s + NRB * 32);            // tokens a row sees, from the end
  const float ks = p.k_scale ? *p.k_scale : 1.f;
  int bad = 0;
  for_each_segment<32, 0>(p, [&](int b, int a, int e, int L, const SegOut&) {
    // a request's pages are its last row's, as its length
    const int* bt = p.bt + ((int64_t)b * p.qrows + p.qrows - 1) * p.bt_stride;
    for (int pass = 0; pass < w.passes; ++pass) {
      const int rbase = pass * NRB * 32;
      __syncthreads();
      for (int x = threadIdx.x; x < NRB * nm * 64; x += NT) {
        const int l = x & 63, m = (x >> 6) % nm, rb = (x >> 6) / nm;
        const int r = rbase + rb * 32 + (l & 31);
        const int c0 = FP8 ? 32 * (m >> 1) + 16 * (l >> 5) + 8 * (m & 1) : 16 * m + 8 * (l >> 5);
        bf16x8 v{};
        if (r < w.rows) {
          const int j = r / p.heads, hd = r - j * p.heads;
          const int64_t row = (int64_t)b * p.qrows + j;
          const int g0 = hd / p.hpg * w.dcg;
          const __bf16* qn = p.q_nope + row * p.qn_sr + hd * p.qn_sh;
          const __bf16* qp = p.q_pe + row * p.qp_sr + hd * p.qp_sh;
          if (c0 >= g0 && c0 + 8 <= g0 + w.dcg) {
            v = load_q8(qn + (c0 - g0), p.q_vec);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int c = c0 + i;
              if (c >= g0 && c < g0 + w.dcg) v[i] = qn[c - g0];
              else if (c >= w.d_c && c < w.cols) v[i] = qp[c - w.d_c];
            }
          }
        }
        qf[x] = v;
      }
      for (int x = threadIdx.x; x < NRB * 32; x += NT) {
        const int r = rbase + x;
        float l = -kNegInf;   // adds nothing
        int lim = 0;
        if (r < w.rows) {
          const int j = r / p.heads, hd = r - j * p.heads;
          l = w.lse[((int64_t)b * p.qrows + j) * w.lse_sr + hd];
          l = is_neg_inf(l) ? -kNegInf : l * kLog2e;
          lim = L - (p.qrows - 1 - j);
        }
        lse_s[x] = l;
        lim_s[x] = lim;
      }
      __syncthreads();
      // byte offset of the divisors of this lane's 4 rows from 8 i4 + 4 h on
      int hoff[NRB][4];
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) hoff[rb][i4] = p.rms_off_b + (rbase + rb * 32 + 8 * i4 + 4 * h) % p.heads * w.rms_b;
      for (int t0 = a + 32 * wave; t0 < e; t0 += 32 * NWV) {
        const int t = t0 + n;
        const int tc = t < e ? t : e - 1;
        const int pg = page_div(p, tc);
        const int id = checked_page(p, bt[pg], bad);
        const char* row = p.kv + id * p.page_stride_b + (int64_t)(tc - pg * p.page_size) * p.token_stride_b;
        const char* krow = row + 16 * h;
        f32x16 s[NRB];
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) s[rb] = f32x16{};
        // columns past the row's keys read as zeros
        auto load = [&](int st) -> i32x4 {
          i32x4 v{};
          const int left = w.cols - (FP8 ? 32 * st + 16 * h : 16 * st + 8 * h);   // valid columns of this load
          if (st < w.steps && left > 0) {
            v = *reinterpret_cast<const i32x4*>(krow + 32 * st);
            constexpr int PER = FP8 ? 16 : 8, CB = FP8 ? 8 : 16;   // columns of a load, bits of a column
            if (left < PER) {
#pragma unroll
              for (int d = 0; d < 4; ++d) {
                const int bits = left * CB - 32 * d;
                v[d] = bits <= 0 ? 0 : bits >= 32 ? v[d] : v[d] & (int)((1u << bits) - 1);
              }
            }
          }
          return v;
        };
        auto use = [&](int st, const i32x4& raw) {
          if (st >= w.steps) return;
          if constexpr (FP8) {
            bf16x8 k0, k1;
            fp8x16_to_bf16(raw, k0, k1);
#pragma unroll
            for (int rb = 0; rb < NRB; ++rb) {
              s[rb] = mfma32(qf[(rb * nm + 2 * st) * 64 + lane], k0, s[rb]);
              s[rb] = mfma32(qf[(rb * nm + 2 * st + 1) * 64 + lane], k1, s[rb]);
            }
          } else {
            const bf16x8 k0 = __builtin_bit_cast(bf16x8, raw);
#pragma unroll
            for (int rb = 0; rb < NRB; ++rb) s[rb] = mfma32(qf[(rb * nm + st) * 64 + lane], k0, s[rb]);
          }
        };
        i32x4 x0[U], x1[U];
#pragma unroll
        for (int i = 0; i < U; ++i) x0[i] = load(i);
        for (int g = 0; g < w.steps; g += 2 * U) {
#pragma unroll
          for (int i = 0; i < U; ++i) x1[i] = load(g + U + i);
#pragma unroll
          for (int i = 0; i < U; ++i) use(g + i, x0[i]);
#pragma unroll
          for (int i = 0; i < U; ++i) x0[i] = load(g + 2 * U + i);
#pragma unroll
          for (int i = 0; i < U; ++i) use(g + U + i, x1[i]);
        }
        const bool edge = t0 + 32 > L - (p.qrows - 1);
        const float f = p.sm_scale * ks;
        float sum = 0.f;
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) {
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            const int x = rb * 32 + 8 * i4 + 4 * h;
            float inv[4];
            if (w.rms_mode == QMLA_RMS_NONE) {
#pragma unroll
              for (int i = 0; i < 4; ++i) inv[i] = 1.f;
            } else {
              uint32_t raw[4];
              if (w.rms4) {
                if (w.rms_b == 1) {
                  const uint32_t v = *reinterpret_cast<const uint32_t*>(row + hoff[rb][i4]);
#pragma unroll
                  for (int i = 0; i < 4; ++i) raw[i] = (v >> (8 * i)) & 0xff;
                } else {
                  const i32x2 v = *reinterpret_cast<const i32x2*>(row + hoff[rb][i4]);
#pragma unroll
                  for (int i = 0; i < 4; ++i) raw[i] = ((uint32_t)v[i >> 1] >> (16 * (i & 1))) & 0xffff;
                }
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const char* at = row + p.rms_off_b + (rbase + x + i) % p.heads * w.rms_b;
                  raw[i] = *(const uint8_t*)at;
                  if (w.rms_b == 2) raw[i] |= (uint32_t)*(const uint8_t*)(at + 1) << 8;
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                inv[i] = w.rms_mode == QMLA_RMS_LOG8 ? fast_exp2(3.0f - (float)raw[i] * (6.0f / 255.0f))
                                                     : 1.f / divisor(raw[i], w.rms_mode, ks);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float v = s[rb][4 * i4 + i] * f * inv[i];
              if (p.logit_cap > 0.f) v = p.logit_cap * (1.0f - 2.0f / (fast_exp2(2.0f * kLog2e * (v / p.logit_cap)) + 1.0f));
              const float l = lse_s[x + i];
              bool dead = __float_as_uint(l) == 0x7f800000u;
              if (edge) dead = dead || t >= lim_s[x + i];
              const float pr = fast_exp2(v * kLog2e - l);
              sum += dead ? 0.f : pr;
            }
          }
        }
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
        sum = __uint_as_float(both[0]) + __uint_as_float(both[1]);
        if (h == 0 && t < e && t < w.width) {
          float* o = w.out + b * w.out_s + t;
          const float before = pass > 0 ? *o : w.win ? w.win[b * w.win_s + t] : 0.f;
          *o = before + sum;
        }
      }
    }
  });
  report_pages(p, bad);
}

template <bool FP8>
static const void* pick(int nrb) {
  switch (nrb) {
    case 1: return (const void*)&weights_kernel<FP8, 1>;
    case 2: return (const void*)&weights_kernel<FP8, 2>;
    case 3: return (const void*)&weights_kernel<FP8, 3>;
    default: return (const void*)&weights_kernel<FP8, 4>;
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
  w.steps = fp8 ? (w.cols + 31) / 32 : (w.cols + 15) / 16;
  const int nm = w.steps * (fp8 ? 2 : 1);
  // the last load of a row may reach past its columns, never past its 16-byte multiple
  const int64_t need = ((int64_t)w.cols * (fp8 ? 1 : 2) + 15) / 16 * 16, ts = (p.page_size > 1 ? p.token_stride : p.page_stride) * (fp8 ? 1 : 2);
  if (ts < need) return QMLA_ERR_SHAPE;
  w.rows = p.qrows * p.heads;
  if ((int64_t)p.qrows * p.heads > 1 << 20) return QMLA_ERR_SHAPE;
  const int blocks = (w.rows + 31) / 32;
  int nrb = blocks < wt::MAXRB ? blocks : wt::MAXRB;
  while (nrb > 1 && nrb * nm * 1024 + nrb * 256 > wt::LDS_MAX) --nrb;
  const int bytes = nrb * nm * 1024 + nrb * 256;
  if (bytes > wt::LDS_MAX) return QMLA_ERR_NOKERNEL;
  w.nrb = nrb;
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
  const int occ = wt::LDS_MAX / bytes < 4 ? wt::LDS_MAX / bytes : 4;
  w.k.nwg = cu_count() * occ;
  w.k.num_splits = 0;
  const void* fn = fp8 ? wt::pick<true>(nrb) : wt::pick<false>(nrb);
  if (bytes > 64 * 1024 && hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return QMLA_ERR_LAUNCH;
  void* args[] = {&w};
  const hipError_t e = hipLaunchKernel(fn, dim3(w.k.nwg), dim3(wt::NT), args, bytes, (hipStream_t)stream);
  return e == hipSuccess ? QMLA_OK : QMLA_ERR_LAUNCH;
}
