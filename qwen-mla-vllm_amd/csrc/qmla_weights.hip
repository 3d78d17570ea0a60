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
// fp32 result.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmla.h"
#include "qmla_common.h"

namespace qmla {
namespace wt {

constexpr int U = 9;             // loads of a group
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
  uint32_t head_mul;   // x / heads
  int head_sh;
  int rms_mode, rms_b;   // divisor bytes of a head
  int rms4;        // 4 heads' divisors load at once
};

// queries may be aligned to their elements only
typedef bf16x8 bf16x8_e __attribute__((aligned(2)));

__device__ __forceinline__ float divisor(uint32_t raw, int mode, float ks) {
  const float r = mode == QMLA_RMS_E4M3 ? fp8_to_f32(raw) * ks : bf16_bits_to_f32(raw);
  return r > 0.f ? r : 1.f;
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
  const float ks = p.k_scale ? *p.k_scale : 1.f;
  int bad = 0;
  for_each_segment<32, 0>(p, [&](int b, int a, int e, int L, const SegOut&) {
    // a request's pages are its last row's, as its length
    const int* bt = p.bt + ((int64_t)b * p.qrows + p.qrows - 1) * p.bt_stride;
    for (int pass = 0; pass < w.passes; ++pass) {
      const int rbase = pass * NRB * 16;
      __syncthreads();
#pragma unroll 6
      for (int x = wave; x < NRB * nm; x += NWV) {
        const int m = x / NRB, rb = x - m * NRB;
        const int r = rbase + rb * 16 + n;
        bf16x8 v{};
        if (r < w.rows) {
          const int j = (int)magic_div((uint32_t)r, w.head_mul, w.head_sh), hd = r - j * p.heads;
          const int64_t row = (int64_t)b * p.qrows + j;
          const int c0 = FP8 ? 64 * (m >> 1) + 16 * lg + 8 * (m & 1) : 32 * m + 8 * lg;
          const int o = c0 - (p.heads > p.hpg && hd >= p.hpg ? hd / p.hpg * w.dcg : 0), q = c0 - w.d_c;
          const __bf16* qn = p.q_nope + row * p.qn_sr + hd * p.qn_sh;
          const __bf16* qp = p.q_pe + row * p.qp_sr + hd * p.qp_sh;
          if (o >= 0 && o + 8 <= w.dcg) {
            v = *reinterpret_cast<const bf16x8_e*>(qn + o);
          } else if (q >= 0 && q + 8 <= p.rope_w) {
            v = *reinterpret_cast<const bf16x8_e*>(qp + q);
          } else if (o + 8 > 0 && c0 < w.cols && (o < w.dcg || q + 8 > 0)) {
            for (int i = 0; i < 8; ++i) {
              __bf16 y = (__bf16)0.f;
              if (o + i >= 0 && o + i < w.dcg) y = qn[o + i];
              else if (q + i >= 0 && q + i < p.rope_w) y = qp[q + i];
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] = k == i ? y : v[k];
            }
          }
        }
        qf[(rb * nm + m) * 64 + lane] = v;
      }
      for (int x = threadIdx.x; x < NRB * 16; x += NT) {
        const int r = rbase + x;
        float l = -kNegInf;   // adds nothing
        int lim = 0, at = p.rms_off_b;
        if (r < w.rows) {
          const int j = r / p.heads, hd = r - j * p.heads;
          l = w.lse[((int64_t)b * p.qrows + j) * w.lse_sr + hd];
          l = is_neg_inf(l) ? -kNegInf : l * kLog2e;
          lim = L - (p.qrows - 1 - j);
          at += hd * w.rms_b;
        }
        lse_s[x] = l;
        lim_s[x] = lim;
        div_s[x] = at;
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
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) {
          {
            const int x = rb * 16 + 4 * lg;
            float inv[4];
            if (w.rms_mode == QMLA_RMS_NONE) {
#pragma unroll
              for (int i = 0; i < 4; ++i) inv[i] = f;
            } else {
              uint32_t raw[4];
              if (w.rms4 && w.rms_b == 1) {
                const uint32_t v = (uint32_t)rraw[rb][0];
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[i] = (v >> (8 * i)) & 0xff;
              } else if (w.rms4) {
                const i32x2 v = rraw[rb];
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[i] = ((uint32_t)v[i >> 1] >> (16 * (i & 1))) & 0xffff;
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint8_t* at = reinterpret_cast<const uint8_t*>(row + div_s[x + i]);
                  raw[i] = at[0];
                  if (w.rms_b == 2) raw[i] |= (uint32_t)at[1] << 8;
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                inv[i] = w.rms_mode == QMLA_RMS_LOG8 ? f * fast_exp2(3.0f - (float)raw[i] * (6.0f / 255.0f))
                                                     : f / divisor(raw[i], w.rms_mode, ks);
            }
            const f32x4 l4 = *reinterpret_cast<const f32x4*>(lse_s + x);
            const i32x4 lim4 = edge ? *reinterpret_cast<const i32x4*>(lim_s + x) : i32x4{};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float v = s[rb][i] * inv[i];
              if (p.logit_cap > 0.f) v = p.logit_cap * (1.0f - 2.0f / (fast_exp2(2.0f * kLog2e * (v / p.logit_cap)) + 1.0f));
              const float l = l4[i];
              bool dead = __float_as_uint(l) == 0x7f800000u;
              if (edge) dead = dead || t >= lim4[i];
              const float pr = fast_exp2(v * kLog2e - l);
              sum += dead ? 0.f : pr;
            }
          }
        }
        sum = sum_lg(sum);
        if (lg == 0 && t < e && t < w.width) *o = before + sum;
      }
    }
  });
  report_pages(p, bad);
}

static int lds_bytes(int nrb, int nm) { return nrb * (nm * 1024 + 16 * 3 * 4); }

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
  page_magic(p.heads, w.head_mul, w.head_sh);
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
