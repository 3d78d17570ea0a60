// Rotary positions of query and key heads (qmla_rotary): half and interleaved pairs, part of the head,
// any table. See include/qmla.h for the formula.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmla.h"
#include "qmla_common.h"

namespace qmla {
namespace rot {

struct RParams {
  qmla_rotary_params p;
  int units;      // vectors of a head a thread handles one of: rot_units pairs of vectors, then the copied ones
  int rot_units;
  int head_units; // (q_heads + k_heads) * units
  uint32_t unit_mul;
  int unit_sh;
};

template <class T>
__device__ __forceinline__ float up(T v) { return (float)v; }

template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// One thread a unit: V pairs (half: V elements of each half; interleaved: V pairs side by side, two
// vectors), or V copied elements. Every element is read and written once, 16 bytes a load, and the table's rows come
// from the L2: bound by the copy rate (12001 tokens of 28 bf16 heads of 256: 80 us, 4.3 TB/s where a copy has 4.9;
// 33 tokens 4 us).
template <class T, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RParams r) {
  const qmla_rotary_params& p = r.p;
  const int t = blockIdx.x;
  const int u = (int)blockIdx.y * 256 + (int)threadIdx.x;
  if (u >= r.head_units) return;
  const int h = (int)magic_div((uint32_t)u, r.unit_mul, r.unit_sh), w = u - h * r.units;
  const bool is_q = h < p.q_heads;
  const int hh = is_q ? h : h - p.q_heads;
  const T* src = is_q ? (const T*)p.q + t * p.q_token_stride + hh * p.q_head_stride
                      : (const T*)p.k + t * p.k_token_stride + hh * p.k_head_stride;
  T* dst = is_q ? (T*)p.q_out + t * p.q_out_token_stride + hh * p.q_out_head_stride
                : (T*)p.k_out + t * p.k_out_token_stride + hh * p.k_out_head_stride;
  typedef Vec<T, V> VT;
  if (w >= r.rot_units) {
    int c = (w - r.rot_units) * V;
    if (c >= p.offset) c += p.rot;
    *(VT*)(dst + c) = *(const VT*)(src + c);
    return;
  }
  const int half = p.rot >> 1, i0 = w * V;
  const int64_t pos = p.positions[t * p.pos_stride];
  const bool ok = pos >= 0 && pos < p.max_pos;
  float c[V], s[V];
  const float* row = p.cos_sin + (ok ? pos : 0) * p.cos_sin_stride + i0;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    c[e] = row[e];
    s[e] = row[half + e];
  }
  const float sign = p.inverse ? -1.f : 1.f, nan = __uint_as_float(0x7fc00000u);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    c[e] = ok ? c[e] : nan;
    s[e] = ok ? s[e] * sign : nan;
  }
  const int xa = p.offset + (INTER ? 2 * i0 : i0), ya = INTER ? xa + V : xa + half;
  VT a = *(const VT*)(src + xa), b = *(const VT*)(src + ya);
  float x[V], y[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    // interleaved: pair e lies at elements 2e and 2e + 1 of the two vectors side by side
    const T xv = INTER ? (2 * e < V ? a.v[2 * e < V ? 2 * e : 0] : b.v[2 * e < V ? 0 : 2 * e - V]) : a.v[e];
    const T yv = INTER ? (2 * e + 1 < V ? a.v[2 * e + 1 < V ? 2 * e + 1 : 0] : b.v[2 * e + 1 < V ? 0 : 2 * e + 1 - V]) : b.v[e];
    x[e] = up(xv) * c[e] - up(yv) * s[e];
    y[e] = up(yv) * c[e] + up(xv) * s[e];
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (INTER) {
      a.v[e] = (T)((e & 1) ? y[e >> 1] : x[e >> 1]);
      b.v[e] = (T)(((V + e) & 1) ? y[(V + e) >> 1] : x[(V + e) >> 1]);
    } else {
      a.v[e] = (T)x[e];
      b.v[e] = (T)y[e];
    }
  }
  *(VT*)(dst + xa) = a;
  *(VT*)(dst + ya) = b;
}

static int elem(int dt) { return dt == QMLA_DT_F32 ? 4 : 2; }

template <class T>
static const void* pick(int v, bool inter) {
  constexpr int W = 16 / sizeof(T);
  if (inter) return v > 1 ? (const void*)&rotary_kernel<T, W, true> : (const void*)&rotary_kernel<T, 1, true>;
  return v > 1 ? (const void*)&rotary_kernel<T, W, false> : (const void*)&rotary_kernel<T, 1, false>;
}

}  // namespace rot
}  // namespace qmla

using namespace qmla;

extern "C" int qmla_rotary(const qmla_rotary_params* p, void* stream) {
  if (!p) return QMLA_ERR_NULL;
  if (p->dtype != QMLA_DT_BF16 && p->dtype != QMLA_DT_F16 && p->dtype != QMLA_DT_F32) return QMLA_ERR_MODE;
  if (p->n < 0 || p->q_heads < 0 || p->k_heads < 0 || p->head_dim <= 0 || p->offset < 0 || p->rot <= 0 || p->rot % 2 ||
      p->rot > p->head_dim - p->offset || p->max_pos <= 0 || p->cos_sin_stride < p->rot)
    return QMLA_ERR_SHAPE;
  const int64_t heads = (int64_t)p->q_heads + p->k_heads;
  if (heads * p->head_dim > 0x7fffffff / 2) return QMLA_ERR_SHAPE;
  if (p->n == 0 || heads == 0) return QMLA_OK;
  if ((p->q_heads && (!p->q || !p->q_out)) || (p->k_heads && (!p->k || !p->k_out)) || !p->positions || !p->cos_sin)
    return QMLA_ERR_NULL;
  const int es = rot::elem(p->dtype), w = 16 / es;
  auto off = [&](const void* a, int64_t st, int64_t sh, int by) {
    return ((uintptr_t)a | (uint64_t)(st * es) | (uint64_t)(sh * es)) % by != 0;
  };
  auto any_off = [&](int by) {
    return (p->q_heads && (off(p->q, p->q_token_stride, p->q_head_stride, by) ||
                           off(p->q_out, p->q_out_token_stride, p->q_out_head_stride, by))) ||
           (p->k_heads && (off(p->k, p->k_token_stride, p->k_head_stride, by) ||
                           off(p->k_out, p->k_out_token_stride, p->k_out_head_stride, by)));
  };
  if (any_off(es) || (uintptr_t)p->cos_sin % 4 || (uintptr_t)p->positions % 8) return QMLA_ERR_ALIGN;
  // 16-byte vectors where every head, the rotated part and its halves lie on them, else single elements
  const bool vec = !any_off(16) && p->head_dim % w == 0 && p->offset % w == 0 && (p->rot / 2) % w == 0;
  auto alias = [](const void* a, const void* b, int64_t s0, int64_t s1, int64_t h0, int64_t h1) {
    return a == b && s0 == s1 && h0 == h1;
  };
  const bool in_place =
      (!p->q_heads || alias(p->q, p->q_out, p->q_token_stride, p->q_out_token_stride, p->q_head_stride, p->q_out_head_stride)) &&
      (!p->k_heads || alias(p->k, p->k_out, p->k_token_stride, p->k_out_token_stride, p->k_head_stride, p->k_out_head_stride));
  rot::RParams r;
  r.p = *p;
  const int v = vec ? w : 1;
  r.rot_units = p->rot / 2 / v;
  r.units = r.rot_units + (in_place ? 0 : (p->head_dim - p->rot) / v);
  r.head_units = (int)heads * r.units;
  page_magic(r.units, r.unit_mul, r.unit_sh);
  const bool inter = p->interleaved != 0;
  const void* fn = p->dtype == QMLA_DT_BF16  ? rot::pick<__bf16>(v, inter)
                   : p->dtype == QMLA_DT_F16 ? rot::pick<_Float16>(v, inter)
                                             : rot::pick<float>(v, inter);
  const int gy = (r.head_units + 255) / 256;
  if (gy > 65535) return QMLA_ERR_SHAPE;
  void* args[] = {&r};
  const hipError_t e = hipLaunchKernel(fn, dim3(p->n, gy), dim3(256), args, 0, (hipStream_t)stream);
  return e == hipSuccess ? QMLA_OK : QMLA_ERR_LAUNCH;
}
