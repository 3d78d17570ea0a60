// Eviction from the paged cache (qmla_evict_select, qmla_cache_compact): the tokens a request keeps and
// their rows moved together. See include/qmla.h.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmla.h"
#include "qmla_common.h"

namespace qmla {
namespace ev {

struct EParams {
  qmla_evict_params p;
  uint32_t page_mul;
  int page_sh;
  uint32_t chunk_mul;   // x / chunks of a row (out of place)
  int chunk_sh;
  int chunks;           // copy units of a row
};

// A weight as an unsigned number that ascends with it; NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t order(float w) {
  if (w != w) w = kNegInf;
  uint32_t u = __float_as_uint(w);
  if (u == 0x80000000u) u = 0;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int NT = 1024, NW = NT / 64;
constexpr int BITS = 11, BINS = 1 << BITS;   // digits of 11, 11 and 10 bits

constexpr int KEYS = 36 * 1024;               // keys LDS holds beside the histogram

// One workgroup a request: the m-th largest key of the middle tokens by three digit histograms, then one
// pass that counts per wave and one that writes. Waves take contiguous runs, so ranks among equal keys
// and output places follow from per-wave counts without a barrier per run. KEPT: the keys stay in LDS after
// the first pass (a request of up to KEYS tokens), else every pass reads the weights again. Bound by the passes of one
// workgroup over a request (40 requests of 2000 .. 32768 tokens: 35 us, 46 with equal bins of a wave added up first; 1 of
// 4100: 11 us).
template <bool KEPT>
__global__ __launch_bounds__(NT) void select_kernel(const EParams e) {
  const qmla_evict_params& p = e.p;
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ uint32_t hist[BINS];
  __shared__ uint32_t sh_digit, sh_need;
  __shared__ int wave_eq[NW], wave_gt[NW], wave_sum[NW];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int L = p.seq_lens[b];
  L = L < 0 ? 0 : L < p.width ? L : p.width;
  int* index = p.index + b * p.index_stride;
  __syncthreads();   // counts may be seq_lens: all have read theirs
  if (tid == 0) p.counts[b] = L < p.keep ? L : p.keep;
  if (L <= p.keep) {
    for (int i = tid; i < p.keep; i += NT) index[i] = i < L ? i : -1;
    return;
  }
  const float* w = p.weights + b * p.weights_stride;
  const int lo = p.sink, hi = L - p.recent, m = p.keep - p.sink - p.recent;
  for (int i = tid; i < lo; i += NT) index[i] = i;
  for (int i = tid; i < p.recent; i += NT) index[lo + m + i] = hi + i;
  if (m == 0) return;
  auto key = [&](int t) { return KEPT ? keys[t - lo] : order(w[t]); };
  // key of rank m among the middle tokens: prefix holds its decided high bits
  uint32_t prefix = 0, need = (uint32_t)m;
  int shift = 32;
  for (int d = 0; d < 3; ++d) {
    const int bits = d < 2 ? BITS : 32 - 2 * BITS;
    shift -= bits;
    for (int i = tid; i < BINS; i += NT) hist[i] = 0;
    __syncthreads();
    constexpr int G = 8;
    for (int base = lo; base < hi; base += G * NT) {
      uint32_t k[G];
#pragma unroll
      for (int q = 0; q < G; ++q) {
        const int t = base + q * NT + tid;
        k[q] = 0;
        if (t < hi) k[q] = d == 0 ? order(w[t]) : key(t);
      }
#pragma unroll
      for (int q = 0; q < G; ++q) {
        const int t = base + q * NT + tid;
        if (KEPT && d == 0 && t < hi) keys[t - lo] = k[q];
        const bool in = t < hi && (d == 0 || (k[q] >> (shift + bits)) == prefix);
        const uint32_t digit = (k[q] >> shift) & ((1u << bits) - 1);
        if (in) atomicAdd(&hist[digit], 1u);
      }
    }
    __syncthreads();
    // the digit whose count from above first reaches `need`: thread i holds bins 2i and 2i + 1
    {
      const int b1 = BINS - 1 - 2 * tid, b0 = b1 - 1;   // descending
      const uint32_t c1 = hist[b1], c0 = hist[b0];
      const int incl = wave_incl_sum((int)(c1 + c0));
      if (lane == 63) wave_sum[wave] = incl;
      __syncthreads();
      int before = 0;
      for (int q = 0; q < wave; ++q) before += wave_sum[q];
      const uint32_t above = (uint32_t)(before + incl) - c1 - c0;
      if (above < need && need <= above + c1) {
        sh_digit = (uint32_t)b1;
        sh_need = need - above;
      } else if (above + c1 < need && need <= above + c1 + c0) {
        sh_digit = (uint32_t)b0;
        sh_need = need - above - c1;
      }
      __syncthreads();
    }
    prefix = (prefix << bits) | sh_digit;
    need = sh_need;
    __syncthreads();
  }
  // keys above `prefix` are kept, and the first `need` tokens equal to it
  const int run = ((hi - lo + NW - 1) / NW + 63) / 64 * 64;
  const int r0 = lo + wave * run, r1 = r0 + run < hi ? r0 + run : hi;
  int gt = 0, eq = 0;
  for (int base = r0; base < r1; base += 256) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int t = base + 64 * q + lane;
      const uint32_t k = t < r1 ? key(t) : 0;
      gt += __builtin_popcountll(__builtin_amdgcn_ballot_w64(t < r1 && k > prefix));
      eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(t < r1 && k == prefix));
    }
  }
  if (lane == 0) {
    wave_gt[wave] = gt;
    wave_eq[wave] = eq;
  }
  __syncthreads();
  int eq0 = 0, at = lo;
  for (int q = 0; q < wave; ++q) {
    const int took = min(wave_eq[q], max(0, (int)need - eq0));
    eq0 += wave_eq[q];
    at += wave_gt[q] + took;
  }
  for (int base = r0; base < r1; base += 64) {
    const int t = base + lane;
    const uint32_t k = t < r1 ? key(t) : 0;
    const uint64_t me = __builtin_amdgcn_ballot_w64(t < r1 && k == prefix);
    const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(me >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)me, 0));
    const bool take = t < r1 && (k > prefix || (k == prefix && eq0 + below < (int)need));
    const uint64_t mt = __builtin_amdgcn_ballot_w64(take);
    const int place = __builtin_amdgcn_mbcnt_hi((uint32_t)(mt >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mt, 0));
    if (take) index[at + place] = t;
    at += __builtin_popcountll(mt);
    eq0 += __builtin_popcountll(me);
  }
}

// Byte offset of token `tok` of request b in pages `table`, or -1 (and `bad` set) outside them.
__device__ __forceinline__ int64_t row_at(const EParams& e, const int* table, int64_t stride, int cols, int b, int tok, int& bad) {
  const qmla_evict_params& p = e.p;
  if (tok < 0) {
    bad = 1;
    return -1;
  }
  const int pg = (int)magic_div((uint32_t)tok, e.page_mul, e.page_sh);
  if (pg >= cols) {
    bad = 1;
    return -1;
  }
  const int id = table[b * stride + pg];
  if ((uint32_t)id >= (uint32_t)p.num_pages) {
    bad = 1;
    return -1;
  }
  return id * p.page_stride + (int64_t)(tok - pg * p.page_size) * p.token_stride;
}

// Out of place: a workgroup copies MR rows of request blockIdx.y, looked up once, MU units a thread under way together.
// What it moves is not read again here, so past the caches. Bound by the copy rate: 40 requests, 522 MB of 1200-byte rows,
// 104 us (a thread a unit that looks its row up itself 143 us).
constexpr int MR = 32, MU = 4;
template <class V>
__global__ __launch_bounds__(256) void move_kernel(const EParams e) {
  __shared__ int64_t from[MR], to[MR];
  const qmla_evict_params& p = e.p;
  const int b = blockIdx.y, i0 = blockIdx.x * MR, tid = threadIdx.x;
  const int rows = min(min(max(p.counts[b], 0), p.keep) - i0, MR);
  if (rows <= 0) return;
  if (tid < rows) {
    const int tok = p.index[b * p.index_stride + i0 + tid], at = (p.first ? p.first[b] : 0) + i0 + tid;
    int bad = 0;
    const int64_t s = row_at(e, p.block_table, p.bt_stride, p.bt_cols, b, tok, bad);
    to[tid] = row_at(e, p.dst_block_table, p.dst_bt_stride, p.dst_bt_cols, b, at, bad);
    from[tid] = to[tid] < 0 ? -1 : s;
    if (p.weights_out && (uint32_t)tok < (uint32_t)p.width && (uint32_t)at < (uint32_t)p.weights_out_width)
      p.weights_out[b * p.weights_out_stride + at] = p.weights[b * p.weights_stride + tok];
    if (bad && p.status) *p.status = QMLA_ERR_PAGE;
  }
  __syncthreads();
  const uint32_t units = (uint32_t)rows * (uint32_t)e.chunks;
  for (uint32_t u0 = tid; u0 < units; u0 += 256u * MU) {
    V v[MU];
    int64_t d[MU];
#pragma unroll
    for (int q = 0; q < MU; ++q) {
      const uint32_t u = u0 + 256u * q, r = u < units ? magic_div(u, e.chunk_mul, e.chunk_sh) : 0, c = u - r * e.chunks;
      const int64_t s = u < units ? from[r] : -1;
      d[q] = s < 0 ? -1 : to[r] + (int64_t)c * (int)sizeof(V);
      if (s >= 0) v[q] = __builtin_nontemporal_load((const V*)((const char*)p.cache + s) + c);
    }
#pragma unroll
    for (int q = 0; q < MU; ++q)
      if (d[q] >= 0) __builtin_nontemporal_store(v[q], (V*)((char*)p.cache + d[q]));
  }
}

// In place: one workgroup owns CW units of every row of a request (blockIdx.x names them; the last
// x owns the weights) and takes the rows in ascending order, STEP at a time: all their loads, a barrier,
// their stores. A kept token moves down or stays, so a store of one step meets no load of a later one,
// and no two workgroups touch the same bytes.
constexpr int CW = 4, RPT = 8, STEP = NT / CW * RPT;
template <class V>
__global__ __launch_bounds__(NT) void move_in_place_kernel(const EParams e) {
  const qmla_evict_params& p = e.p;
  const int b = blockIdx.y, tid = threadIdx.x;
  const int n = min(max(p.counts[b], 0), p.keep);
  const int first = p.first ? p.first[b] : 0;
  const int* index = p.index + b * p.index_stride;
  if ((int)blockIdx.x * CW >= e.chunks) {
    if (!p.weights_out) return;
    for (int i0 = 0; i0 < n; i0 += NT) {
      const int i = i0 + tid, to = first + i;
      const int tok = i < n ? index[i] : -1;
      const bool ok = (uint32_t)tok < (uint32_t)p.width && (uint32_t)to < (uint32_t)p.weights_out_width;
      const float v = ok ? p.weights[b * p.weights_stride + tok] : 0.f;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (ok) p.weights_out[b * p.weights_out_stride + to] = v;
    }
    return;
  }
  const int c = (int)blockIdx.x * CW + tid % CW;
  int bad = 0;
  for (int i0 = 0; i0 < n; i0 += STEP) {
    V v[RPT];
    int64_t d[RPT];
#pragma unroll
    for (int q = 0; q < RPT; ++q) {
      const int i = i0 + q * (NT / CW) + tid / CW;
      d[q] = -1;
      if (i < n && c < e.chunks) {
        const int tok = index[i];
        if (tok != first + i) {
          const int64_t s = row_at(e, p.block_table, p.bt_stride, p.bt_cols, b, tok, bad);
          const int64_t to = row_at(e, p.block_table, p.bt_stride, p.bt_cols, b, first + i, bad);
          if (s >= 0 && to >= 0) {
            v[q] = *((const V*)((const char*)p.cache + s) + c);
            d[q] = to;
          }
        }
      }
    }
    // every load of the step has landed before any store of it
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int q = 0; q < RPT; ++q)
      if (d[q] >= 0) *((V*)((char*)p.cache + d[q]) + c) = v[q];
  }
  if (bad && p.status) *p.status = QMLA_ERR_PAGE;
}

static int check(const qmla_evict_params* p) {
  if (!p) return QMLA_ERR_NULL;
  if (p->requests < 0 || p->width < 0 || p->keep < 0) return QMLA_ERR_SHAPE;
  if (p->requests > 65535) return QMLA_ERR_SHAPE;
  return QMLA_OK;
}

}  // namespace ev
}  // namespace qmla

using namespace qmla;

extern "C" {

int qmla_evict_select(const qmla_evict_params* p, void* stream) {
  const int rc = ev::check(p);
  if (rc) return rc;
  if (p->sink < 0 || p->recent < 0 || (int64_t)p->sink + p->recent > p->keep) return QMLA_ERR_SHAPE;
  if (p->requests == 0) return QMLA_OK;
  if (!p->seq_lens || !p->counts || (p->keep > 0 && !p->index) || (p->width > p->keep && !p->weights)) return QMLA_ERR_NULL;
  ev::EParams e{};
  e.p = *p;
  void* args[] = {&e};
  // the middle tokens of the longest request
  const int64_t most = (int64_t)p->width - p->sink - p->recent;
  const bool kept = most <= ev::KEYS;
  const int bytes = kept && most > 0 ? (int)most * 4 : 0;
  const void* fn = kept ? (const void*)&ev::select_kernel<true> : (const void*)&ev::select_kernel<false>;
  if (bytes > 48 * 1024 && hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return QMLA_ERR_LAUNCH;
  const hipError_t r = hipLaunchKernel(fn, dim3(p->requests), dim3(ev::NT), args, bytes, (hipStream_t)stream);
  return r == hipSuccess ? QMLA_OK : QMLA_ERR_LAUNCH;
}

int qmla_cache_compact(const qmla_evict_params* p, void* stream) {
  const int rc = ev::check(p);
  if (rc) return rc;
  if (p->page_size <= 0 || p->num_pages < 0 || p->row_bytes <= 0 || p->bt_cols < 0 || (p->dst_block_table && p->dst_bt_cols < 0) ||
      p->row_bytes > (1 << 20))
    return QMLA_ERR_SHAPE;
  if (p->row_bytes > p->token_stride && p->page_size > 1) return QMLA_ERR_SHAPE;
  if (p->requests == 0 || p->keep == 0) return QMLA_OK;
  if (!p->cache || !p->index || !p->counts || !p->block_table || (p->weights_out && !p->weights)) return QMLA_ERR_NULL;
  const uint64_t bits = (uint64_t)(uintptr_t)p->cache | (uint64_t)p->page_stride | (uint64_t)p->token_stride | (uint64_t)p->row_bytes;
  const int v = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
  ev::EParams e{};
  e.p = *p;
  e.chunks = (int)(p->row_bytes / v);
  page_magic(p->page_size, e.page_mul, e.page_sh);
  page_magic(e.chunks, e.chunk_mul, e.chunk_sh);
  const bool in_place = !p->dst_block_table;
  if ((int64_t)p->keep * e.chunks > 0x7fffffff - 256) return QMLA_ERR_SHAPE;
  const void* fn = v == 16  ? (in_place ? (const void*)&ev::move_in_place_kernel<i32x4> : (const void*)&ev::move_kernel<i32x4>)
                   : v == 4 ? (in_place ? (const void*)&ev::move_in_place_kernel<int> : (const void*)&ev::move_kernel<int>)
                   : v == 2 ? (in_place ? (const void*)&ev::move_in_place_kernel<short> : (const void*)&ev::move_kernel<short>)
                            : (in_place ? (const void*)&ev::move_in_place_kernel<char> : (const void*)&ev::move_kernel<char>);
  const uint32_t gx = in_place ? (e.chunks + ev::CW - 1) / ev::CW + 1 : (p->keep + ev::MR - 1) / ev::MR;
  void* args[] = {&e};
  const hipError_t r = hipLaunchKernel(fn, dim3(gx, p->requests), dim3(in_place ? ev::NT : 256), args, 0, (hipStream_t)stream);
  return r == hipSuccess ? QMLA_OK : QMLA_ERR_LAUNCH;
}

}  // extern "C"
