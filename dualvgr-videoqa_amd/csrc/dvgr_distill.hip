// dvgr_distill.hip -- include/dvgr_head.h: distillation from a teacher's top logits, value and gradient.
//
//   p = softmax over the K listed entries of v / T         q = softmax over the C classes of z / T
//   loss_r = T^2 sum_k p_k (log p_k - log q_{i_k})         d loss_r / d z_j = T (q_j - sum_{k : i_k = j} p_k)
//
// Bound by memory: the forward reads the logits once (running maximum and sum), the backward reads them once more and writes the
// gradient; the lists are small.  Everything is fp32; the gradient is rounded to the logits' type where it is stored.  4096 x 32000 bf16:
// 51 us forward (5.2 TB/s, see kKeep), 96 us backward (5.5 TB/s of reads and writes).
#include <hip/hip_runtime.h>

#include "../../include/dvgr.h"
#include "../../include/dvgr_head.h"
#include "dvgr_elem.h"

namespace dvgr {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxK = DVGR_DISTILL_MAX_K;
// The backward takes the rows from the last one on: what the forward read last, and not as a stream, is still in the 256 MB cache.  The
// gradients that it writes take room too.  Forward and backward of 4096 x 32000 bf16 / 1023 x 100003 fp16: 152 / 134 us with streams alone,
// 153 / 122 with 96 MB kept, 147 / 117 with 160, 149 / 118 with 232.
constexpr int64_t kKeep = 160000000;

struct Distill {
  const void *z, *v;
  const int64_t* idx;
  int64_t ldz, R, C;
  int K, elem_v, splits;
  int64_t per;                     // classes a split owns (multiple of 16 elements)
  float invT, T;
};

// Per row, for the backward: {max of z, log2 sum of exp((z - max) / T), the same of v}; a row without entries has a maximum of -inf for v
// and neither loss nor gradient.
struct RowStats { float zmax, zlog, vmax, vlog; };

// Running maximum and sum of exp((x - max) / T) = 2^((x - max) c); a maximum of -inf holds nothing.  The maximum is one of the numbers
// themselves and is taken off before the scaling: x c rounded would be off by more than an exponential bears from |x c| = 2^31 on.
struct MaxSum {
  float m = -INFINITY, l = 0.f;
  __device__ __forceinline__ void join(float m2, float l2, float c) {
    const float mn = fmaxf(m, m2);
    if (mn == -INFINITY) { l += l2; return; }                       // (l, l2: 0, or NaN)
    l = l * exp2_fast((m - mn) * c) + l2 * exp2_fast((m2 - mn) * c);
    m = mn;
  }
  template <int N> __device__ __forceinline__ void add(const float (&f)[N], float c) {
    float mx = f[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mx = fmaxf(mx, f[i]);
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += exp2_fast((f[i] - ref) * c);
    l = l * exp2_fast((m - ref) * c) + s;
    m = mn;
  }
};

__device__ __forceinline__ MaxSum wave_join(MaxSum a, float c) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const float m2 = __shfl_xor(a.m, d), l2 = __shfl_xor(a.l, d);
    a.join(m2, l2, c);
  }
  return a;
}

// The elements [c0, c1) of a row, by threads `tid` of kThreads: kUnroll 16-byte vectors at a time (as many loads in flight), single elements
// at the ends (rows of an odd number of classes start at any alignment).
constexpr int kUnroll = 4;
template <typename T, typename FU, typename FE>
__device__ __forceinline__ void for_row(const T* row, int64_t c0, int64_t c1, int tid, FU many, FE one) {
  constexpr int N = Vec16<T>::N;
  const int64_t lead = ((16 - ((uintptr_t)(row + c0) & 15)) & 15) / sizeof(T);
  const int64_t a = c0 + lead < c1 ? c0 + lead : c1;
  const int64_t e = a + (c1 - a) / N * N;
  for (int64_t c = c0 + tid; c < a; c += kThreads) one(c);
  for (int64_t c = a + (int64_t)tid * N; c < e; c += kUnroll * kThreads * N) many(c, e);
  for (int64_t c = e + tid; c < c1; c += kThreads) one(c);
}

template <typename T, bool STREAM>
__device__ __forceinline__ MaxSum row_part(const T* row, int64_t c0, int64_t c1, float c, float (&sh)[8]) {
  MaxSum s;
  constexpr int N = Vec16<T>::N;
  for_row(row, c0, c1, threadIdx.x, [&](int64_t at, int64_t e) {
            typename Vec16<T>::type v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
              const int64_t x = at + (int64_t)u * kThreads * N;
              const typename Vec16<T>::type* p = reinterpret_cast<const typename Vec16<T>::type*>(row + x);
              if (x < e) v[u] = STREAM ? stream_load(p) : *p;
              else v[u] = (T)-INFINITY;
            }
            float f[kUnroll * N];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
#pragma unroll
              for (int i = 0; i < N; ++i) f[u * N + i] = (float)v[u][i];
            s.add(f, c);
          },
          [&](int64_t at) { float f[1] = {(float)row[at]}; s.add(f, c); });
  s = wave_join(s, c);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) { sh[2 * wave] = s.m; sh[2 * wave + 1] = s.l; }
  __syncthreads();
  s.m = sh[0]; s.l = sh[1];
  for (int w = 1; w < kThreads / 64; ++w) s.join(sh[2 * w], sh[2 * w + 1], c);
  return s;
}

__device__ __forceinline__ int entry(const Distill& d, int64_t r, int k, float& v) {        // class of entry k, or -1
  const int64_t i = d.idx[r * d.K + k];
  if (i < 0 || i >= d.C) return -1;
  v = load_elem(d.v, r * d.K + k, d.elem_v);
  return (int)i;
}

// One wave: the teacher's side of a row, up to kHeld entries for each lane.  `fetch` is called before the row is streamed, so that its
// three dependent loads are in flight meanwhile; longer lists load the rest in `finish`.
constexpr int kHeld = 4;
template <typename T> struct Entries {
  float v[kHeld], z[kHeld];
  static __device__ __forceinline__ void one(const Distill& d, int64_t r, int k, float& v, float& z) {
    v = -INFINITY; z = 0.f;
    const int i = k < d.K ? entry(d, r, k, v) : -1;
    if (i >= 0) z = (float)((const T*)d.z)[r * d.ldz + i];
  }
  __device__ __forceinline__ void fetch(const Distill& d, int64_t r, int lane) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) one(d, r, lane + 64 * i, v[i], z[i]);
  }
  __device__ __forceinline__ void finish(const Distill& d, int64_t r, const MaxSum& s, float* loss, RowStats* stats, int lane) const {
    const float c = d.invT * kLog2e, zlog = __log2f(s.l);
    MaxSum t;
    t.add(v, c);
    for (int k = lane + 64 * kHeld; k < d.K; k += 64) {
      float x[1], y;
      one(d, r, k, x[0], y);
      t.add(x, c);
    }
    t = wave_join(t, c);
    if (t.l != t.l) t.m = t.l;                                      // a NaN among the values is the row's loss
    float sum = 0.f;
    if (t.m != -INFINITY) {
      const float vlog = __log2f(t.l);
      const auto add = [&](float x, float y) {
        if (x == -INFINITY) return;                                 // p = 0 adds nothing, whatever the student says there
        const float logp = fmaf(x - t.m, c, -vlog), logq = fmaf(y - s.m, c, -zlog), p = exp2_fast(logp);
        if (p != 0.f) sum += p * (logp - logq);
      };
#pragma unroll
      for (int i = 0; i < kHeld; ++i) add(v[i], z[i]);
      for (int k = lane + 64 * kHeld; k < d.K; k += 64) {
        float x, y;
        one(d, r, k, x, y);
        add(x, y);
      }
      sum = wave_sum(sum);
      t.l = vlog;
    }
    if (lane == 0) {
      loss[r] = sum * kLn2 * d.T * d.T;
      stats[r] = RowStats{s.m, zlog, t.m, t.l};
    }
  }
};

// splits == 1: a workgroup per row does everything.  Otherwise (few rows, many classes) it leaves its share's maximum and sum.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_distill_row(Distill d, float* loss, RowStats* stats, float2* part) {
  __shared__ float sh[8];
  const int64_t r = blockIdx.x / d.splits, c0 = (blockIdx.x % d.splits) * d.per, c1 = c0 + d.per < d.C ? c0 + d.per : d.C;
  Entries<T> e;
  if (d.splits == 1 && threadIdx.x < 64) e.fetch(d, r, threadIdx.x);
  const T* row = (const T*)d.z + r * d.ldz;
  const MaxSum s = (d.R - r) * d.C * (int64_t)sizeof(T) > kKeep ? row_part<T, true>(row, c0, c1, d.invT * kLog2e, sh)
                                                                : row_part<T, false>(row, c0, c1, d.invT * kLog2e, sh);
  if (d.splits > 1) {
    if (threadIdx.x == 0) part[blockIdx.x] = make_float2(s.m, s.l);
  } else if (threadIdx.x < 64) e.finish(d, r, s, loss, stats, threadIdx.x);
}

template <typename T>
__global__ __launch_bounds__(64) void k_distill_join(Distill d, const float2* part, float* loss, RowStats* stats) {
  const int64_t r = blockIdx.x;
  Entries<T> e;
  e.fetch(d, r, threadIdx.x);
  MaxSum s;
  const float c = d.invT * kLog2e;
  for (int i = threadIdx.x; i < d.splits; i += 64) s.join(part[r * d.splits + i].x, part[r * d.splits + i].y, c);
  e.finish(d, r, wave_join(s, c), loss, stats, threadIdx.x);
}

// the sum of the rows' losses (/ number of rows that have an entry); behind the rows' statistics, the factor of a row's gradient
__global__ __launch_bounds__(1024) void k_distill_total(const float* loss, RowStats* stats, int64_t R, int mean, float* total) {
  __shared__ double sh[16];
  __shared__ double shn[16];
  double a = 0.0, n = 0.0;
  for (int64_t r = threadIdx.x; r < R; r += 1024) {
    a += loss[r];
    n += stats[r].vmax == -INFINITY ? 0.0 : 1.0;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) { a += __shfl_xor(a, o); n += __shfl_xor(n, o); }
  if ((threadIdx.x & 63) == 0) { sh[threadIdx.x >> 6] = a; shn[threadIdx.x >> 6] = n; }
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) { a += sh[w]; n += shn[w]; }
  const double f = mean ? (n > 0.0 ? 1.0 / n : 0.0) : 1.0;
  *total = (float)(a * f);
  stats[R].zmax = (float)f;
}

// SAME: z and its gradient have the same alignment, row by row; otherwise elements are written one by one (4096 rows of 50257 classes, bf16,
// forward and backward: 399 us as a slice of rows of 50304, 230 us for dense rows of 50304).  A share is written densely first; the classes the teacher lists
// are then written again with their p, which needs no atomics: entries of the same class all write the same sum.
template <typename T, bool SAME>
__global__ __launch_bounds__(kThreads) void k_distill_bwd(Distill d, const RowStats* stats, const float* up, int up_stride, T* __restrict__ gz, int64_t ldg) {
  __shared__ int32_t sh_i[kMaxK];
  __shared__ float sh_p[kMaxK];
  const int tid = threadIdx.x;
  const unsigned w = gridDim.x - 1 - blockIdx.x;                      // (from the last row on)
  const int64_t r = w / d.splits, c0 = (w % d.splits) * d.per, c1 = c0 + d.per < d.C ? c0 + d.per : d.C;
  const RowStats s = stats[r];
  const T* __restrict__ row = (const T*)d.z + r * d.ldz;
  T* out = gz + r * ldg;
  const float c = d.invT * kLog2e;
  const bool empty = s.vmax == -INFINITY;
  const float f = empty ? 0.f : (up_stride ? up[r] : *up * stats[d.R].zmax) * d.T;
  const auto grad = [&](float z) { return empty ? 0.f : f * exp2_fast(fmaf(z - s.zmax, c, -s.zlog)); };
  for (int k = tid; k < d.K; k += kThreads) {
    float v = -INFINITY;
    const int i = entry(d, r, k, v);
    sh_i[k] = i;
    sh_p[k] = i < 0 || empty ? 0.f : exp2_fast(fmaf(v - s.vmax, c, -s.vlog));
  }
  if (SAME)
    for_row(row, c0, c1, tid, [&](int64_t at, int64_t e) {
      constexpr int N = Vec16<T>::N;
      typename Vec16<T>::type v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (at + (int64_t)u * kThreads * N < e) v[u] = *reinterpret_cast<const typename Vec16<T>::type*>(row + at + (int64_t)u * kThreads * N);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (at + (int64_t)u * kThreads * N >= e) break;
        float g[N];
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = grad((float)v[u][i]);
        stream_store_vec(out + at + (int64_t)u * kThreads * N, g);
      }
    }, [&](int64_t at) { out[at] = (T)grad((float)row[at]); });
  else
    for (int64_t at = c0 + tid; at < c1; at += kThreads) out[at] = (T)grad((float)row[at]);
  __syncthreads();
  for (int k = tid; k < d.K; k += kThreads) {
    const int i = sh_i[k];
    if (i < c0 || i >= c1) continue;
    float p = 0.f;
    for (int j = 0; j < d.K; ++j) p += sh_i[j] == i ? sh_p[j] : 0.f;
    out[i] = (T)(grad((float)row[i]) - f * p);
  }
}

// Few rows of many classes are split until there are about 1024 workgroups, four for each compute unit, but no share is under 8192
// classes; a split of two is not worth the launch that joins it while there are 512 rows.
int split_of(int64_t R, int64_t C, int64_t& per) {
  int64_t s = R >= 512 ? 1 : (1024 + R - 1) / R, most = (C + 8191) / 8192;
  s = s < most ? s : most;
  per = ((C + s - 1) / s + 15) / 16 * 16;
  return (int)((C + per - 1) / per);
}

int check(int64_t R, int64_t C, int64_t ldz, int elem, int elem_v, int K, float T) {
  if (!elem_size(elem) || !elem_size(elem_v)) return DVGR_E_KIND;
  if (R < 0 || R >= (1ll << 22) || C < 1 || C >= (1ll << 31) - 64 || ldz < C || K < 1 || K > kMaxK ||
      !(T >= 1e-6f && T <= 1e6f))
    return DVGR_E_DIMS;
  return 0;
}

Distill problem(const void* z, int64_t ldz, int64_t R, int64_t C, const void* v, int elem_v, const int64_t* idx, int K, float T) {
  Distill d{z, v, idx, ldz, R, C, K, elem_v, 1, 0, 1.f / T, T};
  d.splits = split_of(R, C, d.per);
  return d;
}

template <typename T>
int forward(const Distill& d, float* loss, RowStats* stats, float2* part, hipStream_t st) {
  DVGR_LAUNCH((k_distill_row<T>), dim3((unsigned)(d.R * d.splits)), dim3(kThreads), 0, st, d, loss, stats, part);
  if (d.splits > 1) DVGR_LAUNCH((k_distill_join<T>), dim3((unsigned)d.R), dim3(64), 0, st, d, part, loss, stats);
  return (int)hipGetLastError();
}

template <typename T>
int backward(const Distill& d, const RowStats* stats, const float* up, int up_stride, T* gz, int64_t ldg, hipStream_t st) {
  const bool same = (((uintptr_t)d.z ^ (uintptr_t)gz) & 15) == 0 && ((d.ldz - ldg) * (int64_t)sizeof(T)) % 16 == 0;
  const dim3 grid((unsigned)(d.R * d.splits));
  if (same) DVGR_LAUNCH((k_distill_bwd<T, true>), grid, dim3(kThreads), 0, st, d, stats, up, up_stride, gz, ldg);
  else DVGR_LAUNCH((k_distill_bwd<T, false>), grid, dim3(kThreads), 0, st, d, stats, up, up_stride, gz, ldg);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace dvgr

using namespace dvgr;

extern "C" {

size_t dvgr_distill_workspace_bytes(int64_t R, int64_t C) {
  if (R < 1 || C < 1 || R >= (1ll << 22) || C >= (1ll << 31) - 64) return 0;
  int64_t per;
  const int s = split_of(R, C, per);
  return s > 1 ? (size_t)R * s * sizeof(float2) : 0;
}

int dvgr_distill_forward(const void* logits, int64_t ld, int elem, int64_t R, int64_t C, const void* values, int elem_values, const int64_t* indices,
                         int K, float temperature, int reduction, float* loss_rows, float* total, float* stats, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const int e = check(R, C, ld, elem, elem_values, K, temperature);
  if (e) return e;
  if (reduction < DVGR_DISTILL_NONE || reduction > DVGR_DISTILL_MEAN) return DVGR_E_KIND;
  if (!stats || (reduction && !total) || (R && (!logits || !values || !indices || !loss_rows))) return DVGR_E_NULL;
  const size_t need = dvgr_distill_workspace_bytes(R, C);
  if (need && !workspace) return DVGR_E_NULL;
  if (workspace_bytes < need) return DVGR_E_WORKSPACE;
  if (!ptr16(stats) || !ptr16(workspace) || ((uintptr_t)logits % elem_size(elem)) || ((uintptr_t)values % elem_size(elem_values))) return DVGR_E_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  RowStats* rs = (RowStats*)stats;
  if (R) {
    const Distill d = problem(logits, ld, R, C, values, elem_values, indices, K, temperature);
    const int f = elem == DVGR_ELEM_F32 ? forward<float>(d, loss_rows, rs, (float2*)workspace, st)
                : elem == DVGR_ELEM_BF16 ? forward<bf16_t>(d, loss_rows, rs, (float2*)workspace, st)
                                         : forward<f16_t>(d, loss_rows, rs, (float2*)workspace, st);
    if (f) return f;
  }
  if (reduction) DVGR_LAUNCH(k_distill_total, dim3(1), dim3(1024), 0, st, loss_rows, rs, R, (int)(reduction == DVGR_DISTILL_MEAN), total);
  return (int)hipGetLastError();
}

int dvgr_distill_backward(const void* logits, int64_t ld, int elem, int64_t R, int64_t C, const void* values, int elem_values, const int64_t* indices,
                          int K, float temperature, const float* stats, const float* g_loss, int g_loss_stride, void* g_logits,
                          int64_t ld_g, void* stream) {
  const int e = check(R, C, ld, elem, elem_values, K, temperature);
  if (e) return e;
  if (ld_g < C || g_loss_stride < 0 || g_loss_stride > 1) return DVGR_E_DIMS;
  if (R == 0) return 0;
  if (!logits || !values || !indices || !stats || !g_loss || !g_logits) return DVGR_E_NULL;
  if (!ptr16(stats) || ((uintptr_t)logits % elem_size(elem)) || ((uintptr_t)values % elem_size(elem_values)) || ((uintptr_t)g_logits % elem_size(elem)))
    return DVGR_E_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  const RowStats* rs = (const RowStats*)stats;
  const Distill d = problem(logits, ld, R, C, values, elem_values, indices, K, temperature);
  return elem == DVGR_ELEM_F32 ? backward<float>(d, rs, g_loss, g_loss_stride, (float*)g_logits, ld_g, st)
       : elem == DVGR_ELEM_BF16 ? backward<bf16_t>(d, rs, g_loss, g_loss_stride, (bf16_t*)g_logits, ld_g, st)
                                : backward<f16_t>(d, rs, g_loss, g_loss_stride, (f16_t*)g_logits, ld_g, st);
}

}  // extern "C"
