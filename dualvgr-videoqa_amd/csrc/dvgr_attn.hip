// dvgr_attn.hip -- include/dvgr_attn.h: attention to an encoder's states, forward.
//
// One pass over the keys with the running maximum and sum of the softmax (in powers of two: scale and log2 e are one factor).
// The H / Hk query heads that share a key head are rows of the same tiles, so a key is read once for all of them.  Many rows: a
// workgroup of four waves takes 128 rows and shares tiles of keys in LDS.  Few rows: a workgroup takes 32, its waves go over different
// keys and are joined at the end (dvgr_attn_few.h); the keys are split over workgroups, joined by a second launch, while there are
// few of them.
//
// 2 x 4096 queries over 2048 to 4096 keys, 16 / 4 heads of 128, bf16: 250 to 280 us from card to card, 850 TFLOP/s of products (a large matrix
// product: 1198).  Nothing is full there: matrix units 38 % of the time, LDS 33 % (10 of them conflicts), vector arithmetic about as long as the
// products, while a wave goes through product, softmax, product and two of a SIMD overlap a part of it.  2 x 1024 x 1024, 16 heads of 64,
// fp32: 82 us, matrix units 60 %.  64 x 15 queries over 1024 masked keys, 8 heads of 96, bf16: 32 us, 4.7 TB/s.  One query over
// 65536 keys, 32 / 8 heads of 128, bf16: 47 us, 5.7 TB/s, and 4.7 for the join.
#include "dvgr_attn_few.h"

namespace dvgr {
namespace attn {
namespace {

// Many rows: the maximum moves when a tile exceeds it by 2^kSlack in some row, so the accumulators are scaled again a few times in all
// instead of in every other tile.  p is then at most 2^kSlack, and rounded like any other where it would have been 1 exactly (captions over
// long videos, bf16: 292 -> 272 us; the output off by 0.0023 instead of 0.0019, relative, with half a step 0.0039).  Few rows, which wait
// for memory, move it at once.
constexpr float kSlack = 8.f;

struct Max {
  float at = -INFINITY, cm = 0.f;   // a score; c times it, rounded, 0 where there is none
  bool far = false;                 // the same in all lanes
  float slack;                      // in scores
};

// KS 32-key tiles of a wave's online softmax: s in, probabilities out, m, l and o brought to the new maximum
template <int KS, int NT> __device__ __forceinline__ void softmax_tiles(f32x16 (&s)[KS], unsigned long long bits, float c, Max& m, float& l, f32x16 (&o)[NT], int lane) {
  if (bits != (KS == 2 ? ~0ull : 0xffffffffull)) {
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const uint32_t hb = half_bits((uint32_t)(bits >> (32 * i)), lane);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[i][r] = reg_bit(hb, r) ? s[i][r] : -INFINITY;
    }
  }
  float mx = s[0][0];
#pragma unroll
  for (int i = 0; i < KS; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[i][r]);
  mx = half_max(mx);
  if (__any(mx > m.at + m.slack)) {
    const float mn = fmaxf(m.at, mx), cm = mn == -INFINITY ? 0.f : mn * c;
    m.far = any_far(cm);
    const float f = m.at == -INFINITY ? 0.f : exp2_fast(m.far ? (m.at - mn) * c : m.cm - cm);      // nothing summed yet: o and l are 0
    l *= f;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[u][r] *= f;
    m.at = mn;
    m.cm = cm;
  }
  if (m.far) {                                                      // (in front of the exponentials, which stay in one block with the products behind)
    const float at = m.at == -INFINITY ? 0.f : m.at;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[i][r] -= at;
  }
  const float ref = m.far ? 0.f : m.cm;
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[i][r] = exp2_fast(fmaf(s[i][r], c, -ref));
      sum += s[i][r];
    }
    l += sum;
  }
}

// the row's sum as a score: p = 2^(c (s - log_sum)) in the backward; +inf for a row without keys, so that every p is 0
__device__ __forceinline__ float log_sum(const Args& A, float m, float l) { return l == 0.f ? INFINITY : m + __log2f(l) / A.c; }

// a row's output from o (unnormalised), with what its rounding leaves, and its log-sum
template <typename T, int NT> __device__ __forceinline__ void write_row(const Args& A, int b, int hk, int row, const f32x16 (&o)[NT], float m, float l,
                                                                        int first, int step, bool stats, int lane) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  char* out = const_cast<char*>(q_side(A, A.a.o, b, hk).row(row));
  char* lo = lo_row<T>(A, b, hk, row);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t % step != first) continue;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * t + 8 * g + (lane >> 5) * 4;
      if (d >= A.a.Dh) continue;
      const float x[4] = {o[t][4 * g] * inv, o[t][4 * g + 1] * inv, o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv};
      store4<T>(out + d * sizeof(T), x[0], x[1], x[2], x[3]);
      if (lo) store4<T>(lo + d * sizeof(T), x[0] - (float)(T)x[0], x[1] - (float)(T)x[1], x[2] - (float)(T)x[2], x[3] - (float)(T)x[3]);
    }
  }
  if (A.a.lse && lane < 32 && stats) A.a.lse[row_index(A, b, hk, row)] = log_sum(A, m, l);
}

// ---- many rows: W x 32 of them, tiles of KS x 32 keys -----------------------------------------------------------------------------
template <typename T, int DP, int KS, int W>
__global__ __launch_bounds__(64 * W, (sizeof(T) == 2 ? 2 : 1)) void k_attn_fwd(Args A) {
  typedef Tile<T, DP> Tl;
  constexpr int KT = KS * 32, RT = W * 32, NT = Tl::kNT;
  extern __shared__ __align__(16) char lds[];
  char* lk = lds;
  char* lv = lds + Tl::template bytes<KT>();
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int rtiles = (A.rows + RT - 1) / RT;
  const int64_t w = xcd_work((int64_t)A.a.B * A.a.Hk * rtiles, rtiles);
  if (w < 0) return;
  const int rt = (int)(w % rtiles), hk = (int)(w / rtiles % A.a.Hk), b = (int)(w / rtiles / A.a.Hk);
  const int n = key_count(A, b), dhb = A.a.Dh * A.es, tn = (n + KT - 1) / KT;
  const int row = rt * RT + wave * 32 + (lane & 31);
  const bool live = row < A.rows;
  const Side ks = k_side(A, A.a.k, b, hk), vs = k_side(A, A.a.v, b, hk);
  const uint8_t* mask = A.a.mask ? A.a.mask + (int64_t)b * A.a.mask_stride : nullptr;

  Frag<T> qf[Tl::kSteps];
  {
    const char* qr = q_side(A, A.a.q, b, hk).row(live ? row : 0);
#pragma unroll
    for (int s = 0; s < Tl::kSteps; ++s) qf[s] = Tl::gfrag(qr, s, lane, dhb, live);
    settle(qf);
  }
  f32x16 o[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t] = zero16();
  Max m;
  m.slack = kSlack / A.c;
  float l = 0.f;

  Stage<T, DP, KT, 64 * W> sk, sv;
  uint32_t there = 0;                                               // lane j: key j of the next tile
  const auto fetch = [&](int t) {
    sk.fetch(ks, t * KT, n, dhb, tid);
    sv.fetch(vs, t * KT, n, dhb, tid);
    there = key_there(mask, t * KT + lane, lane < KT ? n : 0);
  };
  if (tn) fetch(0);
  for (int t = 0; t < tn; ++t) {
    const unsigned long long bits = __ballot(there != 0);
    __syncthreads();
    sk.template put<Tl::kStride>(lk, bits, tid);
    sv.template put<Tl::kStrideT>(lv, bits, tid);
    __syncthreads();
    if (t + 1 < tn) fetch(t + 1);
    if (!bits) continue;                                            // (uniform over the workgroup)
    f32x16 s[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) s[i] = zero16();
#pragma unroll
    for (int st = 0; st < Tl::kSteps; ++st)
#pragma unroll
      for (int i = 0; i < KS; ++i) s[i] = mma(Tl::frag(lk + i * 32 * Tl::kStride, st, lane), qf[st], s[i]);
    if (sizeof(T) == 2) reads_ahead<KS * Tl::kSteps>();
    softmax_tiles<KS, NT>(s, bits, A.c, m, l, o, lane);
#pragma unroll
    for (int i = 0; i < KS; ++i) mma_tr<DP>(o, lv + i * 32 * Tl::kStrideT, s[i], lane, T());
  }
  l = half_sum(l);
  if (live) write_row<T>(A, b, hk, row, o, m.at, l, 0, 1, true, lane);
}

// ---- 32 rows: KW waves over different keys -----------------------------------------------------------------------------------------
// (Two waves of a SIMD, in two-byte types, keep twice the loads in flight: the queries are read from LDS for it.)
template <typename T, int DP, int KW>
__global__ __launch_bounds__(64 * KW, (sizeof(T) == 2 ? 2 : 1)) void k_attn_few_fwd(Args A) {
  typedef Tile<T, DP> Tl;
  constexpr int NT = Tl::kNT;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, kw = threadIdx.x >> 6;
  char* lq = lds;
  char* lk = lds + Tl::template bytes<32>() + kw * (Tl::template bytes<32>() + Tl::template bytesT<32>());
  char* lv = lk + Tl::template bytes<32>();
  const FewWork f = few_work<KW>(A, kw);
  if (!f.any) return;
  const int dhb = A.a.Dh * A.es, col = lane & 31, row = f.r0 + col;
  const bool live = row < A.rows;
  const Side ks = k_side(A, A.a.k, f.b, f.hk), vs = k_side(A, A.a.v, f.b, f.hk);
  const uint8_t* mask = A.a.mask ? A.a.mask + (int64_t)f.b * A.a.mask_stride : nullptr;

  f32x16 o[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t] = zero16();
  Max mt;
  mt.slack = 0.f;
  float l = 0.f;
  WaveStage<T, DP> sk, sv;
  uint32_t there = 0;
  const auto fetch = [&](int t) {
    sk.fetch(ks, t * 32, f.n, dhb, A.stream, lane);
    sv.fetch(vs, t * 32, f.n, dhb, A.stream, lane);
    there = key_there(mask, t * 32 + (lane & 31), f.n);
  };
  if (f.t0 < f.t1) fetch(f.t0);
  for (int e = threadIdx.x; e < 32 * Tl::kChunks; e += 64 * KW) {
    const int r = e / Tl::kChunks, c = (e % Tl::kChunks) * 16;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (f.r0 + r < A.rows && c < dhb) x = *reinterpret_cast<const uint4*>(q_side(A, A.a.q, f.b, f.hk).row(f.r0 + r) + c);
    *reinterpret_cast<uint4*>(lq + r * Tl::kStride + c) = x;
  }
  __syncthreads();
  for (int t = f.t0; t < f.t1; t += KW) {
    const uint32_t bits = (uint32_t)__ballot(there != 0);              // (lanes 32 + j say the same as lanes j)
    wave_order();
    sk.template put<Tl::kStride>(lk, bits, lane);
    sv.template put<Tl::kStrideT>(lv, bits, lane);
    wave_order();
    if (t + KW < f.t1) fetch(t + KW);
    if (!bits) continue;
    f32x16 s[1] = {zero16()};
#pragma unroll
    for (int st = 0; st < Tl::kSteps; ++st) s[0] = mma(Tl::frag(lk, st, lane), Tl::frag(lq, st, lane), s[0]);
    softmax_tiles<1, NT>(s, bits, A.c, mt, l, o, lane);
    mma_tr<DP>(o, lv, s[0], lane, T());
  }
  l = half_sum(l);
  float m = mt.at;

  if (KW > 1) {                                                     // join the waves
    __syncthreads();
    float* ml = reinterpret_cast<float*>(lds);                      // [wave][m, l][32]
    float* lo = ml + KW * 64;                                       // [wave][t * 16 + r][lane]
    if (lane < 32) { ml[kw * 64 + lane] = m; ml[kw * 64 + 32 + lane] = l; }
    __syncthreads();
    float mj = -INFINITY;
#pragma unroll
    for (int k = 0; k < KW; ++k) mj = fmaxf(mj, ml[k * 64 + col]);
    const float ref = mj == -INFINITY ? 0.f : mj, fac = exp2_fast((m - ref) * A.c);
    l = 0.f;
#pragma unroll
    for (int k = 0; k < KW; ++k) l += ml[k * 64 + 32 + col] * exp2_fast((ml[k * 64 + col] - ref) * A.c);
    m = mj;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) lo[((kw * NT + t) * 16 + r) * 64 + lane] = o[t][r] * fac;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t % KW != kw) continue;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) a += lo[((k * NT + t) * 16 + r) * 64 + lane];
        o[t][r] = a;
      }
    }
  }
  if (!live) return;
  if (A.splits > 1) {
    const int64_t at = (((int64_t)f.b * A.a.Hk + f.hk) * A.splits + f.split) * A.rows + row;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t % KW != kw) continue;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * t + 8 * g + (lane >> 5) * 4;
        if (d < A.a.Dh) *reinterpret_cast<float4*>(A.part_o + at * A.a.Dh + d) = make_float4(o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]);
      }
    }
    if (lane < 32 && kw == 0) *reinterpret_cast<float2*>(A.part_ml + 2 * at) = make_float2(m, l);
    return;
  }
  write_row<T>(A, f.b, f.hk, row, o, m, l, kw, KW, kw == 0, lane);
}

// Join of the shares of the keys: a workgroup per packed row, its waves take every fourth share, kAtOnce of them in flight, and are added
// in order.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(Args A) {
  constexpr int kAtOnce = 8;
  __shared__ float sh[4][132];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = 2 * lane;
  const int row = (int)(blockIdx.x % A.rows), hk = (int)(blockIdx.x / A.rows % A.a.Hk), b = (int)(blockIdx.x / A.rows / A.a.Hk);
  const int64_t at0 = ((int64_t)b * A.a.Hk + hk) * A.splits * A.rows + row;
  float m = -INFINITY, l = 0.f, x = 0.f, y = 0.f;
  for (int s0 = wave; s0 < A.splits; s0 += 4 * kAtOnce) {
    float2 ml[kAtOnce], o[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int s = s0 + 4 * i;
      ml[i] = make_float2(-INFINITY, 0.f);
      o[i] = make_float2(0.f, 0.f);
      if (s < A.splits) {
        ml[i] = *reinterpret_cast<const float2*>(A.part_ml + 2 * (at0 + (int64_t)s * A.rows));
        if (d < A.a.Dh) o[i] = *reinterpret_cast<const float2*>(A.part_o + (at0 + (int64_t)s * A.rows) * A.a.Dh + d);
      }
    }
    float mn = m;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) mn = fmaxf(mn, ml[i].x);
    const float ref = mn == -INFINITY ? 0.f : mn, f0 = exp2_fast((m - ref) * A.c);
    l *= f0; x *= f0; y *= f0;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const float f = exp2_fast((ml[i].x - ref) * A.c);
      l += ml[i].y * f;
      x += o[i].x * f; y += o[i].y * f;
    }
    m = mn;
  }
  sh[wave][d] = x; sh[wave][d + 1] = y;
  if (lane == 0) { sh[wave][128] = l; sh[wave][129] = m; }
  __syncthreads();
  if (wave) return;
  m = fmaxf(fmaxf(sh[0][129], sh[1][129]), fmaxf(sh[2][129], sh[3][129]));
  const float ref = m == -INFINITY ? 0.f : m;
  x = y = l = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = exp2_fast((sh[w][129] - ref) * A.c);
    x += sh[w][d] * f; y += sh[w][d + 1] * f; l += sh[w][128] * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  x *= inv; y *= inv;
  T* out = (T*)q_side(A, A.a.o, b, hk).row(row);
  T* lo = (T*)lo_row<T>(A, b, hk, row);
  if (d < A.a.Dh) {
    out[d] = (T)x; out[d + 1] = (T)y;
    if (lo) { lo[d] = (T)(x - (float)(T)x); lo[d + 1] = (T)(y - (float)(T)y); }
  }
  if (A.a.lse && lane == 0) A.a.lse[row_index(A, b, hk, row)] = log_sum(A, m, l);
}

template <typename T, int DP, int KS, int W> int launch_many(const Args& A, hipStream_t st) {
  const size_t bytes = Tile<T, DP>::template bytes<KS * 32>() + Tile<T, DP>::template bytesT<KS * 32>();
  static std::atomic<uint32_t> asked{0};
  const auto kern = k_attn_fwd<T, DP, KS, W>;
  const int e = allow_lds(reinterpret_cast<const void*>(kern), bytes, asked);
  if (e) return e;
  DVGR_LAUNCH(kern, dim3(xcd_grid((int64_t)A.a.B * A.a.Hk * ((A.rows + W * 32 - 1) / (W * 32)))), dim3(64 * W), bytes, st, A);
  return (int)hipGetLastError();
}
template <typename T, int DP, int KW> int launch_few(const Args& A, hipStream_t st) {
  typedef Tile<T, DP> Tl;
  size_t bytes = (1 + KW) * Tl::template bytes<32>() + KW * Tl::template bytesT<32>();
  const size_t join = KW > 1 ? (size_t)(KW * 64 + KW * Tl::kNT * 16 * 64) * sizeof(float) : 0;
  bytes = bytes > join ? bytes : join;
  static std::atomic<uint32_t> asked{0};
  const auto kern = k_attn_few_fwd<T, DP, KW>;
  int e = allow_lds(reinterpret_cast<const void*>(kern), bytes, asked);
  if (e) return e;
  DVGR_LAUNCH(kern, dim3(xcd_grid((int64_t)A.a.B * A.a.Hk * A.splits * ((A.rows + 31) / 32))), dim3(64 * KW), bytes, st, A);
  e = (int)hipGetLastError();
  if (e || A.splits == 1) return e;
  DVGR_LAUNCH((k_attn_join<T>), dim3((unsigned)((int64_t)A.a.B * A.a.Hk * A.rows)), dim3(256), 0, st, A);
  return (int)hipGetLastError();
}
// (two-byte types take 64 keys a turn, fp32 32: the same bytes)
template <typename T, int DP> int launch_dp(const Args& A, int KW, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (!KW && many_waves((int64_t)A.a.B * A.a.Hk, A.rows, 2) == 8) return launch_many<T, DP, 2, 8>(A, st);
    if (KW == 8) return launch_few<T, DP, 8>(A, st);
  }
  if (!KW) return launch_many<T, DP, sizeof(T) == 4 ? 1 : 2, 4>(A, st);
  return KW == 1 ? launch_few<T, DP, 1>(A, st) : launch_few<T, DP, 4>(A, st);
}
template <typename T> int launch_t(const Args& A, int KW, hipStream_t st) {
  if (A.a.Dh <= 32) return launch_dp<T, 32>(A, KW, st);
  if (A.a.Dh <= 64) return launch_dp<T, 64>(A, KW, st);
  if (A.a.Dh <= 96) return launch_dp<T, 96>(A, KW, st);
  return launch_dp<T, 128>(A, KW, st);
}

struct Parts { FewPlan few; size_t o_bytes, ml_bytes; };
Parts parts(const dvgr_attn_problem& a) {
  Parts p{};
  const int64_t rows = (int64_t)a.Lq * (a.H / a.Hk);
  p.few = few_plan(a, true);
  if (p.few.splits > 1) {
    p.o_bytes = (size_t)a.B * a.Hk * p.few.splits * rows * a.Dh * sizeof(float);          // (rows of 8 floats at least: 16-byte aligned)
    p.ml_bytes = (size_t)a.B * a.Hk * p.few.splits * rows * 2 * sizeof(float);
  }
  return p;
}

bool view_ok(const dvgr_attn_view& v, int es, int64_t B, int64_t L, int64_t H) {
  const auto bad = [es](int64_t s) { return (s * es) % 16 != 0; };
  return ptr16(v.p) && v.sl >= 0 && v.sl * es < (1ll << 32) && !(B > 1 && bad(v.sb)) && !(L > 1 && bad(v.sl)) && !(H > 1 && bad(v.sh));
}

int check(const dvgr_attn_problem* a) {
  if (!a) return DVGR_E_NULL;
  if (!elem_size(a->elem)) return DVGR_E_KIND;
  if (a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->H < 1 || a->Hk < 1 || a->H % a->Hk || a->Dh < 8 || a->Dh > 128 || a->Dh % 8) return DVGR_E_DIMS;
  if (!(a->scale >= 1e-30f) || !(a->scale <= 1e30f)) return DVGR_E_DIMS;
  const int64_t rows = (int64_t)a->Lq * (a->H / a->Hk), heads = (int64_t)a->B * a->Hk;
  // packed rows and keys are 32-bit numbers, a launch holds fewer than 2^32 threads (256 for 64 rows; 512 for 128 keys, workgroups rounded
  // up to a multiple of 8)
  if (rows >= (1ll << 30) || a->Lk >= (1 << 30) || heads >= (1ll << 22)) return DVGR_E_DIMS;
  if (heads * (rows / 64 + 1) >= (1ll << 24) || heads * (a->Lk / 128 + 1) > (1ll << 23) - 8) return DVGR_E_DIMS;
  return 0;
}
bool empty(const dvgr_attn_problem& a) { return a.B == 0 || a.Lq == 0; }
int check_forward_views(const dvgr_attn_problem& a) {
  const int es = elem_size(a.elem);
  if (empty(a)) return 0;
  if (!a.q.p || !a.o.p || (a.Lk && (!a.k.p || !a.v.p))) return DVGR_E_NULL;
  if (!view_ok(a.q, es, a.B, a.Lq, a.H) || !view_ok(a.o, es, a.B, a.Lq, a.H)) return DVGR_E_ALIGN;
  if (!ptr16(a.o_lo)) return DVGR_E_ALIGN;
  if (a.Lk && (!view_ok(a.k, es, a.B, a.Lk, a.Hk) || !view_ok(a.v, es, a.B, a.Lk, a.Hk))) return DVGR_E_ALIGN;
  return 0;
}

}  // namespace

Args make_args(const dvgr_attn_problem& a) {
  Args A{};
  A.a = a;
  A.G = a.H / a.Hk;
  A.shift = (A.G & (A.G - 1)) == 0 ? __builtin_ctz(A.G) : -1;
  A.rows = a.Lq * A.G;
  A.es = elem_size(a.elem);
  A.splits = A.tiles_per_split = 1;
  A.c = a.scale * kLog2e;
  return A;
}

}  // namespace attn
}  // namespace dvgr

using namespace dvgr;
using namespace dvgr::attn;

extern "C" {

int dvgr_attn_check(const dvgr_attn_problem* a) { return check(a); }

size_t dvgr_attn_forward_workspace_bytes(const dvgr_attn_problem* a) {
  if (check(a) || empty(*a)) return 0;
  const Parts p = parts(*a);
  return p.o_bytes + p.ml_bytes;
}
size_t dvgr_attn_backward_workspace_bytes(const dvgr_attn_problem* a) { return check(a) ? 0 : backward_bytes(*a); }

int dvgr_attn_forward(const dvgr_attn_problem* a, void* workspace, size_t workspace_bytes, void* stream) {
  int e = check(a);
  if (e) return e;
  e = check_forward_views(*a);
  if (e || empty(*a)) return e;
  Args A = make_args(*a);
  const Parts p = parts(*a);
  if (p.o_bytes) {
    if (!workspace) return DVGR_E_NULL;
    if (workspace_bytes < p.o_bytes + p.ml_bytes) return DVGR_E_WORKSPACE;
    if (!ptr16(workspace)) return DVGR_E_ALIGN;
  }
  if (p.few.KW) {
    A.splits = p.few.splits;
    A.tiles_per_split = p.few.tiles_per_split;
  }
  // One word at a time over states that no cache holds (256 MB): 63 -> 51 us for 268 MB; smaller ones stay where the next word finds them.
  A.stream = !a->lse && (double)a->B * a->Lk * a->Hk * a->Dh * A.es * 2 > 256e6;
  A.part_o = (float*)workspace;
  A.part_ml = (float*)((char*)workspace + p.o_bytes);
  hipStream_t st = (hipStream_t)stream;
  return a->elem == DVGR_ELEM_F32 ? launch_t<float>(A, p.few.KW, st) : a->elem == DVGR_ELEM_BF16 ? launch_t<bf16_t>(A, p.few.KW, st)
                                                                                               : launch_t<f16_t>(A, p.few.KW, st);
}

int dvgr_attn_backward(const dvgr_attn_problem* a, const dvgr_attn_grads* g, void* workspace, size_t workspace_bytes, void* stream) {
  int e = check(a);
  if (e) return e;
  if (!g) return DVGR_E_NULL;
  if (a->B == 0 || (a->Lq == 0 && a->Lk == 0)) return 0;
  e = check_forward_views(*a);
  if (e) return e;
  const int es = elem_size(a->elem);
  if (a->Lq == 0) {                                                // (zeros for the keys, which are read all the same)
    if (!a->k.p || !a->v.p) return DVGR_E_NULL;
    if (!view_ok(a->k, es, a->B, a->Lk, a->Hk) || !view_ok(a->v, es, a->B, a->Lk, a->Hk)) return DVGR_E_ALIGN;
  }
  if (a->Lq && (!g->g_o.p || !a->lse)) return DVGR_E_NULL;
  if (!g->g_k.p != !g->g_v.p) return DVGR_E_NULL;
  if (a->Lq && (!view_ok(g->g_o, es, a->B, a->Lq, a->H) || !view_ok(g->g_q, es, a->B, a->Lq, a->H))) return DVGR_E_ALIGN;
  if (a->Lk && (!view_ok(g->g_k, es, a->B, a->Lk, a->Hk) || !view_ok(g->g_v, es, a->B, a->Lk, a->Hk))) return DVGR_E_ALIGN;
  const size_t need = backward_bytes(*a);
  if (need && !workspace) return DVGR_E_NULL;
  if (workspace_bytes < need) return DVGR_E_WORKSPACE;
  if (!ptr16(workspace)) return DVGR_E_ALIGN;
  return launch_backward(make_args(*a), *g, workspace, (hipStream_t)stream);
}

}  // extern "C"
