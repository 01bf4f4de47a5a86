// dvgr_attn_bwd.hip -- include/dvgr_attn.h: attention to an encoder's states, backward.
//
//     P = exp2(c (q.k - lse))     D = rowsum(dO o O)      dS = P o (dO V^T - D)
//     dV = P^T dO      dK = scale dS^T Q      dQ = scale dS K
//
// Many rows: two passes over the scores, neither with atomics: one owns keys and goes over the packed rows (dK, dV; the heads of a
// group are rows of the same reduction), one owns rows and goes over the keys (dQ).  The scores are computed in both: 7 products
// instead of 5, for results that do not depend on the schedule.  Up to 32 rows: one pass over the keys does it all.
//
// 2 x 4096 queries over 2048 to 4096 keys, 16 / 4 heads of 128, bf16: dQ 325 to 355 us from card to card, 990 TFLOP/s of products, matrix units
// 49 % of the time, LDS 37; dK and dV 575 to 625 us, 775, matrix units 43 % of the busy compute units' time, LDS 49 (11 of them conflicts; five
// reads of a tile for its four products), waves waiting 41 %; a quarter of the compute units without work where samples differ in length.
// 2 x 1024 x 1024, 16 heads of 64, fp32: dQ 110 us, dK and dV 171, matrix units 67 and 70 %.
#include "dvgr_attn_few.h"

namespace dvgr {
namespace attn {
namespace {

// fp16 has 5 bits of exponent: the score gradients are scaled by the power of two that puts the largest |dO| of the sample's head
// group into [0.5, 1), so that small upstream gradients do not vanish.  With values near the type's largest they then reach
// p (1 - p) 2 Dh |v| = 2^22: a wave whose tile holds one beyond the type takes that tile's product kHold times smaller, its sums for the
// moment too (powers of two: nothing is rounded).
template <typename T> struct Grad16 { static constexpr bool on = false; };
template <> struct Grad16<f16_t> { static constexpr bool on = true; };
constexpr float kHold = 256.f;
template <typename T> __device__ __forceinline__ bool beyond_type(const f32x16& ds) {          // the same in all lanes
  if (!Grad16<T>::on) return false;
  float top = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
  return __any(top > 65504.f);
}
template <int NT> __device__ __forceinline__ void scale_tiles(f32x16 (&x)[NT], float f) {
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) x[t][r] *= f;
}
// acc[t] += M^T ds (mma_tr) with the score gradients of a tile
template <typename T, int DP> __device__ __forceinline__ void mma_grad(f32x16 (&acc)[DP / 32], const char* at, f32x16& ds, bool beyond, int lane) {
  if (Grad16<T>::on && beyond) {
    scale_tiles(acc, 1.f / kHold);
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] *= 1.f / kHold;
  }
  mma_tr<DP>(acc, at, ds, lane, T());
  if (Grad16<T>::on && beyond) scale_tiles(acc, kHold);
}
__device__ __forceinline__ float grad_scale(uint32_t top) {
  const int e = (int)(top >> 23);                                   // bits of the largest |dO|
  return e == 0 || e >= 255 ? 1.f : ldexpf(1.f, 126 - e);
}

struct BwdArgs {
  Args f;
  dvgr_attn_view g_o, g_q, g_k, g_v;
  float* delta;                     // (B, H, Lq)
  uint32_t* top;                    // (B, Hk): bits of the largest |dO| (fp16)
  Shares rs;                        // of the packed rows, for dK and dV
  float* part_kv;                   // rs.splits > 1: (split, B, Hk, Lk, [dK, dV], Dh)
};

__global__ __launch_bounds__(256) void k_attn_clear(uint32_t* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0u;
}

// D of the packed rows: a workgroup takes kDeltaRows of one key head, 16 lanes a row (one atomic for all of them: one for each row
// took 1.4 ms where few heads have many rows)
constexpr int kDeltaRows = 64;
template <typename T>
__global__ __launch_bounds__(256) void k_attn_delta(BwdArgs B) {
  const Args& A = B.f;
  const int lane = threadIdx.x & 15, tiles = (A.rows + kDeltaRows - 1) / kDeltaRows;
  const int r0 = (int)(blockIdx.x % tiles) * kDeltaRows + (threadIdx.x >> 4), hk = (int)(blockIdx.x / tiles % A.a.Hk), b = (int)(blockIdx.x / tiles / A.a.Hk);
  const Side os = q_side(A, A.a.o, b, hk), gs = q_side(A, B.g_o, b, hk);
  constexpr int N = Vec16<T>::N;
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kDeltaRows / 16; ++i) {
    const int row = r0 + i * 16;
    float s = 0.f;
    if (row < A.rows) {
      const T* o = (const T*)os.row(row);
      const T* g = (const T*)gs.row(row);
      const T* lo = (const T*)lo_row<T>(A, b, hk, row);
      for (int d = lane * N; d < A.a.Dh; d += 16 * N) {
        float x[N], y[N];
        load_vec(o + d, x);
        load_vec(g + d, y);
#pragma unroll
        for (int j = 0; j < N; ++j) { s += x[j] * y[j]; top = fmaxf(top, fabsf(y[j])); }
        if (lo) {
          load_vec(lo + d, x);
#pragma unroll
          for (int j = 0; j < N; ++j) s += x[j] * y[j];
        }
      }
    }
#pragma unroll
    for (int d = 8; d; d >>= 1) s += __shfl_xor(s, d);
    if (lane == 0 && row < A.rows) B.delta[row_index(A, b, hk, row)] = s;
  }
  if (!Grad16<T>::on) return;
  __shared__ float sh[4];
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) atomicMax(&B.top[b * A.a.Hk + hk], __float_as_uint(fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]))));
}

// score gradient as the matrix unit takes it (infinities and NaN stay what they are: a scaled loss that overflows is found by them)
template <typename T> __device__ __forceinline__ float grad16(float ds, float sc) { return Grad16<T>::on ? ds * sc : ds; }

// a row of dQ, or of its part from one share of the keys
template <typename T, int NT> __device__ __forceinline__ void write_dq(const BwdArgs& B, int b, int hk, int split, int row, const f32x16 (&dq)[NT], float f,
                                                                       int first, int step, int lane) {
  const Args& A = B.f;
  char* out = const_cast<char*>(q_side(A, B.g_q, b, hk).row(row));
  float* part = A.part_o + ((((int64_t)b * A.a.Hk + hk) * A.splits + split) * A.rows + row) * A.a.Dh;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t % step != first) continue;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * t + 8 * g + (lane >> 5) * 4;
      if (d >= A.a.Dh) continue;
      const float4 x = make_float4(dq[t][4 * g] * f, dq[t][4 * g + 1] * f, dq[t][4 * g + 2] * f, dq[t][4 * g + 3] * f);
      if (A.splits > 1) *reinterpret_cast<float4*>(part + d) = x;
      else store4<T>(out + d * sizeof(T), x.x, x.y, x.z, x.w);
    }
  }
}

// ---- dK, dV: KW x 32 keys of one key head, RW x RS x 32 packed rows a turn -------------------------------------------------------
// A wave holds 2 DP / 32 x 16 accumulators and its keys' operands; at 128 two-byte values wait in LDS instead (VL), so that two waves of a
// SIMD fit: one alone spent 40 % of its time waiting for LDS.
template <typename T, int DP, int KW, int RW, int RS>
__global__ __launch_bounds__(64 * KW * RW, (sizeof(T) == 2 && KW > 1 ? 2 : 1)) void k_attn_dkv(BwdArgs B) {
  const Args& A = B.f;
  typedef Tile<T, DP> Tl;
  constexpr int RT = RW * RS * 32, KT = KW * 32, NT = Tl::kNT, NTHR = 64 * KW * RW;
  constexpr bool VL = sizeof(T) == 2 && DP == 128 && KW > 1;
  extern __shared__ __align__(16) char lds[];
  char* lq = lds;
  char* lg = lq + Tl::template bytesT<RT>();
  float* lstat = reinterpret_cast<float*>(lg + Tl::template bytesT<RT>());       // [c lse, D, lse, 0][RT]
  char* lval = reinterpret_cast<char*>(lstat + 4 * RT);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kw = wave / RW, rw = wave % RW;
  const int ktiles = (A.a.Lk + KT - 1) / KT;
  const int64_t w = xcd_work((int64_t)A.a.B * A.a.Hk * B.rs.splits * ktiles, ktiles);
  if (w < 0) return;
  const int kt = (int)(w % ktiles), split = (int)(w / ktiles % B.rs.splits);
  const int hk = (int)(w / ktiles / B.rs.splits % A.a.Hk), b = (int)(w / ktiles / B.rs.splits / A.a.Hk);
  const int n = key_count(A, b), dhb = A.a.Dh * A.es;
  const int key = kt * KT + kw * 32 + (lane & 31);
  const uint8_t* mask = A.a.mask ? A.a.mask + (int64_t)b * A.a.mask_stride : nullptr;
  const bool there = key < n && (!mask || mask[key]);

  Frag<T> kf[Tl::kSteps], vf[VL ? 1 : Tl::kSteps];
  lval += kw * Tl::template bytes<32>();
  {
    const char* kr = k_side(A, A.a.k, b, hk).row(there ? key : 0);
    const char* vr = k_side(A, A.a.v, b, hk).row(there ? key : 0);
#pragma unroll
    for (int s = 0; s < Tl::kSteps; ++s) {
      kf[s] = Tl::gfrag(kr, s, lane, dhb, there);
      const Frag<T> x = Tl::gfrag(vr, s, lane, dhb, there);
      if constexpr (!VL) vf[s] = x;
      else if (rw == 0) *reinterpret_cast<Frag<T>*>(lval + (lane & 31) * Tl::kStride + s * 32 + (lane >> 5) * 16) = x;
    }
    settle(kf);
    if constexpr (!VL) settle(vf);
  }
  f32x16 dk[NT], dv[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) dk[t] = dv[t] = zero16();
  const float sc = Grad16<T>::on ? grad_scale(B.top[b * A.a.Hk + hk]) : 1.f;
  const Side qs = q_side(A, A.a.q, b, hk), gs = q_side(A, B.g_o, b, hk);
  const int turns = kt * KT < n ? (A.rows + RT - 1) / RT : 0, t0 = split * B.rs.turns_per_split;           // keys behind the sample's: zeros
  const int t1 = t0 + B.rs.turns_per_split < turns ? t0 + B.rs.turns_per_split : turns;

  Stage<T, DP, RT, NTHR> sq, sg;
  float stat = 0.f;
  const float* from = tid < RT ? A.a.lse : B.delta;
  const auto fetch = [&](int t) {
    sq.fetch(qs, t * RT, A.rows, dhb, tid);
    sg.fetch(gs, t * RT, A.rows, dhb, tid);
    const int r = t * RT + tid % RT;
    if (tid < 2 * RT) stat = from[row_index(A, b, hk, r < A.rows ? r : A.rows - 1)];
  };
  if (tid < RT) lstat[3 * RT + tid] = 0.f;
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();
    sq.template put<Tl::kStrideT>(lq, tid);
    sg.template put<Tl::kStrideT>(lg, tid);
    if (tid < 2 * RT) {
      const float x = t * RT + tid % RT < A.rows ? stat : tid < RT ? INFINITY : 0.f;      // (no row: p = 0)
      lstat[tid] = tid < RT ? x * A.c : x;
      if (tid < RT) lstat[2 * RT + tid] = x;
    }
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
#pragma unroll 1
    for (int i = 0; i < RS; ++i) {
      const char* tq = lq + (rw * RS + i) * 32 * Tl::kStrideT;
      const char* tg = lg + (rw * RS + i) * 32 * Tl::kStrideT;
      const bool far = any_far(lstat[(rw * RS + i) * 32 + (lane & 31)]);
      f32x16 s = zero16(), dp = zero16();                             // rows = packed rows, column = this lane's key
#pragma unroll
      for (int st = 0; st < Tl::kSteps; ++st) s = mma(Tl::fragT(tq, st, lane), kf[st], s);
#pragma unroll
      for (int st = 0; st < Tl::kSteps; ++st) {
        if constexpr (VL) dp = mma(Tl::fragT(tg, st, lane), Tl::frag(lval, st, lane), dp);
        else dp = mma(Tl::fragT(tg, st, lane), vf[st], dp);
      }
      const float* ls = lstat + (rw * RS + i) * 32 + (lane >> 5) * 4;
      if (far) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 e = *reinterpret_cast<const float4*>(ls + 2 * RT + 8 * g);
          const float ee[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) s[4 * g + j] -= ee[j];
        }
      }
      const float* lc = far ? ls + 3 * RT : ls;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 e = *reinterpret_cast<const float4*>(lc + 8 * g), d = *reinterpret_cast<const float4*>(ls + RT + 8 * g);
        const float ee[4] = {e.x, e.y, e.z, e.w}, dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * g + j;
          const float p = exp2_fast(fmaf(s[r], A.c, -ee[j]));       // (a key that is not there: its column alone, cleared at the end)
          s[r] = p;
          dp[r] = grad16<T>(p * (dp[r] - dd[j]), sc);
        }
      }
      mma_tr<DP>(dv, tg, s, lane, T());
      mma_grad<T, DP>(dk, tq, dp, beyond_type<T>(dp), lane);
    }
  }
  if (RW > 1) {                                                     // add the waves that went over other rows, dK then dV
    float* lo = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      f32x16* acc = x ? dv : dk;
      __syncthreads();
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) lo[((wave * NT + t) * 16 + r) * 64 + lane] = acc[t][r];
      __syncthreads();
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t % RW != rw) continue;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float a = 0.f;
#pragma unroll
          for (int k = 0; k < RW; ++k) a += lo[(((kw * RW + k) * NT + t) * 16 + r) * 64 + lane];
          acc[t][r] = a;
        }
      }
    }
  }
  if (key >= A.a.Lk) return;
  if (!there) {
#pragma unroll
    for (int t = 0; t < NT; ++t) dk[t] = dv[t] = zero16();
  }
  const float f = A.a.scale / sc;
  if (B.rs.splits > 1) {
    float* out = B.part_kv + ((((int64_t)split * A.a.B + b) * A.a.Hk + hk) * A.a.Lk + key) * 2 * A.a.Dh;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (RW > 1 && t % RW != rw) continue;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * t + 8 * g + (lane >> 5) * 4;
        if (d >= A.a.Dh) continue;
        *reinterpret_cast<float4*>(out + d) = make_float4(dk[t][4 * g] * f, dk[t][4 * g + 1] * f, dk[t][4 * g + 2] * f, dk[t][4 * g + 3] * f);
        *reinterpret_cast<float4*>(out + A.a.Dh + d) = make_float4(dv[t][4 * g], dv[t][4 * g + 1], dv[t][4 * g + 2], dv[t][4 * g + 3]);
      }
    }
    return;
  }
  char* gk = const_cast<char*>(k_side(A, B.g_k, b, hk).row(key));
  char* gv = const_cast<char*>(k_side(A, B.g_v, b, hk).row(key));
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (RW > 1 && t % RW != rw) continue;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * t + 8 * g + (lane >> 5) * 4;
      if (d >= A.a.Dh) continue;
      store4<T>(gk + d * sizeof(T), dk[t][4 * g] * f, dk[t][4 * g + 1] * f, dk[t][4 * g + 2] * f, dk[t][4 * g + 3] * f);
      store4<T>(gv + d * sizeof(T), dv[t][4 * g], dv[t][4 * g + 1], dv[t][4 * g + 2], dv[t][4 * g + 3]);
    }
  }
}

// dK and dV from the shares of the rows, added in order: 4 elements a thread
template <typename T>
__global__ __launch_bounds__(256) void k_attn_dkv_join(BwdArgs B) {
  const Args& A = B.f;
  const int per = A.a.Dh / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)A.a.B * A.a.Hk * A.a.Lk * 2;
  if (i >= rows * per) return;
  const int d = (int)(i % per) * 4;
  const int64_t row = i / per, key = row / 2;
  const float4* at = reinterpret_cast<const float4*>(B.part_kv + row * A.a.Dh + d);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int s = 0; s < B.rs.splits; ++s) {
    const float4 y = at[(int64_t)s * rows * per];
    x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
  }
  const int b = (int)(key / A.a.Lk / A.a.Hk), hk = (int)(key / A.a.Lk % A.a.Hk);
  char* out = const_cast<char*>(k_side(A, row & 1 ? B.g_v : B.g_k, b, hk).row((int)(key % A.a.Lk)));
  store4<T>(out + d * sizeof(T), x.x, x.y, x.z, x.w);
}

// ---- dQ: W x 32 packed rows, KS x 32 keys a turn (the forward's arrangement) ---------------------------------------------------
template <typename T, int DP, int KS, int W>
__global__ __launch_bounds__(64 * W, (sizeof(T) == 2 ? 2 : 1)) void k_attn_dq(BwdArgs B) {
  const Args& A = B.f;
  typedef Tile<T, DP> Tl;
  constexpr int KT = KS * 32, RT = W * 32, NT = Tl::kNT;
  extern __shared__ __align__(16) char lds[];
  char* lk = lds;
  char* lv = lds + Tl::template bytesT<KT>();
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int rtiles = (A.rows + RT - 1) / RT;
  const int64_t w = xcd_work((int64_t)A.a.B * A.a.Hk * A.splits * rtiles, rtiles);
  if (w < 0) return;
  const int rt = (int)(w % rtiles), split = (int)(w / rtiles % A.splits);
  const int hk = (int)(w / rtiles / A.splits % A.a.Hk), b = (int)(w / rtiles / A.splits / A.a.Hk);
  const int n = key_count(A, b), dhb = A.a.Dh * A.es, turns = (n + KT - 1) / KT, t0 = split * A.tiles_per_split;
  const int t1 = t0 + A.tiles_per_split < turns ? t0 + A.tiles_per_split : turns;
  const int row = rt * RT + wave * 32 + (lane & 31);
  const bool live = row < A.rows;
  const Side ks = k_side(A, A.a.k, b, hk), vs = k_side(A, A.a.v, b, hk);
  const uint8_t* mask = A.a.mask ? A.a.mask + (int64_t)b * A.a.mask_stride : nullptr;

  Frag<T> qf[Tl::kSteps], gf[Tl::kSteps];
  {
    const char* qr = q_side(A, A.a.q, b, hk).row(live ? row : 0);
    const char* gr = q_side(A, B.g_o, b, hk).row(live ? row : 0);
#pragma unroll
    for (int s = 0; s < Tl::kSteps; ++s) { qf[s] = Tl::gfrag(qr, s, lane, dhb, live); gf[s] = Tl::gfrag(gr, s, lane, dhb, live); }
    settle(qf);
    settle(gf);
  }
  const int64_t ri = row_index(A, b, hk, live ? row : 0);
  float stats[2] = {live ? A.a.lse[ri] : INFINITY, live ? B.delta[ri] : 0.f};
  settle(stats);
  const float lse = stats[0], delta = stats[1];
  const bool far = any_far(lse * A.c);
  const float ref = far ? 0.f : lse * A.c;
  const float sc = Grad16<T>::on ? grad_scale(B.top[b * A.a.Hk + hk]) : 1.f;
  f32x16 dq[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) dq[t] = zero16();

  Stage<T, DP, KT, 64 * W> sk, sv;
  uint32_t there = 0;
  const auto fetch = [&](int t) {
    sk.fetch(ks, t * KT, n, dhb, tid);
    sv.fetch(vs, t * KT, n, dhb, tid);
    there = key_there(mask, t * KT + lane, lane < KT ? n : 0);
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    const unsigned long long bits = __ballot(there != 0);
    __syncthreads();
    sk.template put<Tl::kStrideT>(lk, bits, tid);
    sv.template put<Tl::kStride>(lv, bits, tid);
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
#pragma unroll 1
    for (int i = 0; i < KS; ++i) {
      if (!(uint32_t)(bits >> (32 * i))) continue;                  // (uniform over the wave)
      const char* tk = lk + i * 32 * Tl::kStrideT;
      const char* tv = lv + i * 32 * Tl::kStride;
      f32x16 s = zero16(), dp = zero16();                           // rows = keys, column = this lane's packed row
#pragma unroll
      for (int st = 0; st < Tl::kSteps; ++st) s = mma(Tl::fragT(tk, st, lane), qf[st], s);
#pragma unroll
      for (int st = 0; st < Tl::kSteps; ++st) dp = mma(Tl::frag(tv, st, lane), gf[st], dp);
      if (far) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] -= lse;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = grad16<T>(exp2_fast(fmaf(s[r], A.c, -ref)) * (dp[r] - delta), sc);
      if ((uint32_t)(bits >> (32 * i)) != ~0u) {
        const uint32_t hb = half_bits((uint32_t)(bits >> (32 * i)), lane);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = reg_bit(hb, r) ? s[r] : 0.f;
      }
      mma_grad<T, DP>(dq, tk, s, beyond_type<T>(s), lane);
    }
  }
  if (live) write_dq<T>(B, b, hk, split, row, dq, A.a.scale / sc, 0, 1, lane);
}

// ---- up to 32 rows: KW waves over different keys, everything in one pass ---------------------------------------------------------
// The rows' queries and upstream gradients lie in LDS for all waves, with their log-sums and D (computed here: all rows of the head
// group are in the tile, and so is the largest |dO|).  A wave's 32 keys meet all rows at once, so their dK and dV are final and
// leave at once; dQ is added up over the keys.  Its product needs the score gradients transposed, through LDS; two-byte dK and dV leave
// through LDS too, whole rows at a time and past the caches.  The values' tile is free for both once dP is there.  64 x 15 words over
// 1024 frames (8 heads of 96, bf16): 78 us, 4.6 TB/s; with the gradients stored in 8-byte pieces 40 more, through the caches 10 (and the forward of
// the next step 55 instead of 34, while their lines are written back).
template <typename T, int DP> struct FewLds {
  static constexpr bool kOut = sizeof(T) == 2;                      // fp32: values go straight to operands, gradients leave in 16-byte pieces
  static constexpr int kScr = 36;                                   // floats of a scratch row: 16-byte aligned, spread over the banks
  static constexpr int kTile = Tile<T, DP>::template bytes<32>(), kTileT = Tile<T, DP>::template bytesT<32>(), kScrBytes = 32 * kScr * 4;
  static constexpr int kOwn = kTileT + (kOut && kTile > kScrBytes ? kTile : kScrBytes);
  static constexpr int kBytes(int KW) { return 2 * kTileT + 68 * 4 + KW * kOwn; }
};
template <typename T, int DP, int KW>
__global__ __launch_bounds__(64 * KW, (sizeof(T) == 2 && DP <= 96 ? 2 : 1)) void k_attn_few_bwd(BwdArgs B) {
  const Args& A = B.f;
  typedef Tile<T, DP> Tl;
  constexpr int NT = Tl::kNT, kScr = FewLds<T, DP>::kScr;
  constexpr bool kOut = FewLds<T, DP>::kOut;
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, kw = tid >> 6, col = lane & 31, h4 = (lane >> 5) * 4;
  char* lq = lds;
  char* lg = lq + Tl::template bytesT<32>();
  float* stat = reinterpret_cast<float*>(lg + Tl::template bytesT<32>());        // [lse, D][32], largest |dO|
  char* lk = reinterpret_cast<char*>(stat + 68) + kw * FewLds<T, DP>::kOwn;
  char* lx = lk + FewLds<T, DP>::kTileT;                              // values, then score gradients, then dV, then dK
  float* scr = reinterpret_cast<float*>(lx);
  const FewWork f = few_work<KW>(A, kw);
  if (!f.any) return;
  const int dhb = A.a.Dh * A.es;
  const Side ks = k_side(A, A.a.k, f.b, f.hk), vs = k_side(A, A.a.v, f.b, f.hk);
  const Side qs = q_side(A, A.a.q, f.b, f.hk), gs = q_side(A, B.g_o, f.b, f.hk);
  const uint8_t* mask = A.a.mask ? A.a.mask + (int64_t)f.b * A.a.mask_stride : nullptr;

  WaveStage<T, DP> sk, sv;
  Frag<T> vf[kOut ? 1 : Tl::kSteps];
  uint32_t there = 0;
  const auto fetch = [&](int t) {
    const int key = t * 32 + col;
    sk.fetch(ks, t * 32, f.n, dhb, false, lane);
    if constexpr (kOut) sv.fetch(vs, t * 32, f.n, dhb, false, lane);
    else {
      const char* vr = vs.row(key < f.n ? key : 0);
#pragma unroll
      for (int s = 0; s < Tl::kSteps; ++s) vf[s] = Tl::gfrag(vr, s, lane, dhb, key < f.n);
    }
    there = key_there(mask, key, f.n);
  };
  if (f.t0 < f.t1) fetch(f.t0);
  {                                                                 // the rows
    constexpr int per = 2 * KW;                                     // threads of a row
    const int r = tid / per, sub = tid % per;
    const bool live = r < A.rows;
    const char* qr = qs.row(live ? r : 0);
    const char* gr = gs.row(live ? r : 0);
    const char* orow = q_side(A, A.a.o, f.b, f.hk).row(live ? r : 0);
    const char* lo = lo_row<T>(A, f.b, f.hk, live ? r : 0);
    float d = 0.f, top = 0.f;
    for (int c = sub * 16; c < Tl::kRowBytes; c += per * 16) {
      uint4 q = make_uint4(0, 0, 0, 0), g = q;
      if (live && c < dhb) {
        q = *reinterpret_cast<const uint4*>(qr + c);
        g = *reinterpret_cast<const uint4*>(gr + c);
        float x[Vec16<T>::N], y[Vec16<T>::N], z[Vec16<T>::N];
        load_vec(reinterpret_cast<const T*>(orow + c), x);
        load_vec(reinterpret_cast<const T*>(gr + c), y);
        if (lo) load_vec(reinterpret_cast<const T*>(lo + c), z);
#pragma unroll
        for (int i = 0; i < Vec16<T>::N; ++i) {
          d += (lo ? x[i] + z[i] : x[i]) * y[i];
          top = fmaxf(top, fabsf(y[i]));
        }
      }
      *reinterpret_cast<uint4*>(lq + r * Tl::kStrideT + c) = q;
      *reinterpret_cast<uint4*>(lg + r * Tl::kStrideT + c) = g;
    }
#pragma unroll
    for (int o = 1; o < per; o <<= 1) { d += __shfl_xor(d, o); top = fmaxf(top, __shfl_xor(top, o)); }
    if (sub == 0) {
      stat[r] = live ? A.a.lse[row_index(A, f.b, f.hk, r)] : INFINITY;
      stat[32 + r] = d;
    }
    if (Grad16<T>::on) {
      if (tid == 0) stat[64] = 0.f;
      __syncthreads();
      if (sub == 0) atomicMax(reinterpret_cast<int*>(stat + 64), __float_as_int(top));       // (not negative: ordered as integers)
    }
  }
  __syncthreads();
  const float sc = Grad16<T>::on ? grad_scale(__float_as_uint(stat[64])) : 1.f, fac = A.a.scale / sc;
  f32x16 dq[NT], acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) dq[t] = zero16();
  // acc, 32 keys of tile t, to their rows of a gradient
  const auto leave = [&](const dvgr_attn_view& v, int t, float x, uint32_t bits) {
    const Side to = k_side(A, v, f.b, f.hk);
    if (bits != ~0u && !((bits >> col) & 1)) {                      // zeros, where an infinite upstream gradient times p = 0 is NaN
#pragma unroll
      for (int u = 0; u < NT; ++u) acc[u] = zero16();
    }
    if constexpr (kOut) {
      wave_order();
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          store4<T>(lx + col * Tl::kStride + (32 * u + 8 * g + h4) * sizeof(T), acc[u][4 * g] * x, acc[u][4 * g + 1] * x, acc[u][4 * g + 2] * x,
                    acc[u][4 * g + 3] * x);
      wave_order();
#pragma unroll
      for (int i = 0; i < Tl::kChunks / 2; ++i) {
        const int e = lane + i * 64, key = t * 32 + e / Tl::kChunks, c = (e % Tl::kChunks) * 16;
        typedef typename WaveStage<T, DP>::u32x4 u32x4;
        if (key < A.a.Lk && c < dhb)
          stream_store(reinterpret_cast<u32x4*>(const_cast<char*>(to.row(key)) + c), *reinterpret_cast<const u32x4*>(lx + (e / Tl::kChunks) * Tl::kStride + c));
      }
    } else if (t * 32 + col < A.a.Lk) {
      char* out = const_cast<char*>(to.row(t * 32 + col));
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = 32 * u + 8 * g + h4;
          if (d < A.a.Dh) store4<T>(out + d * sizeof(T), acc[u][4 * g] * x, acc[u][4 * g + 1] * x, acc[u][4 * g + 2] * x, acc[u][4 * g + 3] * x);
        }
    }
  };
  int t = f.t0;
  for (; t < f.t1; t += KW) {
    const bool here = there != 0;
    const uint32_t bits = (uint32_t)__ballot(here);
    wave_order();
    sk.template put<Tl::kStrideT>(lk, bits, lane);
    if constexpr (kOut) sv.template put<Tl::kStride>(lx, bits, lane);
    wave_order();
    f32x16 s = zero16(), dp = zero16();                             // rows = packed rows, column = this lane's key
#pragma unroll
    for (int st = 0; st < Tl::kSteps; ++st) {
      if constexpr (kOut) dp = mma(Tl::fragT(lg, st, lane), Tl::frag(lx, st, lane), dp);
      else dp = mma(Tl::fragT(lg, st, lane), vf[st], dp);
    }
    if (t + KW < f.t1) fetch(t + KW);
#pragma unroll
    for (int st = 0; st < Tl::kSteps; ++st) s = mma(Tl::fragT(lq, st, lane), Tl::fragT(lk, st, lane), s);
    wave_order();
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 e = *reinterpret_cast<const float4*>(stat + 8 * g + h4), d = *reinterpret_cast<const float4*>(stat + 32 + 8 * g + h4);
      const float ee[4] = {e.x, e.y, e.z, e.w}, dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * g + j;
        const float p = exp2_fast((s[r] - ee[j]) * A.c);         // (a key that is not there: its column alone, cleared as it leaves)
        s[r] = p;
        dp[r] = here ? grad16<T>(p * (dp[r] - dd[j]), sc) : 0.f;
        scr[(8 * g + h4 + j) * kScr + col] = dp[r];
      }
    }
    wave_order();
    const bool beyond = beyond_type<T>(dp);
    if (B.g_q.p) {
      f32x16 x;                                                     // rows = keys, column = this lane's packed row
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 y = *reinterpret_cast<const float4*>(scr + col * kScr + 8 * g + h4);
        x[4 * g] = y.x; x[4 * g + 1] = y.y; x[4 * g + 2] = y.z; x[4 * g + 3] = y.w;
      }
      mma_grad<T, DP>(dq, lk, x, beyond, lane);
    }
    if (B.g_k.p) {
#pragma unroll
      for (int u = 0; u < NT; ++u) acc[u] = zero16();
      mma_tr<DP>(acc, lg, s, lane, T());
      leave(B.g_v, t, 1.f, bits);
#pragma unroll
      for (int u = 0; u < NT; ++u) acc[u] = zero16();
      mma_grad<T, DP>(acc, lq, dp, beyond, lane);
      leave(B.g_k, t, fac, bits);
    }
  }
  if (B.g_k.p) {                                                    // keys behind the sample's last tile
    const int tiles = (A.a.Lk + 31) / 32, per = A.tiles_per_split * KW, t2 = (f.split + 1) * per < tiles ? (f.split + 1) * per : tiles;
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[u] = zero16();
    for (; t < t2; t += KW) { leave(B.g_v, t, 1.f, ~0u); leave(B.g_k, t, 1.f, ~0u); }
  }
  if (!B.g_q.p) return;
  if (KW > 1) {
    float* lo = reinterpret_cast<float*>(lds);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) lo[((kw * NT + u) * 16 + r) * 64 + lane] = dq[u][r];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      if (u % KW != kw) continue;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) a += lo[((k * NT + u) * 16 + r) * 64 + lane];
        dq[u][r] = a;
      }
    }
  }
  if (col >= A.rows) return;
  write_dq<T>(B, f.b, f.hk, f.split, col, dq, fac, kw, KW, lane);
}

// dQ from the shares of the keys: a workgroup per packed row, its waves take every fourth share, added in the waves' order
template <typename T>
__global__ __launch_bounds__(256) void k_attn_dq_join(BwdArgs B) {
  const Args& A = B.f;
  __shared__ float sh[4][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = 2 * lane;
  const int row = (int)(blockIdx.x % A.rows), hk = (int)(blockIdx.x / A.rows % A.a.Hk), b = (int)(blockIdx.x / A.rows / A.a.Hk);
  const float* at = A.part_o + (((int64_t)b * A.a.Hk + hk) * A.splits * A.rows + row) * A.a.Dh + d;
  float x = 0.f, y = 0.f;
  if (d < A.a.Dh)
#pragma unroll 8
    for (int s = wave; s < A.splits; s += 4) {
      const float2 p = *reinterpret_cast<const float2*>(at + (int64_t)s * A.rows * A.a.Dh);
      x += p.x; y += p.y;
    }
  sh[wave][d] = x; sh[wave][d + 1] = y;
  __syncthreads();
  if (wave || d >= A.a.Dh) return;
  T* out = (T*)const_cast<char*>(q_side(A, B.g_q, b, hk).row(row));
  out[d] = (T)(sh[0][d] + sh[1][d] + sh[2][d] + sh[3][d]);
  out[d + 1] = (T)(sh[0][d + 1] + sh[1][d + 1] + sh[2][d + 1] + sh[3][d + 1]);
}

template <typename K> int launch(K kern, std::atomic<uint32_t>& asked, int64_t work, int threads, size_t bytes, const BwdArgs& B,
                                hipStream_t st) {
  const int e = allow_lds(reinterpret_cast<const void*>(kern), bytes, asked);
  if (e) return e;
  DVGR_LAUNCH(kern, dim3(xcd_grid(work)), dim3(threads), bytes, st, B);
  return (int)hipGetLastError();
}

template <typename T, int DP, int KW, int RW, int RS> int launch_dkv(const BwdArgs& B, hipStream_t st) {
  typedef Tile<T, DP> Tl;
  static std::atomic<uint32_t> asked{0};
  size_t bytes = 2 * Tl::template bytesT<RW * RS * 32>() + 4 * RW * RS * 32 * sizeof(float) + (sizeof(T) == 2 && DP == 128 && KW > 1 ? KW * Tl::template bytes<32>() : 0);
  const size_t join = RW > 1 ? (size_t)KW * RW * Tl::kNT * 16 * 64 * sizeof(float) : 0;
  if (bytes < join) bytes = join;
  const int64_t keys = (int64_t)B.f.a.B * B.f.a.Hk * B.f.a.Lk;
  const int e = launch(k_attn_dkv<T, DP, KW, RW, RS>, asked, (int64_t)B.f.a.B * B.f.a.Hk * B.rs.splits * ((B.f.a.Lk + KW * 32 - 1) / (KW * 32)), 64 * KW * RW,
                       bytes, B, st);
  if (e || B.rs.splits == 1) return e;
  DVGR_LAUNCH((k_attn_dkv_join<T>), dim3((unsigned)((keys * 2 * (B.f.a.Dh / 4) + 255) / 256)), dim3(256), 0, st, B);
  return (int)hipGetLastError();
}
template <typename T> int join_dq(const BwdArgs& B, hipStream_t st) {
  if (B.f.splits == 1 || !B.f.rows) return 0;
  DVGR_LAUNCH((k_attn_dq_join<T>), dim3((unsigned)((int64_t)B.f.a.B * B.f.a.Hk * B.f.rows)), dim3(256), 0, st, B);
  return (int)hipGetLastError();
}
template <typename T, int DP, int KS, int W> int launch_dq(const BwdArgs& B, hipStream_t st) {
  static std::atomic<uint32_t> asked{0};
  const int e = launch(k_attn_dq<T, DP, KS, W>, asked, (int64_t)B.f.a.B * B.f.a.Hk * B.f.splits * ((B.f.rows + W * 32 - 1) / (W * 32)), 64 * W,
                Tile<T, DP>::template bytes<KS * 32>() + Tile<T, DP>::template bytesT<KS * 32>(), B, st);
  return e ? e : join_dq<T>(B, st);
}
template <typename T, int DP, int KW> int launch_few(const BwdArgs& B, hipStream_t st) {
  typedef Tile<T, DP> Tl;
  static std::atomic<uint32_t> asked{0};
  size_t bytes = FewLds<T, DP>::kBytes(KW);
  const size_t join = KW > 1 ? (size_t)KW * Tl::kNT * 16 * 64 * sizeof(float) : 0;
  if (bytes < join) bytes = join;
  const int64_t units = (int64_t)B.f.a.B * B.f.a.Hk;                // (one tile of rows; without rows one that has none)
  const int e = launch(k_attn_few_bwd<T, DP, KW>, asked, units * B.f.splits, 64 * KW, bytes, B, st);
  return e || !B.g_q.p ? e : join_dq<T>(B, st);
}

// 128 keys of a workgroup: four waves, and four more on other rows where two of a SIMD fit (two-byte types).  Few keys for many rows: four
// waves share them and go over different rows.
template <typename T, int DP> int launch_many(const BwdArgs& B, hipStream_t st) {
  constexpr int S = sizeof(T) == 4 ? 1 : 2;                         // a turn: 32 rows (keys) of fp32, 64 of two bytes
  if (B.f.a.Lk && B.g_k.p) {
    const int e = B.f.a.Lk <= 32 ? launch_dkv<T, DP, 1, 4, 1>(B, st) : launch_dkv<T, DP, 4, S, 1>(B, st);
    if (e) return e;
  }
  if (!B.g_q.p) return 0;
  if constexpr (S == 2)
    if (many_waves((int64_t)B.f.a.B * B.f.a.Hk, B.f.rows, 2) == 8) return launch_dq<T, DP, S, 8>(B, st);
  return launch_dq<T, DP, S, 4>(B, st);
}
template <typename T, int DP> int launch_dp(const BwdArgs& B, int KW, hipStream_t st) {
  return KW == 1 ? launch_few<T, DP, 1>(B, st) : KW == 4 ? launch_few<T, DP, 4>(B, st) : launch_many<T, DP>(B, st);
}

template <typename T> int launch_t(const BwdArgs& B, int KW, hipStream_t st) {
  if (!KW) {
    const int64_t groups = (int64_t)B.f.a.B * B.f.a.Hk;
    if (Grad16<T>::on) DVGR_LAUNCH(k_attn_clear, dim3((unsigned)((groups + 255) / 256)), dim3(256), 0, st, B.top, groups);
    DVGR_LAUNCH((k_attn_delta<T>), dim3((unsigned)(groups * ((B.f.rows + kDeltaRows - 1) / kDeltaRows))), dim3(256), 0, st, B);
    const int e = (int)hipGetLastError();
    if (e) return e;
  }
  if (B.f.a.Dh <= 32) return launch_dp<T, 32>(B, KW, st);
  if (B.f.a.Dh <= 64) return launch_dp<T, 64>(B, KW, st);
  if (B.f.a.Dh <= 96) return launch_dp<T, 96>(B, KW, st);
  return launch_dp<T, 128>(B, KW, st);
}

}  // namespace

namespace {
// Workgroups of both passes of many rows: split where there is less than one for each compute unit, in shares of at least four turns.
struct BwdPlan { FewPlan few; Shares ks, rs; size_t delta, top, part_q, part_kv, total; };
BwdPlan bwd_plan(const dvgr_attn_problem& a) {
  BwdPlan p{};
  const int64_t rows = (int64_t)a.Lq * (a.H / a.Hk), heads = (int64_t)a.B * a.Hk;
  const int turn = a.elem == DVGR_ELEM_F32 ? 32 : 64;               // rows or keys of a turn
  p.few = few_plan(a, false);
  p.ks = p.rs = Shares{1, 1 << 30};
  if (p.few.KW) p.ks = Shares{p.few.splits, p.few.tiles_per_split};
  else {
    const int64_t qu = heads * ((rows + 127) / 128), ku = heads * (a.Lk <= 32 ? 1 : (a.Lk + 127) / 128);
    if (qu < 256) p.ks = shares_of(qu, (a.Lk + turn - 1) / turn, 512, 4);
    if (ku < 256) p.rs = shares_of(ku, a.Lk <= 32 ? (rows + 127) / 128 : (rows + turn - 1) / turn, 512, 4);
  }
  size_t o = 0;
  const auto take = [&o](size_t b) { const size_t at = o; o += (b + 255) / 256 * 256; return at; };
  p.delta = take(p.few.KW ? 0 : (size_t)heads * rows * sizeof(float));
  p.top = take(p.few.KW || a.elem != DVGR_ELEM_F16 ? 0 : (size_t)heads * sizeof(uint32_t));
  p.part_q = take(p.ks.splits > 1 ? (size_t)heads * p.ks.splits * rows * a.Dh * sizeof(float) : 0);
  p.part_kv = take(p.rs.splits > 1 ? (size_t)heads * p.rs.splits * a.Lk * 2 * a.Dh * sizeof(float) : 0);
  p.total = o;
  return p;
}
}  // namespace

size_t backward_bytes(const dvgr_attn_problem& a) { return bwd_plan(a).total; }

int launch_backward(const Args& A, const dvgr_attn_grads& g, void* ws, hipStream_t st) {
  const BwdPlan p = bwd_plan(A.a);
  char* at = (char*)ws;
  BwdArgs B{A, g.g_o, g.g_q, g.g_k, g.g_v, (float*)(at + p.delta), (uint32_t*)(at + p.top), p.rs, (float*)(at + p.part_kv)};
  B.f.splits = p.ks.splits;
  B.f.tiles_per_split = p.ks.turns_per_split;
  B.f.part_o = (float*)(at + p.part_q);
  const int KW = p.few.KW;
  return A.a.elem == DVGR_ELEM_F32 ? launch_t<float>(B, KW, st) : A.a.elem == DVGR_ELEM_BF16 ? launch_t<bf16_t>(B, KW, st) : launch_t<f16_t>(B, KW, st);
}

}  // namespace attn
}  // namespace dvgr
