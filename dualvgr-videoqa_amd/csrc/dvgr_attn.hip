// dvgr_attn.hip -- include/dvgr_attn.h: attention to an encoder's states, forward.
//
// One pass over the keys with the running maximum and sum of the softmax (in powers of two: scale and log2 e are one factor).
// A workgroup of four waves takes QW x 32 packed rows of one key head (the H / Hk query heads that share it are rows of the same
// tile, so a key is read once for all of them) and KW x KS x 32 keys a turn: QW = 4 for many rows; KW = 4 for few (a word over a long
// video), where the waves go over different keys and are joined in LDS at the end.
#include "dvgr_attn.h"

namespace dvgr {
namespace attn {
namespace {

template <typename T, int DP, int QW, int KW, int KS>
__global__ __launch_bounds__(kThreads) void k_attn_fwd(Args A) {
  typedef Tile<T, DP> Tl;
  constexpr int KT = KW * KS * 32, RT = QW * 32, NT = Tl::kNT;
  extern __shared__ __align__(16) char lds[];
  char* lk = lds;
  char* lv = lds + Tl::template bytes<KT>();
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, qw = wave / KW, kw = wave % KW;
  const int rtiles = (A.rows + RT - 1) / RT;
  const int64_t w = xcd_work((int64_t)A.a.B * A.a.Hk * A.splits * rtiles);
  if (w < 0) return;
  const int rt = (int)(w % rtiles), split = (int)(w / rtiles % A.splits);
  const int hk = (int)(w / rtiles / A.splits % A.a.Hk), b = (int)(w / rtiles / A.splits / A.a.Hk);
  const int n = key_count(A, b), dhb = A.a.Dh * A.es;
  const int t0 = split * A.tiles_per_split, tn = (n + KT - 1) / KT, t1 = t0 + A.tiles_per_split < tn ? t0 + A.tiles_per_split : tn;
  const int row = rt * RT + qw * 32 + (lane & 31);
  const bool live = row < A.rows;
  const Side ks = k_side(A, A.a.k, b, hk), vs = k_side(A, A.a.v, b, hk);
  const uint8_t* mask = A.a.mask ? A.a.mask + (int64_t)b * A.a.mask_stride : nullptr;

  Frag<T> qf[Tl::kSteps];
  {
    const char* qr = q_side(A, A.a.q, b, hk).row(live ? row : 0, A.G);
#pragma unroll
    for (int s = 0; s < Tl::kSteps; ++s) qf[s] = Tl::gfrag(qr, s, lane, dhb, live);
  }
  f32x16 o[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t] = zero16();
  float m = -INFINITY, l = 0.f;

  Stage<T, DP, KT> sk, sv;
  bool there = false;                                               // lane j: key j of this wave's keys of the next tile
  const auto fetch = [&](int t) {
    sk.fetch(ks, 1, t * KT, n, mask, dhb, tid);
    sv.fetch(vs, 1, t * KT, n, mask, dhb, tid);
    const int j = t * KT + kw * KS * 32 + lane;
    there = lane < KS * 32 && j < n && (!mask || mask[j]);
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();
    sk.put(lk, tid);
    sv.put(lv, tid);
    const unsigned long long bits = __ballot(there);
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
    if (!bits) continue;                                            // (uniform over the wave)
    f32x16 s[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) s[i] = zero16();
#pragma unroll
    for (int st = 0; st < Tl::kSteps; ++st)
#pragma unroll
      for (int i = 0; i < KS; ++i) s[i] = mma(Tl::frag(lk + (kw * KS + i) * 32 * Tl::kStride, st, lane), qf[st], s[i]);
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
    mx = half_max(mx) * A.c;
    if (__any(mx > m)) {
      const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : exp2_fast(m - mn);      // nothing summed yet: o and l are 0
      l *= f;
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[u][r] *= f;
      m = mn;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[i][r] = exp2_fast(fmaf(s[i][r], A.c, -ref));
        sum += s[i][r];
      }
      l += sum;
      mma_tr<DP>(o, lv + (kw * KS + i) * 32 * Tl::kStride, s[i], lane, T());
    }
  }
  l = half_sum(l);

  if (KW > 1) {                                                     // join the waves that went over other keys of the same rows
    __syncthreads();
    float* ml = reinterpret_cast<float*>(lds);                      // [wave][m, l][32]
    float* lo = ml + kWaves * 64;                                   // [wave][t * 16 + r][lane]
    if (lane < 32) { ml[wave * 64 + lane] = m; ml[wave * 64 + 32 + lane] = l; }
    __syncthreads();
    float mj = -INFINITY;
#pragma unroll
    for (int k = 0; k < KW; ++k) mj = fmaxf(mj, ml[(qw * KW + k) * 64 + (lane & 31)]);
    const float ref = mj == -INFINITY ? 0.f : mj, f = exp2_fast(m - ref);
    l = 0.f;
#pragma unroll
    for (int k = 0; k < KW; ++k) l += ml[(qw * KW + k) * 64 + 32 + (lane & 31)] * exp2_fast(ml[(qw * KW + k) * 64 + (lane & 31)] - ref);
    m = mj;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) lo[((wave * NT + t) * 16 + r) * 64 + lane] = o[t][r] * f;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t % KW != kw) continue;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) a += lo[(((qw * KW + k) * NT + t) * 16 + r) * 64 + lane];
        o[t][r] = a;
      }
    }
  }
  if (!live) return;
  const int h4 = (lane >> 5) * 4;
  if (A.splits > 1) {
    const int64_t at = w * RT + qw * 32 + (lane & 31);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (KW > 1 && t % KW != kw) continue;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * t + 8 * g + h4;
        if (d < A.a.Dh) *reinterpret_cast<float4*>(A.part_o + at * A.a.Dh + d) = make_float4(o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]);
      }
    }
    if (lane < 32 && kw == 0) *reinterpret_cast<float2*>(A.part_ml + 2 * at) = make_float2(m, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  char* out = const_cast<char*>(q_side(A, A.a.o, b, hk).row(row, A.G));
  char* lo = lo_row<T>(A, b, hk, row);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (KW > 1 && t % KW != kw) continue;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * t + 8 * g + h4;
      if (d >= A.a.Dh) continue;
      const float x[4] = {o[t][4 * g] * inv, o[t][4 * g + 1] * inv, o[t][4 * g + 2] * inv, o[t][4 * g + 3] * inv};
      store4<T>(out + d * sizeof(T), x[0], x[1], x[2], x[3]);
      if (lo) store4<T>(lo + d * sizeof(T), x[0] - (float)(T)x[0], x[1] - (float)(T)x[1], x[2] - (float)(T)x[2], x[3] - (float)(T)x[3]);
    }
  }
  // log2 of the row's sum, in units of the scaled scores; +inf for a row without keys: every exp2(s - lse) of the backward is 0
  if (A.a.lse && lane < 32 && kw == 0) A.a.lse[row_index(A, b, hk, row)] = l == 0.f ? INFINITY : m + __log2f(l);
}

// join of the shares of the keys: one wave per packed row, shares in their order
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(Args A, int RT) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= (int64_t)A.a.B * A.a.Hk * A.rows) return;
  const int row = (int)(i % A.rows), hk = (int)(i / A.rows % A.a.Hk), b = (int)(i / A.rows / A.a.Hk);
  const int rtiles = (A.rows + RT - 1) / RT;
  const int64_t at0 = (((int64_t)b * A.a.Hk + hk) * A.splits * rtiles + row / RT) * RT + row % RT, step = (int64_t)rtiles * RT;
  float m = -INFINITY;
  for (int s = lane; s < A.splits; s += 64) m = fmaxf(m, A.part_ml[2 * (at0 + s * step)]);
  m = wave_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  const int d = 2 * lane;
  float2 o = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < A.splits; ++s) {
    const int64_t at = at0 + s * step;
    const float2 ml = *reinterpret_cast<const float2*>(A.part_ml + 2 * at);
    const float f = exp2_fast(ml.x - ref);
    l += ml.y * f;
    if (d < A.a.Dh) {
      const float2 p = *reinterpret_cast<const float2*>(A.part_o + at * A.a.Dh + d);
      o.x += p.x * f; o.y += p.y * f;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = (T*)q_side(A, A.a.o, b, hk).row(row, A.G);
  T* lo = (T*)lo_row<T>(A, b, hk, row);
  if (d < A.a.Dh) {
    o.x *= inv; o.y *= inv;
    out[d] = (T)o.x; out[d + 1] = (T)o.y;
    if (lo) { lo[d] = (T)(o.x - (float)(T)o.x); lo[d + 1] = (T)(o.y - (float)(T)o.y); }
  }
  if (A.a.lse && lane == 0) A.a.lse[row_index(A, b, hk, row)] = l == 0.f ? INFINITY : m + __log2f(l);
}

struct Plan { int few, RT, KT, splits, tiles_per_split; int64_t units; size_t o_bytes, ml_bytes; };

// Up to 32 packed rows: the four waves share the rows and split the keys.  The keys are split over workgroups while there are fewer
// workgroups than the chip has room for (two per compute unit), in shares of at least four tiles.
Plan plan(const Args& A) {
  Plan p{};
  p.few = A.rows <= 32;
  p.RT = p.few ? 32 : 128;
  p.KT = p.few ? 128 : A.es == 4 ? 32 : 64;
  const int64_t rtiles = (A.rows + p.RT - 1) / p.RT, tiles = (A.a.Lk + p.KT - 1) / p.KT;
  p.units = (int64_t)A.a.B * A.a.Hk * rtiles;
  int64_t s = p.units ? 512 / p.units : 1;
  if (s > tiles / 4) s = tiles / 4;
  if (s < 1) s = 1;
  p.tiles_per_split = (int)((tiles + s - 1) / s);
  if (p.tiles_per_split < 1) p.tiles_per_split = 1;
  p.splits = (int)((tiles + p.tiles_per_split - 1) / p.tiles_per_split);
  if (p.splits < 1) p.splits = 1;
  if (p.splits > 1) {
    p.o_bytes = (size_t)p.units * p.splits * p.RT * A.a.Dh * sizeof(float);
    p.ml_bytes = (size_t)p.units * p.splits * p.RT * 2 * sizeof(float);
  }
  return p;
}

template <typename T, int DP, int QW, int KW, int KS>
int launch(const Args& A, const Plan& p, hipStream_t st) {
  typedef Tile<T, DP> Tl;
  size_t bytes = 2 * Tl::template bytes<KW * KS * 32>();
  const size_t join = KW > 1 ? (size_t)(kWaves * 64 + kWaves * Tl::kNT * 16 * 64) * sizeof(float) : 0;
  bytes = bytes > join ? bytes : join;
  const auto kern = k_attn_fwd<T, DP, QW, KW, KS>;
  static std::atomic<uint32_t> asked{0};
  const int e = allow_lds(reinterpret_cast<const void*>(kern), bytes, asked);
  if (e) return e;
  DVGR_LAUNCH(kern, dim3(xcd_grid(p.units * p.splits)), dim3(kThreads), bytes, st, A);
  return (int)hipGetLastError();
}
template <typename T, int DP> int launch_dp(const Args& A, const Plan& p, hipStream_t st) {
  if (p.few) return launch<T, DP, 1, 4, 1>(A, p, st);
  return launch<T, DP, 4, 1, sizeof(T) == 4 ? 1 : 2>(A, p, st);
}
template <typename T> int launch_t(const Args& A, const Plan& p, hipStream_t st) {
  int e;
  if (A.a.Dh <= 32) e = launch_dp<T, 32>(A, p, st);
  else if (A.a.Dh <= 64) e = launch_dp<T, 64>(A, p, st);
  else if (A.a.Dh <= 96) e = launch_dp<T, 96>(A, p, st);
  else e = launch_dp<T, 128>(A, p, st);
  if (e || A.splits == 1) return e;
  const int64_t rows = (int64_t)A.a.B * A.a.Hk * A.rows;
  DVGR_LAUNCH((k_attn_join<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, A, p.RT);
  return (int)hipGetLastError();
}

bool view_ok(const dvgr_attn_view& v, int es, int64_t B, int64_t L, int64_t H) {
  const auto bad = [es](int64_t s) { return (s * es) % 16 != 0; };
  return ptr16(v.p) && !(B > 1 && bad(v.sb)) && !(L > 1 && bad(v.sl)) && !(H > 1 && bad(v.sh));
}

int check(const dvgr_attn_problem* a) {
  if (!a) return DVGR_E_NULL;
  if (!elem_size(a->elem)) return DVGR_E_KIND;
  if (a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->H < 1 || a->Hk < 1 || a->H % a->Hk || a->Dh < 8 || a->Dh > 128 || a->Dh % 8) return DVGR_E_DIMS;
  if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return DVGR_E_DIMS;
  const int64_t rows = (int64_t)a->Lq * (a->H / a->Hk);
  // packed rows and keys are 32-bit, a launch holds at most 2^32 threads (a workgroup has 32 rows or keys at least)
  if (rows >= (1ll << 30) || a->Lk >= (1 << 30)) return DVGR_E_DIMS;
  if ((double)a->B * a->Hk * (rows / 4 + 2) >= (double)(1ll << 24) || (double)a->B * a->Hk * (a->Lk / 32 + 2) >= (double)(1ll << 24)) return DVGR_E_DIMS;
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
  const Plan p = plan(make_args(*a));
  return p.o_bytes + p.ml_bytes;
}
size_t dvgr_attn_backward_workspace_bytes(const dvgr_attn_problem* a) { return check(a) ? 0 : backward_bytes(*a); }

int dvgr_attn_forward(const dvgr_attn_problem* a, void* workspace, size_t workspace_bytes, void* stream) {
  int e = check(a);
  if (e) return e;
  e = check_forward_views(*a);
  if (e || empty(*a)) return e;
  Args A = make_args(*a);
  const Plan p = plan(A);
  if (p.splits > 1) {
    if (!workspace) return DVGR_E_NULL;
    if (workspace_bytes < p.o_bytes + p.ml_bytes) return DVGR_E_WORKSPACE;
    if (!ptr16(workspace)) return DVGR_E_ALIGN;
  }
  A.splits = p.splits;
  A.tiles_per_split = p.tiles_per_split;
  A.part_o = (float*)workspace;
  A.part_ml = (float*)((char*)workspace + p.o_bytes);
  hipStream_t st = (hipStream_t)stream;
  return a->elem == DVGR_ELEM_F32 ? launch_t<float>(A, p, st) : a->elem == DVGR_ELEM_BF16 ? launch_t<bf16_t>(A, p, st) : launch_t<f16_t>(A, p, st);
}

int dvgr_attn_backward(const dvgr_attn_problem* a, const dvgr_attn_grads* g, void* workspace, size_t workspace_bytes, void* stream) {
  int e = check(a);
  if (e) return e;
  if (!g) return DVGR_E_NULL;
  if (a->B == 0 || (a->Lq == 0 && a->Lk == 0)) return 0;
  e = check_forward_views(*a);
  if (e) return e;
  const int es = elem_size(a->elem);
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
