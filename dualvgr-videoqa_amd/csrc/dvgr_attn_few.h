// dvgr_attn_few.h -- attention where one 32-row tile holds all packed rows of a key head (a word over a video, a question over its
// frames), or where larger tiles would leave most of the chip idle: bound by the keys' and values' memory, so the waves of a workgroup go
// over different keys at their own pace.  A wave reads its 32 keys a row at a time (whole lines; read straight as operands, 32 bytes of 32
// rows each, they fell out of the cache between the steps) into LDS of its own; nothing waits for another wave before the end.
#pragma once
#include "dvgr_attn.h"

namespace dvgr {
namespace attn {

// 32 rows of a tensor on their way to a wave's own LDS
template <typename T, int DP> struct WaveStage {
  typedef Tile<T, DP> Tl;
  static constexpr int N = Tl::kChunks / 2;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  u32x4 v[N];
  template <bool STREAM> __device__ __forceinline__ void load(const Side& s, int r0, int end, int dh_bytes, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = lane + i * 64, r = r0 + e / Tl::kChunks, c = (e % Tl::kChunks) * 16;
      v[i] = 0;
      if (r < end && c < dh_bytes) {
        const u32x4* p = reinterpret_cast<const u32x4*>(s.row(r) + c);
        v[i] = STREAM ? stream_load(p) : *p;
      }
    }
  }
  __device__ __forceinline__ void fetch(const Side& s, int r0, int end, int dh_bytes, bool stream, int lane) {
    if (stream) load<true>(s, r0, end, dh_bytes, lane);
    else load<false>(s, r0, end, dh_bytes, lane);
  }
  // rows without a bit are zeros, whatever was read
  template <int S> __device__ __forceinline__ void put(char* lds, uint32_t bits, int lane) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = lane + i * 64, r = e / Tl::kChunks;
      *reinterpret_cast<u32x4*>(lds + r * S + (e % Tl::kChunks) * 16) = (bits >> r) & 1 ? v[i] : (u32x4)0;
    }
  }
};

// LDS operations of one wave complete in order; this keeps the compiler from moving them across each other
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// where a wave of a workgroup stands: 32 rows of a key head, share of the keys, its first 32-key tile (it goes on in steps of KW)
struct FewWork {
  int b, hk, split, r0, n, t0, t1;
  bool any;
};
template <int KW> __device__ __forceinline__ FewWork few_work(const Args& A, int kw) {
  FewWork f{};
  const int rtiles = A.rows > 32 ? (A.rows + 31) / 32 : 1;         // (without rows: one tile, for the keys' zeros)
  const int64_t w = xcd_work((int64_t)A.a.B * A.a.Hk * A.splits * rtiles);
  f.any = w >= 0;
  if (!f.any) return f;
  f.r0 = (int)(w % rtiles) * 32;
  f.split = (int)(w / rtiles % A.splits);
  f.hk = (int)(w / rtiles / A.splits % A.a.Hk);
  f.b = (int)(w / rtiles / A.splits / A.a.Hk);
  f.n = key_count(A, f.b);
  const int tiles = (f.n + 31) / 32, per = A.tiles_per_split * KW;
  f.t0 = f.split * per + kw;
  f.t1 = (f.split + 1) * per < tiles ? (f.split + 1) * per : tiles;
  return f;
}

// Work in shares: `units` workgroups of `turns` turns each are split until there are `want` of them (as many as run at once), in shares of
// at least `least` turns.  Where that is no split, up to eight are looked at: 264 workgroups on 256 places are two rounds, 5 x 264 are six
// of a fifth.  A split costs a launch that joins it, about eight turns.  (One query over 33 x 7731 keys, 8 heads of 32, fp32: 176 -> 108 us;
// 40 x 2048 keys, 8 heads of 128, bf16, split for two turns less: 64 -> 70.)
struct Shares { int splits, turns_per_split; };
inline Shares shares_of(int64_t units, int64_t turns, int64_t want, int least) {
  int64_t s = units ? want / units : 1;
  if (s == 1 || (s < 1 && units < 4 * want)) {
    int64_t best = (units + want - 1) / want * turns;
    s = 1;
    for (int64_t x = 2; x <= 8; ++x) {
      const int64_t cost = (units * x + want - 1) / want * ((turns + x - 1) / x) + 8;
      if (cost < best) { best = cost; s = x; }
    }
  }
  if (s > turns / least) s = turns / least;
  if (s < 1) s = 1;
  Shares x{};
  x.turns_per_split = (int)((turns + s - 1) / s);
  if (x.turns_per_split < 1) x.turns_per_split = 1;
  x.splits = turns ? (int)((turns + x.turns_per_split - 1) / x.turns_per_split) : 1;
  return x;
}

// Waves of a workgroup and shares of the keys.  Up to 64 keys one wave does it all; otherwise four, and eight in the forward of two-byte
// types while there are fewer than two workgroups for each compute unit (eight fill its registers as two of four do, with half the
// shares to join).  The keys are split over workgroups while there are fewer than that, in shares of at least two turns.
// KW = 0: the kernels for many rows, which have no need of it: every compute unit has a workgroup of 128 rows.  (The backward adds up
// over all rows at once, so it takes at most 32.)  Where these rows are many and short of that the split keys are not always worth what
// every 32 rows pay to fetch them again.  Forward, here and with the kernel for many rows, us: 8 samples of 8 heads of 64, fp16, 120 queries
// over 512 / 4096 keys 7.6 / 28 and 12.4 / 70, 256 queries 10.4 / 51 and 12.8 / 71; 8 heads of 128, bf16, 1000 queries 11.7 / 45 and 17.3 / 94,
// 2000 queries 22 / 86 and 18 / 95, 3968 queries 47 / 231 and 20 / 102.
struct FewPlan { int KW, splits, tiles_per_split; };
inline FewPlan few_plan(const dvgr_attn_problem& a, bool forward) {
  FewPlan p{};
  const int64_t rows = (int64_t)a.Lq * (a.H / a.Hk), heads = (int64_t)a.B * a.Hk, units = heads * ((rows + 31) / 32);
  if (rows > 32 && (!forward || heads * ((rows + 127) / 128) >= 256)) return p;
  p.KW = a.Lk <= 64 ? 1 : forward && a.elem != DVGR_ELEM_F32 && units < 512 ? 8 : 4;
  const Shares s = shares_of(units, ((int64_t)a.Lk + p.KW * 32 - 1) / (p.KW * 32), p.KW == 8 ? 256 : 512, 2);
  p.splits = s.splits;
  p.tiles_per_split = s.turns_per_split;
  return p;
}

}  // namespace attn
}  // namespace dvgr
