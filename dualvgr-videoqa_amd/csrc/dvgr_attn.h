// dvgr_attn.h -- tiles of the attention kernels (dvgr_attn.hip, dvgr_attn_bwd.hip).
//
// Everything runs on 32 x 32 matrix tiles held by one wave.  With lane = 32 h + c, a tile's accumulator register r of lane (h, c) is
// element (row 8 (r / 4) + 4 h + r % 4, column c).  Scores are computed TRANSPOSED where a query's statistics are wanted (rows = keys,
// column = query): a lane then owns one query, the softmax runs over its registers and one exchange between the wave's halves, and the
// probabilities are already the second product's B operand if that product takes its keys in the order
//     16 s + 8 (j / 4) + 4 h + j % 4                (step s, element j of half h)
// -- the A operand (the values, transposed on the way out of LDS) is read in the same order, so nothing is moved between lanes.
//
// A "step" is 32 bytes of a row: half h of the wave holds bytes 16 h .. 16 h + 15 (one 16-deep MFMA for 2-byte types, four 2-deep
// ones for fp32; the order of the reduction is the same on both sides, so any order is right).
#pragma once
#include "../../include/dvgr_attn.h"
#include "dvgr_elem.h"

namespace dvgr {
namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T> using Frag = typename Vec16<T>::type;

__device__ __forceinline__ f32x16 mma(Frag<bf16_t> a, Frag<bf16_t> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(Frag<f16_t> a, Frag<f16_t> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(Frag<float> a, Frag<float> b, f32x16 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// Waves of a workgroup for many rows, 32 rows each.  Eight fetch and write half as much of a tile each (captions over long videos: forward
// 301 -> 288 us, dQ 400 -> 357), four make twice the workgroups: eight where every compute unit has one of them, and two waves of a SIMD fit
// (two-byte types).
inline int many_waves(int64_t heads, int64_t rows, int es) { return es == 2 && heads * ((rows + 255) / 256) >= 256 ? 8 : 4; }

// One head's side of a tensor: row r of the packed rows (query l, head g of the group, r = l * G + g) or key r (G = 1).  Every thread
// finds several rows' places in every turn, so this is kept to few instructions: a shift where G is a power of two, and products of
// 32 x 32 bits.
struct Side {
  const char* p;
  uint32_t sl;                      // bytes between rows, under 2^32
  int64_t sg;                       // bytes between heads
  int G, shift;                     // shift: log2 G, or -1
  __device__ __forceinline__ const char* row(int r) const {
    if (G == 1) return p + (uint64_t)(uint32_t)r * sl;
    const int l = shift >= 0 ? r >> shift : r / G;
    return p + (uint64_t)(uint32_t)l * sl + (uint32_t)(r - l * G) * sg;
  }
};

template <typename T, int DP> struct Tile {
  static constexpr int kRowBytes = DP * (int)sizeof(T);
  // Bytes between rows in LDS.  16 rows of one 16-byte piece (a row product's operand) fall on different banks if the stride is an odd
  // number of pieces; 4 rows of 4 pieces (an operand across the rows) need it to be 3, 5, 11 or 13 modulo 16 as well.
  static constexpr int kStride = kRowBytes + 16;
  static constexpr int kStrideT = sizeof(T) == 2 && DP == 128 ? kRowBytes + 48 : kStride;          // tiles read across their rows
  static constexpr int kSteps = kRowBytes / 32;
  static constexpr int kChunks = kRowBytes / 16;          // 16-byte pieces of a row
  static constexpr int kNT = DP / 32;                     // 32-wide tiles of the head dimension
  template <int ROWS> static constexpr int bytes() { return ROWS * kStride; }
  template <int ROWS> static constexpr int bytesT() { return ROWS * kStrideT; }

  // operand of a row-wise product: row `lane & 31` of the 32 rows at `at`
  template <int S = kStride> static __device__ __forceinline__ Frag<T> frag(const char* at, int step, int lane) {
    return *reinterpret_cast<const Frag<T>*>(at + (lane & 31) * S + step * 32 + (lane >> 5) * 16);
  }
  static __device__ __forceinline__ Frag<T> fragT(const char* at, int step, int lane) { return frag<kStrideT>(at, step, lane); }
  // the same straight from memory, zeros beyond the head and where `ok` is false
  static __device__ __forceinline__ Frag<T> gfrag(const char* row, int step, int lane, int dh_bytes, bool ok) {
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < Vec16<T>::N; ++i) f[i] = (T)0.f;
    const int at = step * 32 + (lane >> 5) * 16;
    if (ok && at < dh_bytes) f = *reinterpret_cast<const Frag<T>*>(row + at);
    return f;
  }
};

// acc[t] += M^T P: M = 32 rows of LDS at `at` (kStrideT apart, head dimension along the row), P = 32 x 32 in accumulator layout
template <int DP> __device__ __forceinline__ void mma_tr(f32x16 (&acc)[DP / 32], const char* at, const f32x16& p, int lane, float) {
  constexpr int S = Tile<float, DP>::kStrideT;
  const char* base = at + (lane >> 5) * 4 * S + (lane & 31) * 4;
#pragma unroll
  for (int r = 0; r < 16; ++r)
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) {
      const float a = *reinterpret_cast<const float*>(base + (8 * (r / 4) + r % 4) * S + t * 128);
      acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], acc[t], 0, 0, 0);
    }
}
template <typename T, int DP> __device__ __forceinline__ void mma_tr16(f32x16 (&acc)[DP / 32], const char* at, const f32x16& p, int lane) {
  constexpr int S = Tile<T, DP>::kStrideT;
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  // lanes of a group of 16 name 4 rows x 16 columns, 4 elements each, and get one column's 4 rows
  const char* base = at + ((lane >> 5) * 4 + (lane & 15) / 4) * S + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    Frag<T> b;
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = (T)p[8 * s + j];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) {
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(base + (16 * s) * S + t * 64));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(base + (16 * s + 8) * S + t * 64));
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      const s16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      acc[t] = mma(__builtin_bit_cast(Frag<T>, a), b, acc[t]);
    }
  }
}
template <int DP> __device__ __forceinline__ void mma_tr(f32x16 (&acc)[DP / 32], const char* at, const f32x16& p, int lane, bf16_t) { mma_tr16<bf16_t, DP>(acc, at, p, lane); }
template <int DP> __device__ __forceinline__ void mma_tr(f32x16 (&acc)[DP / 32], const char* at, const f32x16& p, int lane, f16_t) { mma_tr16<f16_t, DP>(acc, at, p, lane); }

// ROWS rows of a tensor on their way to LDS: fetched into registers one tile ahead, written behind the barrier that frees the tile.
// Nothing between the two may look at what was fetched: the wait for it would be a wait for memory in every turn.
template <typename T, int DP, int ROWS, int THREADS> struct Stage {
  typedef Tile<T, DP> Tl;
  static constexpr int kPieces = ROWS * Tl::kChunks, N = (kPieces + THREADS - 1) / THREADS;
  static constexpr bool kEven = kPieces % THREADS == 0;             // otherwise the last round is some threads' only
  uint4 v[N];
  // rows r0 .. of which those below `end` exist
  __device__ __forceinline__ void fetch(const Side& s, int r0, int end, int dh_bytes, int tid) {
    const bool whole = kEven && r0 + ROWS <= end && dh_bytes == Tl::kRowBytes;          // (uniform: no zeros to write, no lane to switch off)
    if (whole) load<true>(s, r0, end, dh_bytes, tid);
    else load<false>(s, r0, end, dh_bytes, tid);
  }
  template <bool whole> __device__ __forceinline__ void load(const Side& s, int r0, int end, int dh_bytes, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + i * THREADS, r = r0 + e / Tl::kChunks, c = (e % Tl::kChunks) * 16;
      if (whole) {
        v[i] = *reinterpret_cast<const uint4*>(s.row(r) + c);
        continue;
      }
      v[i] = make_uint4(0, 0, 0, 0);
      if (r < end && c < dh_bytes && (kEven || e < kPieces)) v[i] = *reinterpret_cast<const uint4*>(s.row(r) + c);
    }
  }
  // rows without a bit are zeros, whatever was read
  template <int S> __device__ __forceinline__ void put(char* lds, unsigned long long bits, int tid) const {
    if (bits == (ROWS == 64 ? ~0ull : (1ull << (ROWS & 63)) - 1)) {
      put<S>(lds, tid);
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + i * THREADS, r = e / Tl::kChunks;
      if (kEven || e < kPieces)
        *reinterpret_cast<uint4*>(lds + r * S + (e % Tl::kChunks) * 16) = (bits >> r) & 1 ? v[i] : make_uint4(0, 0, 0, 0);
    }
  }
  template <int S> __device__ __forceinline__ void put(char* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + i * THREADS;
      if (kEven || e < kPieces) *reinterpret_cast<uint4*>(lds + (e / Tl::kChunks) * S + (e % Tl::kChunks) * 16) = v[i];
    }
  }
};

// is key j there, as a number that is not looked at before it is needed
__device__ __forceinline__ uint32_t key_there(const uint8_t* mask, int j, int n) {
  uint32_t x = 0;
  if (j < n) {
    x = 1;
    if (mask) x = mask[j];
  }
  return x;
}

// Operands loaded in front of a loop are waited for here: left to their first use, inside the loop, that wait would also be one for the
// loop's own loads, in every turn.
template <typename F, int N> __device__ __forceinline__ void settle(F (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// Order of a block of matrix products of one LDS read each: kAhead reads in front, then one with every product.  Left to itself the
// compiler reads an operand right in front of its product, which then waits for LDS (captions over long videos, forward: 290 us, 281 with
// four reads in front, 272 with six or eight; dQ the same with and without, dK and dV, whose LDS is busier than its matrix units, slower).
constexpr int kAhead = 6;
template <int PRODUCTS> __device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
  for (int i = 0; i < PRODUCTS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (i + kAhead < PRODUCTS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
}

// the value of both halves of the wave, combined
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A row's maximum m, or its sum as a score, is taken off with the scaling by c = scale log2 e, in one multiply-add, c s - fl(c m), while
// fl(c m) is at most kFar in all rows of the wave.  Its rounding cancels where every term has it, but is 2^-24 of its size: more than an
// exponential bears from 2^31 on.  Beyond kFar m is taken off first, (s - m) c, which costs one operation more (captions over long videos
// with it everywhere: forward 278 us for 275, dQ 329 for 324, dK and dV 621 for 568).
constexpr float kFar = 4096.f;
__device__ __forceinline__ bool any_far(float cm) { return __any(fabsf(cm) > kFar && fabsf(cm) < INFINITY); }

// bit (8 (r / 4) + r % 4) of half h's word: is the key of register r there
__device__ __forceinline__ uint32_t half_bits(uint32_t bits, int lane) { return bits >> ((lane >> 5) * 4); }
__device__ __forceinline__ bool reg_bit(uint32_t hb, int r) { return (hb >> (8 * (r / 4) + r % 4)) & 1; }

// 4 consecutive elements (8 or 16 bytes)
template <typename T> __device__ __forceinline__ void store4(char* p, float a, float b, float c, float d) {
  typedef T v4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<v4*>(p) = v4{(T)a, (T)b, (T)c, (T)d};
}

// An 8-XCD chip hands workgroup i to XCD i % 8: give every XCD a contiguous run of the work, so that the workgroups that read the same
// keys share an L2.  A head with 8 workgroups or more (`tiles`) has one on every XCD instead: samples of different lengths would leave
// XCDs without work (2 x 4096 queries over 2100 and 4000 keys, 16 / 4 heads of 128, bf16: forward 272 us with runs, 214 without; forward and
// backward 1275, 1063).  Without lengths there is little between them: full keys 280, 277 and 1294, 1296; 8 x 2048 x 2048, 16 heads of 64,
// 195, 202 and 827, 855.  -1: nothing to do.
__device__ __forceinline__ int64_t xcd_work(int64_t total, int tiles = 1) {
  if (tiles >= 8) return blockIdx.x < total ? (int64_t)blockIdx.x : -1;
  const int64_t per = (total + 7) / 8, w = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  return (int64_t)(blockIdx.x >> 3) < per && w < total ? w : -1;
}
inline unsigned xcd_grid(int64_t total) { return (unsigned)((total + 7) / 8 * 8); }

struct Args {
  dvgr_attn_problem a;
  int G, shift, rows;               // heads of a group, log2 of it or -1; Lq * G packed rows of one key head
  int es;
  int splits, tiles_per_split;      // the keys of a sample in shares of whole tiles
  float c;                          // scale * log2 e
  bool stream;                      // keys and values are read past the caches
  float *part_o, *part_ml;          // splits > 1: (work, rows of the tile, Dh) and (.., 2)
};
__device__ __forceinline__ Side q_side(const Args& A, const dvgr_attn_view& v, int b, int hk) {
  return Side{(const char*)v.p + ((int64_t)b * v.sb + (int64_t)hk * A.G * v.sh) * A.es, (uint32_t)(v.sl * A.es), v.sh * A.es, A.G, A.shift};
}
__device__ __forceinline__ Side k_side(const Args& A, const dvgr_attn_view& v, int b, int hk) {
  return Side{(const char*)v.p + ((int64_t)b * v.sb + (int64_t)hk * v.sh) * A.es, (uint32_t)(v.sl * A.es), 0, 1, 0};
}
__device__ __forceinline__ int key_count(const Args& A, int b) {
  if (!A.a.lens) return A.a.Lk;
  const int64_t n = A.a.lens[b];
  return n < 0 ? 0 : n > A.a.Lk ? A.a.Lk : (int)n;
}
__device__ __forceinline__ int64_t row_index(const Args& A, int b, int hk, int r) {          // (B, H, Lq) of packed row r
  const int l = A.shift >= 0 ? r >> A.shift : r / A.G;
  return ((int64_t)b * A.a.H + hk * A.G + (r - l * A.G)) * A.a.Lq + l;
}

// row of what the output's rounding left (B, Lq, H, Dh), or nullptr
template <typename T> __device__ __forceinline__ char* lo_row(const Args& A, int b, int hk, int r) {
  if (sizeof(T) == 4 || !A.a.o_lo) return nullptr;
  const int l = A.shift >= 0 ? r >> A.shift : r / A.G;
  return (char*)A.a.o_lo + (((int64_t)b * A.a.Lq + l) * A.a.H + hk * A.G + (r - l * A.G)) * A.a.Dh * (int64_t)sizeof(T);
}

// More than 64 KB of LDS has to be asked for once on a device (`asked`: a bit for each).
inline int allow_lds(const void* kern, size_t bytes, std::atomic<uint32_t>& asked) {
  if (bytes <= 65536) return 0;
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return (int)e;
  if (asked.load(std::memory_order_relaxed) >> (dev & 31) & 1) return 0;
  e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == hipSuccess) asked.fetch_or(1u << (dev & 31), std::memory_order_relaxed);
  return (int)e;
}

Args make_args(const dvgr_attn_problem& a);
int launch_backward(const Args& A, const dvgr_attn_grads& g, void* ws, hipStream_t st);
size_t backward_bytes(const dvgr_attn_problem& a);

}  // namespace attn
}  // namespace dvgr
