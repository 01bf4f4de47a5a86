// dvgr_embed.hip -- include/dvgr_inputs.h: token embedding with scaling, and its gradient by sorted tokens.
//
//   y_i = s E[t_i]                                   G[v] = s sum_{i : t_i = v} dy_i   (i ascending)
//
// Both are bound by memory: the forward reads and writes n rows, the backward reads n rows and writes the whole table.  The
// gradient brings the positions of a token together, adds their rows in fp32 in an order that the tokens alone decide, and rounds
// once: no float atomics, so the result does not depend on the schedule.  Two forms: up to kSmall positions one launch in which
// every workgroup picks the tokens of its own rows of the table; beyond, a stable radix sort of (token, position) pairs.
//
// 65536 positions x 1024 bf16 of 50000 words: forward 27 us, sort 27 in four launches, sums 40, join 14.5; 104 us where 474 MB at a large
// copy's rate take 96.  960 x 300 fp32 of 4000 words: 2.6 and 8.2 us, less than it takes to call them.  Between the two the sort's launches
// weigh (30000 x 300 bf16 of 20000 words: 67 us for both passes, 12 for the bytes; a sort block takes 1024 pairs at least), and rows that are
// no multiple of 16 bytes go in smaller pieces (53291 x 806 fp16: 96 us, 47 for the bytes).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/dvgr.h"
#include "../../include/dvgr_inputs.h"
#include "dvgr_elem.h"

namespace dvgr {
namespace {

// Rows are handled V elements at a time: 16 bytes where rows start at multiples of 16 bytes, otherwise pairs where an even width allows it
// (53291 x 806 fp16 of 19164 words, forward and backward: 198 us by single elements, 112 by pairs), otherwise single elements.  Neighbouring
// lanes take neighbouring pieces.
template <typename T, int V> using Piece = T __attribute__((ext_vector_type(V)));

// One wave per token position, a few pieces in flight.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_embed_fwd(const T* __restrict__ table, int64_t vocab, int wd, const int64_t* __restrict__ tokens, int64_t n,
                                                   float scale, T* __restrict__ y, int32_t* bad) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= n) return;
  const int64_t tok = tokens[row];
  const bool ok = tok >= 0 && tok < vocab;
  if (!ok && lane == 0 && bad) *bad = 1;
  T* dst = y + row * wd;
  const T* src = table + (ok ? tok : 0) * (int64_t)wd;
  constexpr int U = V == Vec16<T>::N ? 2 : 4;
  for (int c0 = lane * V; c0 < wd; c0 += U * 64 * V) {
    Piece<T, V> f[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * 64 * V < wd) f[u] = *reinterpret_cast<const Piece<T, V>*>(src + c0 + u * 64 * V);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c0 + u * 64 * V >= wd) break;
#pragma unroll
      for (int i = 0; i < V; ++i) f[u][i] = (T)(ok ? (float)f[u][i] * scale : 0.f);
      Piece<T, V>* to = reinterpret_cast<Piece<T, V>*>(dst + c0 + u * 64 * V);
      if (V == Vec16<T>::N) stream_store(to, f[u]);
      else *to = f[u];
    }
  }
}

// ---- stable radix sort of (token, position), 8 bits a pass ------------------------------------------------------------------
// A block owns `tile` consecutive elements.  Pass 0 reads the tokens themselves; a token that has no gradient (outside the table,
// or the padding token) gets the key `vocab`, which sorts behind every row.
constexpr int kRadix = 256, kSortThreads = kRadix, kSortBlocks = 256;

struct SortPass {
  const int64_t* tokens;            // pass 0
  const int32_t *key, *pos;         // later passes
  int32_t *key_out, *pos_out;
  int32_t* hist;                    // blocks x kRadix counts
  int64_t n, vocab, padding;
  int tile, blocks, shift;
};

__device__ __forceinline__ int32_t sort_key(const SortPass& s, int64_t i) {
  if (!s.tokens) return s.key[i];
  const int64_t t = s.tokens[i];
  return t < 0 || t >= s.vocab || t == s.padding ? (int32_t)s.vocab : (int32_t)t;
}

__global__ __launch_bounds__(kSortThreads) void k_sort_count(SortPass s) {
  __shared__ int32_t cnt[kRadix];
  const int tid = threadIdx.x;
  for (int d = tid; d < kRadix; d += kSortThreads) cnt[d] = 0;
  __syncthreads();
  const int64_t a = (int64_t)blockIdx.x * s.tile, e = a + s.tile < s.n ? a + s.tile : s.n;
  for (int64_t i = a + tid; i < e; i += kSortThreads) atomicAdd(&cnt[(sort_key(s, i) >> s.shift) & (kRadix - 1)], 1);
  __syncthreads();
  for (int d = tid; d < kRadix; d += kSortThreads) s.hist[(int64_t)blockIdx.x * kRadix + d] = cnt[d];
}

// Stable scatter.  Thread d adds up digit d over all blocks (there are at most kSortBlocks) and over those in front of this one; with the
// digits in front that is the block's first place.  Then rounds of 256 consecutive elements; an element's place is the digit's next
// free place plus the number of equal digits in front of it in the round (earlier waves' counts, then earlier lanes by ballots).
__global__ __launch_bounds__(kSortThreads) void k_sort_scatter(SortPass s) {
  __shared__ int32_t next[kRadix], wcnt[4][kRadix], wsum[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  {
    int32_t all = 0, front = 0;
#pragma unroll 8
    for (int b = 0; b < s.blocks; ++b) {
      const int32_t c = s.hist[b * kRadix + tid];
      all += c;
      front += b < (int)blockIdx.x ? c : 0;
    }
    int32_t inc = all;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t up = __shfl_up(inc, d);
      if (lane >= d) inc += up;
    }
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    int32_t at = inc - all + front;
    for (int w = 0; w < wave; ++w) at += wsum[w];
    next[tid] = at;
  }
  const int64_t a = (int64_t)blockIdx.x * s.tile, e = a + s.tile < s.n ? a + s.tile : s.n;
  for (int64_t i0 = a; i0 < e; i0 += kSortThreads) {
    const int64_t i = i0 + tid;
    const bool live = i < e;
    const int32_t key = live ? sort_key(s, i) : 0;
    const int32_t pos = live ? (s.tokens ? (int32_t)i : s.pos[i]) : 0;
    const int digit = (key >> s.shift) & (kRadix - 1);
    unsigned long long same = __ballot(live);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const unsigned long long m = __ballot((digit >> b) & 1);
      same &= (digit >> b) & 1 ? m : ~m;
    }
    const int before = __popcll(same & ((1ull << lane) - 1ull));
    for (int d = lane; d < kRadix; d += 64) wcnt[wave][d] = 0;
    __syncthreads();
    if (live && before == 0) wcnt[wave][digit] = __popcll(same);
    __syncthreads();
    if (live) {
      int32_t at = next[digit] + before;
      for (int w = 0; w < wave; ++w) at += wcnt[w][digit];
      s.key_out[at] = key;
      s.pos_out[at] = pos;
    }
    __syncthreads();
    for (int d = tid; d < kRadix; d += kSortThreads) next[d] += wcnt[0][d] + wcnt[1][d] + wcnt[2][d] + wcnt[3][d];
    __syncthreads();
  }
}

// ---- rows of one token are consecutive now: sum them ------------------------------------------------------------------------
// One wave owns `kChunk` sorted pairs and 64 lanes x NE elements of the row.  A token whose pairs all lie in the chunk is written at
// once; one that crosses the chunk's ends leaves fp32 partial sums, head (0) and tail (1), which k_embed_join adds in chunk order.
constexpr int kChunk = 32;

template <typename T, int V> struct Cols {
  static constexpr int N = Vec16<T>::N;
  int c0, wd, lane;
  __device__ Cols(int block, int wd_, int lane_) : c0(block * 64 * N), wd(wd_), lane(lane_) {}
  __device__ __forceinline__ int at(int i) const { return c0 + (i / V * 64 + lane) * V + i % V; }
  typedef typename Vec16<T>::type Raw;                              // held as loaded: half the registers of floats for two-byte types
  __device__ __forceinline__ Raw load(const T* row) const {
    Raw v;
    if constexpr (V == N) {
      if (at(0) < wd) return stream_load(reinterpret_cast<const Raw*>(row + at(0)));
      v = (T)0.f;
    } else {
#pragma unroll
      for (int p = 0; p < N; p += V) {
        Piece<T, V> x = (T)0.f;
        if (at(p) < wd) x = *reinterpret_cast<const Piece<T, V>*>(row + at(p));
#pragma unroll
        for (int i = 0; i < V; ++i) v[p + i] = x[i];
      }
    }
    return v;
  }
  static __device__ __forceinline__ void add(float (&acc)[N], const Raw& v) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += (float)v[i];
  }
  __device__ __forceinline__ void store(T* row, const float (&f)[N]) const {
    if constexpr (V == N) {
      if (at(0) < wd) stream_store_vec(row + at(0), f);
    } else {
#pragma unroll
      for (int p = 0; p < N; p += V) {
        Piece<T, V> x;
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (T)f[p + i];
        if (at(p) < wd) *reinterpret_cast<Piece<T, V>*>(row + at(p)) = x;
      }
    }
  }
  // fp32 sums of a row, up to four elements at a time
  static constexpr int VP = V < 4 ? V : 4;
  __device__ __forceinline__ void store_part(float* row, const float (&f)[N]) const {
#pragma unroll
    for (int p = 0; p < N; p += VP) {
      Piece<float, VP> x;
#pragma unroll
      for (int i = 0; i < VP; ++i) x[i] = f[p + i];
      if (at(p) < wd) *reinterpret_cast<Piece<float, VP>*>(row + at(p)) = x;
    }
  }
  __device__ __forceinline__ void add_part(const float* row, float (&f)[N]) const {
#pragma unroll
    for (int p = 0; p < N; p += VP)
      if (at(p) < wd) {
        const Piece<float, VP> x = *reinterpret_cast<const Piece<float, VP>*>(row + at(p));
#pragma unroll
        for (int i = 0; i < VP; ++i) f[p + i] += x[i];
      }
  }
};

// the rows of the table that no pair names are zero: blocks behind those of the sums look their rows up and clear them
template <typename T, int V>
__device__ __forceinline__ void zero_rows(const int32_t* key, int64_t n, int64_t vocab, int wd, int64_t r0, int rows, T* g_table) {
  constexpr int N = Vec16<T>::N;
  __shared__ int sh_there[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid < rows && r0 + tid < vocab) {
    int64_t a = 0, b = n;                                           // first pair of a token >= r0 + tid
    while (a < b) {
      const int64_t m = (a + b) >> 1;
      if (key[m] < r0 + tid) a = m + 1; else b = m;
    }
    sh_there[tid] = a < n && key[a] == r0 + tid;
  }
  __syncthreads();
  for (int r = wave; r < rows && r0 + r < vocab; r += 4) {
    if (sh_there[r]) continue;
    T* row = g_table + (r0 + r) * wd;
    for (int c = lane * V; c < wd; c += 64 * V) {
      const Piece<T, V> z = (T)0.f;
      if (V == N) stream_store(reinterpret_cast<Piece<T, V>*>(row + c), z);
      else *reinterpret_cast<Piece<T, V>*>(row + c) = z;
    }
  }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void k_embed_sum(const T* __restrict__ g_y, const int32_t* key, const int32_t* pos, int64_t n, int64_t vocab, int wd,
                                                   int colblocks, float scale, T* __restrict__ g_table, float* part, int sum_blocks, int zero_per) {
  constexpr int N = Vec16<T>::N, U = 8;
  if ((int)blockIdx.x >= sum_blocks) {
    zero_rows<T, V>(key, n, vocab, wd, (int64_t)((int)blockIdx.x - sum_blocks) * zero_per, zero_per, g_table);
    return;
  }
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t chunk = unit / colblocks, a = chunk * kChunk;
  if (a >= n) return;
  const Cols<T, V> cols((int)(unit % colblocks), wd, lane);
  const int m = (int)(n - a < kChunk ? n - a : kChunk);
  const int32_t mykey = lane < m ? key[a + lane] : (int32_t)vocab;
  const int32_t mypos = lane < m ? pos[a + lane] : 0;
  const int32_t left = a > 0 ? key[a - 1] : -1;                     // the pair in front of the chunk, and the one behind it
  const int32_t right = a + m < n ? key[a + m] : -1;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  int32_t cur = __builtin_amdgcn_readfirstlane(mykey);
  if (cur >= vocab) return;
  bool open_left = cur == left;
  for (int j0 = 0; j0 < m; j0 += U) {
    typename Cols<T, V>::Raw f[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {                                   // (padding pairs of a short chunk read a row that exists: position 0)
      const int32_t p = __builtin_amdgcn_readlane(mypos, (j0 + u) & 63);
      f[u] = cols.load(g_y + (int64_t)p * wd);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j0 + u >= m) break;
      const int32_t k = __builtin_amdgcn_readlane(mykey, (j0 + u) & 63);
      if (k != cur) {
        if (open_left) cols.store_part(part + (2 * chunk) * wd, acc);
        else {
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] *= scale;
          cols.store(g_table + (int64_t)cur * wd, acc);
        }
        cur = k; open_left = false;
        if (cur >= vocab) return;                                   // (sorted: only pairs without a gradient follow)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.f;
      }
      cols.add(acc, f[u]);
    }
  }
  if (open_left) cols.store_part(part + (2 * chunk) * wd, acc);     // a token that fills the chunk and came in from the left: head
  else if (cur == right) cols.store_part(part + (2 * chunk + 1) * wd, acc);
  else {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= scale;
    cols.store(g_table + (int64_t)cur * wd, acc);
  }
}

// Tokens that cross chunks: the chunk where a token starts adds its tail and the heads that follow.  A wave looks at one chunk's end and
// adds up to kAlone heads by itself; a frequent token has hundreds, which the workgroup's waves share, consecutive equal parts each,
// added in order.
constexpr int kJoinWaves = 16, kAlone = 8;
template <typename T, int V>
__global__ __launch_bounds__(64 * kJoinWaves) void k_embed_join(const int32_t* key, int64_t n, int64_t vocab, int wd, int colblocks, float scale,
                                                                T* g_table, const float* part) {
  constexpr int N = Vec16<T>::N;
  __shared__ float sh[kJoinWaves][64 * N];
  __shared__ int32_t sh_long[kJoinWaves], sh_end;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t chunks = (n + kChunk - 1) / kChunk, first = (int64_t)(blockIdx.x / colblocks) * kJoinWaves, mine = first + wave;
  const Cols<T, V> cols((int)(blockIdx.x % colblocks), wd, lane);
  // heads of the token that starts in chunk c and leaves it, up to 64; 0: there is none
  const auto heads_of = [&](int64_t c) {
    const int64_t b = (c + 1) * kChunk;                             // c + 1 is a chunk: b < n
    const int32_t k = key[b - 1];
    if (k >= vocab || key[b] != k || (c > 0 && key[c * kChunk - 1] == k)) return 0;
    const unsigned long long other = __ballot(c + 1 + lane >= chunks || key[(c + 1 + lane) * kChunk] != k);
    return other ? __ffsll(other) - 1 : 64;
  };
  float acc[N];
  int heads = mine + 1 < chunks ? heads_of(mine) : 0;
  if (lane == 0) sh_long[wave] = heads > kAlone;
  if (heads > 0 && heads <= kAlone) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    cols.add_part(part + (2 * mine + 1) * wd, acc);
#pragma unroll 2
    for (int h = 1; h <= heads; ++h) cols.add_part(part + 2 * (mine + h) * wd, acc);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= scale;
    cols.store(g_table + (int64_t)key[(mine + 1) * kChunk] * wd, acc);
  }
  __syncthreads();
  for (int w = 0; w < kJoinWaves; ++w) {
    if (!sh_long[w]) continue;                                      // (uniform over the workgroup)
    const int64_t c = first + w;
    const int32_t k = key[(c + 1) * kChunk];
    int64_t a = c + 1;                                              // first chunk behind c that does not start with k
    for (int got = 64 * kJoinWaves; got == 64 * kJoinWaves; a += got) {
      if (tid == 0) sh_end = 64 * kJoinWaves;
      __syncthreads();
      if (a + tid >= chunks || key[(a + tid) * kChunk] != k) atomicMin(&sh_end, tid);
      __syncthreads();
      got = sh_end;
      __syncthreads();
    }
    const int64_t share = (a - (c + 1) + kJoinWaves - 1) / kJoinWaves;
    const int64_t h0 = c + 1 + wave * share, h1 = h0 + share < a ? h0 + share : a;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    if (wave == 0) cols.add_part(part + (2 * c + 1) * wd, acc);
#pragma unroll 4
    for (int64_t h = h0; h < h1; ++h) cols.add_part(part + (2 * h) * wd, acc);
#pragma unroll
    for (int i = 0; i < N; ++i) sh[wave][i * 64 + lane] = acc[i];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float x = acc[i];
        for (int v = 1; v < kJoinWaves; ++v) x += sh[v][i * 64 + lane];
        acc[i] = x * scale;
      }
      cols.store(g_table + (int64_t)k * wd, acc);
    }
    __syncthreads();
  }
}

// ---- few positions: one launch ----------------------------------------------------------------------------------------------
// Workgroup w of kSmallGroups owns the rows w, w + kSmallGroups, ... (the frequent tokens of a vocabulary are neighbours).  It reads all
// the tokens (they fit the L2 many times over) and keeps the positions of its own in their order.  A wave takes a row and adds its
// positions one after the other; a row of more than kAloneRow positions is shared by the workgroup's waves, consecutive equal parts each,
// added in order.
constexpr int kSmall = 4096, kSmallWaves = 16, kSmallThreads = 64 * kSmallWaves, kSmallRows = 256, kAloneRow = 16, kSmallGroups = 512;

template <typename T, int V>
__global__ __launch_bounds__(kSmallThreads) void k_embed_small(const T* __restrict__ g_y, const int64_t* __restrict__ tokens, int n, int64_t vocab, int wd,
                                                               int colblocks, float scale, int64_t padding, T* __restrict__ g_table) {
  constexpr int N = Vec16<T>::N, U = 4;
  __shared__ uint16_t pos[kSmall], sel[kSmall], row[kSmall];
  __shared__ int32_t cnt[kSmallRows], wcnt[kSmallWaves];
  __shared__ float sh[kSmallWaves][64 * N];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int rows = (int)((vocab - blockIdx.x + kSmallGroups - 1) / kSmallGroups);
  const auto row_at = [&](int r) { return g_table + ((int64_t)r * kSmallGroups + blockIdx.x) * wd; };
  if (tid < kSmallRows) cnt[tid] = 0;
  __syncthreads();
  // puts the elements that are `mine` behind the `have` that are there, in the threads' order; how many there are then
  const auto compact = [&](int have, bool mine, auto put) {
    const unsigned long long b = __ballot(mine);
    if (lane == 0) wcnt[wave] = __popcll(b);
    __syncthreads();
    int at = have + __popcll(b & ((1ull << lane) - 1ull)), all = have;
    for (int w = 0; w < kSmallWaves; ++w) {
      at += w < wave ? wcnt[w] : 0;
      all += wcnt[w];
    }
    if (mine) put(at);
    __syncthreads();
    return all;
  };
  int m = 0;
  for (int i0 = 0; i0 < n; i0 += kSmallThreads) {
    const int i = i0 + tid;
    const int64_t t = i < n ? tokens[i] : -1;
    const bool mine = t >= 0 && t < vocab && t % kSmallGroups == blockIdx.x && t != padding;
    if (mine) atomicAdd(&cnt[t / kSmallGroups], 1);
    m = compact(m, mine, [&](int at) { pos[at] = (uint16_t)i; row[at] = (uint16_t)(t / kSmallGroups); });
  }
  float acc[N];
  for (int r = wave; r < rows; r += kSmallWaves) {
    if (cnt[r] > kAloneRow) continue;
    for (int cb = 0; cb < colblocks; ++cb) {
      const Cols<T, V> cols(cb, wd, lane);
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.f;
      for (int j0 = 0, left = cnt[r]; left; j0 += 64) {             // ends: the list holds cnt[r] of row r
        unsigned long long b = __ballot(j0 + lane < m && row[(j0 + lane) & (kSmall - 1)] == r);
        left -= __popcll(b);
        while (b) {
          typename Cols<T, V>::Raw f[U];
          int have = 0;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (!b) break;
            f[u] = cols.load(g_y + (int64_t)pos[j0 + __ffsll(b) - 1] * wd);
            b &= b - 1;
            ++have;
          }
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (u < have) cols.add(acc, f[u]);
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] *= scale;
      cols.store(row_at(r), acc);
    }
  }
  for (int r = 0; r < rows; ++r) {
    const int k = cnt[r];
    if (k <= kAloneRow) continue;                                   // (uniform over the workgroup)
    int have = 0;
    for (int j0 = 0; j0 < m; j0 += kSmallThreads) {
      const int j = j0 + tid;
      have = compact(have, j < m && row[j & (kSmall - 1)] == r, [&](int at) { sel[at] = pos[j]; });
    }
    const int share = (k + kSmallWaves - 1) / kSmallWaves, a = wave * share, b = a + share < k ? a + share : k;
    for (int cb = 0; cb < colblocks; ++cb) {
      const Cols<T, V> cols(cb, wd, lane);
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.f;
      for (int j = a; j < b; j += U) {
        typename Cols<T, V>::Raw f[U];
#pragma unroll
        for (int u = 0; u < U; ++u) f[u] = cols.load(g_y + (int64_t)sel[j + u < b ? j + u : j] * wd);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (j + u < b) cols.add(acc, f[u]);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) sh[wave][i * 64 + lane] = acc[i];
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          float x = acc[i];
          for (int w = 1; w < kSmallWaves; ++w) x += sh[w][i * 64 + lane];
          acc[i] = x * scale;
        }
        cols.store(row_at(r), acc);
      }
      __syncthreads();
    }
  }
}

// One launch for up to kSmall positions while a workgroup's rows fit its counters.
struct EmbedPlan {
  bool small;
  int tile, blocks, passes, colblocks;
  int64_t chunks;
  size_t key[2], pos[2], hist, part, total;       // byte offsets
};
EmbedPlan embed_plan(int64_t n, int64_t vocab, int wd, int elem) {
  EmbedPlan p{};
  p.small = n <= kSmall && vocab <= (int64_t)kSmallGroups * kSmallRows;
  if (p.small) return p;
  const int64_t tile = (n + kSortBlocks - 1) / kSortBlocks;          // at most kSortBlocks blocks, 1024 pairs each at least
  p.tile = (int)(tile < 1024 ? 1024 : (tile + kSortThreads - 1) / kSortThreads * kSortThreads);
  p.blocks = (int)((n + p.tile - 1) / p.tile);
  for (int64_t v = vocab; v; v >>= 8) ++p.passes;                   // keys are 0 .. vocab
  p.colblocks = (wd + 64 * (16 / elem_size(elem)) - 1) / (64 * (16 / elem_size(elem)));
  p.chunks = (n + kChunk - 1) / kChunk;
  size_t o = 0;
  const auto take = [&o](size_t b) { const size_t at = o; o += (b + 255) / 256 * 256; return at; };
  for (int i = 0; i < 2; ++i) { p.key[i] = take(4 * (size_t)n); p.pos[i] = take(4 * (size_t)n); }
  p.hist = take(4 * (size_t)kRadix * p.blocks);
  p.part = take(2 * (size_t)p.chunks * wd * sizeof(float));
  p.total = o;
  return p;
}

int embed_check(int64_t n, int64_t vocab, int wd, int elem) {
  if (!elem_size(elem)) return DVGR_E_KIND;
  if (vocab < 1 || vocab >= (1ll << 31) - 1 || wd < 1 || wd >= (1 << 30) || n < 0 || n > (1ll << 26) - 64) return DVGR_E_DIMS;
  if (n / kChunk * (wd / 256 + 1) >= (1ll << 23)) return DVGR_E_DIMS;            // a launch holds at most 2^32 threads
  return 0;
}

// f(V as a type): the widest pieces that rows of `wd` elements at both addresses allow
template <typename T, typename F> int by_piece(int wd, const void* a, const void* b, F f) {
  constexpr int N = Vec16<T>::N;
  const uintptr_t at = (uintptr_t)a | (uintptr_t)b;
  if (wd % N == 0 && at % 16 == 0) return f(std::integral_constant<int, N>());
  if (wd % 2 == 0 && at % (2 * sizeof(T)) == 0) return f(std::integral_constant<int, 2>());
  return f(std::integral_constant<int, 1>());
}

template <typename T>
int embed_forward(const T* table, int64_t vocab, int wd, const int64_t* tokens, int64_t n, float scale, T* y, int32_t* bad, hipStream_t st) {
  const dim3 grid((unsigned)((n + 3) / 4));
  by_piece<T>(wd, table, y, [&](auto v) {
    DVGR_LAUNCH((k_embed_fwd<T, decltype(v)::value>), grid, dim3(256), 0, st, table, vocab, wd, tokens, n, scale, y, bad);
    return 0;
  });
  return (int)hipGetLastError();
}

template <typename T, int V>
int embed_sum(const T* g_y, const int32_t* key, const int32_t* pos, int64_t n, int64_t vocab, int wd, const EmbedPlan& p, float scale,
              T* g_table, float* part, hipStream_t st) {
  const int64_t row_bytes = (int64_t)wd * sizeof(T), sum_blocks = (p.chunks * p.colblocks + 3) / 4;
  const int zero_per = row_bytes >= 32768 ? 1 : row_bytes <= 128 ? 256 : (int)(32768 / row_bytes);
  DVGR_LAUNCH((k_embed_sum<T, V>), dim3((unsigned)(sum_blocks + (vocab + zero_per - 1) / zero_per)), dim3(256), 0, st, g_y, key, pos, n, vocab, wd,
              p.colblocks, scale, g_table, part, (int)sum_blocks, zero_per);
  int e = (int)hipGetLastError();
  if (e || p.chunks < 2) return e;
  DVGR_LAUNCH((k_embed_join<T, V>), dim3((unsigned)((p.chunks - 1 + kJoinWaves - 1) / kJoinWaves * p.colblocks)), dim3(64 * kJoinWaves), 0, st, key, n,
              vocab, wd, p.colblocks, scale, g_table, part);
  return (int)hipGetLastError();
}

template <typename T, int V>
int embed_small(const T* g_y, const int64_t* tokens, int n, int64_t vocab, int wd, float scale, int64_t padding, T* g_table, hipStream_t st) {
  const int colblocks = (wd + 64 * Vec16<T>::N - 1) / (64 * Vec16<T>::N);
  DVGR_LAUNCH((k_embed_small<T, V>), dim3((unsigned)(vocab < kSmallGroups ? vocab : kSmallGroups)), dim3(kSmallThreads), 0, st, g_y, tokens, n, vocab, wd, colblocks, scale,
              padding, g_table);
  return (int)hipGetLastError();
}

template <typename T>
int embed_backward(const T* g_y, const int64_t* tokens, int64_t n, int64_t vocab, int wd, float scale, int64_t padding, T* g_table,
                   char* ws, const EmbedPlan& p, hipStream_t st) {
  if (p.small)
    return by_piece<T>(wd, g_y, g_table, [&](auto v) {
      return embed_small<T, decltype(v)::value>(g_y, tokens, (int)n, vocab, wd, scale, padding, g_table, st);
    });
  SortPass s{};
  s.n = n; s.vocab = vocab; s.padding = padding; s.tile = p.tile; s.blocks = p.blocks;
  s.hist = reinterpret_cast<int32_t*>(ws + p.hist);
  int at = 0;
  for (int i = 0; n && i < p.passes; ++i, at ^= 1) {
    s.tokens = i ? nullptr : tokens;
    s.key = reinterpret_cast<int32_t*>(ws + p.key[at]); s.pos = reinterpret_cast<int32_t*>(ws + p.pos[at]);
    s.key_out = reinterpret_cast<int32_t*>(ws + p.key[at ^ 1]); s.pos_out = reinterpret_cast<int32_t*>(ws + p.pos[at ^ 1]);
    s.shift = 8 * i;
    DVGR_LAUNCH(k_sort_count, dim3(p.blocks), dim3(kSortThreads), 0, st, s);
    DVGR_LAUNCH(k_sort_scatter, dim3(p.blocks), dim3(kSortThreads), 0, st, s);
  }
  const int32_t* key = reinterpret_cast<const int32_t*>(ws + p.key[at]);
  const int32_t* pos = reinterpret_cast<const int32_t*>(ws + p.pos[at]);
  float* part = reinterpret_cast<float*>(ws + p.part);
  return by_piece<T>(wd, g_y, g_table, [&](auto v) {
    return embed_sum<T, decltype(v)::value>(g_y, key, pos, n, vocab, wd, p, scale, g_table, part, st);
  });
}

}  // namespace
}  // namespace dvgr

using namespace dvgr;

extern "C" {

int dvgr_embed_forward(const void* table, int64_t vocab, int wd, int elem, const int64_t* tokens, int64_t n, float scale, void* y,
                       int32_t* bad_tokens, void* stream) {
  const int e = embed_check(n, vocab, wd, elem);
  if (e) return e;
  if (n == 0) return 0;
  if (!table || !tokens || !y) return DVGR_E_NULL;
  hipStream_t st = (hipStream_t)stream;
  switch (elem) {
    case DVGR_ELEM_F32: return embed_forward((const float*)table, vocab, wd, tokens, n, scale, (float*)y, bad_tokens, st);
    case DVGR_ELEM_BF16: return embed_forward((const bf16_t*)table, vocab, wd, tokens, n, scale, (bf16_t*)y, bad_tokens, st);
    default: return embed_forward((const f16_t*)table, vocab, wd, tokens, n, scale, (f16_t*)y, bad_tokens, st);
  }
}

size_t dvgr_embed_workspace_bytes(int64_t n, int64_t vocab, int wd, int elem) {
  return embed_check(n, vocab, wd, elem) ? 0 : embed_plan(n, vocab, wd, elem).total;
}

int dvgr_embed_backward(const void* g_y, const int64_t* tokens, int64_t n, int64_t vocab, int wd, int elem, float scale, int64_t padding_idx,
                        void* g_table, void* workspace, size_t workspace_bytes, void* stream) {
  const int e = embed_check(n, vocab, wd, elem);
  if (e) return e;
  const EmbedPlan p = embed_plan(n, vocab, wd, elem);
  if (!g_table || (n && (!g_y || !tokens)) || (p.total && !workspace)) return DVGR_E_NULL;
  if (workspace_bytes < p.total) return DVGR_E_WORKSPACE;
  if (!ptr16(workspace)) return DVGR_E_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  switch (elem) {
    case DVGR_ELEM_F32: return embed_backward((const float*)g_y, tokens, n, vocab, wd, scale, padding_idx, (float*)g_table, ws, p, st);
    case DVGR_ELEM_BF16: return embed_backward((const bf16_t*)g_y, tokens, n, vocab, wd, scale, padding_idx, (bf16_t*)g_table, ws, p, st);
    default: return embed_backward((const f16_t*)g_y, tokens, n, vocab, wd, scale, padding_idx, (f16_t*)g_table, ws, p, st);
  }
}

}  // extern "C"
