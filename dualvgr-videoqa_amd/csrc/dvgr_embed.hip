// dvgr_embed.hip -- include/dvgr_inputs.h: token embedding with scaling, and its gradient by sorted tokens.
//
//   y_i = s E[t_i]                                   G[v] = s sum_{i : t_i = v} dy_i   (i ascending)
//
// Both are bound by memory: the forward reads and writes n rows, the backward reads n rows and writes the whole table.  The
// gradient sorts (token, position) pairs by token with a stable radix sort and adds the rows of a token in the order of their
// positions, in fp32, and rounds once: no float atomics, so the result does not depend on the schedule.
#include <hip/hip_runtime.h>

#include "../../include/dvgr.h"
#include "../../include/dvgr_inputs.h"
#include "dvgr_elem.h"

namespace dvgr {
namespace {

// One wave per token position.  VEC: rows of 16-byte vectors; otherwise single elements, neighbouring lanes on neighbours.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_embed_fwd(const T* table, int64_t vocab, int wd, const int64_t* tokens, int64_t n,
                                                   float scale, T* y, int32_t* bad) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= n) return;
  const int64_t tok = tokens[row];
  const bool ok = tok >= 0 && tok < vocab;
  if (!ok && lane == 0 && bad) *bad = 1;
  T* dst = y + row * wd;
  const T* src = table + (ok ? tok : 0) * (int64_t)wd;
  constexpr int N = Vec16<T>::N;
  if (VEC) {
    for (int c = lane; c < wd / N; c += 64) {
      float f[N];
      load_vec(src + c * N, f);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = ok ? f[i] * scale : 0.f;
      store_vec(dst + c * N, f);
    }
  } else {
    for (int c = lane; c < wd; c += 64) dst[c] = (T)(ok ? (float)src[c] * scale : 0.f);
  }
}

// ---- stable radix sort of (token, position), 8 bits a pass ------------------------------------------------------------------
// A block owns `tile` consecutive elements.  Pass 0 reads the tokens themselves; a token that has no gradient (outside the table,
// or the padding token) gets the key `vocab`, which sorts behind every row.
constexpr int kRadix = 256, kSortThreads = 256;

struct SortPass {
  const int64_t* tokens;            // pass 0
  const int32_t *key, *pos;         // later passes
  int32_t *key_out, *pos_out;
  int32_t* hist;                    // kRadix x blocks: counts, then first places
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
  for (int d = tid; d < kRadix; d += kSortThreads) s.hist[(int64_t)d * s.blocks + blockIdx.x] = cnt[d];
}

// exclusive prefix sum of kRadix x blocks counts, digit-major: one workgroup, each thread a run of consecutive counts
__global__ __launch_bounds__(1024) void k_sort_scan(int32_t* hist, int64_t count) {
  __shared__ int32_t wsum[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t run = (count + 1023) / 1024, a = tid * run, e = a + run < count ? a + run : count;
  int32_t own = 0;
  for (int64_t i = a; i < e; ++i) own += hist[i];
  int32_t inc = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t up = __shfl_up(inc, d);
    if (lane >= d) inc += up;
  }
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  int32_t at = inc - own;
  for (int w = 0; w < wave; ++w) at += wsum[w];
  for (int64_t i = a; i < e; ++i) {
    const int32_t c = hist[i];
    hist[i] = at;
    at += c;
  }
}

// Stable scatter: rounds of 256 consecutive elements; an element's place is the digit's next free place plus the number of equal
// digits in front of it in the round (earlier waves' counts, then earlier lanes by ballots).
__global__ __launch_bounds__(kSortThreads) void k_sort_scatter(SortPass s) {
  __shared__ int32_t next[kRadix], wcnt[4][kRadix];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int d = tid; d < kRadix; d += kSortThreads) next[d] = s.hist[(int64_t)d * s.blocks + blockIdx.x];
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

__global__ __launch_bounds__(256) void k_embed_zero(uint4* g, int64_t n16) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n16; i += (int64_t)gridDim.x * 256) g[i] = make_uint4(0, 0, 0, 0);
}
template <typename T> __global__ __launch_bounds__(256) void k_embed_zero_elems(T* g, int64_t a, int64_t e) {
  for (int64_t i = a + (int64_t)blockIdx.x * 256 + threadIdx.x; i < e; i += (int64_t)gridDim.x * 256) g[i] = (T)0.f;
}

// ---- rows of one token are consecutive now: sum them ------------------------------------------------------------------------
// One wave owns `kChunk` sorted pairs and 64 lanes x NE elements of the row.  A token whose pairs all lie in the chunk is written at
// once; one that crosses the chunk's ends leaves fp32 partial sums, head (0) and tail (1), which k_embed_join adds in chunk order.
constexpr int kChunk = 32;

template <typename T, bool VEC> struct Cols {
  static constexpr int N = Vec16<T>::N;
  int c0, wd, lane;
  __device__ Cols(int block, int wd_, int lane_) : c0(block * 64 * N), wd(wd_), lane(lane_) {}
  __device__ __forceinline__ int at(int i) const { return VEC ? c0 + lane * N + i : c0 + i * 64 + lane; }
  __device__ __forceinline__ void load(const T* row, float (&f)[N]) const {
    if (VEC) {
      if (at(0) < wd) load_vec(row + at(0), f);
      else for (int i = 0; i < N; ++i) f[i] = 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = at(i) < wd ? (float)row[at(i)] : 0.f;
    }
  }
  __device__ __forceinline__ void store(T* row, const float (&f)[N]) const {
    if (VEC) {
      if (at(0) < wd) store_vec(row + at(0), f);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) if (at(i) < wd) row[at(i)] = (T)f[i];
    }
  }
  __device__ __forceinline__ void store_part(float* row, const float (&f)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) if (at(i) < wd) row[at(i)] = f[i];
  }
  __device__ __forceinline__ void add_part(const float* row, float (&f)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) if (at(i) < wd) f[i] += row[at(i)];
  }
};

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_embed_sum(const T* g_y, const int32_t* key, const int32_t* pos, int64_t n, int64_t vocab, int wd,
                                                   int colblocks, float scale, T* g_table, float* part) {
  constexpr int N = Vec16<T>::N, U = 8;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t chunk = unit / colblocks, a = chunk * kChunk;
  if (a >= n) return;
  const Cols<T, VEC> cols((int)(unit % colblocks), wd, lane);
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
    float f[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {                                   // (padding pairs of a short chunk read a row that exists: position 0)
      const int32_t p = __builtin_amdgcn_readlane(mypos, (j0 + u) & 63);
      cols.load(g_y + (int64_t)p * wd, f[u]);
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
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += f[u][i];
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

// Tokens that cross chunks: the workgroup of the chunk where the token starts adds its tail and the following heads.  kJoinWaves waves
// take consecutive, equal shares of the heads (a frequent token has thousands) and are added in order.
constexpr int kJoinWaves = 8;
template <typename T, bool VEC>
__global__ __launch_bounds__(64 * kJoinWaves) void k_embed_join(const int32_t* key, int64_t n, int64_t vocab, int wd, int colblocks, float scale,
                                                                T* g_table, const float* part) {
  constexpr int N = Vec16<T>::N;
  __shared__ float sh[kJoinWaves][64 * N];
  __shared__ int32_t sh_end;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t chunk = blockIdx.x / colblocks, a = chunk * kChunk, b = a + kChunk;      // b < n: the launch leaves the last chunk out
  const int32_t k = key[b - 1];
  if (k >= vocab || key[b] != k) return;                            // nothing crosses this chunk's end,
  if (a > 0 && key[a - 1] == k) return;                             // or it started further left
  const int64_t chunks = (n + kChunk - 1) / kChunk;
  int64_t end = chunk + 1;                                          // the first chunk behind `chunk` that does not start with k
  for (;; ) {
    if (tid == 0) sh_end = 64 * kJoinWaves;
    __syncthreads();
    const int64_t c = end + tid;
    if (c >= chunks || key[c * kChunk] != k) atomicMin(&sh_end, tid);
    __syncthreads();
    const int got = sh_end;
    end += got;
    __syncthreads();
    if (got < 64 * kJoinWaves) break;
  }
  const Cols<T, VEC> cols((int)(blockIdx.x % colblocks), wd, lane);
  const int64_t heads = end - (chunk + 1), share = (heads + kJoinWaves - 1) / kJoinWaves;
  const int64_t h0 = chunk + 1 + wave * share, h1 = h0 + share < end ? h0 + share : end;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  if (wave == 0) cols.add_part(part + (2 * chunk + 1) * wd, acc);
#pragma unroll 4
  for (int64_t h = h0; h < h1; ++h) cols.add_part(part + (2 * h) * wd, acc);
#pragma unroll
  for (int i = 0; i < N; ++i) sh[wave][i * 64 + lane] = acc[i];
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float t = acc[i];
    for (int w = 1; w < kJoinWaves; ++w) t += sh[w][i * 64 + lane];
    acc[i] = t * scale;
  }
  cols.store(g_table + (int64_t)k * wd, acc);
}

struct EmbedPlan {
  int tile, blocks, passes, colblocks;
  int64_t chunks;
  size_t key[2], pos[2], hist, part, total;       // byte offsets
};
EmbedPlan embed_plan(int64_t n, int64_t vocab, int wd, int elem) {
  EmbedPlan p{};
  p.tile = n <= (1 << 18) ? 1024 : 4096;
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
  if (vocab < 1 || vocab >= (1ll << 31) - 1 || wd < 1 || n < 0 || n >= (1ll << 26)) return DVGR_E_DIMS;
  if (n / kChunk * (wd / 256 + 1) >= (1ll << 23)) return DVGR_E_DIMS;            // a launch holds at most 2^32 threads
  return 0;
}

template <typename T>
int embed_forward(const T* table, int64_t vocab, int wd, const int64_t* tokens, int64_t n, float scale, T* y, int32_t* bad, hipStream_t st) {
  const bool vec = wd % Vec16<T>::N == 0 && ptr16(table) && ptr16(y);
  const dim3 grid((unsigned)((n + 3) / 4));
  if (vec) DVGR_LAUNCH((k_embed_fwd<T, true>), grid, dim3(256), 0, st, table, vocab, wd, tokens, n, scale, y, bad);
  else DVGR_LAUNCH((k_embed_fwd<T, false>), grid, dim3(256), 0, st, table, vocab, wd, tokens, n, scale, y, bad);
  return (int)hipGetLastError();
}

template <typename T, bool VEC>
int embed_sum(const T* g_y, const int32_t* key, const int32_t* pos, int64_t n, int64_t vocab, int wd, const EmbedPlan& p, float scale,
              T* g_table, float* part, hipStream_t st) {
  const int64_t units = p.chunks * p.colblocks;
  DVGR_LAUNCH((k_embed_sum<T, VEC>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, g_y, key, pos, n, vocab, wd, p.colblocks, scale,
              g_table, part);
  int e = (int)hipGetLastError();
  if (e || p.chunks < 2) return e;
  DVGR_LAUNCH((k_embed_join<T, VEC>), dim3((unsigned)((p.chunks - 1) * p.colblocks)), dim3(64 * kJoinWaves), 0, st, key, n, vocab, wd, p.colblocks,
              scale, g_table, part);
  return (int)hipGetLastError();
}

template <typename T>
int embed_backward(const T* g_y, const int64_t* tokens, int64_t n, int64_t vocab, int wd, float scale, int64_t padding, T* g_table,
                   char* ws, const EmbedPlan& p, hipStream_t st) {
  const int64_t total = vocab * wd, n16 = ptr16(g_table) ? total * (int64_t)sizeof(T) / 16 : 0;
  if (n16) {
    const int64_t blocks = (n16 + 255) / 256;
    DVGR_LAUNCH(k_embed_zero, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, reinterpret_cast<uint4*>(g_table), n16);
  }
  const int64_t done = n16 * 16 / (int64_t)sizeof(T);
  if (done < total) {                                               // the last elements, or a table that is not 16-byte aligned
    const int64_t blocks = (total - done + 255) / 256;
    DVGR_LAUNCH((k_embed_zero_elems<T>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, g_table, done, total);
  }
  if (n == 0) return (int)hipGetLastError();
  SortPass s{};
  s.n = n; s.vocab = vocab; s.padding = padding; s.tile = p.tile; s.blocks = p.blocks;
  s.hist = reinterpret_cast<int32_t*>(ws + p.hist);
  int at = 0;
  for (int i = 0; i < p.passes; ++i, at ^= 1) {
    s.tokens = i ? nullptr : tokens;
    s.key = reinterpret_cast<int32_t*>(ws + p.key[at]); s.pos = reinterpret_cast<int32_t*>(ws + p.pos[at]);
    s.key_out = reinterpret_cast<int32_t*>(ws + p.key[at ^ 1]); s.pos_out = reinterpret_cast<int32_t*>(ws + p.pos[at ^ 1]);
    s.shift = 8 * i;
    DVGR_LAUNCH(k_sort_count, dim3(p.blocks), dim3(kSortThreads), 0, st, s);
    DVGR_LAUNCH(k_sort_scan, dim3(1), dim3(1024), 0, st, s.hist, (int64_t)kRadix * p.blocks);
    DVGR_LAUNCH(k_sort_scatter, dim3(p.blocks), dim3(kSortThreads), 0, st, s);
  }
  const int32_t* key = reinterpret_cast<const int32_t*>(ws + p.key[at]);
  const int32_t* pos = reinterpret_cast<const int32_t*>(ws + p.pos[at]);
  float* part = reinterpret_cast<float*>(ws + p.part);
  const bool vec = wd % Vec16<T>::N == 0 && ptr16(g_y) && ptr16(g_table);
  return vec ? embed_sum<T, true>(g_y, key, pos, n, vocab, wd, p, scale, g_table, part, st)
             : embed_sum<T, false>(g_y, key, pos, n, vocab, wd, p, scale, g_table, part, st);
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
  return embed_check(n, vocab, wd, elem) || n == 0 ? 0 : embed_plan(n, vocab, wd, elem).total;
}

int dvgr_embed_backward(const void* g_y, const int64_t* tokens, int64_t n, int64_t vocab, int wd, int elem, float scale, int64_t padding_idx,
                        void* g_table, void* workspace, size_t workspace_bytes, void* stream) {
  const int e = embed_check(n, vocab, wd, elem);
  if (e) return e;
  if (!g_table || (n && (!g_y || !tokens || !workspace))) return DVGR_E_NULL;
  const EmbedPlan p = n ? embed_plan(n, vocab, wd, elem) : EmbedPlan{};
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
