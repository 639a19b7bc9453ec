// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   y[t] = s W[id[t]]                      (0 where id[t] is outside [0, V): no entry)
//   dW[v] = s sum_{t: id[t] = v} dy[t]     (every row written, 0 where no token names it)
//
// Forward: one pass of 16-byte loads, memory bound.
//
// Gradient: the tokens are sorted by id, stably, so each row's sum runs over its tokens in token
// order whatever the launch does: no float atomics, the same inputs give the same bits.
//   sort    least-significant-digit radix sort of (id, position), digits of up to 11 bits: one pass up
//           to V = 2047, two up to 4M.  A pass is a histogram per tile of 1024 tokens, a scan of each
//           digit's column of counts, and a scatter that ranks a tile's tokens (lanes with an equal
//           digit find each other by ballots).  Up to 4096 tokens one block does it all in LDS.
//   chunks  64 sorted tokens at a time: where one id fills a chunk, the chunk's sum.  The same again
//           over 64 chunks where one id fills them all.
//   rows    a row's sum, by one lane group or several: its tokens outside full chunks, the sums of its full chunks outside full
//           spans of 64, the sums of those spans.  A row that a million tokens name is so read by
//           the whole device in the chunk pass, and no row walks more than 128 tokens, 128 chunks
//           and tokens / 4096 spans.
// Sums are held in 32 bits and rounded once.
//
// Bound: memory at a million tokens of 128 bf16 values (forward 76 us; gradient 209: sort 69, chunks 26,
// rows 109), launches at 100 000 of 32 fp32 values (forward 6 us; gradient 39 in nine launches).

#include "elem.h"

namespace tts {

constexpr int kEmbBlock = 256;
constexpr int kEmbWaves = kEmbBlock / 64;
constexpr int kSmallPer = 16, kSmallTokens = kSmallPer * kEmbBlock;   // one block sorts up to 4096 tokens
// Tokens a thread and a block of a pass over more: 1024 a block fill the card from 260 000 tokens on
// (4096 a block: scatter of 100 000 tokens 15.4 -> 6.1 us, of a million 28.0 -> 20.8).
constexpr int kPassPer = 4, kPassTokens = kPassPer * kEmbBlock;
constexpr int kMaxDigitBits = 11;
constexpr int kMaxBins = 1 << kMaxDigitBits;
constexpr int kChunk = 64;                             // sorted tokens a chunk, chunks a span
constexpr int kSpan = kChunk * kChunk;

// Sort key of a token: its id, or V (behind every row) where the id names no row.
template <typename I>
__device__ __forceinline__ uint32_t token_key(const I* ids, int64_t t, uint32_t V) {
  const I id = ids[t];
  return id >= 0 && id < (I)V ? (uint32_t)id : V;
}

template <typename T, typename I, int MODE>
__global__ __launch_bounds__(kEmbBlock) void k_emb_fwd(const T* __restrict__ table, uint32_t V,
                                                       int D, const I* __restrict__ ids, int64_t N,
                                                       float scale, T* __restrict__ out, int L) {
  constexpr int VE = kVec<T>;
  const int lig = threadIdx.x & (L - 1), per = kEmbBlock / L;
  for (int64_t t = (int64_t)blockIdx.x * per + threadIdx.x / L; t < N;
       t += (int64_t)gridDim.x * per) {
    const uint32_t k = token_key(ids, t, V);
    const T* src = table + (int64_t)k * D;
    T* dst = out + t * D;
    for (int c = lig * VE; c < D; c += L * VE) {
      float v[VE] = {};
      if (k < V) {
        RowVec<T, MODE> r;
        r.load(src, c, D);
        r.get(c, D, v);
#pragma unroll
        for (int i = 0; i < VE; ++i) v[i] *= scale;
      }
      store_row(dst + c, D - c, v);
    }
  }
}

// Lanes of the wave whose digit equals this lane's, among the lanes with `on`.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool on) {
  uint64_t m = __ballot(on);
  for (int b = 0; b < bits; ++b) {
    const bool s = (digit >> b) & 1;
    const uint64_t z = __ballot(s);
    m &= s ? z : ~z;
  }
  return m;
}

struct SortBuf {
  uint32_t* key[2];
  int32_t* pos[2];
  int32_t* counts;   // [bins][tiles]
  int32_t* totals;   // [bins]
  int2* range;       // [V] first and past-the-last sorted place of each row's tokens
  float* chunk;      // [N / 64][D]
  float* span;       // [N / 4096][D]
};

// Ranks a tile's keys for one digit: cnt[wave][bin] ends as the wave's count of each digit, rank[r]
// is the token's place among the wave's tokens of its digit.  Token r of a lane is at
// wave * 64 PER + r * 64 + lane: order along the tile is (wave, r, lane).
template <int PER>
__device__ __forceinline__ int tile_token(int r) {
  return (int)(threadIdx.x >> 6) * (64 * PER) + r * 64 + (int)(threadIdx.x & 63);
}
template <int PER>
__device__ __forceinline__ void rank_tile(const uint32_t (&key)[PER], int n, int shift, int bits,
                                          int* cnt, int (&rank)[PER]) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, bins = 1 << bits;
  for (int i = threadIdx.x; i < kEmbWaves * bins; i += kEmbBlock) cnt[i] = 0;
  __syncthreads();
  volatile int* c = cnt + wave * bins;
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    const bool on = tile_token<PER>(r) < n;
    const uint32_t d = (key[r] >> shift) & (bins - 1);
    const uint64_t m = same_digit(d, bits, on);
    const int before = __popcll(m & ((1ull << lane) - 1));
    const int base = on ? c[d] : 0;
    rank[r] = base + before;
    __builtin_amdgcn_wave_barrier();   // every lane of the wave has read before one adds
    if (on && before == 0) c[d] = base + __popcll(m);
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
}

// Up to 4096 tokens: the whole sort in one block.  Blocks 1.. clear `range`.
template <typename I>
__global__ __launch_bounds__(kEmbBlock) void k_emb_sort_small(const I* __restrict__ ids, int N,
                                                              uint32_t V, int passes, int bits,
                                                              uint32_t* __restrict__ okey,
                                                              int32_t* __restrict__ opos,
                                                              int2* __restrict__ range) {
  __shared__ int cnt[kEmbWaves * kMaxBins];
  __shared__ uint32_t skey[kSmallTokens];
  __shared__ uint16_t spos[kSmallTokens];
  __shared__ int tmp[kEmbWaves];
  if (gridDim.x > 1) {
    if (blockIdx.x > 0) {
      for (int64_t v = (int64_t)(blockIdx.x - 1) * kEmbBlock + threadIdx.x; v < V;
           v += (int64_t)(gridDim.x - 1) * kEmbBlock)
        range[v] = make_int2(0, 0);
      return;
    }
  } else {
    for (uint32_t v = threadIdx.x; v < V; v += kEmbBlock) range[v] = make_int2(0, 0);
  }
  const int wave = threadIdx.x >> 6, bins = 1 << bits;
  uint32_t key[kSmallPer];
  int pos[kSmallPer], rank[kSmallPer];
#pragma unroll
  for (int r = 0; r < kSmallPer; ++r) {
    const int t = tile_token<kSmallPer>(r);
    key[r] = t < N ? token_key(ids, t, V) : 0;
    pos[r] = t;
  }
  for (int p = 0; p < passes; ++p) {
    rank_tile(key, N, p * bits, bits, cnt, rank);
    // counts -> first place of each (digit, wave): a thread takes bins / 256 digits or one
    const int per = bins > kEmbBlock ? bins / kEmbBlock : 1;
    const int d0 = threadIdx.x * per;
    int sum = 0;
    if (d0 < bins)
      for (int d = d0; d < d0 + per; ++d)
        for (int w = 0; w < kEmbWaves; ++w) sum += cnt[w * bins + d];
    int total;
    int at = block_excl_scan256(sum, tmp, &total);
    if (d0 < bins)
      for (int d = d0; d < d0 + per; ++d)
        for (int w = 0; w < kEmbWaves; ++w) {
          const int c = cnt[w * bins + d];
          cnt[w * bins + d] = at;
          at += c;
        }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSmallPer; ++r) {
      const int t = tile_token<kSmallPer>(r);
      if (t < N) {
        const int to = cnt[wave * bins + ((key[r] >> (p * bits)) & (bins - 1))] + rank[r];
        skey[to] = key[r];
        spos[to] = (uint16_t)pos[r];
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSmallPer; ++r) {
      const int t = tile_token<kSmallPer>(r);
      if (t < N) {
        key[r] = skey[t];
        pos[r] = spos[t];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kSmallPer; ++r) {
    const int t = tile_token<kSmallPer>(r);
    if (t < N) {
      okey[t] = key[r];
      opos[t] = pos[r];
    }
  }
}

// Keys of a pass: from the ids in the first (key null), from the last pass's output after.
template <typename I>
__device__ __forceinline__ uint32_t pass_key(const I* ids, const uint32_t* key, int64_t t,
                                             uint32_t V) {
  return key ? key[t] : token_key(ids, t, V);
}

// counts[digit][tile]; the first pass also clears `range`.
template <typename I>
__global__ __launch_bounds__(kEmbBlock) void k_emb_hist(const I* __restrict__ ids,
                                                        const uint32_t* __restrict__ key, int64_t N,
                                                        uint32_t V, int shift, int bits,
                                                        int32_t* __restrict__ counts,
                                                        int2* __restrict__ range) {
  __shared__ int cnt[kMaxBins];
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < bins; i += kEmbBlock) cnt[i] = 0;
  if (range)
    for (int64_t v = (int64_t)blockIdx.x * kEmbBlock + threadIdx.x; v < V;
         v += (int64_t)gridDim.x * kEmbBlock)
      range[v] = make_int2(0, 0);
  __syncthreads();
  const int64_t t0 = (int64_t)blockIdx.x * kPassTokens;
  uint32_t k[kPassPer];
#pragma unroll
  for (int r = 0; r < kPassPer; ++r) {
    const int64_t t = t0 + r * kEmbBlock + threadIdx.x;
    k[r] = t < N ? pass_key(ids, key, t, V) : 0;
  }
#pragma unroll
  for (int r = 0; r < kPassPer; ++r)
    if (t0 + r * kEmbBlock + threadIdx.x < N) atomicAdd(&cnt[(k[r] >> shift) & (bins - 1)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += kEmbBlock)
    counts[(int64_t)i * gridDim.x + blockIdx.x] = cnt[i];
}

// Exclusive scan of each digit's counts over the tiles, in place; totals[digit].
__global__ __launch_bounds__(kEmbBlock) void k_emb_scan(int32_t* __restrict__ counts, int tiles,
                                                        int32_t* __restrict__ totals) {
  __shared__ int tmp[kEmbWaves];
  int32_t* c = counts + (int64_t)blockIdx.x * tiles;
  int base = 0;
  for (int t0 = 0; t0 < tiles; t0 += kEmbBlock) {
    const int t = t0 + threadIdx.x;
    const int v = t < tiles ? c[t] : 0;
    int total;
    const int e = block_excl_scan256(v, tmp, &total);
    if (t < tiles) c[t] = base + e;
    base += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = base;
}

template <typename I>
__global__ __launch_bounds__(kEmbBlock) void k_emb_scatter(
    const I* __restrict__ ids, const uint32_t* __restrict__ key, const int32_t* __restrict__ pos,
    int64_t N, uint32_t V, int shift, int bits, const int32_t* __restrict__ counts,
    const int32_t* __restrict__ totals, uint32_t* __restrict__ okey, int32_t* __restrict__ opos) {
  __shared__ int cnt[kEmbWaves * kMaxBins];
  __shared__ int tmp[kEmbWaves];
  const int bins = 1 << bits;
  const int64_t t0 = (int64_t)blockIdx.x * kPassTokens;
  const int n = (int)(N - t0 < kPassTokens ? N - t0 : kPassTokens);
  const int wave = threadIdx.x >> 6;
  uint32_t k[kPassPer];
  int p[kPassPer], rank[kPassPer];
#pragma unroll
  for (int r = 0; r < kPassPer; ++r) {
    const int i = tile_token<kPassPer>(r);
    k[r] = i < n ? pass_key(ids, key, t0 + i, V) : 0;
    p[r] = i < n ? (pos ? pos[t0 + i] : (int)(t0 + i)) : 0;
  }
  rank_tile(k, n, shift, bits, cnt, rank);
  // first place of each (digit, wave): tokens of lower digits + this digit's in earlier tiles and waves
  const int per = bins > kEmbBlock ? bins / kEmbBlock : 1;
  const int d0 = threadIdx.x * per;
  int sum = 0;
  if (d0 < bins)
    for (int d = d0; d < d0 + per; ++d) sum += totals[d];
  int total;
  int lower = block_excl_scan256(sum, tmp, &total);
  if (d0 < bins)
    for (int d = d0; d < d0 + per; ++d) {
      int at = lower + counts[(int64_t)d * gridDim.x + blockIdx.x];
      for (int w = 0; w < kEmbWaves; ++w) {
        const int c = cnt[w * bins + d];
        cnt[w * bins + d] = at;
        at += c;
      }
      lower += totals[d];
    }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kPassPer; ++r) {
    const int i = tile_token<kPassPer>(r);
    if (i < n) {
      const int to = cnt[wave * bins + ((k[r] >> shift) & (bins - 1))] + rank[r];
      okey[to] = k[r];
      opos[to] = p[r];
    }
  }
}

// acc += rows src[at(i)], i = first, first + step, .. < last, over the columns [c, c + V) by one lane
// group: eight rows in flight.  Past the last row nothing is read.
template <typename T, int MODE, typename At>
__device__ __forceinline__ void add_rows(const T* src, int D, int c, int first, int last, int step,
                                         At at, float* acc) {
  constexpr int V = kVec<T>, B = 8;
  for (int i = first; i < last; i += B * step) {
    RowVec<T, MODE> r[B];
    int p[B];
#pragma unroll
    for (int u = 0; u < B; ++u)
      if (i + u * step < last) p[u] = at(i + u * step);
#pragma unroll
    for (int u = 0; u < B; ++u)
      if (i + u * step < last) r[u].load(src + (int64_t)p[u] * D, c, D);
#pragma unroll
    for (int u = 0; u < B; ++u) {
      if (i + u * step < last) {
        float v[V];
        r[u].get(c, D, v);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += v[j];
      }
    }
  }
}

// Sum over groups of L lanes up to `end` lanes, the same in each.
template <int N>
__device__ __forceinline__ void add_groups(float (&acc)[N], int L, int end = 64) {
  for (int o = L; o < end; o *= 2)
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] += __shfl_xor(acc[j], o, 64);
}

// Chunk c's sum where one row's tokens fill it (a wave a chunk), and the rows' ranges.
template <typename T, int MODE>
__global__ __launch_bounds__(kEmbBlock) void k_emb_chunk(const uint32_t* __restrict__ key,
                                                         const int32_t* __restrict__ pos, int64_t N,
                                                         uint32_t V, int D,
                                                         const T* __restrict__ dy,
                                                         float* __restrict__ chunk,
                                                         int2* __restrict__ range, int L) {
  constexpr int VE = kVec<T>;
  const int lane = threadIdx.x & 63, lig = lane & (L - 1), grp = lane / L, G = 64 / L;
  const int64_t c0 = (int64_t)blockIdx.x * kEmbWaves + (threadIdx.x >> 6);
  const int64_t t = c0 * kChunk + lane;
  const uint32_t k = t < N ? key[t] : V;
  if (t < N) {
    const uint32_t prev = t > 0 ? key[t - 1] : V;
    const uint32_t next = t + 1 < N ? key[t + 1] : V;
    if (k < V && (t == 0 || prev != k)) range[k].x = (int)t;
    if (k < V && next != k) range[k].y = (int)t + 1;
  }
  if ((c0 + 1) * kChunk > N) return;
  const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)k, 0);
  const uint32_t last = (uint32_t)__builtin_amdgcn_readlane((int)k, 63);
  if (first != last || first >= V) return;
  const int p = pos[t];
  for (int cb = 0; cb < D; cb += L * VE) {
    const int c = cb + lig * VE;
    float acc[VE] = {};
#pragma unroll 8
    for (int i0 = 0; i0 < kChunk; i0 += G) {   // all lanes together: p comes from other lanes
      const int q = __shfl(p, i0 + grp, 64);
      RowVec<T, MODE> r;
      r.load(dy + (int64_t)q * D, c, D);
      float v[VE];
      r.get(c, D, v);
#pragma unroll
      for (int j = 0; j < VE; ++j) acc[j] += v[j];
    }
    add_groups(acc, L);
    if (grp == 0 && c < D)
      for (int j = 0; j < VE && c + j < D; ++j) chunk[c0 * D + c + j] = acc[j];
  }
}

// Span s's sum where one row fills its 64 chunks (a wave a span).
template <int MODE>
__global__ __launch_bounds__(kEmbBlock) void k_emb_span(const uint32_t* __restrict__ key, int64_t N,
                                                        uint32_t V, int D,
                                                        const float* __restrict__ chunk,
                                                        float* __restrict__ span, int L) {
  constexpr int VE = kVec<float>;
  const int lane = threadIdx.x & 63, lig = lane & (L - 1), grp = lane / L, G = 64 / L;
  const int64_t s = (int64_t)blockIdx.x * kEmbWaves + (threadIdx.x >> 6);
  if ((s + 1) * kSpan > N) return;
  const uint32_t first = key[s * kSpan], last = key[(s + 1) * kSpan - 1];
  if (first != last || first >= V) return;
  for (int cb = 0; cb < D; cb += L * VE) {
    const int c = cb + lig * VE;
    float acc[VE] = {};
    if (c < D)
      add_rows<float, MODE>(chunk, D, c, (int)s * kChunk + grp, (int)(s + 1) * kChunk, G,
                            [](int i) { return i; }, acc);
    add_groups(acc, L);
    if (grp == 0 && c < D)
      for (int j = 0; j < VE && c + j < D; ++j) span[s * D + c + j] = acc[j];
  }
}

// dW's rows: G groups of L lanes a row, each in the fixed order head tokens, tail tokens, head chunks,
// spans, tail chunks, of which it takes every G-th; the groups' sums are joined in a tree.
// MODE, FMODE: row modes of the gradient's and of the partial sums' rows.
template <typename T, int MODE, int FMODE>
__global__ __launch_bounds__(kEmbBlock) void k_emb_rows(const int2* __restrict__ range,
                                                        const int32_t* __restrict__ pos,
                                                        uint32_t V, int D,
                                                        const T* __restrict__ dy,
                                                        const float* __restrict__ chunk,
                                                        const float* __restrict__ span, float scale,
                                                        T* __restrict__ dw, int L, int G) {
  constexpr int VE = kVec<T>, VF = kVec<float>;
  const int lig = threadIdx.x & (L - 1), g = threadIdx.x / L & (G - 1), per = kEmbBlock / (L * G);
  for (int64_t v = (int64_t)blockIdx.x * per + threadIdx.x / (L * G); v < V;
       v += (int64_t)gridDim.x * per) {
    const int2 r = range[v];
    // first / last places of: head tokens, head chunks, spans, tail chunks, tail tokens
    const int b = r.x, e = r.y;
    const int c0 = (b + kChunk - 1) / kChunk, c1 = e / kChunk;   // full chunks [c0, c1)
    const int s0 = (b + kSpan - 1) / kSpan, s1 = e / kSpan;      // full spans [s0, s1)
    const bool chunks = c0 < c1, spans = s0 < s1;
    const int tb[2] = {b, chunks ? c1 * kChunk : e}, te[2] = {chunks ? c0 * kChunk : e, e};
    const int cb2[2] = {c0, spans ? s1 * kChunk : c1}, ce[2] = {spans ? s0 * kChunk : c1, c1};
    for (int cb = 0; cb < D; cb += L * VE) {
      const int c = cb + lig * VE;
      float acc[VE] = {};
      if (c < D) {
        for (int k = 0; k < 2; ++k)
          add_rows<T, MODE>(dy, D, c, tb[k] + g, te[k], G, [&](int t) { return pos[t]; }, acc);
        if (chunks) {
          for (int k = 0; k < 3; ++k) {
            const float* src = k == 1 ? span : chunk;
            const int i = k == 1 ? s0 : cb2[k / 2], j = k == 1 ? s1 : ce[k / 2];
            if (k == 1 && !spans) continue;
#pragma unroll
            for (int h = 0; h < VE; h += VF)
              if (c + h < D)
                add_rows<float, FMODE>(src, D, c + h, i + g, j, G, [](int t) { return t; }, acc + h);
          }
        }
      }
      add_groups(acc, L, L * G);
#pragma unroll
      for (int j = 0; j < VE; ++j) acc[j] *= scale;
      if (g == 0 && c < D) store_row(dw + v * D + c, D - c, acc);
    }
  }
}

// Digits of the keys 0..V: passes of equal width.
inline void emb_digits(uint32_t V, int* passes, int* bits) {
  int b = 1;
  while (b < 32 && (V >> b)) ++b;
  *passes = (b + kMaxDigitBits - 1) / kMaxDigitBits;
  *bits = (b + *passes - 1) / *passes;
}

inline size_t emb_layout(int64_t N, int64_t V, int D, char* base, SortBuf* w) {
  int passes, bits;
  emb_digits((uint32_t)V, &passes, &bits);
  const size_t n = (size_t)N, tiles = (n + kPassTokens - 1) / kPassTokens;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char* p = base ? base + off : nullptr;
    off += align256(bytes);
    return p;
  };
  const bool big = N > kSmallTokens;
  char* k0 = take(4 * n);
  char* k1 = take(big && passes > 1 ? 4 * n : 0);
  char* p0 = take(4 * n);
  char* p1 = take(big && passes > 1 ? 4 * n : 0);
  char* co = take(big ? 4 * (tiles << bits) : 0);
  char* to = take(big ? (size_t)4 << bits : 0);
  char* ra = take(sizeof(int2) * (size_t)V);
  char* ch = take(sizeof(float) * (n / kChunk) * D);
  char* sp = take(sizeof(float) * (n / kSpan) * D);
  if (w) {
    w->key[0] = reinterpret_cast<uint32_t*>(k0);
    w->key[1] = reinterpret_cast<uint32_t*>(k1);
    w->pos[0] = reinterpret_cast<int32_t*>(p0);
    w->pos[1] = reinterpret_cast<int32_t*>(p1);
    w->counts = reinterpret_cast<int32_t*>(co);
    w->totals = reinterpret_cast<int32_t*>(to);
    w->range = reinterpret_cast<int2*>(ra);
    w->chunk = reinterpret_cast<float*>(ch);
    w->span = reinterpret_cast<float*>(sp);
  }
  return off;
}

constexpr int64_t kEmbMaxTokens = (int64_t)1 << 30;   // sorted places are 32-bit
constexpr int64_t kEmbMaxRows = (int64_t)1 << 30;
constexpr int kEmbMaxBlocks = 256 * 16;

inline int emb_sizes(int64_t N, int64_t V, int D) {
  if (N < 0 || V < 1 || D < 1) return TTS_EINVAL;
  if (N > kEmbMaxTokens || V > kEmbMaxRows) return TTS_ELENGTH;
  return TTS_OK;
}
inline int emb_blocks(int64_t n) { return (int)(n < kEmbMaxBlocks ? n : kEmbMaxBlocks); }

template <typename T, typename I>
int emb_bwd(const T* dy, const I* ids, int64_t N, int64_t V, int D, float scale, T* dw, SortBuf w,
            hipStream_t stream) {
  int passes, bits;
  emb_digits((uint32_t)V, &passes, &bits);
  const uint32_t v32 = (uint32_t)V;
  int cur = 0;
  if (N <= kSmallTokens) {
    const int nb = 1 + (int)(V > 4096 ? (V / 4096 < 256 ? V / 4096 : 256) : 0);
    k_emb_sort_small<I><<<nb, kEmbBlock, 0, stream>>>(ids, (int)N, v32, passes, bits, w.key[0],
                                                      w.pos[0], w.range);
  } else {
    const int tiles = (int)((N + kPassTokens - 1) / kPassTokens);
    cur = 1;
    for (int p = 0; p < passes; ++p) {
      const uint32_t* key = p ? w.key[cur] : nullptr;
      const int32_t* pos = p ? w.pos[cur] : nullptr;
      cur ^= 1;
      k_emb_hist<I><<<tiles, kEmbBlock, 0, stream>>>(ids, key, N, v32, p * bits, bits, w.counts,
                                                     p ? nullptr : w.range);
      k_emb_scan<<<1 << bits, kEmbBlock, 0, stream>>>(w.counts, tiles, w.totals);
      k_emb_scatter<I><<<tiles, kEmbBlock, 0, stream>>>(ids, key, pos, N, v32, p * bits, bits,
                                                        w.counts, w.totals, w.key[cur], w.pos[cur]);
    }
  }
  const int L = row_lanes((D - 1) / kVec<T> + 1), Lf = row_lanes((D - 1) / kVec<float> + 1);
  if (N > 0) {
    const int64_t nch = (N + kChunk - 1) / kChunk;
    by_row_mode<T>(D, [&](auto mode) {
      k_emb_chunk<T, mode()><<<(int)((nch + kEmbWaves - 1) / kEmbWaves), kEmbBlock, 0, stream>>>(
          w.key[cur], w.pos[cur], N, v32, D, dy, w.chunk, w.range, L);
      return 0;
    });
    const int64_t nsp = N / kSpan;
    if (nsp > 0)
      by_row_mode<float>(D, [&](auto mode) {
        k_emb_span<mode()><<<(int)((nsp + kEmbWaves - 1) / kEmbWaves), kEmbBlock, 0, stream>>>(
            w.key[cur], N, v32, D, w.chunk, w.span, Lf);
        return 0;
      });
  }
  // groups a row: one for every two tokens of a mean row, as far as a wave holds them
  int G = 1;
  while (2 * G * L <= 64 && (int64_t)4 * G * V <= N) G *= 2;
  const int per = kEmbBlock / (L * G);
  return by_row_mode<T>(D, [&](auto mode) {
    return by_row_mode<float>(D, [&](auto fmode) {
      // an even row of a half type is even in fp32, a tiny one in fp32 is tiny in the half types
      if constexpr ((mode() != kRowEven || fmode() == kRowEven) &&
                    (fmode() != kRowTiny || mode() == kRowTiny))
        k_emb_rows<T, mode(), fmode()><<<emb_blocks((V + per - 1) / per), kEmbBlock, 0, stream>>>(
            w.range, w.pos[cur], v32, D, dy, w.chunk, w.span, scale, dw, L, G);
      return launch_status();
    });
  });
}

}  // namespace tts

using namespace tts;

extern "C" {

int tts_embedding_fwd(const void* table, int64_t V, int D, const void* ids, int ids64, int64_t N,
                      float scale, int dtype, void* out, hipStream_t stream) {
  if (N < 0 || V < 1 || D < 1 || !table || (N > 0 && (!ids || !out))) return TTS_EINVAL;
  if (const int e = emb_sizes(N, V, D)) return e;
  if (!elem_dtype_ok(dtype)) return TTS_EDTYPE;
  if (N == 0) return TTS_OK;
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int L = row_lanes((D - 1) / kVec<T> + 1), per = kEmbBlock / L;
    const int nb = emb_blocks((N + per - 1) / per);
    const T* tb = static_cast<const T*>(table);
    T* o = static_cast<T*>(out);
    return by_row_mode<T>(D, [&](auto mode) {
      if (ids64)
        k_emb_fwd<T, int64_t, mode()><<<nb, kEmbBlock, 0, stream>>>(
            tb, (uint32_t)V, D, static_cast<const int64_t*>(ids), N, scale, o, L);
      else
        k_emb_fwd<T, int32_t, mode()><<<nb, kEmbBlock, 0, stream>>>(
            tb, (uint32_t)V, D, static_cast<const int32_t*>(ids), N, scale, o, L);
      return launch_status();
    });
  });
}

size_t tts_embedding_workspace_bytes(int64_t N, int64_t V, int D) {
  if (emb_sizes(N, V, D)) return 0;
  return emb_layout(N, V, D, nullptr, nullptr);
}

int tts_embedding_bwd(const void* dout, const void* ids, int ids64, int64_t N, int64_t V, int D,
                      float scale, int dtype, void* dtable, void* workspace,
                      size_t workspace_bytes, hipStream_t stream) {
  if (N < 0 || V < 1 || D < 1 || !dtable || (N > 0 && (!ids || !dout))) return TTS_EINVAL;
  if (const int e = emb_sizes(N, V, D)) return e;
  if (!elem_dtype_ok(dtype)) return TTS_EDTYPE;
  if (!workspace || workspace_bytes < emb_layout(N, V, D, nullptr, nullptr)) return TTS_EWORKSPACE;
  SortBuf w;
  emb_layout(N, V, D, static_cast<char*>(workspace), &w);
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const T* g = static_cast<const T*>(dout);
    T* o = static_cast<T*>(dtable);
    if (ids64)
      return emb_bwd<T, int64_t>(g, static_cast<const int64_t*>(ids), N, V, D, scale, o, w, stream);
    return emb_bwd<T, int32_t>(g, static_cast<const int32_t*>(ids), N, V, D, scale, o, w, stream);
  });
}

}  // extern "C"
