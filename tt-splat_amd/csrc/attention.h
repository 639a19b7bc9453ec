// Attention: what its kernels share (attention_fwd.hip, attention_dq.hip, attention_dkv.hip).
//
//   S = c Q K^T (masked places -inf),  L = log sum exp S,  P = exp(S - L),  O = P V
//   dV = P^T dO,  dP = dO V^T,  D = rowsum(dO O),  dS = P (dP - D),  dQ = c dS K,  dK = c dS^T Q
//
// Matrix instructions.  All products run on 32x32 results, 16 deep (eight values a lane and operand):
//   A (rows of the result): lane l holds row l % 32, places 8 (l / 32) .. + 7 of the depth
//   B (columns):            lane l holds column l % 32, the same places
//   result:                 lane l holds column l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4, i = 0..15
// The order of places along the depth is free as long as A and B agree.  A result's values 8 c ..
// 8 c + 7 are rows 16 c + 8 (j / 4) + 4 (l / 32) + j % 4 of its column, so they are at once the B
// operand of a product whose depth is those rows: probabilities go from one product to the next
// without leaving their lane.  The A operand of that product is a transposed read of a row-major tile
// in that order (transpose_frag).  Hence each kernel computes the transposes whose column is what the
// wave owns: S^T and O^T, dQ^T with a query row a column; S, dV^T and dK^T with a key a column.  Row
// maxima and sums are then sums over a lane's own values and its partner's in the other half.
//
// Half types take one 16-deep instruction; fp32 takes eight 2-deep ones over the same registers.
//
// Rows.  The query heads that share a key head are rows of one matrix: row r of (batch, key head) is
// position r / grp of query head kvhead * grp + r % grp, so shared heads cost no second read of K
// and V, a single token's heads fill a tile together, and dK, dV sum over the group without atomics.
#pragma once

#include "elem.h"
#include "lds_limit.h"

namespace tts {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
using Frag = T __attribute__((ext_vector_type(8)));
using Acc = float __attribute__((ext_vector_type(16)));

__device__ __forceinline__ Acc mma(Frag<bf16> a, Frag<bf16> b, Acc c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ Acc mma(Frag<f16> a, Frag<f16> b, Acc c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ Acc mma(Frag<float> a, Frag<float> b, Acc c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

// Strides in elements of (batch, head, row).  A row's is below 2^23: a tile's rows are then within 2^31
// bytes of its first; products with a row of the whole axis are 64-bit.
struct AttnStride {
  int64_t b, h;
  int n;
};

struct AttnArgs {
  const void *q, *k, *v, *o, *orest, *dout;
  void *out, *rest, *dq, *dk, *dv;
  float *lse, *delta, *part, *part2;
  const uint8_t* mask;
  int64_t mask_stride;
  AttnStride sq, sk, sv, so, sdo, sdq, sdk, sdv;
  int Hkv, grp, Nq, Nk, D, R;   // R = Nq * grp rows a (batch, key head)
  int D4;                       // D rounded up to 4: row stride of the parts of a split axis
  unsigned grp_mul;             // r / grp = (4 r * grp_mul >> 32) >> grp_shift for r < 2^30
  int grp_shift;
  int causal, off;              // row at position p sees keys up to p + off
  int even_rows;                // tiles of 32 rows start at whole positions, their offsets are 32-bit
  int nsplit;                   // parts of the long axis, joined by a second kernel
  float scale;
};

// Position and head of a row.  grp_mul = ceil(2^(30 + grp_shift) / grp), 2^grp_shift >= grp: the product
// is too large by less than r 2^grp_shift < 2^(30 + grp_shift), less than one in the quotient.
__device__ __forceinline__ void attn_row(const AttnArgs& a, int r, int* pos, int* h) {
  *pos = (int)(__umulhi((unsigned)r << 2, a.grp_mul) >> a.grp_shift);
  *h = r - *pos * a.grp;
}
__device__ __forceinline__ int64_t row_offset(const AttnStride& s, int pos, int h) {
  return h * s.h + (int64_t)pos * s.n;
}

// Eight values at any element's address.
template <typename T>
__device__ __forceinline__ Frag<T> load_whole(const T* p) {
  typedef int Any __attribute__((ext_vector_type(2 * sizeof(T)), aligned(sizeof(T))));
  return __builtin_bit_cast(Frag<T>, *reinterpret_cast<const Any*>(p));
}
// Eight values at p, n of them within the row, zeros behind.
template <typename T>
__device__ __forceinline__ Frag<T> load_frag(const T* p, int n) {
  Frag<T> f;
  if (n >= 8) {
    f = load_whole(p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? p[i] : (T)0.0f;
  }
  return f;
}

// Waits here for a value that was loaded, so that its first use inside a loop does not: that wait would
// be for every load that is in flight there, the next tile's among them.
template <typename F>
__device__ __forceinline__ void arrive(F& f) {
  asm volatile("" : "+v"(f));
}

// Tiles in LDS: row-major, rows longer than their data so that one read's lanes meet different banks.
// Half types: 32 bytes longer: a transposed read's four rows of 32 bytes a clock are apart (115 of 128
// bytes a clock and CU with four waves); a fragment's eight rows of 16 bytes meet in pairs, and pieces
// exchanged within unpadded rows by an exclusive or, which part them too, measured the same in these
// kernels (2500 x 2500: 236 -> 232 us for this form).  fp32: 16 bytes longer; transposed reads
// take 32 values of one row.
template <typename T, int DP>
constexpr int kTileStride = DP + (sizeof(T) == 2 ? 16 : 4);

using Piece = int __attribute__((ext_vector_type(4)));
template <typename T>
using Pieces = int __attribute__((ext_vector_type(2 * sizeof(T))));   // a fragment's, one or two

template <typename T, int DP>
__device__ __forceinline__ Frag<T> tile_frag(const T* tile, int row0, int d0) {
  const int lane = threadIdx.x & 63;
  const T* p = tile + (row0 + (lane & 31)) * kTileStride<T, DP> + d0 + (lane >> 5) * 8;
  if constexpr (sizeof(T) == 2) {
    return __builtin_bit_cast(Frag<T>, *reinterpret_cast<const Piece*>(p));
  } else {
    const Piece lo = *reinterpret_cast<const Piece*>(p), up = *reinterpret_cast<const Piece*>(p + 4);
    return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// A operand whose rows are the tile's columns d0 .. d0 + 31 and whose depth is its rows row0 ..
// row0 + 15, in the order of a result's values: place j is row 8 (j / 4) + 4 (lane / 32) + j % 4.
template <typename T, int DP>
__device__ __forceinline__ Frag<T> transpose_frag(const T* tile, int row0, int d0) {
  const int lane = threadIdx.x & 63, hi = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    // ds_read_tr16_b64: 16 lanes read a 4 x 16 block (lane l: row l / 4, columns 4 (l % 4) ..) and
    // lane l receives column l
    using S4 = short __attribute__((ext_vector_type(4)));
    using LdsPtr = __attribute__((address_space(3))) S4*;
    const T* p = tile + (row0 + 4 * hi + ((lane & 15) >> 2)) * kTileStride<T, DP> + d0 + (lane & 16) +
                 4 * (lane & 3);
    const S4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)p);
    const S4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(p + 8 * kTileStride<T, DP>));
    const short __attribute__((ext_vector_type(8))) r =
        __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(Frag<T>, r);
  } else {
    Frag<T> f;
    const T* p = tile + (row0 + 4 * hi) * kTileStride<T, DP> + d0 + (lane & 31);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = p[(8 * (j >> 2) + (j & 3)) * kTileStride<T, DP>];
    return f;
  }
}

// One tile of BN rows on its way from memory to LDS through registers: load() starts the reads, store()
// writes the tile, zeros for rows not in `live` (masked and missing keys: whatever stands there, NaN
// among it, stays out of the products) and past the head size.  ODD: head sizes that are no multiple
// of eight, read value by value; a branch for them in the same kernel makes the compiler wait for
// the loads at once, which costs the overlap (2500 x 2500 bf16 forward 95 -> 80 us).
template <typename T, int DP, int BN, int NT, bool ODD>
struct TileLoad {
  static constexpr int kPerRow = DP / 8, kN = BN * kPerRow / NT;
  static_assert(kN * NT == BN * kPerRow, "threads must divide the tile");
  Frag<T> r[kN];
  unsigned off[kN];   // bytes from a whole tile's first row, the same for every tile

  // at(i): elements from a whole tile's first row to its row i, below 2^31 bytes
  template <typename At>
  __device__ __forceinline__ void plan(int D, At at) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int v = threadIdx.x + i * NT, d0 = v % kPerRow * 8;
      off[i] = (unsigned)(at(v / kPerRow) + (d0 < D ? d0 : 0)) * (unsigned)sizeof(T);
    }
  }
  __device__ __forceinline__ void load_planned(const T* first) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      r[i] = load_whole(reinterpret_cast<const T*>(reinterpret_cast<const char*>(first) + off[i]));
  }
  // row(i): pointer to the tile's row i (any valid row for rows that are not live)
  template <typename Row>
  __device__ __forceinline__ void load(int D, Row row) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int v = threadIdx.x + i * NT, d0 = v % kPerRow * 8;
      get(i, row(v / kPerRow), d0, D);
    }
  }
  // rows `first` (uniform) + min(n, last) * stride, 32-bit offsets from the first
  __device__ __forceinline__ void load_rows(int D, const T* first, int stride, int last) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int v = threadIdx.x + i * NT, d0 = v % kPerRow * 8, n = min(v / kPerRow, last);
      if constexpr (ODD) {
        get(i, first + n * stride, d0, D);
      } else {
        const unsigned off = (unsigned)(n * stride + (d0 < D ? d0 : 0)) * (unsigned)sizeof(T);
        r[i] = load_whole(reinterpret_cast<const T*>(reinterpret_cast<const char*>(first) + off));
      }
    }
  }
  __device__ __forceinline__ void get(int i, const T* p, int d0, int D) {
    if constexpr (ODD) {
#pragma unroll
      for (int j = 0; j < 8; ++j) r[i][j] = p[d0 + j < D ? d0 + j : 0];
    } else {
      r[i] = load_whole(p + (d0 < D ? d0 : 0));
    }
  }
  __device__ __forceinline__ void store(T* tile, uint64_t live, int D) const {
    if (!ODD && D == DP && live == (BN == 64 ? ~0ull : (1ull << (BN & 63)) - 1)) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int v = threadIdx.x + i * NT;
        write(tile, v, __builtin_bit_cast(Pieces<T>, r[i]));
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int v = threadIdx.x + i * NT, n = v / kPerRow, d0 = v % kPerRow * 8;
      const uint32_t bits = n < 32 ? (uint32_t)live : (uint32_t)(live >> 32);
      const bool on = (bits >> (n & 31) & 1) && d0 < D;
      Frag<T> f = r[i];
      if constexpr (ODD) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = d0 + j < D ? f[j] : (T)0.0f;
      }
      const Pieces<T> w = __builtin_bit_cast(Pieces<T>, f);
      write(tile, v, on ? w : Pieces<T>{});
    }
  }
  // Whole pieces of 16 bytes: byte copies here are taken apart into byte stores by the compiler.
  static __device__ __forceinline__ void write(T* tile, int v, Pieces<T> w) {
    T* p = tile + v / kPerRow * kTileStride<T, DP> + v % kPerRow * 8;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<Piece*>(p) = w;
    } else {
      *reinterpret_cast<Piece*>(p) = __builtin_shufflevector(w, w, 0, 1, 2, 3);
      *reinterpret_cast<Piece*>(p + 4) = __builtin_shufflevector(w, w, 4, 5, 6, 7);
    }
  }
};

// Non-zero bytes of x as four bits.
__device__ __forceinline__ uint32_t byte_bits(uint32_t x) {
  const uint32_t y = ((((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) & 0x80808080u) >> 7;
  return (y * 0x10204080u) >> 28;
}

// Live keys of the tile at key k0 (BN of them), as bits.
template <int BN>
__device__ __forceinline__ uint64_t live_keys(const uint8_t* mask, int k0, int Nk) {
  const int n = Nk - k0;
  if (n <= 0) return 0;
  const uint64_t all = n >= BN ? (BN == 64 ? ~0ull : (1ull << BN) - 1) : (1ull << n) - 1;
  if (!mask) return all;
  uint64_t w = 0;
  if (n >= BN) {
#pragma unroll
    for (int i = 0; i < BN / 16; ++i) {
      uint32_t x[4];
      memcpy(x, mask + k0 + 16 * i, 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) w |= (uint64_t)byte_bits(x[j]) << (16 * i + 4 * j);
    }
  } else {
    for (int i = 0; i < n; ++i) w |= (uint64_t)(mask[k0 + i] != 0) << i;
  }
  return w;
}

// Tiles [t, end) that hold a live key, 64 tiles at a time: lane i holds the bits of tile base + i.
// The same in every wave of a block.
template <int BN>
struct KeyTiles {
  const uint8_t* mask;
  int Nk, base, end;
  uint64_t word, pending;

  __device__ __forceinline__ void start(const uint8_t* m, int nk, int t, int t_end) {
    mask = m;
    Nk = nk;
    base = t;
    end = t_end;
    fill();
  }
  __device__ __forceinline__ void fill() {
    const int t = base + (int)(threadIdx.x & 63);
    word = t < end ? live_keys<BN>(mask, t * BN, Nk) : 0;
    pending = __ballot(word != 0);
  }
  __device__ __forceinline__ bool next(int* tile, uint64_t* live) {
    while (!pending) {
      if (base + 64 >= end) return false;
      base += 64;
      fill();
    }
    const int b = __builtin_ctzll(pending);
    pending &= pending - 1;
    *tile = base + b;
    *live = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)word, b) |
            (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(word >> 32), b) << 32;
    return true;
  }
};

__device__ __forceinline__ float max_halves(float x) {
  const float2 s = swap_halves(x);
  return fmaxf(s.x, s.y);
}
__device__ __forceinline__ float sum_halves(float x) {
  const float2 s = swap_halves(x);
  return s.x + s.y;
}

// Each row's dot product of x and y (fragments of the same 32 rows), in both halves: the diagonal of
// x y^T.  Its terms are added in the order of every product here, so that for a row with one visible
// key, where O = V, rowsum(dO O) equals dO V^T to the last bit and dS is zero.
template <typename T, int KC>
__device__ __forceinline__ float row_dots(const Frag<T> (&x)[KC], const Frag<T> (&y)[KC]) {
  const int col = threadIdx.x & 31, hi = (threadIdx.x & 63) >> 5;
  Acc s = {};
#pragma unroll
  for (int c = 0; c < KC; ++c) s = mma(x[c], y[c], s);
  float r = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) r = 8 * (i >> 2) + 4 * hi + (i & 3) == col ? s[i] : r;
  const float2 w = swap_halves(r);
  return (col >> 2) & 1 ? w.y : w.x;
}

// exp2 by the hardware instruction: exp2(-inf) = 0, one unit in the last place.
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// P of a score from its row's log-sum-exp L: exp(c s - L).  fp32: c s - L with one rounding, small where P
// is not; half types: from c log2(e) s and L log2(e), one operation less and an error far below P's own
// rounding.
template <typename T>
__device__ __forceinline__ float prob(float s, float scale, float c2, float lse, float lse2) {
  if constexpr (sizeof(T) == 4) return exp2_(__builtin_fmaf(s, scale, -lse) * kLog2e);
  return exp2_(__builtin_fmaf(s, c2, -lse2));
}

// Eight of a result's values as an operand, rounded to the operands' type.
template <typename T>
__device__ __forceinline__ Frag<T> acc_frag(const Acc& s, int c) {
  Frag<T> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (T)s[8 * c + j];
  return f;
}

// What that rounding left out, as an operand of a second product.
template <typename T>
__device__ __forceinline__ Frag<T> acc_rest(const Acc& s, int c, Frag<T> f) {
  Frag<T> r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (T)(s[8 * c + j] - (float)f[j]);
  return r;
}
// Half types, odd heads of up to 32 values: the forward's P and dQ's dS go into their products in two parts.
// A row's dS sum to zero, and the fewer values a head has, the more alike are the keys that a row
// weighs most: the terms dS K cancel, while an error of D, which P's rounding in O brings, is multiplied
// by all of sum P K (one value, two rows over 4099 keys, fp16: dQ 1.7 u off in the mean, 1.2 u with dS in
// two parts alone; u = 2^-11).  Costs 12 % at 20 values, 2500 x 2500, 16 heads, bf16, gradients: 189 -> 211 us.
template <typename T, int DP, bool ODD>
constexpr bool kTwoParts = sizeof(T) == 2 && ODD && DP == 32;

// Four consecutive values of a row, n of them within it.
template <typename T>
__device__ __forceinline__ void store4(T* p, int n, float x0, float x1, float x2, float x3) {
  const T v[4] = {(T)x0, (T)x1, (T)x2, (T)x3};
  if (n >= 4) {
    memcpy(p, v, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = v[i];
  }
}
// The result's accumulators set to base[row], as the products' start.
__device__ __forceinline__ Acc acc_rows(const float* base) {
  const int hi = (threadIdx.x & 63) >> 5;
  Acc s;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const float4 x = *reinterpret_cast<const float4*>(base + 8 * g + 4 * hi);
    s[4 * g] = x.x;
    s[4 * g + 1] = x.y;
    s[4 * g + 2] = x.z;
    s[4 * g + 3] = x.w;
  }
  return s;
}

// A column's values (one row of the output in memory): block db of 32 rows of a transposed result.
template <typename T>
__device__ __forceinline__ void store_column(T* row, int D, int db, const Acc& x, float f) {
  const int hi = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int d = db * 32 + 8 * g + 4 * hi;
    store4(row + d, D - d, x[4 * g] * f, x[4 * g + 1] * f, x[4 * g + 2] * f, x[4 * g + 3] * f);
  }
}

// Joins the parts of split rows, in order: G groups of L lanes a row, each of which takes every G-th
// part; the groups' sums are joined in a tree, and where a block takes one row (BLOCK: L G = 256) its
// waves' by way of LDS.  x: four columns' sum from column c on, in group 0.  lse (softmax parts): the
// parts' log-sum-exps weigh them, join_max is their maximum, *l the weights' sum.
constexpr int kJoinLanes = 32;   // 128 columns
struct JoinTeam {
  int lig, g, L, G;
  int64_t row;
  __device__ __forceinline__ JoinTeam(int L_, int G_)
      : lig(threadIdx.x & (L_ - 1)), g(threadIdx.x / L_ & (G_ - 1)), L(L_), G(G_),
        row((int64_t)blockIdx.x * (256 / (L_ * G_)) + threadIdx.x / (L_ * G_)) {}
};
template <bool BLOCK>
__device__ __forceinline__ float join_max(const JoinTeam& t, const float* lse, int64_t rows,
                                          int nsplit) {
  float m = -INFINITY;
  for (int s = t.g * t.L + t.lig; s < nsplit; s += t.L * t.G) m = fmaxf(m, lse[s * rows + t.row]);
  for (int o = 1; o < (BLOCK ? 64 : t.L * t.G); o *= 2) m = fmaxf(m, __shfl_xor(m, o, 64));
  if constexpr (BLOCK) {
    __shared__ float red[4];
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  }
  return m;
}
template <bool SOFT, bool BLOCK = false>
__device__ __forceinline__ void join_parts(const JoinTeam& t, const float* part, const float* lse,
                                           int64_t rows, int nsplit, int D4, int c, float m,
                                           float* l, float (&x)[4]) {
  *l = 0.0f;
  x[0] = x[1] = x[2] = x[3] = 0.0f;
#pragma unroll 4
  for (int s = t.g; s < nsplit; s += t.G) {
    const int64_t i = s * rows + t.row;
    const float4 v = *reinterpret_cast<const float4*>(part + i * D4 + (c < D4 ? c : 0));
    const float w = SOFT ? exp2_((lse[i] - m) * kLog2e) : 1.0f;
    *l += w;
    x[0] += w * v.x;
    x[1] += w * v.y;
    x[2] += w * v.z;
    x[3] += w * v.w;
  }
  for (int o = t.L; o < (BLOCK ? 64 : t.L * t.G); o *= 2) {
    *l += __shfl_xor(*l, o, 64);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] += __shfl_xor(x[j], o, 64);
  }
  if constexpr (BLOCK) {   // L lanes cover the columns: once a row
    __shared__ float red[5][4][kJoinLanes];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (lane < t.L) {
      red[4][wave][lane] = *l;
#pragma unroll
      for (int j = 0; j < 4; ++j) red[j][wave][lane] = x[j];
    }
    __syncthreads();
    if (t.g == 0) {
      auto sum = [&](int j) {
        return (red[j][0][lane] + red[j][1][lane]) + (red[j][2][lane] + red[j][3][lane]);
      };
      *l = sum(4);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = sum(j);
    }
  }
}

// What rounding the output left out: x - (T)x, and nothing where it is below the fp32 sums' own error
// (a row with one key has O = V and no rest).
template <typename T>
__device__ __forceinline__ float rest_of(float x) {
  const float r = x - (float)(T)x;
  return fabsf(r) > fabsf(x) * 0x1p-20f ? r : 0.0f;
}

// ---- host side ----

// Lanes a row's columns and groups a row of a join over `nsplit` parts: groups while the rows alone
// leave the card unfilled (256k threads; 40 000 rows of two parts with two groups 13 us, with one 8.5).
inline void join_shape(int64_t rows, int D, int nsplit, int* L, int* G) {
  *L = row_lanes((D + 3) / 4);
  *G = 1;
  while (*G * 2 <= nsplit && *L * *G < 64 && rows * *L * *G < (1 << 18)) *G *= 2;
}
inline int join_blocks(int64_t rows, int L, int G) { return (int)((rows * L * G + 255) / 256); }

// Head sizes are rounded up to a multiple of 32; those that are no multiple of eight, to 32 or 128.
template <typename F>
inline int by_head(int D, F&& f) {
  using std::bool_constant;
  using std::integral_constant;
  if (D & 7) {
    if (D <= 32) return f(integral_constant<int, 32>{}, bool_constant<true>{});
    return f(integral_constant<int, 128>{}, bool_constant<true>{});
  }
  if (D <= 32) return f(integral_constant<int, 32>{}, bool_constant<false>{});
  if (D <= 64) return f(integral_constant<int, 64>{}, bool_constant<false>{});
  if (D <= 96) return f(integral_constant<int, 96>{}, bool_constant<false>{});
  return f(integral_constant<int, 128>{}, bool_constant<false>{});
}

// Launches a kernel whose dynamic LDS may pass 64 KB.
template <typename K>
inline int launch_lds(K kernel, LdsLimit& lim, int blocks, int threads, size_t lds,
                      const AttnArgs& a, hipStream_t stream) {
  if (lds > 64 * 1024)
    if (const int e = raise_lds_limit(reinterpret_cast<const void*>(kernel), lim)) return e;
  kernel<<<blocks, threads, lds, stream>>>(a);
  return launch_status();
}

constexpr int kAttnMaxSplit = 64;
// Scales whose inverse, and product with the log-sum-exp, stay normal fp32 numbers: a smaller one
// would round to 0, which times a hidden key's -inf is NaN, or give an infinite inverse.
constexpr double kAttnMinScale = 1.0e-30, kAttnMaxScale = 1.0e30;

// Parts of `tiles` steps of the long axis for `waves` waves of work: as many as bring them nearest to
// `fill`, each of `least` steps or more.
inline int attn_splits(int64_t waves, int64_t fill, int tiles, int least) {
  if (waves <= 0) return 1;
  int64_t n = (fill + waves / 2) / waves;
  n = n < tiles / least ? n : tiles / least;
  n = n < kAttnMaxSplit ? n : kAttnMaxSplit;
  return (int)(n < 1 ? 1 : n);
}

// Blocks and splits of each kernel for a shape.
struct AttnPlan {
  int fw, fs, fq;    // forward: waves a block, splits, blocks of 32 rows a wave
  int qw, qs;        // dq
  int kw, ks;        // dk, dv
  int rb_f, rb_q, kb;
};
AttnPlan attn_plan(const AttnArgs& a, int BH, int dtype);

int attn_launch_fwd(const AttnArgs& a, int BH, int dtype, const AttnPlan& p, hipStream_t stream);
int attn_launch_dq(const AttnArgs& a, int BH, int dtype, const AttnPlan& p, hipStream_t stream);
int attn_launch_dkv(const AttnArgs& a, int BH, int dtype, const AttnPlan& p, hipStream_t stream);

}  // namespace tts
