// Attention forward: one pass over the keys with the running maximum and sum of each row's softmax.
//
// A wave owns 32 QB rows (columns of S^T and O^T): Q stays in registers as the B operand, K and V tiles
// of BN keys pass through LDS, read by all waves of the block, the next tile's loads in flight
// while this one is computed.  Rows' maxima and sums are over a lane's own values; the two halves of
// the wave are joined once a tile (maximum) and once at the end (sum).
//
// Roundings: S, the softmax and O are fp32; P is rounded to the operands' type for its product with V
// (half types; odd heads of up to 32 values: kTwoParts), O once at the end.
//
// For a backward in half types the rounding's rest, O - (T)O, is stored beside O: D = rowsum(dO O) then
// carries 16 bits of O, not 8 or 11 (without it dQ and dK of short key axes lose a quarter of a bit).
//
// Bound: at 8040 x 8040, 16 heads of 128 bf16, 717 us (740 TFLOP/s); matrix instructions and LDS reads alone
// 408, without staging and barriers 498, without exponentials 639.  2500 x 2500, 16 heads of 64: 49 us.
//
// Few rows (serving): one wave a block and the keys split over blocks; each part leaves its normalised
// O and its log-sum-exp, and k_attn_join adds the parts by exp(L_part - L).

#include "attention.h"

namespace tts {

template <typename T, int DP, int BN>
constexpr size_t fwd_lds() {
  return (size_t)4 * BN * kTileStride<T, DP> * sizeof(T) + 2 * BN * sizeof(float);
}

template <typename T, int DP, int NW, int BN, int QB, bool ODD>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 && (NW > 1 || DP <= 64) ? 2 : 1)
void k_attn_fwd(AttnArgs a) {
  constexpr int KC = DP / 16, DB = DP / 32, KB = BN / 32, NT = 64 * NW;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* tk = reinterpret_cast<T*>(smem);
  constexpr int kTile = BN * kTileStride<T, DP>;
  T* tv = tk + 2 * kTile;
  float* bias = reinterpret_cast<float*>(tv + 2 * kTile);   // [2][BN] 0, or -inf for hidden keys

  constexpr int kRows = 32 * QB * NW;
  const int nrb = (a.R + kRows - 1) / kRows;
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const int rb = item % nrb, sp = item / nrb % a.nsplit, bh = item / nrb / a.nsplit;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int lane = threadIdx.x & 63, hi = lane >> 5, wave = threadIdx.x >> 6;
  const T* kp = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
  const T* vp = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h;

  const int row0 = (rb * NW + wave) * 32 * QB + (lane & 31);   // the lane's rows: row0 + 32 j
  Frag<T> q[QB][KC];
  int lim[QB];   // the row sees keys up to lim
#pragma unroll
  for (int j = 0; j < QB; ++j) {
    int pos, h;
    attn_row(a, min(row0 + 32 * j, a.R - 1), &pos, &h);
    const T* qp = static_cast<const T*>(a.q) + b * a.sq.b + (int64_t)hk * a.grp * a.sq.h +
                  row_offset(a.sq, pos, h);
#pragma unroll
    for (int c = 0; c < KC; ++c) q[j][c] = load_frag(qp + c * 16 + hi * 8, a.D - c * 16 - hi * 8);
    lim[j] = a.causal ? pos + a.off : a.Nk;
  }
#pragma unroll
  for (int j = 0; j < QB; ++j)
#pragma unroll
    for (int c = 0; c < KC; ++c) arrive(q[j][c]);
  // keys that any row of the block sees
  int nk = a.Nk;
  if (a.causal) {
    int p1, h1;
    attn_row(a, min((rb + 1) * kRows - 1, a.R - 1), &p1, &h1);
    nk = min(nk, max(p1 + a.off + 1, 0));
  }
  // keys up to lim0 are seen by every row of the wave: its first row's, the same in all lanes
  const int lim0 = __builtin_amdgcn_readfirstlane(lim[0]);
  const int tiles = (a.Nk + BN - 1) / BN, need = (nk + BN - 1) / BN;
  const int t0 = (int)((int64_t)tiles * sp / a.nsplit), t1 = (int)((int64_t)tiles * (sp + 1) / a.nsplit);

  Acc o[QB][DB] = {};
  float m[QB], l[QB];
#pragma unroll
  for (int j = 0; j < QB; ++j) {
    m[j] = -INFINITY;
    l[j] = 0.0f;
  }
  const float c2 = a.scale * kLog2e;

  KeyTiles<BN> it;
  it.start(a.mask ? a.mask + b * a.mask_stride : nullptr, a.Nk, t0, min(t1, need));
  int t = 0;
  uint64_t live = 0;
  bool have = it.next(&t, &live);
  TileLoad<T, DP, BN, NT, ODD> lk, lv;
  if constexpr (!ODD) {
    lk.plan(a.D, [&](int n) { return n * a.sk.n; });
    lv.plan(a.D, [&](int n) { return n * a.sv.n; });
  }
  auto fetch = [&](int tile) {
    const int last = a.Nk - 1 - tile * BN;
    const T* k0 = kp + (int64_t)tile * BN * a.sk.n;
    const T* v0 = vp + (int64_t)tile * BN * a.sv.n;
    if (!ODD && last >= BN - 1) {
      lk.load_planned(k0);
      lv.load_planned(v0);
    } else {
      lk.load_rows(a.D, k0, a.sk.n, last);
      lv.load_rows(a.D, v0, a.sv.n, last);
    }
  };
  auto put = [&](int buf, uint64_t bits) {
    lk.store(tk + buf * kTile, bits, a.D);
    lv.store(tv + buf * kTile, bits, a.D);
    if (threadIdx.x < BN) bias[buf * BN + threadIdx.x] = (bits >> threadIdx.x) & 1 ? 0.0f : -INFINITY;
  };
  if (have) {
    fetch(t);
    put(0, live);
  }
  int buf = 0;
  while (have) {
    int tn = 0;
    uint64_t ln = 0;
    const bool more = it.next(&tn, &ln);
    __syncthreads();   // this tile is written, the other buffer is read
    if (more) fetch(tn);
    const T* sk = tk + buf * kTile;
    const T* sv = tv + buf * kTile;

    const uint64_t all = BN == 64 ? ~0ull : (1ull << (BN & 63)) - 1;
    Acc s[KB][QB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const Acc z = live == all ? Acc{} : acc_rows(bias + buf * BN + kb * 32);
#pragma unroll
      for (int j = 0; j < QB; ++j) s[kb][j] = z;
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const Frag<T> f = tile_frag<T, DP>(sk, kb * 32, c * 16);
#pragma unroll
        for (int j = 0; j < QB; ++j) s[kb][j] = mma(f, q[j][c], s[kb][j]);
      }

    if (t * BN + BN - 1 > lim0) {
#pragma unroll
      for (int j = 0; j < QB; ++j) {
        int left = lim[j] - t * BN - 4 * hi;
        asm volatile("" : "+v"(left));   // made here: a branch, not selects in every tile
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (kb * 32 + 8 * (i >> 2) + (i & 3) > left) s[kb][j][i] = -INFINITY;
      }
    }
#pragma unroll
    for (int j = 0; j < QB; ++j) {
      float mx = s[0][j][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][j][i]);
      mx = fmaxf(m[j], max_halves(mx));
      // The exponents' base follows the maximum where it lags by more than 2^8: P up to 256 is as exact
      // as P up to 1, and past a row's first tile O is hardly ever scaled.
      if (__ballot((mx - m[j]) * c2 > 8.0f)) {
        const float f = mx == -INFINITY ? 1.0f : exp2_((m[j] - mx) * c2);
        l[j] *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[j][d][i] *= f;
        m[j] = mx;
      }
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int j = 0; j < QB; ++j) {
        // a row without a key so far keeps -inf and takes 0 for its base: exp2(-inf) = 0
        const float top = m[j] == -INFINITY ? 0.0f : m[j], base = top * c2;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          // fp32: exactly 1 at the maximum, so that a row with one key gives its v to the last bit;
          // half types round P to fewer bits than the one operation less can lose
          s[kb][j][i] = sizeof(T) == 4 ? exp2_((s[kb][j][i] - top) * c2)
                                       : exp2_(__builtin_fmaf(s[kb][j][i], c2, -base));
          l[j] += s[kb][j][i];
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        Frag<T> p[QB], rest[QB];
#pragma unroll
        for (int j = 0; j < QB; ++j) {
          p[j] = acc_frag<T>(s[kb][j], c);
          if constexpr (kTwoParts<T, DP, ODD>) rest[j] = acc_rest(s[kb][j], c, p[j]);
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const Frag<T> f = transpose_frag<T, DP>(sv, kb * 32 + c * 16, d * 32);
#pragma unroll
          for (int j = 0; j < QB; ++j) {
            o[j][d] = mma(f, p[j], o[j][d]);
            if constexpr (kTwoParts<T, DP, ODD>) o[j][d] = mma(f, rest[j], o[j][d]);
          }
        }
      }
    }
    if (more) put(buf ^ 1, ln);
    buf ^= 1;
    t = tn;
    live = ln;
    have = more;
  }

#pragma unroll
  for (int j = 0; j < QB; ++j) {
    const int row = row0 + 32 * j;
    const float sum = sum_halves(l[j]);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const float lse = sum == 0.0f ? -INFINITY : __builtin_fmaf(m[j], a.scale, kLn2 * __log2f(sum));
    if (row >= a.R) continue;
    if (a.nsplit == 1) {
      int pos, h;
      attn_row(a, row, &pos, &h);
      const int hq = hk * a.grp + h;
      T* op = static_cast<T*>(a.out) + b * a.so.b + hq * a.so.h + (int64_t)pos * a.so.n;
#pragma unroll
      for (int d = 0; d < DB; ++d) store_column(op, a.D, d, o[j][d], inv);
      if (sizeof(T) == 2 && a.rest) {
        T* rp = static_cast<T*>(a.rest) + (op - static_cast<T*>(a.out));
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          Acc x;
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = rest_of<T>(o[j][d][i] * inv);
          store_column(rp, a.D, d, x, 1.0f);
        }
      }
      if (a.lse && hi == 0) a.lse[((int64_t)b * a.Hkv * a.grp + hq) * a.Nq + pos] = lse;
    } else {
      const int64_t i = ((int64_t)sp * (gridDim.x / nrb / a.nsplit) + bh) * a.R + row;
#pragma unroll
      for (int d = 0; d < DB; ++d) store_column(a.part + i * a.D4, a.D4, d, o[j][d], inv);
      if (hi == 0) a.part2[i] = lse;
    }
  }
}

// Joins the parts of split rows; BLOCK: a block a row.
template <typename T, bool BLOCK>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a, int BH, int L, int G) {
  const JoinTeam t(L, G);
  const int64_t rows = (int64_t)BH * a.R;
  if (t.row >= rows) return;
  const int bh = (int)(t.row / a.R), row = (int)(t.row - (int64_t)bh * a.R);
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  int pos, h;
  attn_row(a, row, &pos, &h);
  const int hq = hk * a.grp + h;
  const float mx = join_max<BLOCK>(t, a.part2, rows, a.nsplit), m = mx == -INFINITY ? 0.0f : mx;
  T* op = static_cast<T*>(a.out) + b * a.so.b + hq * a.so.h + (int64_t)pos * a.so.n;
  float l = 0.0f;
  for (int c0 = 0; c0 < a.D; c0 += L * 4) {
    const int c = c0 + t.lig * 4;
    float x[4];
    join_parts<true, BLOCK>(t, a.part, a.part2, rows, a.nsplit, a.D4, c, m, &l, x);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (t.g == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] *= inv;
      store4(op + c, a.D - c, x[0], x[1], x[2], x[3]);
      if (sizeof(T) == 2 && a.rest)
        store4(static_cast<T*>(a.rest) + (op + c - static_cast<T*>(a.out)), a.D - c,
               rest_of<T>(x[0]), rest_of<T>(x[1]), rest_of<T>(x[2]), rest_of<T>(x[3]));
    }
  }
  if (a.lse && t.g == 0 && t.lig == 0)
    a.lse[((int64_t)b * a.Hkv * a.grp + hq) * a.Nq + pos] =
        l == 0.0f ? -INFINITY : m + kLn2 * __log2f(l);
}

template <typename T, int DP, int NW, int BN, int QB, bool ODD>
int launch_fwd(const AttnArgs& a, int blocks, hipStream_t stream) {
  static LdsLimit lim;
  return launch_lds(k_attn_fwd<T, DP, NW, BN, QB, ODD>, lim, blocks, 64 * NW, fwd_lds<T, DP, BN>(), a,
                    stream);
}

int attn_launch_fwd(const AttnArgs& a0, int BH, int dtype, const AttnPlan& p, hipStream_t stream) {
  AttnArgs a = a0;
  a.nsplit = p.fs;
  const int blocks = p.rb_f * p.fs * BH;
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int e = by_head(a.D, [&](auto dp, auto odd) {
      if constexpr (!odd())
        if (p.fw == 1) return launch_fwd<T, dp(), 1, 32, 1, false>(a, blocks, stream);
      if constexpr (!odd() && sizeof(T) == 2 && dp() <= 64)
        if (p.fq == 2) return launch_fwd<T, dp(), 4, 64, 2, false>(a, blocks, stream);
      return launch_fwd<T, dp(), 4, 64, 1, odd()>(a, blocks, stream);
    });
    if (e || p.fs == 1) return e;
    int L, G;
    const int64_t rows = (int64_t)BH * a.R;
    join_shape(rows, a.D, a.nsplit, &L, &G);
    // Up to a row a CU, such as single tokens': a block each, where that leaves each group a part or more
    // (64 rows of 64 parts: the join 9.5 -> 4.9 us, a waited-for call 44.5 -> 40.4).
    if (rows <= 256 && a.nsplit * L >= 256) {
      G = 256 / L;
      k_attn_join<T, true><<<(int)rows, 256, 0, stream>>>(a, BH, L, G);
    } else {
      k_attn_join<T, false><<<join_blocks(rows, L, G), 256, 0, stream>>>(a, BH, L, G);
    }
    return launch_status();
  });
}

}  // namespace tts
