// Attention backward, the queries' side: dQ, and D = rowsum(dO O) for the keys' side.
//
// The layout of the forward: a wave owns 32 rows; K and V tiles pass through LDS.  Each tile's
// probabilities are recomputed from S and the forward's log-sum-exp, dS^T is the B operand of
// dQ^T += K^T dS^T, and K's tile is read both ways, by rows and transposed.  Splitting the gradient into
// this kernel and the keys' one computes S and dP twice (7 products in place of 5), and needs no
// atomics, no partial dQ for each block of keys, and gives the same bits every time.
//
// dS is rounded to the operands' type for its product (half types); everything else is fp32.  (Odd heads of up
// to 32 values: kTwoParts.)
//
// Measured: 8040 x 8040, 16 heads of 128 bf16, 870 us (910 TFLOP/s); 2500 x 2500, 16 heads of 64: 66 us.
// Tiles of 32 keys in place of 64: 906 -> 1018.

#include "attention.h"

namespace tts {

template <typename T, int DP, int BN>
constexpr size_t dq_lds() {
  return (size_t)4 * BN * kTileStride<T, DP> * sizeof(T) + 2 * BN * sizeof(float);
}

template <typename T, int DP, int NW, int BN, bool ODD>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 && (NW > 1 || DP <= 64) ? 2 : 1) void k_attn_dq(AttnArgs a) {
  constexpr int KC = DP / 16, DB = DP / 32, KB = BN / 32, NT = 64 * NW;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* tk = reinterpret_cast<T*>(smem);
  constexpr int kTile = BN * kTileStride<T, DP>;
  T* tv = tk + 2 * kTile;
  float* bias = reinterpret_cast<float*>(tv + 2 * kTile);   // [2][BN] 0, or -inf for hidden keys

  const int nrb = (a.R + 32 * NW - 1) / (32 * NW);
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const int rb = item % nrb, sp = item / nrb % a.nsplit, bh = item / nrb / a.nsplit;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int lane = threadIdx.x & 63, hi = lane >> 5, wave = threadIdx.x >> 6;
  const T* kp = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
  const T* vp = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h;

  const int row0 = (rb * NW + wave) * 32, row = row0 + (lane & 31);
  int pos, h;
  attn_row(a, row < a.R ? row : a.R - 1, &pos, &h);
  const int hq = hk * a.grp + h;
  Frag<T> q[KC], go[KC];
  float delta;
  {
    const T* qp = static_cast<const T*>(a.q) + b * a.sq.b + hq * a.sq.h + (int64_t)pos * a.sq.n;
    const T* gp = static_cast<const T*>(a.dout) + b * a.sdo.b + hq * a.sdo.h + (int64_t)pos * a.sdo.n;
    const T* op = static_cast<const T*>(a.o) + b * a.so.b + hq * a.so.h + (int64_t)pos * a.so.n;
    Frag<T> of[KC];
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int d = c * 16 + hi * 8;
      q[c] = load_frag(qp + d, a.D - d);
      go[c] = load_frag(gp + d, a.D - d);
      of[c] = load_frag(op + d, a.D - d);
    }
    delta = row_dots<T, KC>(of, go);
    if (sizeof(T) == 2 && a.orest) {   // what O's rounding left out
      const T* rp = static_cast<const T*>(a.orest) + (op - static_cast<const T*>(a.o));
#pragma unroll
      for (int c = 0; c < KC; ++c) of[c] = load_frag(rp + c * 16 + hi * 8, a.D - c * 16 - hi * 8);
      delta += row_dots<T, KC>(of, go);
    }
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      arrive(q[c]);
      arrive(go[c]);
    }
  }
  const int64_t stat = ((int64_t)b * a.Hkv * a.grp + hq) * a.Nq + pos;
  // exponents' base; a row without a key has L = -inf: +inf here, so that every P is exp2(-inf) = 0
  float lse = a.lse[stat];
  if (lse == -INFINITY) lse = INFINITY;
  asm volatile("" : "+v"(lse));   // here, not in the loop (arrive)
  const float lse2 = lse * kLog2e;
  if (sp == 0 && hi == 0 && row < a.R) a.delta[(int64_t)bh * a.R + row] = delta;

  const int lim = a.causal ? pos + a.off : a.Nk;
  const int lim0 = __builtin_amdgcn_readfirstlane(lim);   // seen by every row of the wave
  int nk = a.Nk;
  if (a.causal) {
    int p1, h1;
    const int last = (rb + 1) * NW * 32 - 1;
    attn_row(a, last < a.R ? last : a.R - 1, &p1, &h1);
    nk = min(nk, max(p1 + a.off + 1, 0));
  }
  const int tiles = (a.Nk + BN - 1) / BN, need = (nk + BN - 1) / BN;
  const int t0 = (int)((int64_t)tiles * sp / a.nsplit), t1 = (int)((int64_t)tiles * (sp + 1) / a.nsplit);

  Acc dq[DB] = {};
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
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      Acc s = live == all ? Acc{} : acc_rows(bias + buf * BN + kb * 32), p = {};
#pragma unroll
      for (int c = 0; c < KC; ++c) s = mma(tile_frag<T, DP>(sk, kb * 32, c * 16), q[c], s);
#pragma unroll
      for (int c = 0; c < KC; ++c) p = mma(tile_frag<T, DP>(sv, kb * 32, c * 16), go[c], p);
      if (t * BN + BN - 1 > lim0) {
        int left = lim - t * BN - 4 * hi;
        asm volatile("" : "+v"(left));   // made here: a branch, not selects in every tile
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kb * 32 + 8 * (i >> 2) + (i & 3) > left) s[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[i] = prob<T>(s[i], a.scale, c2, lse, lse2) * (p[i] - delta);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Frag<T> ds = acc_frag<T>(s, c);
        Frag<T> rest;
        if constexpr (kTwoParts<T, DP, ODD>) rest = acc_rest(s, c, ds);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const Frag<T> f = transpose_frag<T, DP>(sk, kb * 32 + c * 16, d * 32);
          dq[d] = mma(f, ds, dq[d]);
          if constexpr (kTwoParts<T, DP, ODD>) dq[d] = mma(f, rest, dq[d]);
        }
      }
    }
    if (more) put(buf ^ 1, ln);
    buf ^= 1;
    t = tn;
    live = ln;
    have = more;
  }
  if (row >= a.R) return;
  if (a.nsplit == 1) {
    if (!a.dq) return;
    T* op = static_cast<T*>(a.dq) + b * a.sdq.b + hq * a.sdq.h + (int64_t)pos * a.sdq.n;
#pragma unroll
    for (int d = 0; d < DB; ++d) store_column(op, a.D, d, dq[d], a.scale);
  } else {
    const int64_t i = ((int64_t)sp * (gridDim.x / nrb / a.nsplit) + bh) * a.R + row;
#pragma unroll
    for (int d = 0; d < DB; ++d) store_column(a.part + i * a.D4, a.D4, d, dq[d], a.scale);
  }
}

// Sums the parts of split rows.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_dq_join(AttnArgs a, int BH, int L, int G) {
  const JoinTeam t(L, G);
  const int64_t rows = (int64_t)BH * a.R;
  if (t.row >= rows) return;
  const int bh = (int)(t.row / a.R), row = (int)(t.row - (int64_t)bh * a.R);
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  int pos, h;
  attn_row(a, row, &pos, &h);
  T* op = static_cast<T*>(a.dq) + b * a.sdq.b + (hk * a.grp + h) * a.sdq.h + (int64_t)pos * a.sdq.n;
  for (int c0 = 0; c0 < a.D; c0 += L * 4) {
    const int c = c0 + t.lig * 4;
    float x[4], l;
    join_parts<false>(t, a.part, nullptr, rows, a.nsplit, a.D4, c, 0.0f, &l, x);
    if (t.g == 0) store4(op + c, a.D - c, x[0], x[1], x[2], x[3]);
  }
}

template <typename T, int DP, int NW, int BN, bool ODD>
int launch_dq(const AttnArgs& a, int blocks, hipStream_t stream) {
  static LdsLimit lim;
  return launch_lds(k_attn_dq<T, DP, NW, BN, ODD>, lim, blocks, 64 * NW, dq_lds<T, DP, BN>(), a, stream);
}

int attn_launch_dq(const AttnArgs& a0, int BH, int dtype, const AttnPlan& p, hipStream_t stream) {
  AttnArgs a = a0;
  a.nsplit = p.qs;
  const int blocks = p.rb_q * p.qs * BH;
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int e = by_head(a.D, [&](auto dp, auto odd) {
      if constexpr (!odd())
        if (p.qw == 1) return launch_dq<T, dp(), 1, 32, false>(a, blocks, stream);
      return launch_dq<T, dp(), 4, 64, odd()>(a, blocks, stream);
    });
    if (e || p.qs == 1 || !a.dq) return e;
    int L, G;
    join_shape((int64_t)BH * a.R, a.D, a.nsplit, &L, &G);
    k_attn_dq_join<T><<<join_blocks((int64_t)BH * a.R, L, G), 256, 0, stream>>>(a, BH, L, G);
    return launch_status();
  });
}

}  // namespace tts
