// Attention forward: one pass over the keys with the running maximum and sum of each row's softmax.
//
// A wave owns 32 rows (columns of S^T and O^T): Q stays in registers as the B operand, K and V tiles
// of BN keys pass through LDS, read by all waves of the block, the next tile's loads in flight
// while this one is computed.  Rows' maxima and sums are over a lane's own values; the two halves of
// the wave are joined once a tile (maximum) and once at the end (sum).
//
// Roundings: S, the softmax and O are fp32; P is rounded to the operands' type for its product with V
// (half types), O once at the end.
//
// Few rows (serving): one wave a block and the keys split over blocks; each part leaves its normalised
// O and its log-sum-exp, and k_attn_join adds the parts by exp(L_part - L).

#include "attention.h"

namespace tts {

template <typename T, int DP, int BN>
constexpr size_t fwd_lds() {
  return (size_t)4 * BN * kTileStride<T, DP> * sizeof(T) + 2 * BN * sizeof(float);
}

template <typename T, int DP, int NW, int BN, bool ODD>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 && (NW > 1 || DP <= 64) ? 2 : 1) void k_attn_fwd(AttnArgs a) {
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
  Frag<T> q[KC];
  {
    const T* qp = static_cast<const T*>(a.q) + b * a.sq.b + (int64_t)hk * a.grp * a.sq.h +
                  row_offset(a.sq, pos, h);
#pragma unroll
    for (int c = 0; c < KC; ++c) q[c] = load_frag(qp + c * 16 + hi * 8, a.D - c * 16 - hi * 8);
#pragma unroll
    for (int c = 0; c < KC; ++c) arrive(q[c]);
  }
  const int lim = a.causal ? pos + a.off : a.Nk;   // the row sees keys up to lim
  // keys that any row of the block sees
  int nk = a.Nk;
  if (a.causal) {
    int p1, h1;
    const int last = (rb + 1) * NW * 32 - 1;
    attn_row(a, last < a.R ? last : a.R - 1, &p1, &h1);
    nk = min(nk, max(p1 + a.off + 1, 0));
  }
  int lim0 = a.Nk;   // keys up to lim0 are seen by every row of the wave
  if (a.causal) {
    int p0, h0;
    attn_row(a, row0 < a.R ? row0 : a.R - 1, &p0, &h0);
    lim0 = p0 + a.off;
  }
  const int tiles = (a.Nk + BN - 1) / BN, need = (nk + BN - 1) / BN;
  const int t0 = (int)((int64_t)tiles * sp / a.nsplit), t1 = (int)((int64_t)tiles * (sp + 1) / a.nsplit);

  Acc o[DB] = {};
  float m = -INFINITY, l = 0.0f;
  const float c2 = a.scale * kLog2e;

  KeyTiles<BN> it;
  it.start(a.mask ? a.mask + b * a.mask_stride : nullptr, a.Nk, t0, min(t1, need));
  int t = 0;
  uint64_t live = 0;
  bool have = it.next(&t, &live);
  TileLoad<T, DP, BN, NT, ODD> lk, lv;
  auto fetch = [&](int tile) {
    const int last = a.Nk - 1 - tile * BN;
    const T* k0 = kp + (int64_t)tile * BN * a.sk.n;
    const T* v0 = vp + (int64_t)tile * BN * a.sv.n;
    lk.load(a.D, [&](int n) { return k0 + (int64_t)min(n, last) * a.sk.n; });
    lv.load(a.D, [&](int n) { return v0 + (int64_t)min(n, last) * a.sv.n; });
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
    Acc s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) s[kb] = live == all ? Acc{} : acc_rows(bias + buf * BN + kb * 32);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int c = 0; c < KC; ++c) s[kb] = mma(tile_frag<T, DP>(sk, kb * 32, c * 16), q[c], s[kb]);

    if (t * BN + BN - 1 > lim0) {
      const int left = lim - t * BN - 4 * hi;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kb * 32 + 8 * (i >> 2) + (i & 3) > left) s[kb][i] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = fmaxf(m, max_halves(mx));
    // a row without a key so far keeps -inf and takes 0 for its exponents' base: exp2(-inf) = 0
    const float top = mx == -INFINITY ? 0.0f : mx, base = top * c2;
    if (__ballot(mx > m)) {
      const float f = exp2_((m - top) * c2);
      l *= f;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= f;
      m = mx;
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        // fp32: exactly 1 at the maximum, so that a row with one key gives its v to the last bit;
        // half types round P to fewer bits than the one operation less can lose
        s[kb][i] = sizeof(T) == 4 ? exp2_((s[kb][i] - top) * c2)
                                  : exp2_(__builtin_fmaf(s[kb][i], c2, -base));
        l += s[kb][i];
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Frag<T> p = acc_frag<T>(s[kb], c);
#pragma unroll
        for (int d = 0; d < DB; ++d)
          o[d] = mma(transpose_frag<T, DP>(sv, kb * 32 + c * 16, d * 32), p, o[d]);
      }
    }
    if (more) put(buf ^ 1, ln);
    buf ^= 1;
    t = tn;
    live = ln;
    have = more;
  }

  l = sum_halves(l);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const float lse = l == 0.0f ? -INFINITY : m * a.scale + kLn2 * __log2f(l);
  if (row >= a.R) return;
  if (a.nsplit == 1) {
    const int hq = hk * a.grp + h;
    T* op = static_cast<T*>(a.out) + b * a.so.b + hq * a.so.h + (int64_t)pos * a.so.n;
#pragma unroll
    for (int d = 0; d < DB; ++d) store_column(op, a.D, d, o[d], inv);
    if (a.lse && hi == 0) a.lse[((int64_t)b * a.Hkv * a.grp + hq) * a.Nq + pos] = lse;
  } else {
    const int64_t i = ((int64_t)sp * (gridDim.x / nrb / a.nsplit) + bh) * a.R + row;
#pragma unroll
    for (int d = 0; d < DB; ++d) store_column(a.part + i * a.D, a.D, d, o[d], inv);
    if (hi == 0) a.part2[i] = lse;
  }
}

// Joins the parts of split rows: L lanes a row, parts in order.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a, int BH, int L) {
  const int lig = threadIdx.x & (L - 1);
  const int64_t rows = (int64_t)BH * a.R, i = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (i >= rows) return;
  const int bh = (int)(i / a.R), row = (int)(i - (int64_t)bh * a.R);
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  int pos, h;
  attn_row(a, row, &pos, &h);
  const int hq = hk * a.grp + h;
  float m = -INFINITY, l = 0.0f;
  for (int s = 0; s < a.nsplit; ++s) m = fmaxf(m, a.part2[s * rows + i]);
  const float base = m == -INFINITY ? 0.0f : m;
  // a NaN in any part reaches the sum, as it does in one pass
  for (int s = 0; s < a.nsplit; ++s) l += exp2_((a.part2[s * rows + i] - base) * kLog2e);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* op = static_cast<T*>(a.out) + b * a.so.b + hq * a.so.h + (int64_t)pos * a.so.n;
  for (int c = lig * 4; c < a.D; c += L * 4) {
    float x[4] = {};
#pragma unroll 4
    for (int s = 0; s < a.nsplit; ++s) {
      const float w = exp2_((a.part2[s * rows + i] - base) * kLog2e);
      float v[4];
      load_row(a.part + (s * rows + i) * a.D + c, a.D - c, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] += w * v[j];
    }
    store4(op + c, a.D - c, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  }
  if (a.lse && lig == 0)
    a.lse[((int64_t)b * a.Hkv * a.grp + hq) * a.Nq + pos] =
        l == 0.0f ? -INFINITY : base + kLn2 * __log2f(l);
}

template <typename T, int DP, int NW, int BN, bool ODD>
int launch_fwd(const AttnArgs& a, int blocks, hipStream_t stream) {
  static LdsLimit lim;
  return launch_lds(k_attn_fwd<T, DP, NW, BN, ODD>, lim, blocks, 64 * NW, fwd_lds<T, DP, BN>(), a,
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
        if (p.fw == 1) return launch_fwd<T, dp(), 1, 32, false>(a, blocks, stream);
      return launch_fwd<T, dp(), 4, 64, odd()>(a, blocks, stream);
    });
    if (e || p.fs == 1) return e;
    const int L = row_lanes((a.D + 3) / 4);
    const int64_t rows = (int64_t)BH * a.R;
    k_attn_join<T><<<(int)((rows * L + 255) / 256), 256, 0, stream>>>(a, BH, L);
    return launch_status();
  });
}

}  // namespace tts
