// Attention backward, the keys' side: dK and dV; and the C entry points.
//
// A wave owns 32 keys (columns of S, dV^T and dK^T): K and V stay in registers as B operands and the
// rows' Q and dO pass through LDS, 32 rows a tile, with their log-sum-exp, D and (causal) last
// visible key.  S gives P, dO V^T gives dP; P and dS are the B operands of dV^T += dO^T P and
// dK^T += Q^T dS, whose A operands are transposed reads of the same tiles.  Rows of all query heads of
// the group follow one another, so the sum over shared heads is the loop's.
//
// Bound: one wave a SIMD at 128 values a head, so what is not a matrix instruction adds to them: 8040 x 8040,
// 16 heads, bf16 1487 us (710 TFLOP/s), the matrix instructions alone 580, without staging 1170, without LDS
// reads 1090, without VALU work 1312.  2500 x 2500, 16 heads of 64: 87 us.
//
// Few keys and many rows (gaussians over a view's tokens): the rows are split over blocks, and
// k_attn_dkv_join adds the parts in order.

#include "attention.h"

namespace tts {

constexpr int kDkvRows = 64;   // rows a tile with four waves a block

template <typename T, int DP, int BM>
constexpr size_t dkv_lds() {
  return (size_t)4 * BM * kTileStride<T, DP> * sizeof(T) + 2 * 3 * BM * sizeof(float);
}

template <typename T, int DP, int NW, int BM, bool ODD, bool CAUSAL>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 && DP <= 64 ? 2 : 1) void k_attn_dkv(AttnArgs a) {
  constexpr int KC = DP / 16, DB = DP / 32, NT = 64 * NW;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int kTile = BM * kTileStride<T, DP>;
  T* tq = reinterpret_cast<T*>(smem);
  T* tg = tq + 2 * kTile;
  float* stat = reinterpret_cast<float*>(tg + 2 * kTile);   // [2][-L (/ scale in half types), -D, last key][BM]

  const int nkb = (a.Nk + 32 * NW - 1) / (32 * NW);
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const int kb = item % nkb, sp = item / nkb % a.nsplit, bh = item / nkb / a.nsplit;
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int lane = threadIdx.x & 63, hi = lane >> 5, wave = threadIdx.x >> 6;
  const int key0 = kb * 32 * NW, key = key0 + wave * 32 + (lane & 31);
  const T* qp = static_cast<const T*>(a.q) + b * a.sq.b + (int64_t)hk * a.grp * a.sq.h;
  const T* gp = static_cast<const T*>(a.dout) + b * a.sdo.b + (int64_t)hk * a.grp * a.sdo.h;

  bool on = key < a.Nk;
  if (on && a.mask) on = a.mask[b * a.mask_stride + key] != 0;
  const bool busy = __ballot(on) != 0;   // the wave has a live key
  Frag<T> k[KC], v[KC];
  {
    const int64_t kk = min(key, a.Nk - 1);
    const T* kp = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h + kk * a.sk.n;
    const T* vp = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h + kk * a.sv.n;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int d = c * 16 + hi * 8;
      k[c] = load_frag(kp + d, on ? a.D - d : 0);
      v[c] = load_frag(vp + d, on ? a.D - d : 0);
    }
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      arrive(k[c]);
      arrive(v[c]);
    }
  }
  Acc dk[DB] = {}, dv[DB] = {};
  const float c2 = a.scale * kLog2e, inv_scale = 1.0f / a.scale;

  // rows of this part; causal: none before the first that sees the block's first key
  const int tiles = (a.R + BM - 1) / BM;
  int t = (int)((int64_t)tiles * sp / a.nsplit);
  int t1 = (int)((int64_t)tiles * (sp + 1) / a.nsplit);
  if constexpr (CAUSAL) {
    const int64_t first = (int64_t)max(key0 - a.off, 0) * a.grp / BM;
    t = (int)(first > t ? (first < t1 ? first : t1) : t);
  }
  {   // no live key in the block: no rows
    int* any = reinterpret_cast<int*>(stat);
    if (lane == 0) any[wave] = busy;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) n |= any[w];
    __syncthreads();
    if (!n) t1 = t;
  }

  TileLoad<T, DP, BM, NT, ODD> lq, lg;
  // even rows: a whole tile's addresses are its first row's and offsets that are the same for every tile
  // (half types: the offsets would push fp32 tiles of 128 values out of the registers)
  constexpr bool kPlan = !ODD && sizeof(T) == 2;
  int lse_off, lim_off;
  if constexpr (kPlan) {
    auto at = [&](const AttnStride& s) {
      return [&](int n) {
        int pos, h;
        attn_row(a, n, &pos, &h);
        return (int)(h * s.h) + pos * s.n;
      };
    };
    if (a.even_rows) {
      lq.plan(a.D, at(a.sq));
      lg.plan(a.D, at(a.sdo));
    }
  }
  {
    int pos, h;
    attn_row(a, threadIdx.x & (BM - 1), &pos, &h);
    lse_off = h * a.Nq + pos;   // below R, which is below 2^30
    lim_off = pos + a.off;
  }
  const float* lsep = a.lse + (int64_t)bh * a.grp * a.Nq;
  float st0 = 0.0f, st1 = 0.0f;
  int st2 = 0;
  auto fetch = [&](int tile) {
    if (kPlan && a.even_rows && (tile + 1) * BM <= a.R) {
      int pos0, h0;
      attn_row(a, tile * BM, &pos0, &h0);
      pos0 = __builtin_amdgcn_readfirstlane(pos0);
      lq.load_planned(qp + (int64_t)pos0 * a.sq.n);
      lg.load_planned(gp + (int64_t)pos0 * a.sdo.n);
      st0 = lsep[pos0 + lse_off];
      st1 = a.delta[(int64_t)bh * a.R + tile * BM + (int)(threadIdx.x & (BM - 1))];
      st2 = pos0 + lim_off;
      return;
    }
    lq.load(a.D, [&](int n) {
      int pos, h;
      attn_row(a, min(tile * BM + n, a.R - 1), &pos, &h);
      return qp + row_offset(a.sq, pos, h);
    });
    lg.load(a.D, [&](int n) {
      int pos, h;
      attn_row(a, min(tile * BM + n, a.R - 1), &pos, &h);
      return gp + row_offset(a.sdo, pos, h);
    });
    const int r = min(tile * BM + (int)(threadIdx.x & (BM - 1)), a.R - 1);
    int pos, h;
    attn_row(a, r, &pos, &h);
    st0 = lsep[(int64_t)h * a.Nq + pos];
    st1 = a.delta[(int64_t)bh * a.R + r];
    st2 = pos + a.off;
  };
  auto put = [&](int tile, int buf) {
    const int n = a.R - tile * BM;
    const uint64_t rows = n >= BM ? (BM == 64 ? ~0ull : (1ull << (BM & 63)) - 1) : (1ull << n) - 1;
    lq.store(tq + buf * kTile, rows, a.D);
    lg.store(tg + buf * kTile, rows, a.D);
    if (threadIdx.x < BM) {
      float* s = stat + buf * 3 * BM;
      // rows without a key (L = -inf) and rows past the last: every P is exp2(-inf) = 0
      const bool none = st0 == -INFINITY || (int)threadIdx.x >= n;
      s[threadIdx.x] = none ? -INFINITY : sizeof(T) == 4 ? -st0 : -st0 * inv_scale;
      s[BM + threadIdx.x] = (int)threadIdx.x >= n ? 0.0f : -st1;
      reinterpret_cast<int*>(s)[2 * BM + threadIdx.x] = st2;
    }
  };
  if (t < t1) {
    fetch(t);
    put(t, 0);
  }
  int buf = 0;
  for (; t < t1; ++t) {
    const bool more = t + 1 < t1;
    __syncthreads();   // this tile is written, the other buffer is read
    if (more) fetch(t + 1);
    const T* sq = tq + buf * kTile;
    const T* sg = tg + buf * kTile;
    const float* st = stat + buf * 3 * BM;
    if (busy) {
#pragma unroll
      for (int rb = 0; rb < BM; rb += 32) {
        // Half types: S starts from -L / scale, no subtraction after it; fp32 would lose bits of S to the
        // larger number (P 1e-6 off in place of 2e-7).  dP does not start from -D: its sum and D's are the
        // same terms in the same order for a row with one key, and dS = 0 (row_dots).
        Acc s = {}, p = {};
        if constexpr (sizeof(T) == 2) s = acc_rows(st + rb);
#pragma unroll
        for (int c = 0; c < KC; ++c) s = mma(tile_frag<T, DP>(sq, rb, c * 16), k[c], s);
#pragma unroll
        for (int c = 0; c < KC; ++c) p = mma(tile_frag<T, DP>(sg, rb, c * 16), v[c], p);
        if constexpr (CAUSAL) {
          const Acc lim = acc_rows(st + 2 * BM + rb);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (key > __builtin_bit_cast(int, (float)lim[i])) s[i] = -INFINITY;
        }
        if constexpr (sizeof(T) == 4) {
          const Acc ml = acc_rows(st + rb);
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = prob<T>(s[i], a.scale, c2, -ml[i], 0.0f);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = exp2_(s[i] * c2);
        }
        const Acc md = acc_rows(st + BM + rb);
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = (p[i] + md[i]) * s[i];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const Frag<T> pf = acc_frag<T>(s, c), df = acc_frag<T>(p, c);
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            dv[d] = mma(transpose_frag<T, DP>(sg, rb + c * 16, d * 32), pf, dv[d]);
            dk[d] = mma(transpose_frag<T, DP>(sq, rb + c * 16, d * 32), df, dk[d]);
          }
        }
      }
    }
    if (more) put(t + 1, buf ^ 1);
    buf ^= 1;
  }
  if (!on) {   // a hidden key's column holds products with zeros
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[d] = dv[d] = Acc{};
  }
  if (key >= a.Nk) return;
  if (a.nsplit == 1) {
    if (a.dk) {
      T* kp = static_cast<T*>(a.dk) + b * a.sdk.b + hk * a.sdk.h + (int64_t)key * a.sdk.n;
#pragma unroll
      for (int d = 0; d < DB; ++d) store_column(kp, a.D, d, dk[d], a.scale);
    }
    if (a.dv) {
      T* vp = static_cast<T*>(a.dv) + b * a.sdv.b + hk * a.sdv.h + (int64_t)key * a.sdv.n;
#pragma unroll
      for (int d = 0; d < DB; ++d) store_column(vp, a.D, d, dv[d], 1.0f);
    }
  } else {
    const int64_t i = (((int64_t)sp * (gridDim.x / nkb / a.nsplit) + bh) * a.Nk + key) * 2;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      store_column(a.part2 + i * a.D4, a.D4, d, dk[d], a.scale);
      store_column(a.part2 + (i + 1) * a.D4, a.D4, d, dv[d], 1.0f);
    }
  }
}

// Sums the parts of split keys; a row is a (key, dk or dv).
template <typename T>
__global__ __launch_bounds__(256) void k_attn_dkv_join(AttnArgs a, int BH, int L, int G) {
  const JoinTeam t(L, G);
  const int64_t rows = (int64_t)BH * a.Nk * 2;
  if (t.row >= rows) return;
  const int bh = (int)(t.row / 2 / a.Nk), key = (int)(t.row / 2 - (int64_t)bh * a.Nk);
  const int b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const AttnStride& s = t.row & 1 ? a.sdv : a.sdk;
  T* op = static_cast<T*>(t.row & 1 ? a.dv : a.dk);
  if (!op) return;
  op += b * s.b + hk * s.h + (int64_t)key * s.n;
  for (int c0 = 0; c0 < a.D; c0 += L * 4) {
    const int c = c0 + t.lig * 4;
    float x[4], l;
    join_parts<false>(t, a.part2, nullptr, rows, a.nsplit, a.D4, c, 0.0f, &l, x);
    if (t.g == 0) store4(op + c, a.D - c, x[0], x[1], x[2], x[3]);
  }
}

template <typename T, int DP, int NW, int BM, bool ODD>
int launch_dkv(const AttnArgs& a, int blocks, hipStream_t stream) {
  static LdsLimit lim, lim_causal;
  constexpr size_t lds = dkv_lds<T, DP, BM>();
  if (a.causal)
    return launch_lds(k_attn_dkv<T, DP, NW, BM, ODD, true>, lim_causal, blocks, 64 * NW, lds, a,
                      stream);
  return launch_lds(k_attn_dkv<T, DP, NW, BM, ODD, false>, lim, blocks, 64 * NW, lds, a, stream);
}

int attn_launch_dkv(const AttnArgs& a0, int BH, int dtype, const AttnPlan& p, hipStream_t stream) {
  AttnArgs a = a0;
  a.nsplit = p.ks;
  const int blocks = p.kb * p.ks * BH;
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int e = by_head(a.D, [&](auto dp, auto odd) {
      if constexpr (!odd())
        if (p.kw == 1) return launch_dkv<T, dp(), 1, 32, false>(a, blocks, stream);
      // fp32 with 128 values a head: half the rows a tile, which leaves its registers unspilled
      constexpr int kRows = sizeof(T) == 4 && dp() == 128 ? kDkvRows / 2 : kDkvRows;
      return launch_dkv<T, dp(), 4, kRows, odd()>(a, blocks, stream);
    });
    if (e || p.ks == 1) return e;
    int L, G;
    join_shape((int64_t)BH * a.Nk * 2, a.D, a.nsplit, &L, &G);
    k_attn_dkv_join<T><<<join_blocks((int64_t)BH * a.Nk * 2, L, G), 256, 0, stream>>>(a, BH, L, G);
    return launch_status();
  });
}

// Up to 32 rows (keys) one wave a block holds them all; past that four waves share the tiles they
// read.  Half types with head sizes up to 64 give a wave 64 rows in the forward once that leaves a wave
// for every second SIMD: each fragment of K and V then feeds two products (2500 x 2500, 16 heads of
// 64: 77 -> 62 us with its join; 128 values a head leave it one wave a SIMD, 735 -> 810).  Then the
// long axis is split until the waves that have work fill the card, two a SIMD: one where the keys'
// kernel needs a SIMD's registers for itself.
AttnPlan attn_plan(const AttnArgs& a, int BH, int dtype) {
  AttnPlan p;
  const bool odd = a.D % 8 != 0;
  const int64_t row_waves = (int64_t)((a.R - 1) / 32 + 1) * BH;
  const int64_t key_waves = (int64_t)((a.Nk - 1) / 32 + 1) * BH;
  p.fw = p.qw = a.R <= 32 && !odd ? 1 : 4;
  p.fq = p.fw == 4 && !odd && dtype != TTS_F32 && a.D <= 64 && row_waves >= 1024 ? 2 : 1;
  p.rb_f = (a.R - 1) / (32 * p.fw * p.fq) + 1;
  p.rb_q = (a.R - 1) / (32 * p.qw) + 1;
  const int tiles = (a.Nk - 1) / (p.fw == 1 ? 32 : 64) + 1;
  p.fs = attn_splits(row_waves / p.fq, 2048, tiles, p.fw == 1 ? 2 : 4);
  p.qs = attn_splits(row_waves, 2048, tiles, p.qw == 1 ? 2 : 4);
  p.kw = a.Nk <= 32 && !odd ? 1 : 4;
  p.kb = (a.Nk - 1) / (32 * p.kw) + 1;
  p.ks = attn_splits(key_waves, a.D <= 64 ? 2048 : 1024, (a.R - 1) / (p.kw == 1 ? 32 : kDkvRows) + 1,
                     2);
  return p;
}

// Sub-buffers of the workspaces: forward's parts; backward's D, then parts of dQ and of dK, dV.
size_t attn_fwd_layout(AttnArgs& a, int64_t BH, const AttnPlan& p, char* base) {
  if (p.fs == 1) return 0;
  const size_t o = align256((size_t)p.fs * BH * a.R * a.D4 * sizeof(float));
  a.part = reinterpret_cast<float*>(base);
  a.part2 = reinterpret_cast<float*>(base + o);
  return o + align256((size_t)p.fs * BH * a.R * sizeof(float));
}
size_t attn_bwd_layout(AttnArgs& a, int64_t BH, const AttnPlan& p, char* base) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char* r = base + off;
    off += align256(bytes);
    return reinterpret_cast<float*>(r);
  };
  a.delta = take((size_t)BH * a.R * sizeof(float));
  a.part = take(p.qs > 1 ? (size_t)p.qs * BH * a.R * a.D4 * sizeof(float) : 0);
  a.part2 = take(p.ks > 1 ? (size_t)p.ks * BH * a.Nk * 2 * a.D4 * sizeof(float) : 0);
  return off;
}

// Checks a shape's numbers and sets what both directions take from it.
int attn_shape(const tts_attention_shape* s, AttnArgs* a, int* BH) {
  if (s->batch < 0 || s->kv_heads < 1 || s->heads < 1 || s->queries < 0 || s->keys < 0 ||
      !(s->scale >= kAttnMinScale) || !(s->scale <= kAttnMaxScale))
    return TTS_EINVAL;
  if (s->head_dim < 1 || s->head_dim > 128 || s->heads % s->kv_heads) return TTS_EHEADS;
  if (s->dtype < 0 || s->dtype > 2) return TTS_EDTYPE;
  const int64_t grp = s->heads / s->kv_heads, lim = (int64_t)1 << 30;
  if (grp > lim || s->queries > lim / grp || s->keys > lim || s->batch > lim ||
      s->kv_heads > lim || (s->batch > 0 && s->kv_heads > lim / s->batch))
    return TTS_ELENGTH;
  *a = AttnArgs{};
  for (const int64_t* x : {s->q, s->k, s->v, s->o, s->dout, s->dq, s->dk, s->dv})
    if (x[2] < 0 || x[2] >= (int64_t)1 << 23) return TTS_ELENGTH;
  auto st = [](const int64_t* x) { return AttnStride{x[0], x[1], (int)x[2]}; };
  a->sq = st(s->q);
  a->sk = st(s->k);
  a->sv = st(s->v);
  a->so = st(s->o);
  a->sdo = st(s->dout);
  a->sdq = st(s->dq);
  a->sdk = st(s->dk);
  a->sdv = st(s->dv);
  a->mask_stride = s->mask_stride;
  a->Hkv = (int)s->kv_heads;
  a->grp = (int)grp;
  a->Nq = (int)s->queries;
  a->Nk = (int)s->keys;
  a->D = (int)s->head_dim;
  a->D4 = (a->D + 3) & ~3;
  a->R = (int)(s->queries * grp);
  while ((1 << a->grp_shift) < grp) ++a->grp_shift;
  a->grp_mul = (unsigned)((((uint64_t)1 << (30 + a->grp_shift)) + grp - 1) / grp);
  a->causal = s->causal != 0;
  a->off = (int)(s->keys - s->queries);
  a->scale = (float)s->scale;
  const int64_t far = (int64_t)1 << 31, e = (int64_t)elem_size((int)s->dtype);
  a->even_rows = 32 % grp == 0;
  for (const int64_t* x : {s->q, s->dout})
    if (x[1] < 0 || x[1] >= far || ((grp - 1) * x[1] + 64 * x[2] + 128) * e >= far) a->even_rows = 0;
  *BH = (int)(s->batch * s->kv_heads);
  return TTS_OK;
}

// Blocks of a launch are 32-bit.
bool attn_fits(const AttnArgs& a, int64_t BH, const AttnPlan& p) {
  const int64_t lim = (int64_t)1 << 30;
  return (int64_t)p.rb_f * p.fs * BH < lim && (int64_t)p.kb * p.ks * BH < lim &&
         BH * a.R < lim && BH * a.Nk < lim;
}

}  // namespace tts

using namespace tts;

extern "C" {

size_t tts_attention_workspace_bytes(const tts_attention_shape* shape, int backward) {
  AttnArgs a;
  int BH;
  if (!shape || attn_shape(shape, &a, &BH) || !BH || !a.R || !a.Nk) return 0;
  const AttnPlan p = attn_plan(a, BH, (int)shape->dtype);
  return backward ? attn_bwd_layout(a, BH, p, nullptr) : attn_fwd_layout(a, BH, p, nullptr);
}

int tts_attention_fwd(const tts_attention_shape* shape, const void* q, const void* k,
                      const void* v, const uint8_t* key_mask, void* out, void* rest, float* lse,
                      void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (!shape) return TTS_EINVAL;
  AttnArgs a;
  int BH;
  if (const int e = attn_shape(shape, &a, &BH)) return e;
  if (!BH || !a.R) return TTS_OK;
  if (!q || !out || (a.Nk > 0 && (!k || !v))) return TTS_EINVAL;
  AttnPlan p = {};
  if (a.Nk > 0) {
    p = attn_plan(a, BH, (int)shape->dtype);
  } else {   // no keys: rows of zeros, no tile is read
    p.fw = 4;
    p.rb_f = (a.R - 1) / 128 + 1;
    p.fs = 1;
    p.kb = p.ks = 1;
    key_mask = nullptr;
  }
  if (!attn_fits(a, BH, p)) return TTS_ELENGTH;
  a.q = q;
  a.k = k;
  a.v = v;
  a.mask = key_mask;
  a.out = out;
  a.rest = rest;
  a.lse = lse;
  const size_t need = attn_fwd_layout(a, BH, p, static_cast<char*>(workspace));
  if (need && (!workspace || workspace_bytes < need)) return TTS_EWORKSPACE;
  return attn_launch_fwd(a, BH, (int)shape->dtype, p, stream);
}

int tts_attention_bwd(const tts_attention_shape* shape, const void* q, const void* k,
                      const void* v, const uint8_t* key_mask, const void* out, const void* rest,
                      const float* lse, const void* dout, void* dq, void* dk, void* dv, void* workspace,
                      size_t workspace_bytes, hipStream_t stream) {
  if (!shape) return TTS_EINVAL;
  AttnArgs a;
  int BH;
  if (const int e = attn_shape(shape, &a, &BH)) return e;
  if (!BH || !a.R || !a.Nk) return TTS_EINVAL;   // no product to differentiate
  if (!q || !k || !v || !out || !lse || !dout || (!dq && !dk && !dv)) return TTS_EINVAL;
  const AttnPlan p = attn_plan(a, BH, (int)shape->dtype);
  if (!attn_fits(a, BH, p)) return TTS_ELENGTH;
  a.q = q;
  a.k = k;
  a.v = v;
  a.mask = key_mask;
  a.o = out;
  a.orest = rest;
  a.lse = const_cast<float*>(lse);
  a.dout = dout;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  const size_t need = attn_bwd_layout(a, BH, p, static_cast<char*>(workspace));
  if (!workspace || workspace_bytes < need) return TTS_EWORKSPACE;
  if (const int e = attn_launch_dq(a, BH, (int)shape->dtype, p, stream)) return e;
  if (!dk && !dv) return TTS_OK;
  return attn_launch_dkv(a, BH, (int)shape->dtype, p, stream);
}

}  // extern "C"
