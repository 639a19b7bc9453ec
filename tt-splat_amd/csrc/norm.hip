// Layer norm over the rows of x [rows, cols], forward and backward.
//
//   m = mean x,  r = 1 / sqrt(mean (x - m)^2 + eps),  xh = (x - m) r,  y = xh w + b
//   g = dy w,    dx = r (g - mean g - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Everything is held in 32 bits; y and dx are rounded once to x's type, dw and db once to w's.
//
// Bound: memory.  Rows of up to 256 vectors of 16 bytes (1024 fp32 or 2048 half values) are held in
// the registers of L lanes, L the power of two that covers them (eight rows of 64 half values share
// a wave), so x, dy are read once and y, dx written once, and the variance is the mean of squared
// deviations, not a difference of two large sums.  Wider rows take a block each and are read again
// from the caches for each of their passes.
//
// dw and db: each block walks its share of the rows with the columns' sums in registers, joins its
// waves in LDS in wave order and writes one row of partials; k_ln_join adds the blocks in order.
// No atomics: the same inputs give the same bits.
//
// Measured: 1M x 64 bf16 forward 44 us (6.0 TB/s of its 0.26 GB, part of it still in the caches), backward
// 75 + 6; 8040 x 1003 fp16 12 and 15 + 4.

#include "elem.h"

namespace tts {

constexpr int kLnBlock = 256;
constexpr int kLnWaves = kLnBlock / 64;
constexpr int kLnFwdBlocks = 2048;  // eight blocks a CU walk the rows
constexpr int kLnBwdBlocks = 1024;  // four a CU; each leaves one row of partials behind
constexpr int kLnShare = 4;         // rows a lane group or more where the card is full without
constexpr int kLnRegVecs = 256;     // rows of up to this many vectors stay in registers

// Weights of one lane's vectors at [c, c + kVec), `fill` where there is none.
template <typename T, int MODE>
__device__ __forceinline__ void ln_weight(const void* w, int wf32, int c, int cols, float fill,
                                          float* out) {
  constexpr int V = kVec<T>, VF = kVec<float>;
  if (!w) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = fill;
  } else if (wf32) {
#pragma unroll
    for (int h = 0; h < V; h += VF) {   // a tiny row of a half type may hold more than four values
      RowVec<float, MODE> r;
      r.load(static_cast<const float*>(w), c + h, cols);
      r.get(c + h, cols, out + h);
    }
  } else {
    RowVec<T, MODE> r;
    r.load(static_cast<const T*>(w), c, cols);
    r.get(c, cols, out);
  }
}
template <typename T, int L, int NV, int MODE>
__device__ __forceinline__ void ln_load_weight(const void* w, int wf32, int cols, int lig,
                                               float fill, float (&out)[NV][kVec<T>]) {
#pragma unroll
  for (int j = 0; j < NV; ++j)
    ln_weight<T, MODE>(w, wf32, (lig + j * L) * kVec<T>, cols, fill, out[j]);
}

template <typename T, int L, int NV, int MODE>
__global__ __launch_bounds__(kLnBlock) void k_ln_fwd(const T* __restrict__ x, int64_t xs,
                                                     const void* __restrict__ w,
                                                     const void* __restrict__ b, int wf32,
                                                     int64_t rows, int cols, float eps,
                                                     T* __restrict__ y, float2* __restrict__ stats) {
  constexpr int V = kVec<T>, G = kLnBlock / L;
  const int lig = threadIdx.x & (L - 1), grp = threadIdx.x / L;
  float wt[NV][V], bi[NV][V];
  ln_load_weight<T, L, NV, MODE>(w, wf32, cols, lig, 1.0f, wt);
  ln_load_weight<T, L, NV, MODE>(b, wf32, cols, lig, 0.0f, bi);
  const float inv = 1.0f / (float)cols;
  for (int64_t row = (int64_t)blockIdx.x * G + grp; row < rows; row += (int64_t)gridDim.x * G) {
    const T* xr = x + row * xs;
    float v[NV][V], s = 0.0f;
    RowVec<T, MODE> rv[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) rv[j].load(xr, (lig + j * L) * V, cols);
#pragma unroll
    for (int j = 0; j < NV; ++j) rv[j].get((lig + j * L) * V, cols, v[j]);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[j][i];
    const float m = group_sum<L>(s) * inv;
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[j][i] -= m;
        if ((lig + j * L) * V + i < cols) q += v[j][i] * v[j][i];
      }
    const float r = 1.0f / sqrtf(group_sum<L>(q) * inv + eps);
    T* yr = y + row * cols;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = v[j][i] * r * wt[j][i] + bi[j][i];
      store_row(yr + (lig + j * L) * V, cols - (lig + j * L) * V, o);
    }
    if (stats && lig == 0) stats[row] = make_float2(m, r);
  }
}

// Rows of more than kLnRegVecs vectors: a block a row, three passes over it.
template <typename T>
__global__ __launch_bounds__(kLnBlock) void k_ln_fwd_wide(const T* __restrict__ x, int64_t xs,
                                                          const void* __restrict__ w,
                                                          const void* __restrict__ b, int wf32,
                                                          int64_t rows, int cols, float eps,
                                                          T* __restrict__ y,
                                                          float2* __restrict__ stats) {
  constexpr int V = kVec<T>;
  __shared__ float tmp[kLnWaves];
  const float inv = 1.0f / (float)cols;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * xs;
    T* yr = y + row * cols;
    float s = 0.0f, v[V];
    for (int64_t c = (int64_t)threadIdx.x * V; c < cols; c += kLnBlock * V) {
      load_row(xr + c, (int)(cols - c), v);
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[i];
    }
    const float m = block_sum256(s, tmp) * inv;
    float q = 0.0f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < cols; c += kLnBlock * V) {
      load_row(xr + c, (int)(cols - c), v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = v[i] - m;
        if (c + i < cols) q += d * d;
      }
    }
    const float r = 1.0f / sqrtf(block_sum256(q, tmp) * inv + eps);
    for (int64_t c = (int64_t)threadIdx.x * V; c < cols; c += kLnBlock * V) {
      float wt[V], bi[V];
      const int n = (int)(cols - c);
      load_row(xr + c, n, v);
      ln_weight<T, kRowTail>(w, wf32, (int)c, cols, 1.0f, wt);
      ln_weight<T, kRowTail>(b, wf32, (int)c, cols, 0.0f, bi);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (v[i] - m) * r * wt[i] + bi[i];
      store_row(yr + c, n, v);
    }
    if (stats && threadIdx.x == 0) stats[row] = make_float2(m, r);
  }
}

// dy w, rounded: fused into g - mean g its rounding's rest would stay where they are equal (rows of one
// column have dx = 0).
__device__ __forceinline__ float ln_weighted(float dy, float w) {
#pragma clang fp contract(off)
  return dy * w;
}

// dx of the block's rows and its partial sums of dy xh and dy, part[block][2][cols].
template <typename T, int L, int NV, int MODE>
__global__ __launch_bounds__(kLnBlock) void k_ln_bwd(const T* __restrict__ x, int64_t xs,
                                                     const void* __restrict__ w, int wf32,
                                                     const T* __restrict__ dy, int64_t dys,
                                                     const float2* __restrict__ stats,
                                                     int64_t rows, int cols, T* __restrict__ dx,
                                                     float* __restrict__ part) {
  constexpr int V = kVec<T>, G = kLnBlock / L;
  __shared__ float red[2 * L * NV * V];
  const int lig = threadIdx.x & (L - 1), grp = threadIdx.x / L;
  float wt[NV][V], aw[NV][V] = {}, ab[NV][V] = {};
  ln_load_weight<T, L, NV, MODE>(w, wf32, cols, lig, 1.0f, wt);
  const float inv = 1.0f / (float)cols;
  for (int64_t row = (int64_t)blockIdx.x * G + grp; row < rows; row += (int64_t)gridDim.x * G) {
    const T* xr = x + row * xs;
    const T* gr = dy + row * dys;
    const float2 st = stats[row];
    float v[NV][V], g[NV][V];
    RowVec<T, MODE> rv[NV], rg[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      rv[j].load(xr, (lig + j * L) * V, cols);
      rg[j].load(gr, (lig + j * L) * V, cols);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      rv[j].get((lig + j * L) * V, cols, v[j]);
      rg[j].get((lig + j * L) * V, cols, g[j]);
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[j][i] = (v[j][i] - st.x) * st.y;   // past the row: g is zero there, so it adds nothing
        aw[j][i] += g[j][i] * v[j][i];
        ab[j][i] += g[j][i];
        g[j][i] = ln_weighted(g[j][i], wt[j][i]);
        s1 += g[j][i];
        s2 += g[j][i] * v[j][i];
      }
    if (dx) {
      s1 = group_sum<L>(s1) * inv;
      s2 = group_sum<L>(s2) * inv;
      T* dr = dx + row * cols;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float o[V];
        const int c = (lig + j * L) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = st.y * (g[j][i] - s1 - v[j][i] * s2);
        store_row(dr + c, cols - c, o);
      }
    }
  }
  if (!part) return;
  // the wave's row groups, then the waves, in order
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int o = L; o < 64; o *= 2) {
        aw[j][i] += __shfl_xor(aw[j][i], o, 64);
        ab[j][i] += __shfl_xor(ab[j][i], o, 64);
      }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int k = 0; k < kLnWaves; ++k) {
    if (wave == k && lane < L) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int c = (lig + j * L) * V + i;
          red[c] = (k ? red[c] : 0.0f) + aw[j][i];
          red[L * NV * V + c] = (k ? red[L * NV * V + c] : 0.0f) + ab[j][i];
        }
    }
    __syncthreads();
  }
  float* p = part + (int64_t)blockIdx.x * 2 * cols;
  for (int c = threadIdx.x; c < cols; c += kLnBlock) {
    p[c] = red[c];
    p[cols + c] = red[L * NV * V + c];
  }
}

template <typename T>
__global__ __launch_bounds__(kLnBlock) void k_ln_bwd_wide(const T* __restrict__ x, int64_t xs,
                                                          const void* __restrict__ w, int wf32,
                                                          const T* __restrict__ dy, int64_t dys,
                                                          const float2* __restrict__ stats,
                                                          int64_t rows, int cols,
                                                          T* __restrict__ dx) {
  constexpr int V = kVec<T>;
  __shared__ float tmp[kLnWaves];
  const float inv = 1.0f / (float)cols;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * xs;
    const T* gr = dy + row * dys;
    T* dr = dx + row * cols;
    const float2 st = stats[row];
    float v[V], g[V], wt[V], s1 = 0.0f, s2 = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {
      for (int64_t c = (int64_t)threadIdx.x * V; c < cols; c += kLnBlock * V) {
        const int n = (int)(cols - c);
        load_row(xr + c, n, v);
        load_row(gr + c, n, g);
        ln_weight<T, kRowTail>(w, wf32, (int)c, cols, 1.0f, wt);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[i] = (v[i] - st.x) * st.y;
          g[i] = ln_weighted(g[i], wt[i]);
          if (pass == 0) {
            s1 += g[i];
            s2 += g[i] * v[i];
          } else {
            v[i] = st.y * (g[i] - s1 - v[i] * s2);
          }
        }
        if (pass) store_row(dr + c, n, v);
      }
      if (pass == 0) {
        s1 = block_sum256(s1, tmp) * inv;
        s2 = block_sum256(s2, tmp) * inv;
      }
    }
  }
}

// Wide rows' partial sums: block (strip of 256 vectors' columns, share of the rows).
template <typename T>
__global__ __launch_bounds__(kLnBlock) void k_ln_bwd_cols(const T* __restrict__ x, int64_t xs,
                                                          const T* __restrict__ dy, int64_t dys,
                                                          const float2* __restrict__ stats,
                                                          int64_t rows, int cols,
                                                          float* __restrict__ part) {
  constexpr int V = kVec<T>;
  const int64_t c = ((int64_t)blockIdx.x * kLnBlock + threadIdx.x) * V;
  if (c >= cols) return;
  const int n = (int)(cols - c);
  float aw[V] = {}, ab[V] = {}, v[V], g[V];
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float2 st = stats[row];
    load_row(x + row * xs + c, n, v);
    load_row(dy + row * dys + c, n, g);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      aw[i] += g[i] * ((v[i] - st.x) * st.y);
      ab[i] += g[i];
    }
  }
  float* p = part + (int64_t)blockIdx.y * 2 * cols + c;
  for (int i = 0; i < V && i < n; ++i) {
    p[i] = aw[i];
    p[cols + i] = ab[i];
  }
}

// dw, db = the partials' sums over the blocks: 16 columns a block, 16 threads a column, joined in
// thread order.
template <typename T>
__global__ __launch_bounds__(kLnBlock) void k_ln_join(const float* __restrict__ part, int nblk,
                                                      int cols, int wf32, void* dw, void* db) {
  __shared__ float red[16][17];
  const int64_t c = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
  const int t = threadIdx.x >> 4;
  float s = 0.0f;
  if (c < 2 * (int64_t)cols) {
#pragma unroll 8
    for (int k = t; k < nblk; k += 16) s += part[(int64_t)k * 2 * cols + c];
  }
  red[t][threadIdx.x & 15] = s;
  __syncthreads();
  if (t || c >= 2 * (int64_t)cols) return;
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; ++k) s += red[k][threadIdx.x];
  void* out = c < cols ? dw : db;
  const int64_t i = c < cols ? c : c - cols;
  if (!out) return;
  if (wf32)
    static_cast<float*>(out)[i] = s;
  else
    static_cast<T*>(out)[i] = (T)s;
}

// Blocks of `per` rows at a time: as many as there are rows for up to two a CU, from there on each takes
// kLnShare rows a lane group before another is added, so that weights are read (and partial sums
// left) once for several rows.
inline int64_t ln_blocks(int64_t rows, int64_t per, int64_t most) {
  const int64_t want = (rows + per - 1) / per;
  int64_t n = (want + kLnShare - 1) / kLnShare;
  n = n < 512 ? 512 : n;
  n = n < want ? n : want;
  return n < most ? n : most;
}

// Blocks of the backward over `rows` rows of `cols` values of `esize` bytes.
inline int ln_bwd_blocks(int64_t rows, int cols, int esize) {
  const int nvec = (int)(((int64_t)cols * esize + 15) / 16);
  if (rows <= 0) return 0;
  if (nvec <= kLnRegVecs) return (int)ln_blocks(rows, kLnBlock / row_lanes(nvec), kLnBwdBlocks);
  // wide rows: strips of 256 vectors' columns by shares of at least 16 rows
  const int64_t strips = (nvec + kLnBlock - 1) / kLnBlock, share = (rows + 15) / 16;
  const int64_t cap = strips < kLnBwdBlocks ? kLnBwdBlocks / strips : 1;
  return (int)(share < cap ? share : cap);
}

// f(lanes a row, vectors a lane, row mode) for rows of nvec vectors.
template <typename T, typename F>
inline int ln_by_width(int cols, int nvec, F&& f) {
  using std::integral_constant;
  return by_row_mode<T>(cols, [&](auto mode) {
#define TTS_LN(L, NV) return f(integral_constant<int, L>{}, integral_constant<int, NV>{}, mode)
    if constexpr (mode() != kRowTiny) {
      if (nvec > 128) TTS_LN(64, 4);
      if (nvec > 64) TTS_LN(64, 2);
      if (nvec > 32) TTS_LN(64, 1);
      if (nvec > 16) TTS_LN(32, 1);
      if (nvec > 8) TTS_LN(16, 1);
      if (nvec > 4) TTS_LN(8, 1);
      if (nvec > 2) TTS_LN(4, 1);
      if (nvec > 1) TTS_LN(2, 1);
    }
    TTS_LN(1, 1);
#undef TTS_LN
  });
}

}  // namespace tts

using namespace tts;

extern "C" {

int tts_layer_norm_fwd(const void* x, int64_t x_stride, const void* weight, const void* bias,
                       int64_t rows, int cols, float eps, int dtype, int w_dtype, void* y,
                       float* stats, hipStream_t stream) {
  if (rows < 0 || cols < 1 || (rows > 0 && (!x || !y))) return TTS_EINVAL;
  if (!elem_dtype_ok(dtype) || (w_dtype != dtype && w_dtype != TTS_F32)) return TTS_EDTYPE;
  if (rows == 0) return TTS_OK;
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int nvec = (cols - 1) / kVec<T> + 1, wf32 = w_dtype == TTS_F32;
    const T* xp = static_cast<const T*>(x);
    T* yp = static_cast<T*>(y);
    float2* st = reinterpret_cast<float2*>(stats);
    if (nvec > kLnRegVecs) {
      const int64_t nb = rows < kLnFwdBlocks ? rows : kLnFwdBlocks;
      k_ln_fwd_wide<T><<<(int)nb, kLnBlock, 0, stream>>>(xp, x_stride, weight, bias, wf32, rows,
                                                         cols, eps, yp, st);
      return launch_status();
    }
    return ln_by_width<T>(cols, nvec, [&](auto L, auto NV, auto mode) {
      const int64_t nb = ln_blocks(rows, kLnBlock / L(), kLnFwdBlocks);
      k_ln_fwd<T, L(), NV(), mode()><<<(int)nb, kLnBlock, 0, stream>>>(xp, x_stride, weight, bias, wf32,
                                                               rows, cols, eps, yp, st);
      return launch_status();
    });
  });
}

size_t tts_layer_norm_workspace_bytes(int64_t rows, int cols, int dtype) {
  if (rows < 0 || cols < 1 || !elem_dtype_ok(dtype)) return 0;
  return (size_t)ln_bwd_blocks(rows, cols, (int)elem_size(dtype)) * 2 * cols * sizeof(float);
}

int tts_layer_norm_bwd(const void* x, int64_t x_stride, const void* weight, const void* dy,
                       int64_t dy_stride, const float* stats, int64_t rows, int cols, int dtype,
                       int w_dtype, void* dx, void* dweight, void* dbias, void* workspace,
                       size_t workspace_bytes, hipStream_t stream) {
  if (rows < 0 || cols < 1 || (rows > 0 && (!x || !dy || !stats))) return TTS_EINVAL;
  if (!dx && !dweight && !dbias) return TTS_EINVAL;
  if (!elem_dtype_ok(dtype) || (w_dtype != dtype && w_dtype != TTS_F32)) return TTS_EDTYPE;
  const bool sums = dweight || dbias;
  const size_t need = sums ? tts_layer_norm_workspace_bytes(rows, cols, dtype) : 0;
  if (need && (!workspace || workspace_bytes < need)) return TTS_EWORKSPACE;
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int nvec = (cols - 1) / kVec<T> + 1, wf32 = w_dtype == TTS_F32;
    const int nb = ln_bwd_blocks(rows, cols, (int)sizeof(T));
    const T* xp = static_cast<const T*>(x);
    const T* gp = static_cast<const T*>(dy);
    const float2* st = reinterpret_cast<const float2*>(stats);
    T* dxp = static_cast<T*>(dx);
    float* part = sums ? static_cast<float*>(workspace) : nullptr;
    if (rows > 0 && nvec > kLnRegVecs) {
      const int64_t nr = rows < kLnFwdBlocks ? rows : kLnFwdBlocks;
      if (dx)
        k_ln_bwd_wide<T><<<(int)nr, kLnBlock, 0, stream>>>(xp, x_stride, weight, wf32, gp,
                                                           dy_stride, st, rows, cols, dxp);
      if (sums) {
        const dim3 g((nvec + kLnBlock - 1) / kLnBlock, nb);
        k_ln_bwd_cols<T><<<g, kLnBlock, 0, stream>>>(xp, x_stride, gp, dy_stride, st, rows, cols,
                                                     part);
      }
    } else if (rows > 0) {
      ln_by_width<T>(cols, nvec, [&](auto L, auto NV, auto mode) {
        k_ln_bwd<T, L(), NV(), mode()><<<nb, kLnBlock, 0, stream>>>(xp, x_stride, weight, wf32, gp,
                                                            dy_stride, st, rows, cols, dxp, part);
        return 0;
      });
    }
    if (sums)
      k_ln_join<T><<<(int)((2 * (int64_t)cols + 15) / 16), kLnBlock, 0, stream>>>(
          part, nb, cols, wf32, dweight, dbias);
    return launch_status();
  });
}

}  // extern "C"
