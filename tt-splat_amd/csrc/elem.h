// Element types of the token operators (attention, layer norm, embedding): 32-bit, half and
// bfloat16 values in memory, 32-bit values in registers, 16 bytes a lane and load.
#pragma once

#include <string.h>

#include <type_traits>

#include "tts_common.h"

namespace tts {

using bf16 = __bf16;
using f16 = _Float16;

// Elements of one 16-byte vector.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// 16 bytes at any element's address: rows of odd sizes start at addresses that are multiples of
// the element only, and global loads and stores of gfx950 take those (one instruction each).
template <typename T>
struct Pack {
  T v[kVec<T>];
};
template <typename T>
__device__ __forceinline__ Pack<T> load_pack(const T* p) {
  Pack<T> r;
  memcpy(&r, p, 16);
  return r;
}
// How a row of `cols` values divides into vectors: evenly, with a tail, or shorter than one.
enum RowMode { kRowEven, kRowTail, kRowTiny };
template <typename T>
inline RowMode row_mode(int cols) {
  return cols % kVec<T> == 0 ? kRowEven : cols < kVec<T> ? kRowTiny : kRowTail;
}
// f(integral_constant) by the row's mode.
template <typename T, typename F>
inline int by_row_mode(int cols, F&& f) {
  switch (row_mode<T>(cols)) {
    case kRowEven: return f(std::integral_constant<int, kRowEven>{});
    case kRowTail: return f(std::integral_constant<int, kRowTail>{});
    default: return f(std::integral_constant<int, kRowTiny>{});
  }
}

// Values [c, c + kVec) of a row of `cols`.  load() is one unconditional 16-byte load (tiny rows aside),
// so that several are in flight at once: a branch with a conversion in it waits for each.  A tail's
// vector is read so that it ends with the row, one past the row from the row's start; get() gives
// its values as floats, shifted to their places, zeros past the row.
template <typename T, int MODE>
struct RowVec {
  static constexpr int V = kVec<T>;
  Pack<T> r;
  __device__ __forceinline__ void load(const T* row, int c, int cols) {
    if constexpr (MODE == kRowTiny) {
#pragma unroll
      for (int i = 0; i < V; ++i) r.v[i] = c + i < cols ? row[c + i] : (T)0.0f;
    } else {
      r = load_pack(row + (c + V <= cols ? c : MODE == kRowTail ? cols - V : 0));
    }
  }
  __device__ __forceinline__ void get(int c, int cols, float* out) const {
    const int n = cols - c;
    if constexpr (MODE == kRowTail) {
      const int s = n > 0 && n < V ? V - n : 0;
      uint32_t w[4];
      memcpy(w, &r, 16);
      constexpr int kTop = sizeof(T) == 2 ? 4 : 2;   // elements of two words
      if (s & kTop) {
        w[0] = w[2];
        w[1] = w[3];
      }
      if (s & (kTop / 2)) {
        w[0] = w[1];
        w[1] = w[2];
        w[2] = w[3];
      }
      if (sizeof(T) == 2 && (s & 1)) {
        w[0] = w[0] >> 16 | w[1] << 16;
        w[1] = w[1] >> 16 | w[2] << 16;
        w[2] = w[2] >> 16 | w[3] << 16;
        w[3] >>= 16;
      }
      Pack<T> q;
      memcpy(&q, w, 16);
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = i < n ? (float)q.v[i] : 0.0f;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = n > 0 ? (float)r.v[i] : 0.0f;
    }
  }
};
// The first n values at p as floats, zeros behind (joins of partial sums; n >= 1).
template <typename T>
__device__ __forceinline__ void load_row(const T* p, int n, float* out) {
  Pack<T> r;
  if (n >= kVec<T>) {
    r = load_pack(p);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) r.v[i] = i < n ? p[i] : (T)0.0f;
  }
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) out[i] = (float)r.v[i];
}
template <typename T>
__device__ __forceinline__ void store_row(T* p, int n, const float* in) {
  if (n >= kVec<T>) {
    Pack<T> r;
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) r.v[i] = (T)in[i];
    memcpy(p, &r, 16);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (i < n) p[i] = (T)in[i];
  }
}

// The two halves of a wave exchanged: {own lower half in both halves, own upper half in both}.
__device__ __forceinline__ float2 swap_halves(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return make_float2(__builtin_bit_cast(float, (uint32_t)r[0]),
                     __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float2 swap_rows16(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return make_float2(__builtin_bit_cast(float, (uint32_t)r[0]),
                     __builtin_bit_cast(float, (uint32_t)r[1]));
}

// Sum over groups of L consecutive lanes (a power of two), the same in each lane of the group: DPP
// moves inside 16 lanes, lane swaps past that.  All lanes of a group must call together.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (L >= 2) v = dpp_add<0xB1, 0xf>(v);   // quad_perm 1,0,3,2
  if constexpr (L >= 4) v = dpp_add<0x4E, 0xf>(v);   // quad_perm 2,3,0,1
  if constexpr (L >= 8) v = dpp_add<0x141, 0xf>(v);  // row_half_mirror: quads are uniform by now
  if constexpr (L >= 16) v = dpp_add<0x140, 0xf>(v); // row_mirror
  if constexpr (L >= 32) {
    const float2 s = swap_rows16(v);
    v = s.x + s.y;
  }
  if constexpr (L >= 64) {
    const float2 s = swap_halves(v);
    v = s.x + s.y;
  }
  return v;
}

inline bool elem_dtype_ok(int dtype) {
  return dtype == TTS_F32 || dtype == TTS_F16 || dtype == TTS_BF16;
}
inline size_t elem_size(int dtype) { return dtype == TTS_F32 ? 4 : 2; }

// f(float{} | f16{} | bf16{}) by the type code.
template <typename F>
inline int by_dtype(int dtype, F&& f) {
  switch (dtype) {
    case TTS_F32: return f(float{});
    case TTS_F16: return f(f16{});
    case TTS_BF16: return f(bf16{});
    default: return TTS_EDTYPE;
  }
}

// Lanes a row: the smallest power of two that covers its vectors, 64 at most.
inline int row_lanes(int nvec) {
  int l = 1;
  while (l < nvec && l < 64) l *= 2;
  return l;
}

}  // namespace tts
