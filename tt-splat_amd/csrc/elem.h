// Element types of the token operators (attention, layer norm, embedding): 32-bit, half and
// bfloat16 values in memory, 32-bit values in registers, 16 bytes a lane and load.
#pragma once

#include <string.h>

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
// Elements [0, n) of the vector at p as floats, zeros behind them.  The last vector of a row is
// read element by element: nothing past the row is touched.
template <typename T>
__device__ __forceinline__ void load_row(const T* p, int n, float* out) {
  if (n >= kVec<T>) {
    const Pack<T> r = load_pack(p);
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) out[i] = (float)r.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) out[i] = i < n ? (float)p[i] : 0.0f;
  }
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
