// What the prologue's forward and backward kernels share: rows of 8 values per
// lane, and the exchange with the rotation partner's lane.
#pragma once

#include "lanes.hpp"

namespace inl {

namespace {

__device__ __forceinline__ float round_bf16(float v) { return (float)(bf16)v; }

template <typename TI>
__device__ __forceinline__ void load8(const char* p, float (&v)[8]) {
  if constexpr (sizeof(TI) == 2) {
    u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __builtin_bit_cast(float, w[j] << 16);
      v[2 * j + 1] = __builtin_bit_cast(float, w[j] & 0xffff0000u);
    }
  } else {
    f32x4 a = *reinterpret_cast<const f32x4*>(p);
    f32x4 b = *reinterpret_cast<const f32x4*>(p + 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
  }
}

// A lane's 8 input values kept as loaded (bf16: one 16-byte vector, f32:
// two) until the head step that uses them, so that the HB heads in flight
// cost half the registers in bf16.
struct Raw8 {
  u32x4 a, b;
};
template <typename TI>
__device__ __forceinline__ void load_raw(const char* p, Raw8& r) {
  r.a = *reinterpret_cast<const u32x4*>(p);
  if constexpr (sizeof(TI) != 2) r.b = *reinterpret_cast<const u32x4*>(p + 16);
}
template <typename TI>
__device__ __forceinline__ void unpack8(const Raw8& r, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t a = r.a[j];
    if constexpr (sizeof(TI) == 2) {
      v[2 * j] = __builtin_bit_cast(float, a << 16);
      v[2 * j + 1] = __builtin_bit_cast(float, a & 0xffff0000u);
    } else {
      const uint32_t b = r.b[j];
      v[j] = __builtin_bit_cast(float, a);
      v[4 + j] = __builtin_bit_cast(float, b);
    }
  }
}

template <typename TO>
__device__ __forceinline__ void store8(char* p, const float (&v)[8]) {
  if constexpr (sizeof(TO) == 2) {
    bf16x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (bf16)v[j];
    *reinterpret_cast<bf16x8*>(p) = o;
  } else {
    f32x4 a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
    *reinterpret_cast<f32x4*>(p) = a;
    *reinterpret_cast<f32x4*>(p + 16) = b;
  }
}

// out[e] = in[e] of lane (lane ^ m), for m a power of two below 64
// (uniform): one switch for the 8 values. Called with every lane of the
// wave active (a DPP read of a lane outside exec returns 0).
__device__ __forceinline__ void xor_lanes8(const float (&in)[8], float (&out)[8], int m, int lane) {
  switch (m) {
    case 1:
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = dpp<0xB1>(in[e]);      // quad_perm [1, 0, 3, 2]
      break;
    case 2:
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = dpp<0x4E>(in[e]);      // quad_perm [2, 3, 0, 1]
      break;
    case 4: {
      const bool hi = lane & 4;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float down = dpp<0x114>(in[e]);   // row_shr:4: lane i - 4
        const float up = dpp<0x104>(in[e]);     // row_shl:4: lane i + 4
        out[e] = hi ? down : up;
      }
      break;
    }
    case 8:
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = dpp<0x128>(in[e]);     // row_ror:8
      break;
    case 16: {
      const bool odd = lane & 16;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float a = in[e], b = in[e];   // a: rows (0, 0, 2, 2), b: rows (1, 1, 3, 3)
        asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
        out[e] = odd ? a : b;
      }
      break;
    }
    default: {
      const bool upper = lane & 32;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float a = in[e], b = in[e];   // a: halves (0, 0), b: halves (1, 1)
        asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
        out[e] = upper ? a : b;
      }
    }
  }
}

}  // namespace

// Checks of inl_norm_rope_desc that the forward and the backward have in
// common: types, head_dim, the rotation and its tables.
int norm_rope_check(const inl_norm_rope_desc* d, const int32_t* rows, const float* cos, const float* sin,
                    const float* cos2, const float* sin2);

}  // namespace inl
