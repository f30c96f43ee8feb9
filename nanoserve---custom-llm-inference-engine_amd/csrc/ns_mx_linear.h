// Products of MX rows with the rows of a 4-bit MX weight, on gfx950's scaled matrix instruction.
//
//   out[i][j] = round( sum over 32-blocks b of 2^(sx[i][b] - 127) 2^(sw[j][b] - 127) sum_{c in b} x[i][c] w[j][c] )
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 16 rows of each side and 128 columns, the codes as they are stored and for each
// row and block of 32 its scale byte.  The weight is its first operand: a lane then holds four consecutive outputs of
// one token.  Lane l = 16 g + r serves row r: of 4-bit codes the 16 bytes of columns 32 g .. 32 g + 31; of 8-bit codes
// two pieces of 16, columns 16 g .. + 15 and 64 + 16 g .. + 15; and the scale of block g either way.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ns_mx.h"

namespace ns_mx {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct Bf16 {
  uint16_t bits;
};
struct F16 {
  uint16_t bits;
};

template <typename T> __device__ __forceinline__ float widen(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (__is_same(T, Bf16)) return __uint_as_float((uint32_t)x.bits << 16);
  else return (float)__builtin_bit_cast(_Float16, x.bits);
}
template <typename T> __device__ __forceinline__ void widen2(uint32_t w, float& a, float& b) {
  if constexpr (__is_same(T, Bf16)) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
  } else {
    const f16x2 h = __builtin_bit_cast(f16x2, w);
    a = (float)h[0];
    b = (float)h[1];
  }
}
// to nearest even
template <typename T> __device__ __forceinline__ uint32_t narrow2(float a, float b) {
  if constexpr (__is_same(T, Bf16)) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
}
template <typename T> __device__ __forceinline__ T narrow(float a) {
  if constexpr (sizeof(T) == 4) return a;
  else return T{(uint16_t)narrow2<T>(a, 0.0f)};
}
template <typename T> __device__ __forceinline__ float rounded(float a) { return widen<T>(narrow<T>(a)); }

// ---- one 16 x 16 tile a wave ------------------------------------------------------------------------------------

template <int XF> __device__ __forceinline__ f32x4 products(u32x4 w, const u32x4 (&x)[2], int sw, int sx, f32x4 c) {
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  if constexpr (XF == NS_MX_FP8) {
    const i32x8 b = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3], (int)x[1][0], (int)x[1][1], (int)x[1][2], (int)x[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, sw, 0, sx);
  } else {
    const i32x8 b = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, 0, sw, 0, sx);
  }
}

template <typename T, int XF> __global__ __launch_bounds__(256) void linear_kernel(ns_mx_linear_args a) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int64_t n0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16, m0 = (int64_t)blockIdx.y * 16;
  if (n0 >= a.n) return;
  // rows past the ends read the last one; nothing of theirs is stored
  const int64_t wr = min(n0 + r, a.n - 1), xr = min(m0 + r, a.m - 1);
  const unsigned char* wc = static_cast<const unsigned char*>(a.weight.codes) + wr * a.weight.stride_codes + 16 * g;
  const uint8_t* ws = a.weight.scales + wr * a.weight.stride_scales + g;
  const unsigned char* xc = static_cast<const unsigned char*>(a.x.codes) + xr * a.x.stride_codes + 16 * g;
  const uint8_t* xs = a.x.scales + xr * a.x.stride_scales + g;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int k = 0; k < a.k; k += 128) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(wc + k / 2);
    u32x4 x[2];
    if constexpr (XF == NS_MX_FP8) {
      x[0] = *reinterpret_cast<const u32x4*>(xc + k);
      x[1] = *reinterpret_cast<const u32x4*>(xc + k + 64);
    } else {
      x[0] = *reinterpret_cast<const u32x4*>(xc + k / 2);
    }
    acc = products<XF>(w, x, ws[k / 32], xs[k / 32], acc);
  }
  if (m0 + r >= a.m) return;
  T* out = static_cast<T*>(a.out) + (m0 + r) * a.stride_out + n0 + 4 * g;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n0 + 4 * g + e < a.n) out[e] = narrow<T>(acc[e]);
}

template <typename T, int XF> const char* launch_linear_t(const ns_mx_linear_args& a, hipStream_t stream) {
  if (a.m > 16 * 65535) return "m must be at most 1048560";
  hipLaunchKernelGGL((linear_kernel<T, XF>), dim3((unsigned)((a.n + 63) / 64), (unsigned)((a.m + 15) / 16)), dim3(256), 0, stream, a);
  return nullptr;
}
template <typename T> const char* launch_linear_x(const ns_mx_linear_args& a, hipStream_t stream) {
  return a.x.format == NS_MX_FP8 ? launch_linear_t<T, NS_MX_FP8>(a, stream) : launch_linear_t<T, NS_MX_FP4>(a, stream);
}
// NULL, or why the call is refused
inline const char* launch_linear(const ns_mx_linear_args& a, hipStream_t stream) {
  return a.dtype == NS_MX_F32 ? launch_linear_x<float>(a, stream) : a.dtype == NS_MX_BF16 ? launch_linear_x<Bf16>(a, stream)
                                                                                          : launch_linear_x<F16>(a, stream);
}

}  // namespace ns_mx
