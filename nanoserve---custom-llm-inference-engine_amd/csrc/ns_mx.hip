// The layer operators around attention and logits for gfx950: the root-mean-square norm of hidden rows with the
// residual's addition, the gated activation, MX quantisation in their epilogues and by itself, and the products of MX
// rows with 4-bit weights (ns_mx_linear.h).

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "ns_mx.h"
#include "ns_mx_linear.h"

namespace {

using namespace ns_mx;

thread_local char g_err[512];

int fail(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
int fail(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return 1;
}

int64_t padded(int64_t cols) { return (cols + NS_MX_ROW_ALIGN - 1) / NS_MX_ROW_ALIGN * NS_MX_ROW_ALIGN; }

// ---- rows of 8 values a thread ------------------------------------------------------------------------------

template <typename T> __device__ __forceinline__ void load8(const void* base, int64_t at, int left, float (&v)[8]) {
  load_words<T>(base, at, left).get(v);
}

// ---- MX codes -------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t quad_max(uint32_t x) {   // over the four lanes of a quad
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true));
  return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true));
}

// Values 8 t .. 8 t + 7 of a row by lane t: a quad of lanes holds a block.  The magnitudes are compared as bits, which
// orders NaN above infinity above the finite ones.  With x = 2^(b - 127) <= max < 2x the scale byte is s = b - emax and the
// factor 2^(127 - s) multiplies exactly (what it takes below the least normal float is far below the least code); the
// conversions round to nearest even, and the 8-bit one, which makes NaN of what is too large, gets at most 448.
template <int FORMAT> __device__ __forceinline__ void store_codes(const ns_mx_rows& to, int64_t row, int chunk, const float (&v)[8]) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
  most = quad_max(most);
  const bool fine = most < 0x7f800000u;
  const int s = max((int)(most >> 23) - (FORMAT == NS_MX_FP4 ? 2 : 8), 0);
  const float by = __uint_as_float((uint32_t)(254 - s) << 23);
  unsigned char* codes = static_cast<unsigned char*>(to.codes) + row * to.stride_codes;
  if constexpr (FORMAT == NS_MX_FP4) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0] * by, v[1] * by, 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2] * by, v[3] * by, 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4] * by, v[5] * by, 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6] * by, v[7] * by, 1.0f, 3);
    *reinterpret_cast<uint32_t*>(codes + 4 * chunk) = fine ? w : 0u;
  } else {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = __builtin_amdgcn_fmed3f(v[i] * by, -448.0f, 448.0f);
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    *reinterpret_cast<u32x2*>(codes + 8 * chunk) = fine ? u32x2{(uint32_t)lo, (uint32_t)hi} : u32x2{0u, 0u};
  }
  if ((threadIdx.x & 3) == 0) to.scales[row * to.stride_scales + (chunk >> 2)] = fine ? (uint8_t)s : (uint8_t)255;
}

template <typename T>
__device__ __forceinline__ void store_row8(const ns_mx_rows& mx, void* out, int64_t at, int64_t row, int chunk, int left,
                                           const float (&v)[8]) {
  if (mx.format == NS_MX_FP8) store_codes<NS_MX_FP8>(mx, row, chunk, v);
  else if (mx.format == NS_MX_FP4) store_codes<NS_MX_FP4>(mx, row, chunk, v);
  else if (left > 0) store8<T>(out, at + 8 * chunk, left, v);
}

// ---- norm -----------------------------------------------------------------------------------------------------

// n / d for 32-bit n by a multiplication (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994)
struct Divide {
  uint32_t m = 0, shift1 = 0, shift2 = 0;
  Divide() = default;
  explicit Divide(uint32_t d) {
    uint32_t l = 0;
    while (((uint64_t)1 << l) < d) ++l;
    m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - d)) / d + 1);
    shift1 = l < 1 ? l : 1;
    shift2 = l < 1 ? 0 : l - 1;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    const uint32_t t = __umulhi(m, n);
    return (t + ((n - t) >> shift1)) >> shift2;
  }
};

// A row by a group of `group` threads (a power of two up to 64: several rows to a workgroup; else the whole workgroup).
// Thread t takes the row's values 8 (c group + t) .. + 7 for c < CH and keeps them, as they were rounded to the type,
// until the row's sum is known, so memory is read once; CH = 0 reads a row of any width a second time.  The squares are
// added in float64: a float32's square neither overflows nor vanishes there.
// Bound by memory: 8192 x 4096 bfloat16 rows with residual and sum to 8-bit MX rows move 236 MB in 45 us, 5.2 TB/s, a large
// copy's rate; 4096 rows of 40 float16 heads of 128, 84 MB in 19 us, 17.6 one after another.  One row of 4096 takes 3.2 us.
// Float32 rows of 32 values a thread keep ten registers in scratch (a workgroup of 1024 threads has 128 for each): 8192 x 8192 to
// float32 take 111 us, 4.8 TB/s, 8192 x 4096 by 16 values 48, 5.6.
template <typename T, int CH>
__global__ __launch_bounds__(1024) void norm_kernel(ns_mx_norm_args a, int group, int width, double one_over_cols, Divide by_heads) {
  __shared__ double s_part[16];
  const int t = threadIdx.x & (group - 1 | -(int)(group > 64)), lane = threadIdx.x & 63;
  const int64_t i = group > 64 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (blockDim.x / group) + threadIdx.x / group;
  const bool there = i < a.n * a.heads;
  int64_t row = there ? i : 0;
  int head = 0;
  if (a.heads > 1) {
    const uint32_t q = by_heads((uint32_t)row);
    head = (int)((uint32_t)row - q * (uint32_t)a.heads);
    row = q;
  }
  int64_t from = row;
  if (a.rows != nullptr) from = a.rows[row];
  const bool valid = from >= 0 && from < a.n_x;
  if (!valid) from = 0;
  const int64_t x_at = from * a.stride_x + head * a.stride_x_head;
  const int64_t r_at = from * a.stride_residual + head * a.stride_residual_head;
  const int64_t s_at = row * a.stride_sum + head * a.stride_sum_head;
  const int64_t o_at = row * a.stride_out + head * a.stride_out_head;
  const auto load = [&](int chunk) {
    const int left = there ? a.cols - 8 * chunk : 0;
    Words<T> h = load_words<T>(a.x, x_at + 8 * chunk, left);
    if (a.residual != nullptr || !valid) {
      float v[8], r[8];
      h.get(v);
      if (a.residual != nullptr) {
        load_words<T>(a.residual, r_at + 8 * chunk, left).get(r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
      }
      if (!valid) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? __uint_as_float(0x7fc00000u) : 0.0f;
      }
      h.put(v);
    }
    return h;
  };
  const auto keep_sum = [&](int chunk, const Words<T>& h) {
    const int left = there ? a.cols - 8 * chunk : 0;
    if (a.sum != nullptr && left > 0) store_words<T>(a.sum, s_at + 8 * chunk, left, h);
  };
  const auto put = [&](int chunk, const Words<T>& h, double root, float by) {
    float v[8], w[8];
    const int left = a.cols - 8 * chunk;
    if (a.weight_dtype == NS_MX_F32) load8<float>(a.weight, 8 * chunk, left, w);
    else load8<T>(a.weight, 8 * chunk, left, w);
    h.get(v);
    if (by != 0.0f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * by * w[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (float)((double)v[e] * root) * w[e];
    }
    if (left < 8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < left ? v[e] : 0.0f;
    }
    store_row8<T>(a.out_mx, a.out, o_at, row, chunk, left, v);
  };
  // the row's sum of what its threads have
  const auto total = [&](double square) {
    for (int o = 1; o < min(group, 64); o <<= 1) square += __shfl_xor(square, o);
    if (group > 64) {
      if (lane == 0) s_part[threadIdx.x >> 6] = square;
      __syncthreads();
      square = 0.0;
      for (int w = 0; w < (int)(blockDim.x >> 6); ++w) square += s_part[w];
    }
    return square;
  };
  const auto add_squares = [](const Words<T>& h, double square) {
    float v[8];
    h.get(v);
#pragma unroll
    for (int e = 0; e < 8; ++e) square = fma((double)v[e], (double)v[e], square);
    return square;
  };
  // a factor that float32 holds badly or not at all (rows near its ends, eps of 0) is kept in float64, by is 0
  const auto factor = [&](double square, double& root) {
    const double mean = fma(square, one_over_cols, (double)a.eps);
    root = __builtin_amdgcn_rsq(mean);   // right to 2^-26 or better; one step of Newton's doubles that
    if (mean > 0.0 && mean < (double)INFINITY) root = root * fma(-0.5 * mean * root, root, 1.5);
    return root > 0x1p-120 && root < 0x1p120 ? (float)root : 0.0f;
  };
  double root;
  if constexpr (CH > 0) {
    Words<T> h[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) h[c] = load(c * group + t);
    double square = 0.0;
    if constexpr (sizeof(T) == 2) {
      // A 16-bit value's square is exact in float32, so a pair's sum is rounded once; only the pairs' sums are float64's, whose
      // additions of every value alone took 6 of 55 us (8192 x 4096).  A row whose squares leave float32 is added up again.
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float v[8];
        h[c].get(v);
#pragma unroll
        for (int e = 0; e < 8; e += 2) square += (double)fmaf(v[e], v[e], v[e + 1] * v[e + 1]);
        keep_sum(c * group + t, h[c]);
      }
      square = total(square);
      if (!(square > 0x1p-90 && square < 0x1p120)) {
        if (group > 64) __syncthreads();
        square = 0.0;
#pragma unroll
        for (int c = 0; c < CH; ++c) square = add_squares(h[c], square);
        square = total(square);
      }
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        square = add_squares(h[c], square);
        keep_sum(c * group + t, h[c]);
      }
      square = total(square);
    }
    const float by = factor(square, root);
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (there && 8 * (c * group + t) < width) put(c * group + t, h[c], root, by);
  } else {
    double square = 0.0;
    for (int chunk = t; 8 * chunk < a.cols; chunk += group) {
      const Words<T> h = load(chunk);
      square = add_squares(h, square);
      keep_sum(chunk, h);
    }
    const float by = factor(total(square), root);
    for (int chunk = t; 8 * chunk < width; chunk += group)
      put(chunk, a.sum != nullptr ? load_words<T>(a.sum, s_at + 8 * chunk, a.cols - 8 * chunk) : load(chunk), root, by);   // as this thread wrote it
  }
}

template <typename T> int launch_norm(const ns_mx_norm_args& a, hipStream_t stream) {
  const int width = a.out_mx.format ? (int)padded(a.cols) : a.cols;
  const int64_t rows = a.n * a.heads, need = (width + 7) / 8;
  int group = 4, threads = 256;
  void (*kernel)(ns_mx_norm_args, int, int, double, Divide) = norm_kernel<T, 1>;
  if (need <= 64) {
    while (group < need) group *= 2;
  } else {
    // 256 threads of up to 32 values fill the memory's queues best when there are rows enough (8192 x 4096: 46 us, 52 with 512
    // threads of 8); few rows are done sooner by more threads (one row: 0.5 us)
    const int64_t most = rows <= 1024 ? 1024 : 256;
    const int64_t per = need <= most ? 1 : need <= 2 * most ? 2 : need <= 4096 ? 4 : 0;
    group = per ? (int)(((need + per - 1) / per + 63) / 64 * 64) : 1024;
    threads = group;
    kernel = per == 1 ? norm_kernel<T, 1> : per == 2 ? norm_kernel<T, 2> : per == 4 ? norm_kernel<T, 4> : norm_kernel<T, 0>;
  }
  const int64_t per_block = group > 64 ? 1 : threads / group;
  const int64_t blocks = (rows + per_block - 1) / per_block;
  if (blocks >= (int64_t)1 << 31 || (a.heads > 1 && rows >= (int64_t)1 << 32)) return fail("too many rows");
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, stream, a, group, width, 1.0 / a.cols, Divide((uint32_t)a.heads));
  return 0;
}

// ---- gated activation, quantisation ---------------------------------------------------------------------------

constexpr int kGate = 256;

// exp(-x), 0 <= x <= 80: 2^t by the instruction (within 2 units of 2^-24), t = -x log2(e) rounded, times 1 + ln(2) (the rest of
// -x log2(e)), which rounds once more: 3 units.  The library's function takes three times the instructions, and 8 of them a
// value and a division bound the kernel (8192 x 8192 values: 85 us with them).
__device__ __forceinline__ float exp_minus(float x) {
  constexpr float kLog2e = 0x1.715476p+0f, kLog2eRest = 0x1.4ae0c0p-26f, kLn2 = 0x1.62e430p-1f;
  const float t = -x * kLog2e;
  const float rest = fmaf(-x, kLog2eRest, fmaf(-x, kLog2e, -t));
  const float p = __builtin_amdgcn_exp2f(t);
  return fmaf(p, rest * kLn2, p);
}

// A workgroup takes kGate / 2^shift rows by 2^shift threads' 8 values; blockIdx.y: the next ones along the rows.  A quad of
// lanes has an MX block, so no value passes through LDS.  Bound by memory: 4096 x 16384 bfloat16 gates to 8-bit rows
// move 338 MB in 63 us, 5.4 TB/s; 128256 x 2048 bfloat16 weights to 4-bit rows 665 MB in 119 us, 5.6 TB/s (a large copy: 5.2).
template <typename T, bool GATED>
__global__ __launch_bounds__(kGate) void gate_kernel(ns_mx_gate_args a, int shift, int width) {
  const int chunk = (int)(threadIdx.x & ((1u << shift) - 1)) + ((int)blockIdx.y << shift);
  const int64_t row = ((int64_t)blockIdx.x << (8 - shift)) + (threadIdx.x >> shift);
  if (row >= a.n || 8 * chunk >= width) return;
  int64_t from = row;
  if (a.rows != nullptr) from = a.rows[row];
  const bool valid = from >= 0 && from < a.n_x;
  if (!valid) from = 0;
  const int left = a.cols - 8 * chunk;
  float v[8];
  load8<T>(a.gate, from * a.stride_gate + 8 * chunk, left, v);
  if constexpr (GATED) {
    float u[8];
    load8<T>(a.up, from * a.stride_up + 8 * chunk, left, u);
    // far negative gates take the exponential that does not overflow, and keep their small products
    if constexpr (sizeof(T) == 4) {   // float32 results show each rounding: one exponential, one sum, one quotient, one product
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool far = v[e] < -80.0f;
        const float t = expf(far ? v[e] : -v[e]);
        v[e] = (far ? v[e] * t : v[e]) / (1.0f + t) * u[e];
      }
    } else {
      float most = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
      if (most <= 80.0f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float small = exp_minus(fabsf(v[e])), d = 1.0f + small;
          float over = __builtin_amdgcn_rcpf(d);             // within 2 units of 2^-24, one step takes it to 1
          over = fmaf(fmaf(-d, over, 1.0f), over, over);
          v[e] = v[e] * (v[e] < 0.0f ? small * over : over) * u[e];
        }
      } else {   // exponentials below the normal numbers, infinities, NaN
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float small = expf(-fabsf(v[e]));
          v[e] = v[e] * ((v[e] < 0.0f ? small : 1.0f) / (1.0f + small)) * u[e];
        }
      }
    }
  }
  if (!valid) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? __uint_as_float(0x7fc00000u) : 0.0f;
  }
  store_row8<T>(a.out_mx, a.out, row * a.stride_out, row, chunk, left, v);
}

template <typename T, bool GATED> int launch_gate(const ns_mx_gate_args& a, hipStream_t stream) {
  const int width = a.out_mx.format ? (int)padded(a.cols) : a.cols;
  const int need = (width + 7) / 8;
  int shift = 2;
  while (shift < 8 && (1 << shift) < need) ++shift;
  const int64_t blocks = (a.n + (kGate >> shift) - 1) / (kGate >> shift), along = (need + (1 << shift) - 1) >> shift;
  if (blocks >= (int64_t)1 << 31) return fail("too many rows");
  hipLaunchKernelGGL((gate_kernel<T, GATED>), dim3((unsigned)blocks, (unsigned)along), dim3(kGate), 0, stream, a, shift, width);
  return 0;
}

// ---- dequantisation -------------------------------------------------------------------------------------------

// With PAST the values are stored past the caches: results larger than these hold push out what is read.  Bound by memory: 128256
// x 2048 values of 4 bits to bfloat16, 665 MB in 122 us, 5.4 TB/s.
template <typename T, bool PAST>
__global__ __launch_bounds__(kGate) void values_kernel(ns_mx_rows r, int64_t n, int cols, void* out, int64_t stride_out, int shift) {
  const int chunk = (int)(threadIdx.x & ((1u << shift) - 1)) + ((int)blockIdx.y << shift);
  const int64_t row = ((int64_t)blockIdx.x << (8 - shift)) + (threadIdx.x >> shift);
  if (row >= n || 8 * chunk >= cols) return;
  const unsigned char* codes = static_cast<const unsigned char*>(r.codes) + row * r.stride_codes;
  const uint32_t s = r.scales[row * r.stride_scales + (chunk >> 2)];
  const float scale = __uint_as_float(s == 255 ? 0x7fc00000u : s == 0 ? 0x00400000u : s << 23);
  float v[8];
  f32x2 p[4];
  if (r.format == NS_MX_FP4) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + 4 * chunk);
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(codes + 8 * chunk);
    p[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false);
    p[1] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true);
    p[2] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false);
    p[3] = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = p[e >> 1][e & 1] * scale;
  store8<T, PAST>(out, row * stride_out + 8 * chunk, cols - 8 * chunk, v);
}

// ---- checks ---------------------------------------------------------------------------------------------------

bool is_float(int32_t t) { return t == NS_MX_F32 || t == NS_MX_BF16 || t == NS_MX_F16; }

// of n rows of k values (padded)
int check_mx(const ns_mx_rows& r, const char* name, int64_t n, int64_t k) {
  if (r.format != NS_MX_FP4 && r.format != NS_MX_FP8) return fail("%s: format must be NS_MX_FP4 or NS_MX_FP8 (got %d)", name, r.format);
  if (!r.codes || !r.scales) return fail("%s: a pointer is NULL", name);
  if ((uintptr_t)r.codes % 16 != 0 || r.stride_codes % 16 != 0 || r.stride_codes < 0)
    return fail("%s: codes must be 16-byte aligned, row by row", name);
  if ((uintptr_t)r.scales % 4 != 0 || r.stride_scales % 4 != 0 || r.stride_scales < 0)
    return fail("%s: scales must be 4-byte aligned, row by row", name);
  if (n > 1 && (r.stride_codes < (r.format == NS_MX_FP4 ? k / 2 : k) || r.stride_scales < k / 32))
    return fail("%s: strides must be as wide as the rows", name);
  return 0;
}

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("launch failed: %s", hipGetErrorString(e));
}

int check_out(const void* out, const ns_mx_rows& mx, int64_t n, int64_t cols) {
  if (!out == !mx.format) return fail("one of out and out_mx is needed");
  return mx.format ? check_mx(mx, "out_mx", n, padded(cols)) : 0;
}

}  // namespace

extern "C" {

int ns_mx_abi_version(void) { return NS_MX_ABI_VERSION; }

const char* ns_mx_last_error(void) { return g_err; }

int ns_mx_rms_norm(const ns_mx_norm_args* a, hipStream_t stream) {
  if (!a) return fail("args is NULL");
  if (!is_float(a->dtype)) return fail("dtype must be NS_MX_F32, _BF16 or _F16 (got %d)", a->dtype);
  if (a->weight_dtype != a->dtype && a->weight_dtype != NS_MX_F32) return fail("weight_dtype must be dtype or NS_MX_F32");
  if (a->n < 0 || a->n_x < 0 || a->heads < 1) return fail("n and n_x must be >= 0 and heads > 0");
  if (a->cols < 1 || a->cols > (1 << 30)) return fail("cols must lie in 1 .. 2^30 (got %d)", a->cols);
  if (!(a->eps >= 0.0f)) return fail("eps must be >= 0");
  if (a->n == 0) return 0;
  if (!a->x || !a->weight) return fail("a tensor pointer is NULL");
  if (!a->rows && a->n != a->n_x) return fail("without rows there are as many output rows as input rows");
  if (a->rows && a->n_x == 0) return fail("rows of an empty input");
  if (a->out_mx.format && a->heads != 1) return fail("MX rows are of whole rows: heads must be 1");
  if (check_out(a->out, a->out_mx, a->n, a->cols)) return 1;
  if (a->stride_x < 0 || a->stride_x_head < 0 || a->stride_residual < 0 || a->stride_residual_head < 0 || a->stride_sum < 0 ||
      a->stride_sum_head < 0 || a->stride_out < 0 || a->stride_out_head < 0)
    return fail("strides must not be negative");
  const int rc = a->dtype == NS_MX_F32 ? launch_norm<float>(*a, stream) : a->dtype == NS_MX_BF16 ? launch_norm<Bf16>(*a, stream)
                                                                                                  : launch_norm<F16>(*a, stream);
  return rc ? rc : launched();
}

static int check_gate(const ns_mx_gate_args* a) {
  if (!a) return fail("args is NULL");
  if (!is_float(a->dtype)) return fail("dtype must be NS_MX_F32, _BF16 or _F16 (got %d)", a->dtype);
  if (a->n < 0 || a->n_x < 0) return fail("n and n_x must be >= 0");
  if (a->cols < 1 || a->cols > (1 << 26)) return fail("cols must lie in 1 .. 2^26 (got %d)", a->cols);
  if (a->n == 0) return 0;
  if (!a->gate) return fail("a tensor pointer is NULL");
  if (!a->rows && a->n != a->n_x) return fail("without rows there are as many output rows as input rows");
  if (a->rows && a->n_x == 0) return fail("rows of an empty input");
  if (a->stride_gate < 0 || a->stride_up < 0 || a->stride_out < 0) return fail("strides must not be negative");
  return check_out(a->out, a->out_mx, a->n, a->cols);
}

int ns_mx_silu_mul(const ns_mx_gate_args* a, hipStream_t stream) {
  if (check_gate(a)) return 1;
  if (a->n == 0) return 0;
  if (!a->up) return fail("a tensor pointer is NULL");
  if (a->rows) return fail("ns_mx_silu_mul takes no rows");
  const int rc = a->dtype == NS_MX_F32    ? launch_gate<float, true>(*a, stream)
                 : a->dtype == NS_MX_BF16 ? launch_gate<Bf16, true>(*a, stream)
                                          : launch_gate<F16, true>(*a, stream);
  return rc ? rc : launched();
}

int ns_mx_quantize(const ns_mx_gate_args* a, hipStream_t stream) {
  if (check_gate(a)) return 1;
  if (a->up || a->out) return fail("ns_mx_quantize takes neither up nor out");
  if (a->n == 0) return 0;
  const int rc = a->dtype == NS_MX_F32    ? launch_gate<float, false>(*a, stream)
                 : a->dtype == NS_MX_BF16 ? launch_gate<Bf16, false>(*a, stream)
                                          : launch_gate<F16, false>(*a, stream);
  return rc ? rc : launched();
}

int ns_mx_dequantize(const ns_mx_rows* r, int64_t n, int32_t cols, void* out, int64_t stride_out, int32_t dtype, hipStream_t stream) {
  if (!r) return fail("rows is NULL");
  if (!is_float(dtype)) return fail("dtype must be NS_MX_F32, _BF16 or _F16 (got %d)", dtype);
  if (n < 0) return fail("n must be >= 0");
  if (cols < 1 || cols > (1 << 26)) return fail("cols must lie in 1 .. 2^26 (got %d)", cols);
  if (n > 1 && stride_out < cols) return fail("stride_out must be at least cols");
  if (n == 0) return 0;
  if (!out) return fail("out is NULL");
  if (check_mx(*r, "rows", n, padded(cols))) return 1;
  const int need = (cols + 7) / 8;
  int shift = 2;
  while (shift < 8 && (1 << shift) < need) ++shift;
  const int64_t blocks = (n + (kGate >> shift) - 1) / (kGate >> shift), along = (need + (1 << shift) - 1) >> shift;
  if (blocks >= (int64_t)1 << 31) return fail("too many rows");
  // more than the memory-side cache of 256 MB holds: 525 MB of values (128256 x 2048) take 101 us this way, 124 the other
  const bool past = n * cols * (dtype == NS_MX_F32 ? 4 : 2) > (int64_t)256 << 20;
  const auto kernel = dtype == NS_MX_F32    ? past ? values_kernel<float, true> : values_kernel<float, false>
                      : dtype == NS_MX_BF16 ? past ? values_kernel<Bf16, true> : values_kernel<Bf16, false>
                                            : past ? values_kernel<F16, true> : values_kernel<F16, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)along), dim3(kGate), 0, stream, *r, n, cols, out, stride_out, shift);
  return launched();
}

int ns_mx_linear(const ns_mx_linear_args* a, hipStream_t stream) {
  if (!a) return fail("args is NULL");
  if (!is_float(a->dtype)) return fail("dtype must be NS_MX_F32, _BF16 or _F16 (got %d)", a->dtype);
  if (a->m < 0 || a->n < 0 || a->m > INT32_MAX || a->n > INT32_MAX) return fail("m and n must lie in 0 .. 2^31 - 1");
  if (a->k < NS_MX_ROW_ALIGN || a->k % NS_MX_ROW_ALIGN != 0) return fail("k must be a positive multiple of %d (got %d)", NS_MX_ROW_ALIGN, a->k);
  if (a->m == 0 || a->n == 0) return 0;
  if (check_mx(a->x, "x", a->m, a->k) || check_mx(a->weight, "weight", a->n, a->k)) return 1;
  // a workgroup's 256 rows are addressed by 32 bits
  if ((a->m > 1 && (a->x.stride_codes >= 1 << 23 || a->x.stride_scales >= 1 << 23)) ||
      (a->n > 1 && (a->weight.stride_codes >= 1 << 23 || a->weight.stride_scales >= 1 << 23)))
    return fail("strides must be below 2^23 bytes");
  if (a->weight.format != NS_MX_FP4) return fail("weight: format must be NS_MX_FP4");
  if (!a->out) return fail("out is NULL");
  if (a->m > 1 && a->stride_out < a->n) return fail("stride_out must be at least n");
  if (const char* why = launch_linear(*a, stream)) return fail("%s", why);
  return launched();
}

}  // extern "C"
