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

template <typename T> __device__ __forceinline__ void store8(void* base, int64_t at, int left, const float (&v)[8]) {
  T* p = static_cast<T*>(base) + at;
  if (left >= 8) {
    if constexpr (sizeof(T) == 4) {
      typedef uint32_t words __attribute__((ext_vector_type(4), aligned(4)));
      words a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = __float_as_uint(v[i]);
        b[i] = __float_as_uint(v[4 + i]);
      }
      *reinterpret_cast<words*>(p) = a;
      *reinterpret_cast<words*>(p + 4) = b;
    } else {
      typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));
      words a;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = narrow2<T>(v[2 * i], v[2 * i + 1]);
      *reinterpret_cast<words*>(p) = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = narrow<T>(v[i]);
  }
}

// ---- operands ---------------------------------------------------------------------------------------------------

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

typedef __attribute__((address_space(3))) void lds_void;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}
// `rows` rows from row `first` on
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const void* base, int64_t first, int64_t stride, int rows, int width) {
  return rsrc(static_cast<const unsigned char*>(base) + first * stride, (uint32_t)((rows - 1) * stride + width));
}
__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t voff, int soff) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, soff, 0));
}
__device__ __forceinline__ int load1(__amdgpu_buffer_rsrc_t r, uint32_t voff, int soff) {
  return (int)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, (int)voff, soff, 0);
}
// One direct load: 16 (4) bytes a lane from the buffer at voff + soff, to LDS at dst + 16 (4) lane (dst the same for the wave).
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t r, unsigned char* dst, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)dst, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void load_lds4(__amdgpu_buffer_rsrc_t r, unsigned char* dst, uint32_t voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)dst, 4, voff, soff, 0, 0);
}

// ---- few rows: the weight streamed through registers ------------------------------------------------------------

// vmcnt(n) alone
#define NS_MX_VMCNT(n) (((n) & 15) | (7 << 4) | (15 << 8) | (((n) >> 4) << 14))

// A workgroup of eight waves computes 16 TM rows of x by 32 outputs for each of its 8 / KW waves side by side, and goes on
// to further outputs; KW waves share one set of outputs, their columns dealt out in groups of 512 (four stages of 128).
// The weight goes from memory into the operand registers of the one wave that uses it: a stage's registers are refilled
// with the wave's next group as soon as its products are issued, whatever output it is of, so that 8 KB stay in flight per
// wave.  x lies in LDS, in two halves of KS stages: where its columns fit they stay there and the waves run on their own;
// else the halves take turns, one filled by direct loads while the other is used, with a barrier for each.  Sums of KW
// waves meet in LDS and are added in the waves' order.
//
// LDS rows are the stage's codes of a row of x: 8 (8-bit) or 4 pieces of 16 bytes, piece c of row r at c ^ f(r), so that 16
// lanes that read one piece of 16 rows, and either 8 of them, meet every bank once: f = (r & 7) ^ (r >> 3 & 1) for 8
// pieces, (r >> 1 & 3) ^ (r >> 3 & 1) for 4.  The weight's rows go to the instruction in an order that leaves a lane with 8
// consecutive outputs: of a pair of its 16-row operands, row 8 a + 4 p + e is row 4 a + e of operand p.
template <int PIECES> __device__ __forceinline__ int x_swizzle(int row) {
  return PIECES == 8 ? (row & 7) ^ (row >> 3 & 1) : (row >> 1 & 3) ^ (row >> 3 & 1);
}

template <int XF, int TM, int KS> struct Stream {
  static constexpr int XP = XF == NS_MX_FP8 ? 8 : 4;
  static constexpr int XSTEP = 16 * TM * XP * 16;                  // bytes of a stage's codes
  static constexpr int XB = KS * XSTEP, SB = KS * 16 * TM * 4;     // of a half's codes and scales
  static constexpr int FILLS = XB / 1024 / 8;                      // 16-byte direct loads of a thread
  static_assert(FILLS * 8192 == XB, "tiling");
};

template <typename T, int XF, int TM, int KW, int KS>
__global__ __launch_bounds__(512, TM < 4 ? 4 : 2) void stream_kernel(const ns_mx_linear_args a, int blocks_n) {
  using C = Stream<XF, TM, KS>;
  constexpr int XP = C::XP, NW = 8 / KW, GROUPS = KS / 4;
  static_assert(GROUPS % KW == 0, "tiling");
  __shared__ __attribute__((aligned(16))) unsigned char s0[C::XB + C::SB], s1[C::XB + C::SB];
  __shared__ float sums[KW > 1 ? 8 * TM * 8 * 64 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
  const int kw = wave % KW, nw = wave / KW;
  const int64_t m0 = (int64_t)(blockIdx.x / blocks_n) * (16 * TM);
  const int mrows = (int)min((int64_t)(16 * TM), a.m - m0), xw = XF == NS_MX_FP8 ? a.k : a.k / 2;
  const __amdgpu_buffer_rsrc_t xr = rows_buffer(a.x.codes, m0, a.x.stride_codes, mrows, xw);
  const __amdgpu_buffer_rsrc_t xsr = rows_buffer(a.x.scales, m0, a.x.stride_scales, mrows, a.k / 32);
  const int nst = a.k / 128, ng = (nst + 3) / 4, nc = (nst + KS - 1) / KS;
  const bool resident = nc <= 2;

  const auto fill = [&](int c, unsigned char* to) {
    const int base = c * KS;
#pragma unroll
    for (int j = 0; j < C::FILLS; ++j) {
      const int at = (j * 8 + wave) * 64 + lane, step = at / (16 * TM * XP), row = at / XP % (16 * TM), p = at % XP;
      const int st = min(base + step, nst - 1);
      load_lds16(xr, to + (j * 8 + wave) * 1024,
                 (uint32_t)(row * a.x.stride_codes + st * (XP * 16) + 16 * (p ^ x_swizzle<XP>(row))), 0);
    }
    for (int j = wave; j < KS * TM / 4; j += 8) {
      const int at = j * 64 + lane, step = at / (16 * TM), row = at % (16 * TM), st = min(base + step, nst - 1);
      load_lds4(xsr, to + C::XB + j * 256, (uint32_t)(row * a.x.stride_scales + st * 4), 0);
    }
  };

  const int tiles = (int)((a.n + 31) / 32), step_tiles = blocks_n * NW;
  int tile = (int)(blockIdx.x % blocks_n) * NW + nw;
  uint32_t wo[2], wso[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int row = 8 * (r >> 2) + 4 * p + (r & 3);
    wo[p] = (uint32_t)(row * a.weight.stride_codes + 16 * g);
    wso[p] = (uint32_t)(row * a.weight.stride_scales);
  }
  u32x4 w[4][2], scale[2], next[2];
  __amdgpu_buffer_rsrc_t wr, wsr;
  const auto aim = [&](int t) {   // at a set of outputs; past the last: at nothing, which reads as zeros
    const int64_t n0 = (int64_t)t * 32;
    const int rows = t < tiles ? (int)min((int64_t)32, a.n - n0) : 0;
    wr = rsrc(static_cast<const unsigned char*>(a.weight.codes) + (rows ? n0 : 0) * a.weight.stride_codes,
              rows ? (uint32_t)((rows - 1) * a.weight.stride_codes + a.k / 2) : 0u);
    wsr = rsrc(a.weight.scales + (rows ? n0 : 0) * a.weight.stride_scales,
               rows ? (uint32_t)((rows - 1) * a.weight.stride_scales + a.k / 32) : 0u);
  };
  const auto load_stage = [&](int s, int q) {
#pragma unroll
    for (int p = 0; p < 2; ++p) w[s][p] = load16(wr, wo[p] + 64 * s, q * 256);
  };
  f32x4 acc[TM][2];
  const int xf = x_swizzle<XP>(r);
  const int x_at = r * (XP * 16) + 16 * (g ^ xf), x_at2 = r * (XP * 16) + 16 * ((4 + g) ^ xf);
  const int sx_at = C::XB + r * 4 + g;

  // the products of group q, and the loads of the group that this wave takes next
  const auto group = [&](int q, const unsigned char* from) {
    const bool here = q + KW < ng;
    const int then = here ? q + KW : kw;
    if (!here) aim(tile + step_tiles);
#pragma unroll
    for (int p = 0; p < 2; ++p) next[p] = load16(wsr, wso[p], then * 16);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (4 * q + s < nst) {
        const int st = (4 * q + s) % KS;
        const unsigned char *xs = from + st * C::XSTEP + x_at, *xs2 = from + st * C::XSTEP + x_at2, *sx = from + st * (16 * TM * 4) + sx_at;
        const int sw[2] = {(int)(scale[0][s] >> (8 * g)), (int)(scale[1][s] >> (8 * g))};
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          u32x4 x[2];
          x[0] = *reinterpret_cast<const u32x4*>(xs + i * (XP * 256));
          if constexpr (XP == 8) x[1] = *reinterpret_cast<const u32x4*>(xs2 + i * (XP * 256));
          const int f = sx[i * 64];
#pragma unroll
          for (int p = 0; p < 2; ++p) acc[i][p] = products<XF>(w[s][p], x, sw[p], f, acc[i][p]);
        }
      }
      load_stage(s, then);
    }
    scale[0] = next[0];
    scale[1] = next[1];
  };

  fill(0, s0);
  if (resident && nc > 1) fill(1, s1);
  aim(kw < ng ? tile : tiles);
  scale[0] = load16(wsr, wso[0], kw * 16);
  scale[1] = load16(wsr, wso[1], kw * 16);
#pragma unroll
  for (int s = 0; s < 4; ++s) load_stage(s, kw);
  bool started = true;    // whether a group's ten loads are newer than the last fill's
  int half = 0;
  const auto chunk = [&](int c, unsigned char* from, unsigned char* other, bool wait, bool more) {
    if (wait) {
      if (started) __builtin_amdgcn_s_waitcnt(NS_MX_VMCNT(10));
      else __builtin_amdgcn_s_waitcnt(NS_MX_VMCNT(0));
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
      if (more) {
        fill(c + 1 < nc ? c + 1 : 0, other);
        started = false;
      }
    }
#pragma unroll 1
    for (int j = 0; j < GROUPS / KW; ++j) {
      const int q = c * GROUPS + kw + KW * j;
      if (q < ng) {
        group(q, from);
        started = true;
      }
    }
  };
  const int rounds = (tiles - (tile - nw) + step_tiles - 1) / step_tiles;   // the same for every wave
  for (int round = 0; round < rounds; ++round, tile += step_tiles) {
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[i][0] = acc[i][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = 0; c < nc; ++c) {
      const bool wait = !resident || (round == 0 && c == 0), more = !resident && (c + 1 < nc || round + 1 < rounds);
      if (half == 0) chunk(c, s0, s1, wait, more);
      else chunk(c, s1, s0, wait, more);
      half = nc > 1 ? half ^ 1 : 0;
    }
    if (resident) half = 0;
    const int64_t col = (int64_t)tile * 32 + 8 * g, left = a.n - col;
    if constexpr (KW == 1) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int64_t row = m0 + 16 * i + r;
        const float v[8] = {acc[i][0][0], acc[i][0][1], acc[i][0][2], acc[i][0][3], acc[i][1][0], acc[i][1][1], acc[i][1][2], acc[i][1][3]};
        if (row < a.m && left > 0) store8<T>(a.out, row * a.stride_out + col, left < 8 ? (int)left : 8, v);
      }
    } else {
      float* mine = sums + wave * (TM * 8 * 64) + lane;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) mine[(i * 8 + e) * 64] = acc[i][e >> 2][e & 3];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
      for (int i = kw; i < TM; i += KW) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = 0.0f;
#pragma unroll
          for (int z = 0; z < KW; ++z) v[e] += sums[(nw * KW + z) * (TM * 8 * 64) + (i * 8 + e) * 64 + lane];
        }
        const int64_t row = m0 + 16 * i + r;
        if (row < a.m && left > 0) store8<T>(a.out, row * a.stride_out + col, left < 8 ? (int)left : 8, v);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
      __builtin_amdgcn_s_barrier();   // before the next round's sums
    }
  }
  __builtin_amdgcn_s_waitcnt(0);   // nothing may land in LDS after the workgroup ends
}

template <typename T, int XF, int TM, int KW, int KS>
const char* launch_stream(const ns_mx_linear_args& a, int per_cu, hipStream_t stream) {
  constexpr int NW = 8 / KW;
  const int64_t wanted = ((a.n + 31) / 32 + NW - 1) / NW, along = (a.m + 16 * TM - 1) / (16 * TM);
  const int64_t blocks_n = wanted < 256 * per_cu ? wanted : 256 * per_cu;
  hipLaunchKernelGGL((stream_kernel<T, XF, TM, KW, KS>), dim3((unsigned)(blocks_n * along)), dim3(512), 0, stream, a, (int)blocks_n);
  return nullptr;
}

// ---- tiles through LDS ------------------------------------------------------------------------------------------

// A workgroup computes BM rows of x by BN rows of the weight, its WM x WN waves 16 TI by 16 TJ each.  Stages of 128
// columns go to LDS by direct loads, two stages ahead, in a ring of three: at stage t a wave waits for its own share of
// stage t, the barrier makes everyone's visible and says that everyone is past stage t - 1, whose place stage t + 2 takes.
// The three places are three arrays and the loop is unrolled by three: the compiler sees that a stage's reads touch none
// that a direct load is filling, and waits for none of those.
//
// LDS rows are the stage's codes of a matrix row: 8 (8-bit) or 4 pieces of 16 bytes.  Piece c of row r lies at c ^ f(r), so
// that 16 lanes that read one piece of 16 rows, and either 8 of them, meet every bank once: f = (r & 7) ^ (r >> 3 & 1) for
// 8 pieces, and for the weight's 4 f = (r >> 3 & 3) ^ (r & 2).  The weight's rows go to the instruction in an order that leaves
// a lane with 8 consecutive outputs: of a pair of its 16-row operands, row 8 a + 4 p + e is row 4 a + e of operand p.
template <typename T, int XF, int BM, int BN, int WM, int WN>
struct Tile {
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int TI = BM / WM / 16, TJ = BN / WN / 16;
  static constexpr int XP = XF == NS_MX_FP8 ? 8 : 4;            // pieces of an x row in a stage
  static constexpr int XB = BM * XP * 16, WB = BN * 4 * 16;     // bytes of a stage
  static constexpr int XL = XB / 1024 / WAVES, WL = WB / 1024 / WAVES, SL = (BM + BN + THREADS - 1) / THREADS;
  static constexpr int SB = SL * THREADS * 4;                   // scales: 4 bytes of every row
  static constexpr int BYTES = XB + WB + SB;
  static_assert(XL * 1024 * WAVES == XB && WL * 1024 * WAVES == WB && TJ % 2 == 0 && BM % 64 == 0 && BN % 64 == 0, "tiling");
};

template <typename T, int XF, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void tile_kernel(const ns_mx_linear_args a) {
  using C = Tile<T, XF, BM, BN, WM, WN>;
  constexpr int TI = C::TI, TJ = C::TJ, XP = C::XP;
  __shared__ __attribute__((aligned(16))) unsigned char s0[C::BYTES], s1[C::BYTES], s2[C::BYTES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int nx = (int)((a.m + BM - 1) / BM);
  const int64_t m0 = (int64_t)(blockIdx.x % nx) * BM, n0 = (int64_t)(blockIdx.x / nx) * BN;
  const int mrows = (int)min((int64_t)BM, a.m - m0), nrows = (int)min((int64_t)BN, a.n - n0);
  // rows past the ends lie behind the buffers' ends and read as zeros
  const __amdgpu_buffer_rsrc_t xr = rows_buffer(a.x.codes, m0, a.x.stride_codes, mrows, XF == NS_MX_FP8 ? a.k : a.k / 2);
  const __amdgpu_buffer_rsrc_t wr = rows_buffer(a.weight.codes, n0, a.weight.stride_codes, nrows, a.k / 2);
  const __amdgpu_buffer_rsrc_t xsr = rows_buffer(a.x.scales, m0, a.x.stride_scales, mrows, a.k / 32);
  const __amdgpu_buffer_rsrc_t wsr = rows_buffer(a.weight.scales, n0, a.weight.stride_scales, nrows, a.k / 32);
  uint32_t xo[C::XL], wo[C::WL], so[C::SL];
#pragma unroll
  for (int j = 0; j < C::XL; ++j) {
    const int at = j * C::THREADS + tid, row = at / XP, c = at % XP;
    const int f = XP == 8 ? (row & 7) ^ (row >> 3 & 1) : (row >> 1 & 3) ^ (row >> 3 & 1);
    xo[j] = (uint32_t)(row * a.x.stride_codes + 16 * (c ^ f));
  }
#pragma unroll
  for (int j = 0; j < C::WL; ++j) {
    const int at = j * C::THREADS + tid, row = at / 4, c = at % 4;
    wo[j] = (uint32_t)(row * a.weight.stride_codes + 16 * (c ^ ((row >> 3 & 3) ^ (row & 2))));
  }
#pragma unroll
  for (int j = 0; j < C::SL; ++j) {
    const int row = j * C::THREADS + tid;
    so[j] = (uint32_t)(row < BM ? row * a.x.stride_scales : row < BM + BN ? (row - BM) * a.weight.stride_scales : 0);
  }
  const int nst = a.k / 128;
  const auto load = [&](int stage, unsigned char* to) {   // stages past the last are it again
    const int st = stage < nst ? stage : nst - 1;
#pragma unroll
    for (int j = 0; j < C::XL; ++j)
      load_lds16(xr, to + (j * C::WAVES + wave) * 1024, xo[j], st * XP * 16);
#pragma unroll
    for (int j = 0; j < C::WL; ++j)
      load_lds16(wr, to + C::XB + (j * C::WAVES + wave) * 1024, wo[j], st * 64);
#pragma unroll
    for (int j = 0; j < C::SL; ++j)
      load_lds4((j * C::WAVES + wave) * 64 < BM ? xsr : wsr, to + C::XB + C::WB + (j * C::WAVES + wave) * 256, so[j], st * 4);
  };
  const int wm = wave % WM, wn = wave / WM;
  const int x_row = wm * (16 * TI) + r;                              // of operand 0; operand i: 16 i more
  const int w_row = wn * (16 * TJ) + 8 * (r >> 2) + (r & 3);         // of operand 0; operand 2 q + p: 32 q + 4 p more
  const int xf = XP == 8 ? (x_row & 7) ^ (x_row >> 3 & 1) : (x_row >> 1 & 3) ^ (x_row >> 3 & 1);
  const int wf = (w_row >> 3 & 3) ^ (w_row & 2);
  const int x_at = x_row * (XP * 16) + 16 * (g ^ xf), x_at2 = x_row * (XP * 16) + 16 * ((4 + g) ^ xf);
  const int w_at = C::XB + w_row * 64 + 16 * (g ^ wf);
  const int sx_at = C::XB + C::WB + x_row * 4 + g, sw_at = C::XB + C::WB + (BM + w_row) * 4 + g;
  f32x4 acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int LOADS = C::XL + C::WL + C::SL;
  constexpr int WAIT = (LOADS & 15) | (7 << 4) | (15 << 8) | ((LOADS >> 4) << 14);   // vmcnt(LOADS) alone
  const auto stage = [&](int st, const unsigned char* from, unsigned char* to) {
    __builtin_amdgcn_s_waitcnt(WAIT);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    load(st + 2, to);
    __builtin_amdgcn_sched_barrier(0);
    const unsigned char *xs = from + x_at, *xs2 = from + x_at2, *ws = from + w_at, *sx0 = from + sx_at, *sw0 = from + sw_at;
    u32x4 w[TJ];
    int sw[TJ];
#pragma unroll
    for (int j = 0; j < TJ; ++j) {   // f is the same for all: 32 and 4 leave its bits alone
      const int row = 32 * (j >> 1) + 4 * (j & 1);
      w[j] = *reinterpret_cast<const u32x4*>(ws + row * 64);
      sw[j] = sw0[row * 4];
    }
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      u32x4 x[2];
      x[0] = *reinterpret_cast<const u32x4*>(xs + i * (XP * 256));
      if constexpr (XP == 8) x[1] = *reinterpret_cast<const u32x4*>(xs2 + i * (XP * 256));
      const int sx = sx0[i * 64];
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[i][j] = products<XF>(w[j], x, sw[j], sx, acc[i][j]);
    }
  };
  load(0, s0);
  load(1, s1);
  int st = 0;
  for (; st + 3 <= nst; st += 3) {
    stage(st, s0, s2);
    stage(st + 1, s1, s0);
    stage(st + 2, s2, s1);
  }
  if (st < nst) stage(st, s0, s2);
  if (st + 1 < nst) stage(st + 1, s1, s0);
  __builtin_amdgcn_s_waitcnt(0);   // nothing may land in LDS after the workgroup ends
  // operand pair q, token r: outputs 32 q + 8 g .. + 7
#pragma unroll
  for (int i = 0; i < TI; ++i) {
    const int64_t row = m0 + x_row + 16 * i;
    if (row >= a.m) continue;
#pragma unroll
    for (int q = 0; q < TJ / 2; ++q) {
      const int64_t col = n0 + wn * (16 * TJ) + 32 * q + 8 * g;
      const float v[8] = {acc[i][2 * q][0], acc[i][2 * q][1], acc[i][2 * q][2], acc[i][2 * q][3],
                          acc[i][2 * q + 1][0], acc[i][2 * q + 1][1], acc[i][2 * q + 1][2], acc[i][2 * q + 1][3]};
      const int64_t left = a.n - col;
      if (left > 0) store8<T>(a.out, row * a.stride_out + col, left < 8 ? (int)left : 8, v);
    }
  }
}

template <typename T, int XF, int BM, int BN, int WM, int WN> const char* launch_tile(const ns_mx_linear_args& a, hipStream_t stream) {
  const int64_t blocks = ((a.m + BM - 1) / BM) * ((a.n + BN - 1) / BN);
  if (blocks >= (int64_t)1 << 31) return "too many rows";
  hipLaunchKernelGGL((tile_kernel<T, XF, BM, BN, WM, WN>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0, stream, a);
  return nullptr;
}

template <typename T, int XF> const char* launch_linear_t(const ns_mx_linear_args& a, hipStream_t stream) {
  if (a.m > 64) return launch_tile<T, XF, 256, 256, 4, 2>(a, stream);
  const int64_t tiles = (a.n + 31) / 32;
  if (tiles >= 2048) {
    if (a.m <= 16) return launch_stream<T, XF, 1, 1, 16>(a, 2, stream);
    if (a.m <= 32) return launch_stream<T, XF, 2, 1, 8>(a, 2, stream);
    return launch_stream<T, XF, 4, 1, 8>(a, 1, stream);
  }
  if (tiles >= 1024) return launch_stream<T, XF, 1, 2, 16>(a, 1, stream);
  if (tiles >= 512) return launch_stream<T, XF, 1, 4, 16>(a, 1, stream);
  return launch_stream<T, XF, 1, 8, 32>(a, 1, stream);
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
