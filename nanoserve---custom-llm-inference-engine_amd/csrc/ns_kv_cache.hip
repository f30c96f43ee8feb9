// The paged KV cache for gfx950: the store of new key and value rows with their rotation by position
// (nanoserve/model/rope.py:78-91 and attention.py:55-72 in one launch), and the pages: extending, forking, freeing,
// releasing behind a window, copying and compacting (nanoserve/cache/block_allocator.py:14-47 keeps a free list on the
// host; here counts and tables live on the device and every operator is a launch or two).

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "ns_kv_cache.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

thread_local char g_err[512];

int fail(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
int fail(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return 1;
}

__device__ __forceinline__ void flag(int32_t* status, int bit) {
  if (status != nullptr) atomicOr(status, bit);
}

// ---- store ------------------------------------------------------------------------------------------------

struct Bf16 {};
struct F16 {};
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// 16 bytes of a row: N elements
template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int N = 4, bytes = 4;
  static __device__ __forceinline__ void get(u32x4 w, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ u32x4 put(const float (&x)[N]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __float_as_uint(x[i]);
    return w;
  }
};
template <> struct Elem<Bf16> {
  static constexpr int N = 8, bytes = 2;
  static __device__ __forceinline__ void get(u32x4 w, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ u32x4 put(const float (&x)[N]) {   // to nearest even
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x[2 * i], x[2 * i + 1]}, bf16x2_t));
    return w;
  }
};
template <> struct Elem<F16> {
  static constexpr int N = 8, bytes = 2;
  static __device__ __forceinline__ void get(u32x4 w, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = w[i];   // a bit cast of a vector's element takes its first one
      const f16x2_t h = __builtin_bit_cast(f16x2_t, u);
      x[2 * i] = (float)h[0];
      x[2 * i + 1] = (float)h[1];
    }
  }
  static __device__ __forceinline__ u32x4 put(const float (&x)[N]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x[2 * i], x[2 * i + 1]}, f16x2_t));
    return w;
  }
};

constexpr int kStoreThreads = 256;

// The sequence of token i by the whole wave, 64 entries of query_start_loc at a time: the largest s with
// query_start_loc[s] <= i.
__device__ __forceinline__ int find_seq(const int32_t* qsl, int num_seqs, int i) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = num_seqs;
  for (;;) {
    const int stride = (len + 63) / 64;
    const int at = lane * stride;
    const int below = __popcll(__ballot(at < len && qsl[lo + (at < len ? at : 0)] <= i));
    const int skip = (below > 0 ? below - 1 : 0) * stride;
    lo += skip;
    if (stride == 1) return lo;
    len = min(stride, len - skip);
  }
}

// A workgroup of four waves takes T tokens.  A wave first places one of them (its sequence, position, page and slot)
// and, a lane per frequency, forms the angles: p * inv_freq / (2 pi) in 64 bits less its nearest whole number, so that
// positions of millions keep their angle to 2^-26 of a turn.  Then all threads take items: 16 bytes of a head's
// lower half and the 16 bytes half a head above, which the rotation pairs; a value head's two pieces are only copied.
// Bound: memory.  8192 tokens of 24 / 8 heads of 128 dims (bf16, rotated; 168 MB read and written) take 30 us, 5.6 TB/s;
// 64 tokens 3.6 us: a launch and four trips to memory after one another (the starts that are searched, the sequence's
// length, the table entry, the rows, which wait at the barrier although their own addresses do not need the place).
template <typename T, int D, int TOK>
__global__ __launch_bounds__(kStoreThreads) void store_kernel(ns_kv_store_args a) {
  using E = Elem<T>;
  constexpr int N = E::N;
  constexpr int HALF = D / 2;
  constexpr int LPH = HALF / N;   // items of a head
  __shared__ float s_cos[TOK][HALF], s_sin[TOK][HALF];
  __shared__ int64_t s_k[TOK], s_v[TOK];   // element offsets of the token's slot, -1: none
  __shared__ int s_live[TOK];

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int first = blockIdx.x * TOK;
  for (int w = wave; w < TOK; w += kStoreThreads / 64) {
    const int i = first + w;
    int64_t k = -1, v = -1;
    bool live = false;
    if (i < a.total) {
      const int s = find_seq(a.query_start_loc, a.num_seqs, i);
      const int nth = i - a.query_start_loc[s], len = a.query_lens[s];
      const int pos = a.seq_lens[s] - len + nth;
      live = nth >= 0 && nth < len && pos >= 0;
      if (live) {
        const int col = pos / a.block_size, slot = pos - col * a.block_size;
        const int page = col < a.max_blocks_per_seq ? a.block_tables[(int64_t)s * a.stride_bt_seq + col] : -1;
        if (page >= 0 && page < a.num_blocks) {
          k = (int64_t)page * a.stride_k_block + (int64_t)slot * a.stride_k_token;
          v = (int64_t)page * a.stride_v_block + (int64_t)slot * a.stride_v_token;
        } else if (lane == 0) {
          flag(a.status, NS_KV_STATUS_BAD_PAGE);
        }
        if (a.inv_freq != nullptr && lane < HALF) {
          constexpr double kTurn = 0.15915494309189533577;   // 1 / (2 pi)
          const double turns = (double)pos * (double)a.inv_freq[lane] * kTurn;
          float sn, cs;
          sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
          s_cos[w][lane] = cs;
          s_sin[w][lane] = sn;
        }
      }
    }
    if (lane == 0) {
      s_live[w] = live;
      s_k[w] = k;
      s_v[w] = v;
    }
  }
  __syncthreads();

  const int hq = a.query != nullptr ? a.num_heads_q : 0;
  const int heads = hq + 2 * a.num_kv_heads;
  const bool turn = a.inv_freq != nullptr;
  for (int it = threadIdx.x; it < TOK * heads * LPH; it += kStoreThreads) {
    const int c = it % LPH, th = it / LPH;
    const int w = th / heads, h = th - w * heads;
    if (!s_live[w]) continue;
    const int64_t tok = first + w;
    const void* src;
    void* dst;
    int64_t from, to;
    if (h < hq) {
      src = a.query;
      dst = a.out;
      from = tok * a.stride_q_token + (int64_t)h * a.stride_q_head;
      to = tok * a.stride_o_token + (int64_t)h * a.stride_o_head;
    } else {
      const bool val = h >= hq + a.num_kv_heads;
      const int kh = h - hq - (val ? a.num_kv_heads : 0);
      if (s_k[w] < 0) continue;
      src = val ? a.value : a.key;
      dst = val ? a.v_cache : a.k_cache;
      from = val ? tok * a.stride_value_token + (int64_t)kh * a.stride_value_head
                 : tok * a.stride_key_token + (int64_t)kh * a.stride_key_head;
      to = val ? s_v[w] + (int64_t)kh * a.stride_v_head : s_k[w] + (int64_t)kh * a.stride_k_head;
    }
    const char* sp = reinterpret_cast<const char*>(src) + (from + c * N) * E::bytes;
    char* dp = reinterpret_cast<char*>(dst) + (to + c * N) * E::bytes;
    u32x4 lo = *reinterpret_cast<const u32x4*>(sp), hi = *reinterpret_cast<const u32x4*>(sp + HALF * E::bytes);
    if (turn && h < hq + a.num_kv_heads) {
      float x[N], y[N], u[N], v[N];
      E::get(lo, x);
      E::get(hi, y);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float cs = s_cos[w][c * N + i], sn = s_sin[w][c * N + i];
        u[i] = fmaf(-y[i], sn, x[i] * cs);
        v[i] = fmaf(x[i], sn, y[i] * cs);
      }
      lo = E::put(u);
      hi = E::put(v);
    }
    *reinterpret_cast<u32x4*>(dp) = lo;
    *reinterpret_cast<u32x4*>(dp + HALF * E::bytes) = hi;
  }
}

// ---- pages ------------------------------------------------------------------------------------------------

constexpr int kPlan = 1024;          // threads of a planning workgroup
constexpr int kPlanWaves = kPlan / 64;
constexpr int kGroup = 1024;         // pages that a wave looks at together, 16 consecutive ones a lane
constexpr int kCopy = 256;
constexpr int kMaxRows = NS_KV_MAX_ROWS;

__device__ __forceinline__ int pages_of(int tokens, int block_size) {
  return tokens > 0 ? (tokens - 1) / block_size + 1 : 0;
}
// the columns of a row that hold pages
__device__ __forceinline__ int held_cols(const ns_kv_pool& p, int len) { return min(pages_of(len, p.block_size), p.num_cols); }

// A barrier behind which the workgroup sees what its threads stored, also by atomics that other XCDs' caches pass by:
// the barrier alone waits for LDS only.
__device__ __forceinline__ void sync_memory() {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
}

// Sum of a wave's shares before this wave (every lane passes its wave's); *total: of all waves.
__device__ __forceinline__ int wave_prefix(int x, int* total) {
  __shared__ int s_sum[kPlanWaves];
  const int wave = threadIdx.x >> 6;
  __syncthreads();   // an earlier call's sums are read
  if ((threadIdx.x & 63) == 0) s_sum[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    before += w < wave ? s_sum[w] : 0;
    all += s_sum[w];
  }
  *total = all;
  return before;
}
// Exclusive prefix sum of x over the workgroup's threads; *total: the sum.
__device__ __forceinline__ int block_prefix(int x, int* total) {
  const int lane = threadIdx.x & 63;
  int in = x;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int y = __shfl_up(in, s);
    if (lane >= s) in += y;
  }
  return wave_prefix(__shfl(in, 63), total) + in - x;
}

// Which of a lane's 16 pages p0 .. p0 + 15 have pred(page, count): bit i for page p0 + i.
template <typename Pred>
__device__ __forceinline__ uint32_t pages_with(const int32_t* refs, int n, int64_t p0, Pred pred) {
  i32x4 x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = i32x4{0, 0, 0, 0};
    if (p0 + 4 * j + 3 < n) {
      x[j] = *reinterpret_cast<const i32x4*>(refs + p0 + 4 * j);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (p0 + 4 * j + i < n) x[j][i] = refs[p0 + 4 * j + i];
    }
  }
  uint32_t bits = 0u;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (p0 + j < n && pred((int)(p0 + j), x[j / 4][j % 4])) bits |= 1u << j;
  return bits;
}

__device__ __forceinline__ int wave_inclusive(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int y = __shfl_up(x, s);
    if (lane >= s) x += y;
  }
  return x;
}

// What a planning kernel leaves in the pool's scratch memory for the kernel after it: a line for each list entry, and of
// every group of 1024 pages which are free and how many.
struct Plan {
  int32_t* total;    // pages that the list asks for
  int32_t* off;      // by list entry: the first rank that falls to it
  int32_t* row;      // its row, -1: nothing to do
  int32_t* col;      // the column that the first of its pages goes to
  int32_t* len;      // its new length
  i32x4* pair;       // of a fork: parent's row, tokens (0: nothing to do), the copy's rank (-1: none), its source
  int32_t* count;    // by group
  uint16_t* free;    // by 16 pages, 64 a group
  int groups;
  __device__ __forceinline__ explicit Plan(const ns_kv_pool& p) {
    total = p.scratch;
    off = total + 4;
    row = off + kMaxRows;
    col = row + kMaxRows;
    len = col + kMaxRows;
    pair = reinterpret_cast<i32x4*>(off);
    count = off + 4 * kMaxRows;
    groups = (int)(((int64_t)p.num_pages + kGroup - 1) / kGroup);
    free = reinterpret_cast<uint16_t*>(count + groups);
  }
};
constexpr uint64_t plan_ints(uint64_t pages) { return 4 + 4 * (uint64_t)kMaxRows + (pages + kGroup - 1) / kGroup * 33; }

// The groups' free pages, a group a wave, by the workgroups after the first.
__device__ __forceinline__ void find_free(const ns_kv_pool& p, const Plan& plan) {
  const int lane = threadIdx.x & 63;
  const int64_t g = (int64_t)(blockIdx.x - 1) * kPlanWaves + (threadIdx.x >> 6);
  if (g >= plan.groups) return;
  const uint32_t bits = pages_with(p.page_refs, p.num_pages, g * kGroup + 16 * lane, [](int, int refs) { return refs == 0; });
  plan.free[g * 64 + lane] = (uint16_t)bits;
  const int upto = wave_inclusive(__popc(bits));
  if (lane == 63) plan.count[g] = upto;
}

// The request that rank r falls to: the largest i with off[i] <= r, at least lo.
__device__ __forceinline__ int request_of(const int* off, int lo, int n, int r) {
  int hi = n;   // off[lo] <= r, off[hi] > r
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A list's rows, each counted where it is listed first: a table of the list's places, hashed by row, in LDS (places of
// one row meet in one slot, which keeps the lowest).
constexpr int kSlots = 2 * kMaxRows;   // a power of two, at most half full
constexpr int kEach = kMaxRows / kPlan;   // list entries a thread takes at most, consecutive ones
struct Rows {
  int row[kMaxRows];   // -1: not in the tables
  int slot[kSlots];
};
static_assert((kSlots & (kSlots - 1)) == 0 && kEach * kPlan == kMaxRows, "sizes");

// Fills row with the thread's entries first .. last - 1 (-1: not in the tables); bit k of the result set where entry
// first + k is its row's first listing.
__device__ __forceinline__ uint32_t first_listings(Rows& s, const int32_t* rows, int num_rows, int first, int last,
                                                   int (&row)[kEach]) {
  for (int i = threadIdx.x; i < kSlots; i += kPlan) s.slot[i] = -1;
  int at[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    row[k] = first + k < last ? rows[first + k] : -1;
    if (row[k] >= num_rows || row[k] < 0) row[k] = -1;
    if (first + k < last) s.row[first + k] = row[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    at[k] = (int)(((uint32_t)row[k] * 2654435769u) >> 16) & (kSlots - 1);
    while (row[k] >= 0) {   // at most half of the slots are taken, so one is met that is free or the row's own
      const int held = atomicCAS(&s.slot[at[k]], -1, first + k);
      if (held < 0) break;
      if (s.row[held] == row[k]) {
        atomicMin(&s.slot[at[k]], first + k);
        break;
      }
      at[k] = (at[k] + 1) & (kSlots - 1);
    }
  }
  __syncthreads();
  uint32_t own = 0u;
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (row[k] >= 0 && s.slot[at[k]] == first + k) own |= 1u << k;
  return own;
}

// Extending takes two launches.  The first: one workgroup sums up what the rows ask for, the others find the free
// pages.  All of it in one workgroup is bound by what one CU gets through (2.8 us for 16,384 pages' counts): a call for
// 10,400 pages took 18.6 us with 27,000 pages and 38.9 with 160,000 of which a tenth were free, one page 9.1; so 11.6,
// 11.6 and 10.1 (each with the 5 us that an idle queue takes to start it).
__global__ __launch_bounds__(kPlan) void extend_plan_kernel(ns_kv_pool p, const int32_t* rows, const int32_t* lens, int n) {
  __shared__ Rows s;
  const Plan plan(p);
  if (blockIdx.x > 0) {
    find_free(p, plan);
    return;
  }
  const int per = (n + kPlan - 1) / kPlan;
  const int first = min(n, (int)threadIdx.x * per), last = min(n, first + per);
  int row[kEach], need[kEach], mine = 0;
  const uint32_t own = first_listings(s, rows, p.num_rows, first, last, row);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    need[k] = 0;
    if (first + k >= last) continue;
    int col = 0, now = 0;
    if ((own >> k) & 1u) {
      const int old = p.seq_lens[row[k]];
      now = lens[first + k];
      if (old < 0 || now < old || now > (int64_t)p.num_cols * p.block_size) {
        flag(p.status, NS_KV_STATUS_BAD_LENGTH);
        row[k] = -1;
      } else {
        col = pages_of(old, p.block_size);
        need[k] = pages_of(now, p.block_size) - col;
        mine += need[k];
      }
    } else {
      flag(p.status, NS_KV_STATUS_BAD_ROW);
      row[k] = -1;
    }
    plan.row[first + k] = row[k];
    plan.col[first + k] = col;
    plan.len[first + k] = now;
  }
  int total;
  int at = block_prefix(mine, &total);
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (first + k < last) {
      plan.off[first + k] = at;
      at += need[k];
    }
  if (threadIdx.x == 0) *plan.total = total;
}

// The second: a wave a group of pages.  Its free pages' ranks follow from the counts of the groups before it; each goes
// to the row and column that its rank falls to, if all that the row asks for is there.  The first workgroup also sets
// the rows' lengths.
__global__ __launch_bounds__(kCopy) void extend_kernel(ns_kv_pool p, int n) {
  __shared__ int s_off[kMaxRows];
  const Plan plan(p);
  const int lane = threadIdx.x & 63;
  const int64_t g = (int64_t)blockIdx.x * (kCopy / 64) + (threadIdx.x >> 6);
  const uint32_t bits = g < plan.groups ? plan.free[g * 64 + lane] : 0u;
  for (int i = threadIdx.x; i < n; i += kCopy) s_off[i] = plan.off[i];
  const int total = *plan.total;
  int found = 0, before = 0;
  for (int c = lane; c < plan.groups; c += 64) {
    const int x = plan.count[c];
    found += x;
    before += c < g ? x : 0;
  }
  found = __shfl(wave_inclusive(found), 63);
  before = __shfl(wave_inclusive(before), 63);
  __syncthreads();
  auto end_of = [&](int i) -> int { return i + 1 < n ? s_off[i + 1] : total; };
  const int most = min(total, found);
  int r = before + wave_inclusive(__popc(bits)) - __popc(bits);
  int i = -1, end = 0;
  int32_t* to = nullptr;
  for (uint32_t left = bits; left != 0u && r < most; left &= left - 1u, ++r) {
    if (i < 0 || r >= end) {
      i = request_of(s_off, max(i, 0), n, r);
      end = end_of(i);
      if (end > found) break;   // not served, nor are those after it
      to = p.block_tables + (int64_t)plan.row[i] * p.stride_bt_row + plan.col[i] - s_off[i];
    }
    const int page = (int)(g * kGroup) + 16 * lane + __ffs(left) - 1;
    to[r] = page;
    p.page_refs[page] = 1;
  }
  if (blockIdx.x > 0) return;
  for (int k = threadIdx.x; k < n; k += kCopy) {
    const int row = plan.row[k];
    if (row < 0) continue;
    if (end_of(k) == s_off[k] || end_of(k) <= found) p.seq_lens[row] = plan.len[k];
    else flag(p.status, NS_KV_STATUS_NO_PAGES);
  }
}

// A fork's first launch, as extending's.  Both: 3.8 us and 4.9 for one pair of 32 tensors (latency); 96 pairs of 56
// tensors, up to 15 slots of 2 KB each, 29 us (5.6 TB/s of reads and writes, pages shared by siblings read once).
__global__ __launch_bounds__(kPlan) void fork_plan_kernel(ns_kv_pool p, const int32_t* parents, const int32_t* children, int n) {
  __shared__ Rows s;
  const Plan plan(p);
  if (blockIdx.x > 0) {
    find_free(p, plan);
    return;
  }
  const int per = (n + kPlan - 1) / kPlan;
  const int first = min(n, (int)threadIdx.x * per), last = min(n, first + per);
  int row[kEach], mine = 0;
  const uint32_t own = first_listings(s, children, p.num_rows, first, last, row);
  i32x4 x[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    x[k] = i32x4{0, 0, -1, -1};
    if (first + k >= last) continue;
    const int parent = parents[first + k];
    if (!((own >> k) & 1u) || parent < 0 || parent >= p.num_rows || p.seq_lens[row[k]] != 0) {
      flag(p.status, NS_KV_STATUS_BAD_ROW);
      continue;
    }
    x[k][0] = parent;
    x[k][1] = max(0, (int)min((int64_t)p.seq_lens[parent], (int64_t)p.num_cols * p.block_size));
    if (x[k][1] % p.block_size != 0) {
      x[k][3] = p.block_tables[(int64_t)parent * p.stride_bt_row + x[k][1] / p.block_size];
      if (x[k][3] >= 0 && x[k][3] < p.num_pages) ++mine;
      else x[k][3] = -1;
    }
  }
  int total;
  int at = block_prefix(mine, &total);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    if (first + k >= last) continue;
    if (x[k][3] >= 0) x[k][2] = at++;
    plan.pair[first + k] = x[k];
  }
}

// The free page of rank r, by a whole wave; -1: there are no more than r.
__device__ __forceinline__ int free_page(const Plan& plan, int r) {
  const int lane = threadIdx.x & 63;
  for (int g0 = 0; g0 < plan.groups; g0 += 64) {
    const int x = g0 + lane < plan.groups ? plan.count[g0 + lane] : 0;
    const int upto = wave_inclusive(x);
    const uint64_t past = __ballot(upto > r);
    if (past == 0ull) {
      r -= __shfl(upto, 63);
      continue;
    }
    const int at = __ffsll((unsigned long long)past) - 1;
    r -= __shfl(upto - x, at);
    uint32_t bits = plan.free[(int64_t)(g0 + at) * 64 + lane];
    const int sum = wave_inclusive(__popc(bits));
    const int who = __ffsll((unsigned long long)__ballot(sum > r)) - 1;
    r -= __shfl(sum - __popc(bits), who);
    bits = __shfl(bits, who);
    for (; r > 0; --r) bits &= bits - 1u;
    return (g0 + at) * kGroup + 16 * who + __ffs(bits) - 1;
  }
  return -1;
}

// `bytes` (a multiple of 16) from src to dst by the workgroup, eight loads a thread in flight
__device__ __forceinline__ void copy_bytes(char* dst, const char* src, int64_t bytes) {
  constexpr int kStep = kCopy * 16;
  int64_t i = (int64_t)threadIdx.x * 16;
  for (; i + 7 * kStep < bytes; i += 8 * kStep) {
    u32x4 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + i + u * kStep));
#pragma unroll
    for (int u = 0; u < 8; ++u) __builtin_nontemporal_store(x[u], reinterpret_cast<u32x4*>(dst + i + u * kStep));
  }
  for (; i < bytes; i += kStep) *reinterpret_cast<u32x4*>(dst + i) = *reinterpret_cast<const u32x4*>(src + i);
}

// A fork's second launch.  blockIdx.x: the pair; blockIdx.y 0: the child's table row and length and the shared pages'
// counts, else the copy in one tensor.  Every wave finds the copy's page for itself.
__global__ __launch_bounds__(kCopy) void fork_kernel(ns_kv_pool p, const int32_t* children) {
  const int i = blockIdx.x, t = (int)blockIdx.y - 1;
  const Plan plan(p);
  const i32x4 x = plan.pair[i];
  if (x[1] == 0 || (t >= 0 && x[2] < 0)) return;
  const int page = x[2] >= 0 ? free_page(plan, x[2]) : -1;
  if (x[2] >= 0 && page < 0) {   // no page was left: the child stays empty
    if (t < 0 && threadIdx.x == 0) flag(p.status, NS_KV_STATUS_NO_PAGES);
    return;
  }
  if (t >= 0) {
    const uint64_t base = p.tensors[2 * t], stride = p.tensors[2 * t + 1];
    copy_bytes(reinterpret_cast<char*>(base + page * stride), reinterpret_cast<const char*>(base + x[3] * stride),
               (int64_t)(x[1] % p.block_size) * p.slot_bytes);
    return;
  }
  const int32_t* from = p.block_tables + (int64_t)x[0] * p.stride_bt_row;
  int32_t* to = p.block_tables + (int64_t)children[i] * p.stride_bt_row;
  const int last = page >= 0 ? x[1] / p.block_size : -1;
  const int cols = held_cols(p, x[1]);
  for (int j = threadIdx.x; j < cols; j += kCopy) {
    if (j == last) {
      to[j] = page;
      p.page_refs[page] = 1;
      continue;
    }
    int e = from[j];
    if (e >= p.num_pages) {
      flag(p.status, NS_KV_STATUS_BAD_PAGE);
      e = -1;
    }
    to[j] = e;
    if (e >= 0) atomicAdd(p.page_refs + e, 1);
  }
  if (threadIdx.x == 0) p.seq_lens[children[i]] = x[1];
}

// A workgroup a listed row: its entries in [first, last) of its columns become -1, their pages' counts fall.  An entry
// is taken out by an exchange, so that a row listed twice gives its pages up once.  2.4 us for one row, 3.5 for 40 of 8192
// tokens: a launch, then reads, exchanges and counts one after the other.
template <bool ALL>
__global__ __launch_bounds__(kCopy) void drop_kernel(ns_kv_pool p, const int32_t* rows, int window, int sinks) {
  const int row = rows[blockIdx.x];
  if (row < 0 || row >= p.num_rows) {
    if (threadIdx.x == 0) flag(p.status, NS_KV_STATUS_BAD_ROW);
    return;
  }
  const int len = p.seq_lens[row];
  int first = 0, last = held_cols(p, len);
  if (!ALL) {
    first = sinks > 0 ? (sinks - 1) / p.block_size + 1 : 0;
    const int64_t gone = (int64_t)len - window + 1;   // positions below it are behind the window
    last = gone > 0 ? min((int64_t)last, gone / p.block_size) : 0;
  }
  int32_t* bt = p.block_tables + (int64_t)row * p.stride_bt_row;
  // eight columns a thread at a time: their reads, then the exchanges, then the counts
  for (int j0 = first + threadIdx.x; j0 < last; j0 += 8 * kCopy) {
    int e[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = j0 + u * kCopy;
      e[u] = j < last ? bt[j] : -1;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (e[u] >= 0) e[u] = atomicExch(bt + j0 + u * kCopy, -1);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (e[u] < 0) continue;
      if (e[u] >= p.num_pages) flag(p.status, NS_KV_STATUS_BAD_PAGE);
      else atomicSub(p.page_refs + e[u], 1);
    }
  }
  if (ALL) {
    __syncthreads();
    if (threadIdx.x == 0) p.seq_lens[row] = 0;
  }
}

__global__ __launch_bounds__(kCopy) void copy_kernel(ns_kv_pool p, const uint64_t* to, int to_pages, const int32_t* src,
                                                     const int32_t* dst) {
  const int s = src[blockIdx.x], d = dst[blockIdx.x], t = blockIdx.y;
  if (s < 0 || s >= p.num_pages || d < 0 || d >= to_pages) {
    if (threadIdx.x == 0 && t == 0) flag(p.status, NS_KV_STATUS_BAD_PAGE);
    return;
  }
  copy_bytes(reinterpret_cast<char*>(to[2 * t] + (uint64_t)d * to[2 * t + 1]),
             reinterpret_cast<const char*>(p.tensors[2 * t] + (uint64_t)s * p.tensors[2 * t + 1]),
             p.slot_bytes * p.block_size);
}

// Planning a compaction.  With m pages in use, the free pages below m (holes) and the used ones from m on (movers) are
// as many, and one ascending scan lists both: list[0 .. h-1] holes, list[h .. 2h-1] movers.  head[0]: moves, or all
// pages in use with `to`; -1: `to` is too small.
__global__ __launch_bounds__(kPlan) void compact_plan_kernel(ns_kv_pool p, int32_t* to_refs, int to_pages, int32_t* map) {
  int32_t* head = p.scratch;
  int32_t* list = head + 4;
  const int tid = threadIdx.x;
  int mine = 0;
  for (int i = tid; i < p.num_pages; i += kPlan) mine += p.page_refs[i] != 0;
  int m;
  block_prefix(mine, &m);
  if (to_refs != nullptr && m > to_pages) {
    if (tid == 0) {
      flag(p.status, NS_KV_STATUS_NO_PAGES);
      head[0] = -1;
    }
    for (int i = tid; i < p.num_pages; i += kPlan) map[i] = -1;
    return;
  }
  // 16 groups at a time, each a wave's
  int both = 0;
  for (int64_t c0 = 0; c0 < p.num_pages; c0 += kPlanWaves * kGroup) {
    const int64_t p0 = c0 + 16 * tid;
    const uint32_t bits =
        pages_with(p.page_refs, p.num_pages, p0, [m](int page, int refs) { return (page < m) == (refs == 0); });
    int all;
    int r = both + block_prefix(__popc(bits), &all);
    for (uint32_t left = bits; left != 0u; left &= left - 1u) list[r++] = (int)p0 + __ffs(left) - 1;
    both += all;
  }
  const int h = both / 2;
  for (int i = tid; i < p.num_pages; i += kPlan) map[i] = i < m && p.page_refs[i] != 0 ? i : -1;
  if (to_refs != nullptr)
    for (int i = tid; i < to_pages; i += kPlan) to_refs[i] = i < m ? p.page_refs[i] : 0;
  if (tid == 0) {
    head[0] = h;
    head[1] = m;
  }
  sync_memory();
  for (int r = tid; r < h; r += kPlan) {
    const int hole = list[r], mover = list[h + r];
    map[mover] = hole;
    if (to_refs != nullptr) {
      to_refs[hole] = p.page_refs[mover];
    } else {
      p.page_refs[hole] = p.page_refs[mover];
      p.page_refs[mover] = 0;
    }
  }
}

// The first num_rows workgroups rewrite a table row each; the others take (page, tensor) pieces in turn.  Bound: memory.
// 1.7 GB of pages moved take 682 us, 4.98 TB/s of reads and writes; a large copy reaches 4.95.
__global__ __launch_bounds__(kCopy) void compact_kernel(ns_kv_pool p, ns_kv_pool to, const int32_t* map, int into) {
  const int32_t* head = p.scratch;
  const int32_t* list = head + 4;
  const int h = head[0];
  if (h < 0) return;
  if ((int)blockIdx.x < p.num_rows) {
    const int row = blockIdx.x;
    const int32_t* from = p.block_tables + (int64_t)row * p.stride_bt_row;
    int32_t* bt = into ? to.block_tables + (int64_t)row * to.stride_bt_row : p.block_tables + (int64_t)row * p.stride_bt_row;
    const int len = p.seq_lens[row], cols = held_cols(p, len);
    for (int j = threadIdx.x; j < (into ? p.num_cols : cols); j += kCopy) {
      int e = j < cols ? from[j] : -1;
      if (e >= p.num_pages) {
        flag(p.status, NS_KV_STATUS_BAD_PAGE);
        e = -1;
      }
      bt[j] = e >= 0 ? map[e] : -1;
    }
    if (into && threadIdx.x == 0) to.seq_lens[row] = len;
    return;
  }
  const int64_t bytes = p.slot_bytes * p.block_size;
  const int64_t pieces = (int64_t)(into ? head[1] : h) * p.num_tensors;
  for (int64_t u = blockIdx.x - p.num_rows; u < pieces; u += gridDim.x - p.num_rows) {
    const int k = (int)(u / p.num_tensors), t = (int)(u - (int64_t)k * p.num_tensors);
    int src, dst = into ? k : list[k];
    if (into) {   // page k of the compact cache: page k itself, or the mover that fills the hole
      src = k;
      if (map[k] != k) {
        int lo = 0, hi = h;   // list[0 .. h-1] ascends
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (list[mid] <= k) lo = mid;
          else hi = mid;
        }
        src = list[h + lo];
      }
    } else {
      src = list[h + k];
    }
    copy_bytes(reinterpret_cast<char*>((into ? to.tensors : p.tensors)[2 * t] +
                                       (uint64_t)dst * (into ? to.tensors : p.tensors)[2 * t + 1]),
               reinterpret_cast<const char*>(p.tensors[2 * t] + (uint64_t)src * p.tensors[2 * t + 1]), bytes);
  }
}

// ---- host side ----------------------------------------------------------------------------------------------

// Four tokens a workgroup, a wave a token to place, from 4096 on; below, one, so that few tokens spread over more CUs.  In
// us, one and four (from a graph): 24 / 8 heads of 128 dims, rotated, bf16: 64 tokens 3.6, 5.3; 512 4.4, 6.0; 2048 9.4,
// 9.8; 4096 16.0, 15.5; 8192 31.4, 30.4.  32 / 8 of 64, f16: 512 3.6, 4.6; 2048 6.5, 7.3; 4096 11.6, 10.9; 8192 18.8, 18.1;
// keys and values alone 512 3.0, 3.2; 2048 3.8, 3.7; 4096 6.0, 5.2; 8192 9.7, 8.3.  4 / 1 of 64: 512 3.4, 3.5; 2048 3.9,
// 3.8; 4096 5.9, 4.2.
template <typename T, int D>
void launch_store(const ns_kv_store_args& a, hipStream_t stream) {
  if (a.total >= 4096)
    hipLaunchKernelGGL((store_kernel<T, D, 4>), dim3((a.total + 3) / 4), dim3(kStoreThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((store_kernel<T, D, 1>), dim3(a.total), dim3(kStoreThreads), 0, stream, a);
}

template <typename T>
void launch_store_d(const ns_kv_store_args& a, hipStream_t stream) {
  if (a.head_dim == 64) launch_store<T, 64>(a, stream);
  else launch_store<T, 128>(a, stream);
}

uint64_t scratch_bytes(int32_t num_pages) {
  // a plan, or a compaction's head and list
  const uint64_t plan = plan_ints(num_pages), list = 4ull + (uint64_t)num_pages;
  return 4ull * (plan > list ? plan : list);
}

int plan_groups(int32_t num_pages) { return 1 + (int)(((int64_t)num_pages + kPlanWaves * kGroup - 1) / (kPlanWaves * kGroup)); }

int check_pool(const ns_kv_pool* p) {
  if (!p) return fail("pool is NULL");
  if (p->num_rows < 1 || p->num_cols < 1 || p->num_pages < 1 || p->num_tensors < 1 || p->block_size < 1)
    return fail("a pool needs rows, columns, pages, tensors and a block size (got %d, %d, %d, %d, %d)", p->num_rows,
                p->num_cols, p->num_pages, p->num_tensors, p->block_size);
  if (p->num_tensors > 65534) return fail("at most 65534 tensors (got %d)", p->num_tensors);
  if (!p->block_tables || !p->seq_lens || !p->page_refs || !p->tensors || !p->scratch)
    return fail("a pool pointer is NULL");
  if (p->stride_bt_row < p->num_cols) return fail("stride_bt_row (%lld) is below num_cols (%d)", (long long)p->stride_bt_row, p->num_cols);
  if (p->slot_bytes < 16 || p->slot_bytes % 16 != 0) return fail("slot_bytes must be a positive multiple of 16 (got %lld)", (long long)p->slot_bytes);
  if ((uintptr_t)p->page_refs % 16 != 0 || (uintptr_t)p->scratch % 16 != 0)
    return fail("page_refs and scratch must be 16-byte aligned");
  if (p->scratch_bytes < scratch_bytes(p->num_pages))
    return fail("scratch of %llu bytes needed (got %llu)", (unsigned long long)scratch_bytes(p->num_pages),
                (unsigned long long)p->scratch_bytes);
  return 0;
}

int check_list(const ns_kv_pool* p, const void* a, const void* b, int32_t n, int32_t most) {
  if (check_pool(p)) return 1;
  if (n < 0) return fail("the list's length must be >= 0 (got %d)", n);
  if (n > most) return fail("a call takes at most %d rows (got %d)", most, n);
  if (n > 0 && (!a || !b)) return fail("a list is NULL");
  return 0;
}

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("kernel launch failed: %s", hipGetErrorString(e));
}

}  // namespace

extern "C" {

int ns_kv_abi_version(void) { return NS_KV_ABI_VERSION; }

const char* ns_kv_last_error(void) { return g_err; }

int ns_kv_store(const ns_kv_store_args* a, hipStream_t stream) {
  if (!a) return fail("args is NULL");
  if (a->dtype != NS_KV_DTYPE_F32 && a->dtype != NS_KV_DTYPE_BF16 && a->dtype != NS_KV_DTYPE_F16)
    return fail("dtype must be NS_KV_DTYPE_F32, _BF16 or _F16 (got %d)", a->dtype);
  if (a->head_dim != 64 && a->head_dim != 128) return fail("head_dim must be 64 or 128 (got %d)", a->head_dim);
  if (a->total < 0) return fail("total must be >= 0 (got %d)", a->total);
  if (a->num_kv_heads < 1 || a->num_kv_heads > 65535) return fail("num_kv_heads must lie in 1 .. 65535 (got %d)", a->num_kv_heads);
  if (a->query && (a->num_heads_q < 1 || a->num_heads_q > 65535))
    return fail("num_heads_q must lie in 1 .. 65535 (got %d)", a->num_heads_q);
  if (a->query && !a->inv_freq) return fail("a query is there to be rotated: it needs inv_freq");
  if (!a->query != !a->out) return fail("query and out come together");
  if (a->total == 0) return 0;
  if (a->num_seqs < 1) return fail("num_seqs must be > 0 when there are tokens (got %d)", a->num_seqs);
  if (a->block_size < 1 || a->num_blocks < 1) return fail("block_size and num_blocks must be > 0");
  if (a->max_blocks_per_seq < 0 || a->stride_bt_seq < 0) return fail("max_blocks_per_seq and stride_bt_seq must be >= 0");
  if (!a->key || !a->value || !a->k_cache || !a->v_cache || !a->block_tables || !a->seq_lens || !a->query_start_loc ||
      !a->query_lens)
    return fail("a tensor pointer is NULL");
  const int esz = a->dtype == NS_KV_DTYPE_F32 ? 4 : 2;
  const int64_t strides[] = {a->query ? a->stride_q_token : 0, a->query ? a->stride_q_head : 0,
                             a->query ? a->stride_o_token : 0, a->query ? a->stride_o_head : 0,
                             a->stride_key_token, a->stride_key_head, a->stride_value_token, a->stride_value_head,
                             a->stride_k_block, a->stride_k_token, a->stride_k_head, a->stride_v_block,
                             a->stride_v_token, a->stride_v_head};
  for (int64_t s : strides)
    if (s < 0 || (s * esz) % 16 != 0) return fail("row strides must be multiples of 16 bytes, not negative");
  if (((uintptr_t)a->query | (uintptr_t)a->key | (uintptr_t)a->value | (uintptr_t)a->out | (uintptr_t)a->k_cache |
       (uintptr_t)a->v_cache) % 16 != 0)
    return fail("tensors must be 16-byte aligned");
  switch (a->dtype) {
    case NS_KV_DTYPE_F32: launch_store_d<float>(*a, stream); break;
    case NS_KV_DTYPE_BF16: launch_store_d<Bf16>(*a, stream); break;
    default: launch_store_d<F16>(*a, stream); break;
  }
  return launched();
}

int ns_kv_scratch_bytes(int32_t num_pages, uint64_t* bytes) {
  if (!bytes) return fail("bytes is NULL");
  if (num_pages < 1) return fail("a pool needs pages (got %d)", num_pages);
  *bytes = scratch_bytes(num_pages);
  return 0;
}

int ns_kv_extend(const ns_kv_pool* p, const int32_t* rows, const int32_t* lens, int32_t n, hipStream_t stream) {
  if (check_list(p, rows, lens, n, kMaxRows)) return 1;
  if ((int64_t)n * p->num_cols >= ((int64_t)1 << 31)) return fail("rows times columns must lie below 2^31");
  if (n == 0) return 0;
  hipLaunchKernelGGL(extend_plan_kernel, dim3(plan_groups(p->num_pages)), dim3(kPlan), 0, stream, *p, rows, lens, n);
  const int64_t groups = ((int64_t)p->num_pages + kGroup - 1) / kGroup;
  hipLaunchKernelGGL(extend_kernel, dim3((unsigned)((groups + kCopy / 64 - 1) / (kCopy / 64))), dim3(kCopy), 0, stream, *p, n);
  return launched();
}

int ns_kv_fork(const ns_kv_pool* p, const int32_t* parents, const int32_t* children, int32_t n, hipStream_t stream) {
  if (check_list(p, parents, children, n, kMaxRows)) return 1;
  if (n == 0) return 0;
  hipLaunchKernelGGL(fork_plan_kernel, dim3(plan_groups(p->num_pages)), dim3(kPlan), 0, stream, *p, parents, children, n);
  hipLaunchKernelGGL(fork_kernel, dim3(n, p->num_tensors + 1), dim3(kCopy), 0, stream, *p, children);
  return launched();
}

int ns_kv_free(const ns_kv_pool* p, const int32_t* rows, int32_t n, hipStream_t stream) {
  if (check_list(p, rows, rows, n, INT32_MAX)) return 1;
  if (n == 0) return 0;
  hipLaunchKernelGGL((drop_kernel<true>), dim3(n), dim3(kCopy), 0, stream, *p, rows, 0, 0);
  return launched();
}

int ns_kv_release(const ns_kv_pool* p, const int32_t* rows, int32_t n, int32_t window, int32_t sinks, hipStream_t stream) {
  if (check_list(p, rows, rows, n, INT32_MAX)) return 1;
  if (window < 1) return fail("window must be at least 1 (got %d)", window);
  if (sinks < 0) return fail("sinks must be >= 0 (got %d)", sinks);
  if (n == 0) return 0;
  hipLaunchKernelGGL((drop_kernel<false>), dim3(n), dim3(kCopy), 0, stream, *p, rows, window, sinks);
  return launched();
}

int ns_kv_copy(const ns_kv_pool* p, const ns_kv_pool* to, const int32_t* src, const int32_t* dst, int32_t n,
               hipStream_t stream) {
  if (check_list(p, src, dst, n, INT32_MAX)) return 1;
  if (check_pool(to)) return 1;
  if (to->num_tensors != p->num_tensors || to->block_size != p->block_size || to->slot_bytes != p->slot_bytes)
    return fail("the two pools' pages differ");
  if (n == 0) return 0;
  hipLaunchKernelGGL(copy_kernel, dim3(n, p->num_tensors), dim3(kCopy), 0, stream, *p, to->tensors, to->num_pages, src, dst);
  return launched();
}

int ns_kv_compact(const ns_kv_pool* p, const ns_kv_pool* to, int32_t* page_map, hipStream_t stream) {
  if (check_pool(p)) return 1;
  if (!page_map) return fail("page_map is NULL");
  if (to) {
    if (check_pool(to)) return 1;
    if (to->num_tensors != p->num_tensors || to->block_size != p->block_size || to->slot_bytes != p->slot_bytes)
      return fail("the two pools' pages differ");
    if (to->num_rows != p->num_rows || to->num_cols != p->num_cols) return fail("the two pools' tables differ in size");
    if (to->page_refs == p->page_refs || to->block_tables == p->block_tables || to->seq_lens == p->seq_lens ||
        to->tensors == p->tensors)
      return fail("the two pools share a table or their tensors");
  }
  const ns_kv_pool q = to ? *to : *p;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlan), 0, stream, *p, to ? q.page_refs : nullptr, q.num_pages, page_map);
  hipLaunchKernelGGL(compact_kernel, dim3(p->num_rows + 2048), dim3(kCopy), 0, stream, *p, q, page_map, to ? 1 : 0);
  return launched();
}

}  // extern "C"
