// Attention with a sliding window and sinks, query tiles on the matrix core: part of ns_paged_attention.hip.
//
// The tiles, the steps of 64 positions, the operand layouts and the two-part weights are pa_prefill_kernel's.  A tile
// walks virtual positions: the sinks, then from the first token's window on (Hole), with what lies between left out.
// What differs, and what it measured (four 512-token chunks of 24 / 8 heads of 128 dims, bf16, window 2048, four sinks; the
// walk in runs of equal length with scalar row addresses, as without a window, 118.8 us):
//   * A step's rows are placed a lane a position: each lane maps its position, reads its block-table entry and checks
//     it, and the lanes that load the row take block and offset from it by a lane exchange: 116 us.  Placed by scalar
//     instructions, a load's four rows at a time, a step took some 700 of them a wave, more than its products.
//   * The window makes the tiles alike, so a workgroup takes a (tile, KV head): 113.6 us, with what follows and on a warm
//     GPU 105 to 107; or one of f.parts even parts of its steps where there are few of them: one chunk alone 73 us, 47 in
//     two parts (pw_parts_for has more).
//   * LDS reads run a few ahead of their products, and the weights of the next 16 positions are made between the
//     products of these, in an order that the compiler is held to: by itself it waits for each read before its product.
//     On the first walk that order changed nothing (119); it stays for its registers, which are known.
//   * Rows that no token of the tile sees are zeroed on their way to LDS, and a column whose output is not finite is
//     computed again in float arithmetic (plain_column): a weight of 0 times an infinite or NaN value that only other
//     tokens of the tile see must not reach it.
// Bound: the two waves of a SIMD between them, no pipe alone.  Without the weights' low parts (a third of the products)
// the first walk took 102 us, without the exponentials no less than with them, and with every step's rows read from the
// same place no less either.
#pragma once

namespace {

constexpr int kAheadK = 4, kAheadV = 2;   // LDS reads ahead of their products

// One query column of a tile by one wave in float arithmetic, 64 positions at a time: a lane a position for the scores,
// D / 64 dims a lane for the values.  What the windowed kernel falls back to for a column whose output is not finite
// though its sum is.
template <typename T, int D>
__device__ __forceinline__ void plain_column(const PaParams& p, const PfTile& t, int c, int G, int kvh, int lane) {
  using M = Mma<T>;
  constexpr int E = D / 64;
  const int tok = c / G, h = kvh * G + c % G;
  auto element = [](const void* base, int64_t at) -> float {
    return M::lo(reinterpret_cast<const uint16_t*>(base)[at]);
  };
  const int64_t q0 = (int64_t)(t.t0 + tok) * p.sq_tok + (int64_t)h * p.sq_head;
  const int n = min(t.kv_pos0 + tok + 1 - t.hole.gap, t.lt), h1 = t.hole.h1 + tok;
  const int32_t* bt_row = p.bt + (int64_t)t.seq * p.sbt;
  float o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  for (int v0 = 0; v0 < n; v0 += 64) {
    if (v0 >= p.sinks && v0 + 64 <= h1) continue;   // hidden
    const int v = v0 + lane, j = t.hole.position(min(v, n - 1));
    const int bi = j / p.block_size, off = j - bi * p.block_size;
    int blk = v < n && (v < p.sinks || v >= h1) && bi < p.max_blocks_per_seq ? bt_row[bi] : -1;
    if (blk >= p.num_blocks) blk = -1;
    const uint64_t seen = __ballot(blk >= 0);
    const int64_t krow = (int64_t)max(blk, 0) * p.sk_blk + (int64_t)off * p.sk_tok + (int64_t)kvh * p.sk_head;
    const int64_t vrow = (int64_t)max(blk, 0) * p.sv_blk + (int64_t)off * p.sv_tok + (int64_t)kvh * p.sv_head;
    float s = 0.f;
#pragma unroll 4
    for (int d = 0; d < D; d += 8) {
      const u32x4 a = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.q) + q0 + d);
      const u32x4 b = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.k) + krow + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s = fmaf(M::lo(a[i]) * p.scale_log2, M::lo(b[i]), s);
        s = fmaf(M::hi(a[i]) * p.scale_log2, M::hi(b[i]), s);
      }
    }
    if (blk < 0) s = -INFINITY;
    const float mn = fmaxf(m, wave_max(s));
    const float alpha = mn == -INFINITY ? 0.f : exp2f(m - mn), w = mn == -INFINITY ? 0.f : exp2f(s - mn);
    m = mn;
    l = fmaf(l, alpha, wave_sum(w));
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = alpha == 1.f ? o[i] : o[i] * alpha;
    for (int k0 = 0; k0 < 64; k0 += 16) {   // sixteen rows' loads together
      float x[16][E];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const uint64_t row = (uint32_t)__builtin_amdgcn_readlane((int)vrow, k0 + k) |
                             (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(vrow >> 32), k0 + k) << 32;
#pragma unroll
        for (int i = 0; i < E; ++i) x[k][i] = element(p.v, (int64_t)row + lane * E + i);
      }
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if ((seen >> (k0 + k)) & 1ull) {
          const float wk = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), k0 + k));
#pragma unroll
          for (int i = 0; i < E; ++i) o[i] = fmaf(wk, x[k][i], o[i]);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i)
    store_one<T>(p.out, (int64_t)(t.t0 + tok) * p.so_tok + (int64_t)h * p.so_head + lane * E + i,
                 quotient<true>(o[i], l));
}

template <typename T, int D, int G>
__global__ __launch_bounds__(kPfThreads) __attribute__((amdgpu_waves_per_eu(D == 128 ? 2 : 3, D == 128 ? 2 : 3))) void pa_window_kernel(PaParams p,
                                                                                                      PfParams f) {
  using M = Mma<T>;
  using vec = typename M::vec;
  constexpr int BQ = kPfCols / G;                 // tokens per tile
  constexpr int KS = D / 16;                      // k-steps of S^T = K Q^T
  constexpr int DB = D / 32;                      // 32-dim blocks of O^T
  constexpr int CPP = D / 8;                      // 16-byte chunks of a key or value row
  constexpr int LPT = kPfPos * CPP / kPfThreads;  // chunks of each kind a thread loads per step
  constexpr int PK = D * 2 + 16, PV = D * 2 + 64;   // bytes per staged row, as in pa_prefill_kernel
  static_assert(LPT * kPfThreads == kPfPos * CPP && kPfPos == 64, "a step's chunks split evenly, its positions are the lanes");
  __shared__ __align__(16) unsigned char s_k[2][kPfPos * PK];
  __shared__ __align__(16) unsigned char s_v[2][kPfPos * PV];
  __shared__ int s_last;

  // consecutive workgroups, which run on different XCDs, take a tile's KV heads
  const int kvh = (int)(blockIdx.x % p.hkv), tile = (int)(blockIdx.x / p.hkv % f.n_tiles);
  const int part = (int)(blockIdx.x / p.hkv / f.n_tiles);
  const PfTile t = pf_tile<true>(p, f, tile, BQ);
  if (threadIdx.x == 0 && kvh == 0 && part == 0 && p.status) {
    if (t.steps == 0) atomicOr(p.status, NS_PA_STATUS_BAD_TILE);
    if (t.cut) atomicOr(p.status, NS_PA_STATUS_SEQ_TOO_LONG);
  }
  // steps of a part: those of a tile shared evenly, none for some parts of a tile of few steps
  auto first_step = [&](int i) -> int { return (int)((int64_t)t.steps * i / f.parts); };
  const int off = first_step(part), take = first_step(part + 1) - off;
  if (take == 0) return;

  const float scale = f.scale_log2;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  uint64_t todo = 0ull;   // lanes whose columns' outputs are not finite though their sums are
  {
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c32 = lane & 31;
    const int dc0 = lane % CPP;   // every chunk of the thread has dims 8 dc0 .. + 7
    // the transposing read, as in pa_prefill_kernel
    const int tr_pos = 4 * h + ((lane & 15) >> 2), tr_dim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);

    const int j0 = off * kPfPos;
    const int j1 = t.lt < j0 + take * kPfPos ? t.lt : j0 + take * kPfPos;
    // the lane's column: token tok, head hd.  Visible virtual positions: below kvl (-1: a padding column, never
    // written), and not in [sinks, kvl - window); hidden from every token of the tile: [sinks, h1_t)
    const int c = wv * 32 + c32;
    const int tok = c / G, hd = c % G;
    const int h1_t = t.hole.h1;
    int kvl = -1;
    if (c < BQ * G && tok < t.nq) {
      const int seen = t.kv_pos0 + tok + 1 - t.hole.gap;
      const int kl = seen < t.lt ? seen : t.lt;
      kvl = kl > 0 ? kl : 0;
    }
    // the wave's tokens: positions from hi on and [sinks, h1_lo) are hidden from all of them, those from lo on and
    // [sinks, h1_hi) from some
    const int tok_lo = wv * 32 / G, tok_hi = min((wv * 32 + 31) / G, t.nq - 1);
    const bool live = tok_lo <= tok_hi;   // a wave of padding columns only loads rows
    const int h1_lo = h1_t + tok_lo, h1_hi = h1_t + tok_hi;
    const int lo = min(max(t.kv_pos0 + tok_lo + 1 - t.hole.gap, 0), j1);
    const int hi = t.kv_pos0 + tok_hi + 1 - t.hole.gap;
    const int32_t* bt_row = p.bt + (int64_t)t.seq * p.sbt;
    const char* kbase = reinterpret_cast<const char*>(p.k) + ((int64_t)kvh * p.sk_head + 8 * dc0) * 2;
    const char* vbase = reinterpret_cast<const char*>(p.v) + ((int64_t)kvh * p.sv_head + 8 * dc0) * 2;

    // Q^T operand: column c, dims 16 ks + 8 h .. + 7 (zeros for a padding column)
    vec qop[KS];
    {
      const int64_t qoff = (int64_t)(t.t0 + tok) * p.sq_tok + (int64_t)(kvh * G + hd) * p.sq_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        u32x4 x = {0u, 0u, 0u, 0u};
        if (kvl >= 0) x = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(p.q) + (qoff + 16 * ks + 8 * h) * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (x[i] & f.q_and) ^ f.q_xor;
        qop[ks] = __builtin_bit_cast(vec, x);
      }
    }

    // A step's positions, one a lane (every wave places all of them): the block-table entry is read one step ahead of
    // the rows, the rows one step ahead of the products.  Past the segment, its last position again.
    int entry = 0, slot = 0;   // of the step whose rows are loaded next
    auto place = [&](int jt) {
      const int j = t.hole.position(min(jt + lane, j1 - 1));
      int bi;
      if (p.bs_shift >= 0) { bi = j >> p.bs_shift; slot = j & (p.block_size - 1); }
      else { bi = j / p.block_size; slot = j - bi * p.block_size; }
      entry = bi < p.max_blocks_per_seq ? bt_row[bi] : -1;
    };
    u32x4 kreg[LPT], vreg[LPT];
    uint64_t gone = 0ull;   // positions of the loaded step whose block is invalid
    auto load_rows = [&](int jt) {
      gone = __ballot((uint32_t)entry >= (uint32_t)p.num_blocks);
      if (__builtin_expect(gone != 0ull, 0)) {
        // block 0 stands in, the rows are not used; flagged unless the window hides the block
        if ((uint32_t)entry >= (uint32_t)p.num_blocks) {
          const int bi = t.hole.position(min(jt + lane, j1 - 1)) / p.block_size;
          if (p.status && !hidden_block(p, bi, t.kv_pos0)) atomicOr(p.status, NS_PA_STATUS_BAD_BLOCK);
          entry = 0;
        }
      }
#pragma unroll
      for (int r = 0; r < LPT; ++r) {
        const int pos = (tid + kPfThreads * r) / CPP;
        const uint32_t b = (uint32_t)__shfl(entry, pos), o = (uint32_t)__shfl(slot, pos);
        // a slot's offset fits 32 bits (host)
        kreg[r] = *reinterpret_cast<const u32x4*>(kbase + ((int64_t)b * p.sk_blk + o * (uint32_t)p.sk_tok) * 2);
        vreg[r] = *reinterpret_cast<const u32x4*>(vbase + ((int64_t)b * p.sv_blk + o * (uint32_t)p.sv_tok) * 2);
      }
    };
    auto store_rows = [&](int jt, int buf) {
      // weight 0 times a row that is not of this sequence, or that no token of the tile sees, must be 0
      if (gone != 0ull || jt + kPfPos > j1 || (jt < h1_t && jt + kPfPos > p.sinks)) {
#pragma unroll
        for (int r = 0; r < LPT; ++r) {
          const int pos = (tid + kPfThreads * r) / CPP, j = jt + pos;
          if (((gone >> pos) & 1ull) || j >= j1 || (j >= p.sinks && j < h1_t)) vreg[r] = u32x4{0u, 0u, 0u, 0u};
        }
      }
#pragma unroll
      for (int r = 0; r < LPT; ++r) {
        const int pos = (tid + kPfThreads * r) / CPP;
        *reinterpret_cast<u32x4*>(s_k[buf] + pos * PK + dc0 * 16) = kreg[r];
        *reinterpret_cast<u32x4*>(s_v[buf] + pos * PV + dc0 * 16) = vreg[r];
      }
    };

    f32x16_t acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[db][e] = 0.f;
    float m = -INFINITY, l = 0.f;

    if (t.lt > 0) {
      place(j0);
      load_rows(j0);
      place(j0 + kPfPos);
      store_rows(j0, 0);
      __syncthreads();
    }
    int buf = 0;
    for (int jt = j0; jt < j1; jt += kPfPos, buf ^= 1) {
      // the next step's rows and the table entries of the one after it, in flight across this step's arithmetic
      const bool more = jt + kPfPos < j1;
      const uint64_t skip = gone;
      if (more) {
        load_rows(jt + kPfPos);
        place(jt + 2 * kPfPos);
      }
      if (live && jt < hi && (jt + kPfPos > h1_lo || jt < p.sinks)) {   // some column sees some of the step
        const unsigned char* kt = s_k[buf] + c32 * PK + 16 * h;
        const unsigned char* vt = s_v[buf] + tr_pos * PV + tr_dim * 2;
        // S^T = K Q^T for the step's two 32-position row blocks (i & 1)
        f32x16_t st[2];
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
          for (int e = 0; e < 16; ++e) st[rb][e] = 0.f;
        u32x4 kx[kAheadK];
        auto read_k = [&](int i) { kx[i % kAheadK] = *reinterpret_cast<const u32x4*>(kt + 32 * (i & 1) * PK + 32 * (i >> 1)); };
#pragma unroll
        for (int i = 0; i < kAheadK; ++i) read_k(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) {
          st[i & 1] = M::mma(__builtin_bit_cast(vec, kx[i % kAheadK]), qop[i >> 1], st[i & 1]);
          if (i + kAheadK < 2 * KS) read_k(i + kAheadK);
          __builtin_amdgcn_sched_barrier(0);
        }
        // element e of block rb: position 32 rb + 8 (e / 4) + 4 h + e % 4 of the step
        if (jt + kPfPos > lo || (jt < h1_hi && jt + kPfPos > p.sinks) || skip != 0ull) {   // one hidden from some column
          const int end = min(kvl, j1) - jt - 4 * h;
          const uint32_t hlen = (uint32_t)max(kvl - p.window - p.sinks, 0);
          const int from = jt + 4 * h - p.sinks;
          const uint64_t mask = skip >> (4 * h);
#pragma unroll
          for (int rb = 0; rb < 2; ++rb)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int r = 32 * rb + 8 * (e >> 2) + (e & 3);
              float x = st[rb][e];
              x = r < end ? x : -INFINITY;
              x = (uint32_t)(from + r) >= hlen ? x : -INFINITY;
              st[rb][e] = (uint32_t)(mask >> r) & 1u ? -INFINITY : x;
            }
        }
        // the online softmax, as in pa_prefill_kernel: a column's reference moves only for a score well above it
        float mt = -INFINITY;
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
          for (int e = 0; e < 16; ++e) mt = fmaxf(mt, st[rb][e]);
        mt = fmaxf(mt, __shfl_xor(mt, 32)) * scale;
        const bool move = mt > m + (M::kLift + M::kGap);
        const float mn = move ? mt - M::kLift : m;
        const float msub = mn == -INFINITY ? 0.f : mn;
        const float alpha = move ? __builtin_amdgcn_exp2f(m - msub) : 1.f;
        m = mn;
        if (__ballot(move) != 0ull) {
          l *= alpha;
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[db][e] *= alpha;
        }
        // per 16-position k-step s: P as the hi / lo B operands, then O^T += V^T P^T; the weights of k-step s + 1 are
        // made between the products of s
        u32x4 wh[2], wl[2];
        float ls = 0.f;   // a step's sum by itself: added to l one by one, equal weights err to one side in their thousands
        auto weigh = [&](int s, int i2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(st[s >> 1][8 * (s & 1) + 2 * i2], scale, -msub));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(st[s >> 1][8 * (s & 1) + 2 * i2 + 1], scale, -msub));
          ls += p0 + p1;
          const uint32_t x = M::pack2(p0, p1);
          wh[s & 1][i2] = x;
          wl[s & 1][i2] = M::pack2(p0 - M::lo(x), p1 - M::hi(x));
        };
        u32x4 vx[kAheadV];
        auto read_v = [&](int i) {   // k-step i / DB, dims 32 (i % DB) .. + 31
          const unsigned char* src = vt + 16 * (i / DB) * PV + 64 * (i % DB);
          const u32x2 lo4 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                          (__attribute__((address_space(3))) i16x4*)(src)));
          const u32x2 hi4 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                          (__attribute__((address_space(3))) i16x4*)(src + 8 * PV)));
          vx[i % kAheadV] = u32x4{lo4[0], lo4[1], hi4[0], hi4[1]};
        };
#pragma unroll
        for (int i = 0; i < kAheadV; ++i) read_v(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i2 = 0; i2 < 4; ++i2) weigh(0, i2);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4 * DB; ++i) {
          const int s = i / DB, db = i % DB;
          const vec x = __builtin_bit_cast(vec, vx[i % kAheadV]);
          acc[db] = M::mma(x, __builtin_bit_cast(vec, wh[s & 1]), acc[db]);
          acc[db] = M::mma(x, __builtin_bit_cast(vec, wl[s & 1]), acc[db]);
          if (i + kAheadV < 4 * DB) read_v(i + kAheadV);
          if (s < 3) {
#pragma unroll
            for (int i2 = db * 4 / DB; i2 < (db + 1) * 4 / DB; ++i2) weigh(s + 1, i2);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        l += ls;
      }
      if (more) store_rows(jt + kPfPos, buf ^ 1);
      __syncthreads();   // the next step staged, this one read
    }
    l += __shfl_xor(l, 32);   // the other half's positions

    // O^T layout: lane, element e -> column c, dim 32 db + 8 (e / 4) + 4 h + e % 4
    auto write_out = [&](const f32x16_t (&o)[DB], float sum) -> bool {
      if (kvl < 0) return false;
      const int64_t obase = (int64_t)(t.t0 + tok) * p.so_tok + (int64_t)(kvh * G + hd) * p.so_head + 4 * h;
      const float inv = sum != 0.f ? 1.f / sum : 0.f;   // no visible key: zeros; NaN scores: NaN
      float z = 0.f;   // NaN with an output that is not finite
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = sum != 0.f ? o[db][4 * e4 + i] * inv : 0.f;
            z = fmaf(o[db][4 * e4 + i], 0.f, z);
          }
          const int64_t d = obase + 32 * db + 8 * e4;
          if (f.out_vec) {
            *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + d) =
                u32x2{M::pack2(x[0], x[1]), M::pack2(x[2], x[3])};
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) store_one<T>(p.out, d + i, x[i]);
          }
        }
      return z != 0.f && sum == sum;   // with a NaN among the column's scores it all is NaN
    };
    if (take == t.steps) {
      todo = __ballot(write_out(acc, l));
    } else {
      // a tile in parts: this one's partials to its slot, in the lanes' accumulator layout (agent-scope stores: the
      // parts' workgroups run on different XCDs)
      const int th = kvh * f.n_tiles + tile;
      constexpr int SW = D / 2 * 64;   // floats of a slot per wave
      const int64_t slot0 = (int64_t)th * f.parts;
      if (live) {
        float* dst = f.ws_acc + ((slot0 + part) * kPfWaves + wv) * SW + 2 * lane;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 16; e += 2) st_dev2(dst + (db * 16 + e) * 64, acc[db][e], acc[db][e + 1]);
        if (h == 0) st_dev2(f.ws_ml + ((slot0 + part) * kPfCols + c) * 2, m, l);
      }
      // the last part to arrive merges (the partials crossed through agent-scope atomic stores completed by the
      // s_waitcnt, read back through agent-scope loads)
      const int arrivals = t.steps < f.parts ? t.steps : f.parts;
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      int32_t* counter = f.counters + th;
      if (tid == 0) s_last = atomicAdd(counter, 1) == arrivals - 1;
      __syncthreads();
      if (!s_last) return;
      if (tid == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (live) {
        float mx = -INFINITY;
        for (int i = 0; i < f.parts; ++i)
          if (first_step(i) < first_step(i + 1)) mx = fmaxf(mx, ld_dev2(f.ws_ml + ((slot0 + i) * kPfCols + c) * 2)[0]);
        float L = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[db][e] = 0.f;
        for (int i = 0; i < f.parts; ++i) {
          if (first_step(i) == first_step(i + 1)) continue;
          const float* src = f.ws_acc + ((slot0 + i) * kPfWaves + wv) * SW + 2 * lane;
          const f32x2 ml = ld_dev2(f.ws_ml + ((slot0 + i) * kPfCols + c) * 2);
          f32x2 x[D / 4];   // all of a part's loads issued before the first is used
#pragma unroll
          for (int e = 0; e < D / 4; ++e) x[e] = ld_dev2(src + e * 128);
          // a part whose keys were all skipped (m = -inf) weighs 0
          const float wt = ml[0] == -INFINITY ? 0.f : exp2f(ml[0] - mx);
          L = fmaf(wt, ml[1], L);
#pragma unroll
          for (int e = 0; e < D / 4; ++e) {
            acc[e / 8][2 * (e % 8)] = fmaf(wt, x[e][0], acc[e / 8][2 * (e % 8)]);
            acc[e / 8][2 * (e % 8) + 1] = fmaf(wt, x[e][1], acc[e / 8][2 * (e % 8) + 1]);
          }
        }
        todo = __ballot(write_out(acc, L));
      }
    }
  }
  if (__builtin_expect(todo != 0ull, 0)) {
    // An infinite or NaN value makes NaN of the zero weight that a token of the tile has which does not see it, and of
    // the two parts of one that does where infinity is right: those columns again, over the outputs just written.  (The
    // arguments are read anew, hidden from the compiler, which would hold them in registers throughout.)
    __builtin_amdgcn_s_waitcnt(0);
    uint64_t args = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    const PaParams pa = *reinterpret_cast<const PaParams*>(args);
    for (todo = (todo | todo >> 32) & 0xffffffffull; todo != 0ull; todo &= todo - 1ull)
      plain_column<T, D>(pa, t, 32 * wv + __ffsll((unsigned long long)todo) - 1, G, kvh, (int)threadIdx.x & 63);
  }
}

}  // namespace
