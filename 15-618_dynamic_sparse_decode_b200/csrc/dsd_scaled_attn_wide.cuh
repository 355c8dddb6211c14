// dsd_scaled_attn_wide.cuh -- attention over the scaled 8-bit cache for many query
// rows per key head (prompt chunks, drafted tokens, large groups): 128 rows at a
// time on the fp16 tensor cores.
//
//   S[row][token] = Q[row][d] K[token][d]^T      O[row][d] += P[row][token] V[token][d]
//
// With many rows the tile's codes are worth widening once: e4m3 and int8 are exact
// in fp16, so four warps write each K and V tile as fp16 operands and one product
// does what the narrow kernel needs three 8-bit pieces for.  Queries are scaled by
// a power of two of their row into fp16's range (exact for fp16 and for bf16 within
// 2^-29 of the row's largest).
//
// A weight carries its value scale: P = 2^(s - r) vs, fp16, back in TMEM as the A
// operand of the second product, so that O / sum is the output as it stands.  The
// row's reference r bounds the largest weight that it SEES from above.  Where every
// row sees a whole tile and the tile's value scales lie within 2^8 of one another,
// the largest logit and the largest scale bound it closely enough, and a column has
// two constants, its scales (with the exponent of vs in the logits, as in the narrow
// kernel, it had four: chunks 522 us, with two 489 us).  Elsewhere r comes from each
// seen token's own logit and exponent: what a row does not see must not move its
// weights, and a token with a large scale and next to no weight must not push the
// others out of fp16 (chunks 502 us with the first bound for every tile, 507 us so).
// A weight keeps its bits down to 2^-11 of the row's largest and an absolute 2^-22
// of it below.
//
// The reference stays while nothing has grown past it by more than 2^8, which fp16
// weights bear, so a tile is one pass over its logits; else the eight warps vote, O
// is rescaled in TMEM and the weights are made again (a pass for the maximum every
// tile: 544 us).  A thread owns half a row of S, 32 columns at a time: 64 values
// kept in registers left none to load ahead with (759 us), and sixteen warps with a
// quarter each came out at 766 us.
//
// Bound: the softmax warps' latency (the tensor cores are 20% busy, ex2 21%); three
// requests of 300-700 queries over 5000-9000 tokens, 32 heads over 8: 0.50-0.51 ms, 467
// TFLOP/s of the 1679 a bf16 product reaches.
//
// Roles: warps 0-7 softmax, 8-11 widen the codes, 12 TMA, 13 MMA issue, 14 token
// data, 15 units.
#pragma once

#include "dsd_scaled_attn_tc.cuh"

namespace dsds {

constexpr int kWideThreads = 512;
constexpr int kWideRows = 128;
constexpr float kWideGrow = 8.0f;     // log2 of how far a maximum may run behind
constexpr float kWideOne = 6.0f;      // log2 of the largest weight on a fresh reference

// PP: fp16 pieces of a weight.  One for bf16, whose outputs are far coarser than a
// weight's 2^-12; two for fp16, or the weights' rounding would add to the output's
// own.  fp32 rows stay with the narrow kernel: the accumulator's adds truncate, and
// sums over 60000 tokens in it came out 1.6e-5 off, against 3e-7 there.
template <int PP>
struct WideShape {
  static constexpr int kStages = 2;
  static constexpr int kTile16 = 2 * kTcTileBytes;   // a tile of 128 x 128 fp16
  static constexpr size_t kSmem = 1024 + size_t(kStages) * 2 * kTcTileBytes + 4 * size_t(kTile16);
  // TMEM columns: S twice, O, P
  static constexpr int kO = 256, kP = 384, kColumns = 512;
};

__device__ __forceinline__ bool wide_sync_or(bool flag) {
  uint32_t any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(any) : "r"(uint32_t(flag)) : "memory");
  return any != 0;
}

// D (fp32) [128][n], A and B fp16; b_n_major: B's columns are adjacent.
__device__ __forceinline__ uint32_t wide_desc(int n, bool b_n_major) {
  return (1u << 4) | (b_n_major ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"(uint32_t(add)) : "memory");
}
__device__ __forceinline__ void mma_f16_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(desc), "r"(uint32_t(add)) : "memory");
}
// 64 fp16 columns (128 bytes) a row, swizzled; the second 64 lie 16 KiB behind.
__device__ __forceinline__ uint64_t operand16_desc(uint32_t addr) {
  return (uint64_t(addr >> 4) & 0x3FFF) | (uint64_t(kTcTileBytes >> 4) << 16) | (uint64_t(64) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}

__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&x)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(addr), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(x[8]),
               "r"(x[9]), "r"(x[10]), "r"(x[11]), "r"(x[12]), "r"(x[13]), "r"(x[14]), "r"(x[15]) : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two fp32 values in a register pair (packed fp32 instructions).
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t x;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
  return x;
}
__device__ __forceinline__ uint64_t pair(uint32_t a, uint32_t b) {
  uint64_t x;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "r"(a), "r"(b));
  return x;
}
__device__ __forceinline__ void unpair(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t x;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(x) : "l"(a), "l"(b), "l"(c));
  return x;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t x;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(a), "l"(b));
  return x;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t x;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(a), "l"(b));
  return x;
}
__device__ __forceinline__ uint64_t ex2_pair(uint64_t x) {
  float a, b;
  unpair(x, a, b);
  return pair(ex2(a), ex2(b));
}
__device__ __forceinline__ float max_pair(float m, uint64_t x) {
  float a, b;
  unpair(x, a, b);
  return fmaxf(m, fmaxf(a, b));
}
// w * x, 0 where w is 0 whatever x is
__device__ __forceinline__ uint64_t seen_product(uint64_t w, uint64_t x) {
  float a, b, c, d;
  unpair(w, a, b);
  unpair(x, c, d);
  return pair(a != 0.0f ? a * c : 0.0f, b != 0.0f ? b * d : 0.0f);
}

// 16 codes as fp16, exactly.
template <bool I8>
__device__ __forceinline__ void widen16(uint4 c, uint4& lo, uint4& hi) {
  const uint32_t in[4] = {c.x, c.y, c.z, c.w};
  uint32_t out[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (I8) {
      // 0x64uu is 1024 + u: with u = code + 128, less 1152
      const uint32_t u = in[i] ^ 0x80808080u;
      const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
      uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
      const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off), y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
      out[2 * i] = *reinterpret_cast<const uint32_t*>(&x);
      out[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
    } else {
      asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
          : "=r"(out[2 * i]), "=r"(out[2 * i + 1]) : "r"(in[i]));
    }
  }
  lo = make_uint4(out[0], out[1], out[2], out[3]);
  hi = make_uint4(out[4], out[5], out[6], out[7]);
}

// Row `t` of a swizzled code tile into the fp16 tile; all loads before the first use.
template <bool I8>
__device__ __forceinline__ void widen_row(const uint8_t* codes, uint8_t* wide, int t, bool zero) {
  uint4 raw[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) raw[j] = *reinterpret_cast<const uint4*>(codes + (t * 128 + (j << 4) ^ (t & 7) << 4));
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint4 lo, hi;
    if (zero) raw[j] = make_uint4(0, 0, 0, 0);   // code 0 is 0 in both formats
    widen16<I8>(raw[j], lo, hi);
    uint8_t* to = wide + (j >> 2) * kTcTileBytes;
    *reinterpret_cast<uint4*>(to + (t * 128 + ((2 * j & 7) << 4) ^ (t & 7) << 4)) = lo;
    *reinterpret_cast<uint4*>(to + (t * 128 + ((2 * j & 7) + 1 << 4) ^ (t & 7) << 4)) = hi;
  }
}

// Exponent that bounds a value scale from above, in the range of token_scale().
__device__ __forceinline__ int scale_bound(float vs) {
  return min(max(static_cast<int>(__float_as_uint(vs) >> 23 & 255) - 126, -64), 100);
}
constexpr int kWideSpread = 8;   // log2 of how far a tile's value scales may lie apart under one bound

// A tile's tokens as the softmax reads them, four at a time.
struct __align__(16) Columns {   // its size too: float4 reads of the second one
  float ks[kTile], vs[kTile], bound[kTile];   // bound: scale_bound(vs), with one piece
  uint32_t valid[4];   // a bit per token
  int largest[4], least[4];   // bounding exponents of each 32 tokens' value scales
  int place, open;     // open: every row sees every token that is there
};

template <bool I8, int PP>
__global__ void __launch_bounds__(kWideThreads, 1)
attn_wide_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap k_map,
                 const __grid_constant__ CUtensorMap v_map, int head_first) {
  using Shape = WideShape<PP>;
  constexpr int STAGES = Shape::kStages;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* base = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
  uint8_t* k_ring = base;
  uint8_t* v_ring = k_ring + STAGES * kTcTileBytes;
  uint8_t* k16 = v_ring + STAGES * kTcTileBytes;
  uint8_t* v16 = k16 + Shape::kTile16;
  uint8_t* q16 = v16 + 2 * Shape::kTile16;
  __shared__ uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
  __shared__ uint64_t k16_full, k16_empty, v16_full[2], v16_empty[2], s_full[2], s_empty[2], p_full, o_full, q_full;
  __shared__ uint64_t cols_full[2], cols_empty[2], unit_full[2], unit_empty[2];
  __shared__ uint64_t token_full[kTokenStages], token_empty[kTokenStages], drained;
  __shared__ TileInfo info[kTokenStages];
  __shared__ __align__(16) uint8_t token_smem[kTokenBytes];
  __shared__ __align__(16) Columns cols[2];
  __shared__ float red[2][2][kWideRows];
  __shared__ UnitInfo units[2];
  __shared__ uint32_t tmem_base;
  __shared__ int stop;
  __shared__ Walk walk_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = blockIdx.x, head = cta % p.Hk;

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 4);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&v16_full[i], 4);
      mbar_init(&v16_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 8);
      mbar_init(&cols_full[i], 4);
      mbar_init(&cols_empty[i], 8);
      mbar_init(&unit_full[i], 1);
      mbar_init(&unit_empty[i], 9);   // the softmax warps and the MMA warp
    }
    mbar_init(&k16_full, 4);
    mbar_init(&k16_empty, 1);
    mbar_init(&p_full, 8);
    mbar_init(&o_full, 1);
    mbar_init(&q_full, 8);
    for (int i = 0; i < kTokenStages; ++i) {
      mbar_init(&token_full[i], 64);
      mbar_init(&token_empty[i], 4);
    }
    mbar_init(&drained, 1);
    stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
  }
  pdl_wait();
  pdl_trigger();
  if (tid == 0) p.meta[cta] = make_int4(0, 0, -1, 0);
  plan_walk<kWideThreads>(p, cta / p.Hk, reinterpret_cast<int*>(k_ring), &walk_s);
  Walk w = walk_s;
  if (w.left == 0) return;
  proxy_fence();   // the plan's scratch lay in the ring
  if (warp == 13) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                 "r"(Shape::kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  if (warp == 12) {
    walk_boxes<STAGES>(p, w, head, k_map, v_map, head_first, k_ring, v_ring, k_full, k_empty, v_full, v_empty, &stop);
  } else if (warp == 14) {
    walk_tokens(p, w, head, TokenRing(token_smem, p), info, token_full, token_empty, &stop);
  } else if (warp == 15) {
    // ---- units
    bool ok = true;
#pragma unroll 1
    for (uint32_t unit = 0; ok; ++unit) {
      const int u = unit & 1;
      const bool end = w.left <= 0;
      const Request r = w.r;
      const Span span = w.span;
      const int slots = slots_of(span);
      const Segment seg = segment_of(w, slots);
      ok = __all_sync(~0u, mbar_wait(&unit_empty[u], (unit >> 1 & 1) ^ 1, &stop, p.status));
      if (!ok) break;
      if (lane == 0) {
        UnitInfo& x = units[u];
        x.tiles = end ? -1 : span.n == 0 ? 0 : seg.n;
        x.b = w.b;
        x.qt = w.qt;
        x.rows = r.rows;
        x.q0 = r.q0;
        x.base_pos = r.len - r.nq;
        x.opens = seg.opens;
        x.ends = seg.ends;
        x.last_slot = w.at - w.slot + slots - 1;
        mbar_arrive(&unit_full[u]);
      }
      __syncwarp();
      if (end) break;
      next_unit(p, seg, w);
    }
  } else if (warp == 13) {
    // ---- MMA issue
    const bool leader = elect_one();
    const uint32_t s_desc = wide_desc(kTile, false), o_desc = wide_desc(p.D, true);
    const uint64_t k_d = operand16_desc(smem_addr(k16)), v_d = operand16_desc(smem_addr(v16)), q_d = operand16_desc(smem_addr(q16));
    const auto all = [&](uint64_t* bar, int parity) { return __all_sync(~0u, mbar_wait(bar, parity, &stop, p.status)) != 0; };
    uint32_t g = 0, unit = 0, with_tiles = 0;
    int left = 0;
    bool ok = true, owed = false, owed_first = false, first = false, end = false;
    const auto weigh = [&]() {   // O of tile g - 1
      const int t = g - 1;
      owed = false;
      ok = ok && all(&p_full, t & 1) && all(&v16_full[t & 1], t >> 1 & 1);
      if (!ok) return;
      tc_fence_after();
      if (leader) {
        const uint64_t v = v_d + (t & 1) * (Shape::kTile16 >> 4);
#pragma unroll
        for (int piece = 0; piece < PP; ++piece)
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mma_f16_tmem(tmem + Shape::kO, tmem + Shape::kP + piece * 64 + 8 * k, v + 128 * k, o_desc, !owed_first || k > 0 || piece > 0);
        mma_commit(&v16_empty[t & 1]);
        mma_commit(&o_full);
      }
      __syncwarp();
    };
#pragma unroll 1
    while (ok && !(end && !owed)) {
      if (left == 0 && !end) {
        if (owed) {
          weigh();   // the next queries overwrite nothing that it reads, but wait for its result
          continue;
        }
        const int u = unit & 1;
        ok = all(&unit_full[u], unit >> 1 & 1);
        if (!ok) break;
        left = units[u].tiles;
        __syncwarp();
        if (lane == 0) mbar_arrive(&unit_empty[u]);
        ++unit;
        end = left < 0;
        first = true;
        if (left > 0) {
          ok = all(&q_full, with_tiles & 1);
          ++with_tiles;
        }
        continue;
      }
      const bool more = !end;
      if (more) {
        const int buf = g & 1;
        ok = all(&k16_full, g & 1) && all(&s_empty[buf], (g >> 1 & 1) ^ 1);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const int steps = p.D / 16;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < steps) {
              const int at = (k >> 2) * (kTcTileBytes >> 4) + 2 * (k & 3);
              mma_f16(tmem + buf * kTile, q_d + at, k_d + at, s_desc, k > 0);
            }
          mma_commit(&k16_empty);
          mma_commit(&s_full[buf]);
        }
        __syncwarp();
        --left;
      }
      if (owed) weigh();
      if (more) {
        owed = true;
        owed_first = first;
        first = false;
        ++g;
      }
    }
    if (!ok) {
      int never = 0;
      if (leader) mma_commit(&drained);
      mbar_wait_slow(&drained, 0, &never, nullptr);
      __syncwarp();
    }
  } else if (warp >= 8) {
    // ---- widen: thread = token; its data, then its K row, then its V row
    const TokenRing ring(token_smem, p);
    const int t = tid - 256, here = p.tpp ? kTile : p.ppt * p.P;
    const int my_entry = t / p.by_block, my_place = t % p.by_block;
    int ts = 0, tp = 0, s = 0, sp = 0;   // stage and phase of the token and code rings
    uint32_t g = 0;
    bool ok = true;
    // of the units only the number of tiles matters here
    int tiles_left = 0;
#pragma unroll 1
    while (w.left > 0) {
      const Span span = w.span;
      const Segment seg = segment_of(w, slots_of(span));
      tiles_left += span.n == 0 ? 0 : seg.n;
      next_unit(p, seg, w);
    }
#pragma unroll 1
    for (; tiles_left > 0 && ok; --tiles_left, ++g) {
      const int cb = g & 1;
      ok = ok && mbar_wait(&token_full[ts], tp, &stop, p.status);
      const TileInfo tile = info[ts];
      int entry = my_entry, in_block = my_place;
      if (tile.lead) {
        entry = (tile.lead + t) / p.by_block;
        in_block = (tile.lead + t) % p.by_block;
      }
      entry += ts * ring.entries;
      const bool valid = t < here && in_block < ring.limit[entry];
      const float2 scales = ring.scales[entry];
      __syncwarp();
      if (lane == 0) mbar_arrive(&token_empty[ts]);
      if (++ts == ring.stages) {
        ts = 0;
        tp ^= 1;
      }
      const uint8_t* k_codes = k_ring + s * kTcTileBytes;
      const uint8_t* v_codes = v_ring + s * kTcTileBytes;
      ok = ok && mbar_wait(&k_full[s], sp, &stop, p.status) && mbar_wait(&k16_empty, (g & 1) ^ 1, &stop, p.status);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      widen_row<I8>(k_codes, k16, t, !valid);
      proxy_fence();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&k16_full);
        mbar_arrive(&k_empty[s]);
      }
      // see the narrow kernel: a value row with NaN that some row must not see
      bool nan_row = false;
      if (!I8 && !tile.open) {
        ok = ok && mbar_wait(&v_full[s], sp, &stop, p.status);
        nan_row = valid && row_has_nan(reinterpret_cast<const uint4*>(v_codes + t * 128), lane);
      }
      const float vs = !valid ? 0.0f : nan_row ? NAN : scales.y;
      const uint32_t present = __ballot_sync(~0u, valid);
      const int largest = __reduce_max_sync(~0u, scale_bound(vs)), least = __reduce_min_sync(~0u, scale_bound(vs));
      ok = ok && mbar_wait(&cols_empty[cb], (g >> 1 & 1) ^ 1, &stop, p.status);
      Columns& c = cols[cb];
      c.ks[t] = valid ? scales.x : 0.0f;
      c.vs[t] = vs;
      if constexpr (PP == 1) c.bound[t] = static_cast<float>(scale_bound(vs));
      if (lane == 0) {
        c.valid[t >> 5] = present;
        c.largest[t >> 5] = largest;
        c.least[t >> 5] = least;
      }
      if (t == 0) {
        c.place = tile.place;
        c.open = tile.open;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&cols_full[cb]);
      ok = ok && mbar_wait(&v_full[s], sp, &stop, p.status) && mbar_wait(&v16_empty[cb], (g >> 1 & 1) ^ 1, &stop, p.status);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      widen_row<I8>(v_codes, v16 + cb * Shape::kTile16, t, !valid || nan_row);
      proxy_fence();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&v16_full[cb]);
        mbar_arrive(&v_empty[s]);
      }
      if (++s == STAGES) {
        s = 0;
        sp ^= 1;
      }
    }
  } else {
    // ---- softmax: row = lane of the warp's quarter, half of the tile's columns
    const int row = tid & 127, half = tid >> 7;
    const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
    const int d_half = (p.D / 2 + 15) / 16 * 16;   // output elements of the first half, in steps of 16
    // 16-byte accesses where every row starts on their boundary
    const bool q_aligned = reinterpret_cast<uintptr_t>(p.q) % 16 == 0 && p.qst[0] % 8 == 0 && p.qst[1] % 8 == 0;
    const bool out_aligned = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.ost[0] % 8 == 0 && p.ost[1] % 8 == 0;
    uint32_t g = 0;
    bool ok = true;
#pragma unroll 1
    for (uint32_t unit = 0; ok; ++unit) {
      const int u = unit & 1;
      ok = !wide_sync_or(!mbar_wait(&unit_full[u], unit >> 1 & 1, &stop, p.status));
      if (!ok) break;
      const UnitInfo x = units[u];
      if (x.tiles < 0) break;
      const int row0 = x.qt * kWideRows, gr = min(row0 + row, x.rows - 1);
      const bool mine = row0 + row < x.rows;
      const int qi = gr / p.by_group, q_head = head * p.G + gr % p.by_group;
      const int pos = x.base_pos + qi;
      float factor = 0.0f;
      if (x.tiles > 0) {
        // queries: half a row a thread, scaled by the row's power of two
        const uint16_t* q = static_cast<const uint16_t*>(p.q) + 1ll * (x.q0 + qi) * p.qst[0] + 1ll * q_head * p.qst[1] + 64 * half;
        const int n = mine ? min(max(p.D - 64 * half, 0), 64) : 0;   // a multiple of 16
        uint4 raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = make_uint4(0, 0, 0, 0);
        if (q_aligned) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (8 * i < n) raw[i] = reinterpret_cast<const uint4*>(q)[i];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (8 * i < n)
              raw[i] = make_uint4(q[8 * i] | q[8 * i + 1] << 16, q[8 * i + 2] | q[8 * i + 3] << 16,
                                  q[8 * i + 4] | q[8 * i + 5] << 16, q[8 * i + 6] | q[8 * i + 7] << 16);
        }
        const auto values = [&](int i, int j) {   // elements 8 i + 4 j to + 3
          return widen_four(make_uint4(j ? raw[i].z : raw[i].x, j ? raw[i].w : raw[i].y, 0, 0), p.dtype);
        };
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float4 y = values(i / 2, i & 1);
          top = max(top, max(max(__float_as_uint(fabsf(y.x)), __float_as_uint(fabsf(y.y))),
                             max(__float_as_uint(fabsf(y.z)), __float_as_uint(fabsf(y.w)))));
        }
        red[0][half][row] = __uint_as_float(top);
        wide_sync_or(false);
        top = max(__float_as_uint(red[0][0][row]), __float_as_uint(red[0][1][row]));
        const int e = max(static_cast<int>(top >> 23) - 127, -100);
        // a negative scale turns the query: the largest product is the largest logit then
        const float f = copysignf(__uint_as_float(uint32_t(14 - e + 127) << 23), p.scale_log2);
        factor = top >= 0x7f800000u ? NAN : fabsf(p.scale_log2) * __uint_as_float(uint32_t(e - 14 + 127) << 23);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t out[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float4 y = values(i, j);
            const __half2 a = __floats2half2_rn(y.x * f, y.y * f), b = __floats2half2_rn(y.z * f, y.w * f);
            out[2 * j] = *reinterpret_cast<const uint32_t*>(&a);
            out[2 * j + 1] = *reinterpret_cast<const uint32_t*>(&b);
          }
          *reinterpret_cast<uint4*>(q16 + half * kTcTileBytes + row * 128 + ((i ^ (row & 7)) << 4)) =
              make_uint4(out[0], out[1], out[2], out[3]);
        }
        proxy_fence();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full);
        wide_sync_or(false);   // `red` is free again
      }

      float m = -INFINITY, l = 0.0f;   // the reference of the weights; the sum
#pragma unroll 1
      for (int i = 0; i < x.tiles && ok; ++i, ++g) {
        const int buf = g & 1;
        const Columns& c = cols[buf];
        bool in = mbar_wait(&cols_full[buf], g >> 1 & 1, &stop, p.status);
        in = mbar_wait(&s_full[buf], g >> 1 & 1, &stop, p.status) && in;
        __syncwarp();
        tc_fence_after();
        const uint4 valid = *reinterpret_cast<const uint4*>(c.valid);
        const int4 largest = *reinterpret_cast<const int4*>(c.largest), least = *reinterpret_cast<const int4*>(c.least);
        const int up = max(max(largest.x, largest.y), max(largest.z, largest.w));
        // every row sees all places, and 2^up bounds their value scales closely
        const bool open = c.open != 0 && (valid.x & valid.y & valid.z & valid.w) == ~0u &&
                          up - min(min(least.x, least.y), min(least.z, least.w)) <= kWideSpread;
        // P and O are the last tile's until its product is done
        if (i > 0) {
          in = mbar_wait(&o_full, (g - 1) & 1, &stop, p.status) && in;
          __syncwarp();
          tc_fence_after();
        }
        // The half's weights under the reference r, into P; their sum and what bounds the
        // largest: of an open tile the largest product S ks, else of what the row sees the
        // largest logit with its scale's exponent.  Values lie two to a register pair: one
        // instruction for both.
        const auto weigh = [&](float r, float& top) {
          const uint64_t factor2 = pair(factor, factor), r2 = pair(-r, -r);
          float sum = 0.0f;
#pragma unroll 1
          for (int at = 64 * half; at < 64 * half + 64; at += 32) {
            uint32_t raw[32];
            tmem_load<32>(lanes + buf * kTile + at, raw);
            ulonglong2 k[8], v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) k[j] = *reinterpret_cast<const ulonglong2*>(&c.ks[at + 4 * j]);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = *reinterpret_cast<const ulonglong2*>(&c.vs[at + 4 * j]);
            tmem_load_wait();
            float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            uint64_t sums[2] = {0, 0}, s[16];
            if (open) {
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const uint64_t x = mul2(pair(raw[2 * j], raw[2 * j + 1]), j & 1 ? k[j / 2].y : k[j / 2].x);
                t[j & 3] = max_pair(t[j & 3], x);
                const uint64_t w = ex2_pair(fma2(x, factor2, r2));
                sums[j & 1] = add2(sums[j & 1], w);
                s[j] = mul2(w, j & 1 ? v[j / 2].y : v[j / 2].x);
              }
            } else {
              // columns lo .. hi are the row's to see
              const int hi = (p.causal ? pos - c.place : kTile) - at;
              const int lo = (p.window ? max(max(pos - c.place, -1) - p.window + 1, 0) : 0) - at;
              const uint32_t there = c.valid[at / 32];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                float a, b;
                unpair(mul2(pair(raw[2 * j], raw[2 * j + 1]), j & 1 ? k[j / 2].y : k[j / 2].x), a, b);
                const bool see_a = (there >> (2 * j) & 1) && 2 * j <= hi && 2 * j >= lo;
                const bool see_b = (there >> (2 * j + 1) & 1) && 2 * j + 1 <= hi && 2 * j + 1 >= lo;
                // from shared memory chunks take 507 us, made here 517; with two pieces 576 and 562
                float2 bound;
                if constexpr (PP == 1) {
                  bound = *reinterpret_cast<const float2*>(&c.bound[at + 2 * j]);
                } else {
                  unpair(j & 1 ? v[j / 2].y : v[j / 2].x, bound.x, bound.y);
                  bound = make_float2(static_cast<float>(scale_bound(bound.x)), static_cast<float>(scale_bound(bound.y)));
                }
                t[j & 3] = fmaxf(t[j & 3], fmaxf(see_a ? fmaf(a, factor, bound.x) : -INFINITY,
                                                 see_b ? fmaf(b, factor, bound.y) : -INFINITY));
                const uint64_t w = pair(see_a ? ex2(fmaf(a, factor, -r)) : 0.0f, see_b ? ex2(fmaf(b, factor, -r)) : 0.0f);
                sums[j & 1] = add2(sums[j & 1], w);
                // the scale of a place that the row does not see may be NaN
                s[j] = seen_product(w, j & 1 ? v[j / 2].y : v[j / 2].x);
              }
            }
            top = fmaxf(top, fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])));
            float x0, x1;
            unpair(add2(sums[0], sums[1]), x0, x1);
            sum += x0 + x1;
#pragma unroll
            for (int piece = 0; piece < PP; ++piece) {
              uint32_t out[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                unpair(s[j], x0, x1);
                const __half2 h = __floats2half2_rn(x0, x1);
                out[j] = *reinterpret_cast<const uint32_t*>(&h);
                if (piece + 1 < PP) {
                  const float2 b = __half22float2(h);
                  s[j] = pair(x0 - b.x, x1 - b.y);
                }
              }
              tmem_store16(lanes + Shape::kP + piece * 64 + at / 2, out);
            }
          }
          return sum;
        };
        // One pass on the reference of the tiles so far; where a row's largest weight
        // has grown past what fp16 bears (seldom after the first tile), all eight warps
        // agree on new references and make the weights again.
        float top = -INFINITY;
        float sum = weigh(m == -INFINITY ? 0.0f : m, top);
        // the reference that this tile alone would take (-inf: the row sees nothing of it)
        const auto fresh = [&](float t) {
          return t == -INFINITY ? -INFINITY : (open ? fmaf(t, factor, float(up)) : t) - kWideOne;
        };
        const auto grown = [&](float f) { return f > m + kWideGrow || (m == -INFINITY && f > m); };
        if (wide_sync_or(grown(fresh(top)) || !in)) {
          ok = !wide_sync_or(!in);
          if (!ok) break;
          red[buf][half][row] = top;
          wide_sync_or(false);
          const float now = fresh(fmaxf(top, red[buf][half ^ 1][row]));
          float a = 1.0f;
          if (grown(now)) {
            a = ex2(m - now);   // 0 from -inf
            l *= a;
            m = now;
          }
          sum = weigh(m == -INFINITY ? 0.0f : m, top);
          if (i > 0) {
#pragma unroll 1
            for (int at = half ? d_half : 0; at < (half ? p.D : d_half); at += 16) {
              uint32_t o[16];
              tmem_load<16>(lanes + Shape::kO + at, o);
              tmem_load_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * a);
              tmem_store16(lanes + Shape::kO + at, o);
            }
          }
        }
        l += sum;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[buf]);
        tmem_store_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&cols_empty[buf]);
          mbar_arrive(&p_full);
        }
      }
      if (x.tiles > 0 && ok) {
        ok = mbar_wait(&o_full, (g - 1) & 1, &stop, p.status);
        __syncwarp();
        tc_fence_after();
      }
      // both halves' sums; the tile loop's last use of `red` lies behind a product of all warps
      red[0][half][row] = l;
      ok = !wide_sync_or(!ok);
      if (!ok) break;
      l = red[0][0][row] + red[0][1][row];
      const bool whole = x.opens && x.ends;
      const float one = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
      const long long piece_at = (2ll * cta + x.opens) * p.R + row;
      const long long out_at = 1ll * (x.q0 + qi) * p.ost[0] + 1ll * q_head * p.ost[1];
#pragma unroll 1
      for (int at = half ? d_half : 0; at < (half ? p.D : d_half); at += 16) {
        uint32_t o[16];
        if (x.tiles > 0) {
          tmem_load<16>(lanes + Shape::kO + at, o);
          tmem_load_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = 0;
        }
        if (!mine) continue;
        if (whole) {
          uint32_t packed[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float y0 = l == 0.0f ? 0.0f : __uint_as_float(o[2 * j]) * one;
            const float y1 = l == 0.0f ? 0.0f : __uint_as_float(o[2 * j + 1]) * one;
            if (p.dtype == DSD_TYPE_BF16) {
              const __nv_bfloat162 h = __floats2bfloat162_rn(y0, y1);
              packed[j] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
              const __half2 h = __floats2half2_rn(y0, y1);
              packed[j] = *reinterpret_cast<const uint32_t*>(&h);
            }
          }
          uint16_t* to = static_cast<uint16_t*>(p.out) + out_at + at;
          if (out_aligned) {
            reinterpret_cast<uint4*>(to)[0] = make_uint4(packed[0], packed[1], packed[2], packed[3]);
            reinterpret_cast<uint4*>(to)[1] = make_uint4(packed[4], packed[5], packed[6], packed[7]);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) to[j] = static_cast<uint16_t>(packed[j / 2] >> (j & 1 ? 16 : 0));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; j += 4)
            *reinterpret_cast<float4*>(&p.part_o[piece_at * p.D + at + j]) =
                make_float4(__uint_as_float(o[j]) * one, __uint_as_float(o[j + 1]) * one, __uint_as_float(o[j + 2]) * one,
                            __uint_as_float(o[j + 3]) * one);
        }
      }
      if (half == 0 && mine) {
        if (!whole) {
          p.part_ml[2 * piece_at] = m;
          p.part_ml[2 * piece_at + 1] = l;
        } else if (p.lse) {
          p.lse[1ll * (x.q0 + qi) * p.H + q_head] = l == 0.0f ? -INFINITY : ((m == -INFINITY ? 0.0f : m) + log2f(l)) * kLn2;
        }
      }
      if (x.opens && !x.ends && tid == 0) p.meta[cta] = make_int4(x.b, x.qt, gang_of(p, x.last_slot, w.total), 0);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&unit_empty[u]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 13)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Shape::kColumns));
}

}  // namespace dsds
