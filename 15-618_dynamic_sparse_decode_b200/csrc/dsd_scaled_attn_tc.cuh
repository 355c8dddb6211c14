// dsd_scaled_attn_tc.cuh -- attention over the scaled 8-bit cache on the tensor
// cores (tcgen05), the 8-bit codes as operands where TMA put them.
//
// The cache's bytes never pass through registers.  A tile of 128 tokens is the
// 128-row operand of both products:
//   S^T[token][row] = K[token][d]    Q'[row][d]^T    (K rows as they lie, K-major)
//   O^T[d][row]     = V[token][d]^T  P'[row][token]^T (V read M-major, the same bytes)
// and Q', P' are made 8-bit too, without losing what the other operand cannot
// carry: a query row (or weight row) is the sum of a few 8-bit pieces, each its
// own column of the product,
//   e4m3: x = h0 + h1/16 + h2/256 ..., h_j the nearest e4m3 of the remainder * 16^j
//   int8: x = round(x 2^20) in base-128 digits (sums are exact integers)
// three pieces hold 12 (20) bits of fp16/bf16 rows, six (four) an fp32 row.  The
// products are exact and add in fp32 (int32); a query row's own power of two and
// the cache's scales are applied to the logits and weights in fp32.
// The pieces cost columns of a product that a decode step leaves idle anyway:
// with 8 query rows per key head, S and O have 24 of their up to 256 columns.
//
// Bound: HBM.  64 requests of 16-32k tokens, 32 heads over 8, token-major pages of
// 32: 0.50-0.52 ms, 6.2-6.4 TB/s (0.94-0.98 of the measured copy rate).  Some 20 us of
// a call are its plan (2.5), a CTA's first tile (4-5), the spread of the ranges' ends
// (5-11) and the join (4-9), so smaller calls reach less.  Two CTAs per SM with three
// stages each, two stages for 8 rows of four pieces or more; three CTAs with two stages
// measured the same for 1 or 2 rows and a fifth slower for 4 (80 registers).
//
// Roles: warps 0-3 softmax (thread = token for S^T, = element d for O^T), warp 4
// TMA, warp 5 MMA issue, warp 6 token data (page, scales, masks of a tile), warp 7
// the next unit's queries.  Warps 4, 6 and 7 walk the CTA's range ahead of the
// softmax, across units, so that a unit's first tile finds its operands ready.
// S and O are double-buffered in TMEM: S of the next tile is issued before the
// weights of this one are ready.  O^T leaves TMEM every tile and adds up in
// registers in fp32, rescaled by the running maximum there.
#pragma once

#include <cuda.h>
#include <limits.h>

#include "dsd_scaled_common.cuh"

namespace dsds {

constexpr int kTcThreads = 256;
constexpr int kTokenBytes = 2816;   // shared memory for token data, see TokenRing
constexpr int kTokenStages = 8;     // tiles of token data ahead at most
constexpr int kTcTileBytes = kTile * 128;
constexpr size_t kTcStatic = 4096;  // static shared memory of a narrow CTA at most

__host__ __device__ constexpr int pad16(int n) { return (n + 15) / 16 * 16; }
__host__ __device__ constexpr int pow2_at_least(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : 512; }

template <int R, int PIECES>
struct TcShape {
  static constexpr int N = pad16(R * PIECES);           // columns of S and of O
  static constexpr int kColumns = pow2_at_least(4 * N);
  static constexpr int kOperand = (R * PIECES + 7) / 8 * 1024;   // bytes of Q' (and of one P')
  // CTAs per SM, and as many ring stages as shared memory then allows: an SM has 228 KiB,
  // of which each CTA takes 1 KiB for the system and up to kTcStatic for its own variables.
  // The host checks on its first call that this many CTAs fit: with one, the ranges cut for
  // two run one after the other (64 requests of 1024-4096 tokens, 64 heads over 8: 128 us,
  // with two 96).
  static constexpr int kCtas = 2;
  static constexpr size_t bytes(int stages) { return 1024 + size_t(stages) * 2 * kTcTileBytes + 4 * kOperand; }
  static constexpr int kStages = bytes(3) + kTcStatic + 1024 <= 228 * 1024 / kCtas ? 3 : 2;
  static constexpr size_t kSmem = bytes(kStages);
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint64_t* b, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t* b, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* b, int parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_addr(b)), "r"(parity) : "memory");
  return ok != 0;
}
// The same, asleep for up to 20 us at a time: spinning warps took issue slots from
// the softmax.
__device__ __forceinline__ bool mbar_sleep(uint64_t* b, int parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_addr(b)), "r"(parity), "r"(20000) : "memory");
  return ok != 0;
}
// Bounded: gives up after about a second, or once another role has.
__device__ __noinline__ bool mbar_wait_slow(uint64_t* b, int parity, volatile int* stop, int* status) {
  const long long until = clock64() + (1ll << 31);
  while (!mbar_sleep(b, parity)) {
    if (*stop) return false;
    if (clock64() > until) {
      *stop = 1;
      if (status) atomicOr(status, DSD_SCALED_TIMEOUT);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool mbar_wait(uint64_t* b, int parity, volatile int* stop, int* status) {
  if (mbar_try(b, parity)) return true;
  return mbar_wait_slow(b, parity, stop, status);
}

__device__ __forceinline__ void tma_box(const CUtensorMap* map, uint32_t dst, uint64_t* bar, int c1, int c2, int page) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(dst), "l"(map), "r"(0), "r"(c1), "r"(c2), "r"(page), "r"(smem_addr(bar)) : "memory");
}

// Shared-memory operand in the 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return (uint64_t(addr >> 4) & 0x3FFF) | (uint64_t(64) << 16) | (uint64_t(64) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

// D (fp32 or int32) [128][N], A and B 8-bit; a_m_major: A's rows are adjacent.
template <bool I8, int N>
__host__ __device__ constexpr uint32_t mma_desc(bool a_m_major) {
  return (I8 ? (2u << 4) | (1u << 7) | (1u << 10) : (1u << 4)) | (a_m_major ? 1u << 15 : 0u) | (uint32_t(N >> 3) << 17) |
         (uint32_t(128 >> 4) << 24);
}

template <bool I8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
  if constexpr (I8)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"(uint32_t(add)) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"(uint32_t(add)) : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&x)[N]) {
  static_assert(N == 1 || N == 2 || N == 4 || N == 8 || N % 16 == 0);
  if constexpr (N == 1)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(x[0]) : "r"(addr));
  else if constexpr (N == 2)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(addr));
  else if constexpr (N == 4)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(addr));
  else if constexpr (N == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]) : "r"(addr));
  else {
    // 16 columns a load
#pragma unroll
    for (int i = 0; i < N; i += 16)
      asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                   : "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]),
                     "=r"(x[i + 7]), "=r"(x[i + 8]), "=r"(x[i + 9]), "=r"(x[i + 10]), "=r"(x[i + 11]), "=r"(x[i + 12]),
                     "=r"(x[i + 13]), "=r"(x[i + 14]), "=r"(x[i + 15])
                   : "r"(addr + i));
  }
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// The four softmax warps; returns whether any thread's flag was set.
__device__ __forceinline__ bool softmax_sync_or(bool flag) {
  uint32_t any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(any) : "r"(uint32_t(flag)) : "memory");
  return any != 0;
}

// Sum of a product's pieces: columns j * R + r hold piece j of row r.
template <bool I8, int PIECES>
__device__ __forceinline__ float add_pieces(float sum, uint32_t x, int j) {
  // first piece last: Horner from the smallest
  if constexpr (I8) return fmaf(sum, 1.0f / 128, static_cast<float>(static_cast<int>(x)));
  return fmaf(sum, 1.0f / 16, __uint_as_float(x));
}

// Two values x in [-256, 256] (e4m3) or two integers (int8) cut into PIECES bytes each.
template <int PIECES>
__device__ __forceinline__ void cut_e4m3(float a, float b, uint16_t (&piece)[PIECES]) {
#pragma unroll
  for (int j = 0; j < PIECES; ++j) {
    const __nv_fp8x2_storage_t h = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    piece[j] = h;
    if (j + 1 < PIECES) {
      const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3)));
      a = (a - f.x) * 16.0f;   // exact: the remainder has fewer bits
      b = (b - f.y) * 16.0f;
    }
  }
}
template <int PIECES>
__device__ __forceinline__ void cut_int(int a, int b, uint16_t (&piece)[PIECES]) {
#pragma unroll
  for (int j = 0; j < PIECES; ++j) {
    const int shift = 7 * (PIECES - 1 - j);
    const int x = j ? (a >> shift) & 127 : a >> shift, y = j ? (b >> shift) & 127 : b >> shift;
    piece[j] = static_cast<uint16_t>((x & 255) | (y & 255) << 8);
  }
}

// The e4m3 row of 128 codes at `row` (swizzled or not): does it hold a NaN code?
__device__ __forceinline__ bool row_has_nan(const uint4* row, int lane) {
  uint32_t hit = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint4 x = row[(i + lane) & 7];         // lanes start apart: no bank conflicts
    const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      hit |= ((y[j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;   // 0x7f + 1 carries into the sign's place
  }
  return hit != 0;
}

// What the softmax warps know of a unit, from warp 7.
struct UnitInfo {
  int tiles;          // -1: the range ends
  int b, qt;
  int rows;           // query rows from the unit's first on (wide: the request's)
  int q0, base_pos;   // wide: first query row, place of the first query
  int opens, ends;    // the segment has the unit's first / last slot
  int last_slot;      // of the unit, on the axis
};

// Token data of a tile, from warp 6.  A scale covers a block of bt tokens, so a
// tile has at most 128 / bt + 1 entries: the two scales and how many of the
// block's tokens are there.  As many tiles ahead as the ring has room for: the
// scales come from far apart in memory, and one tile ahead left the softmax
// waiting for them (64 requests x 16-32k: 1.01 ms, with eight ahead 0.62 ms).
struct TokenRing {
  float2* scales;    // [stages][entries]
  int* limit;        // [stages][entries]
  int entries, stages;

  __device__ __forceinline__ TokenRing(uint8_t* smem, const AttnParams& p) {
    entries = p.token_entries;
    stages = p.token_stages;
    scales = reinterpret_cast<float2*>(smem);
    limit = reinterpret_cast<int*>(scales + stages * entries);
  }
};
struct TileInfo { int place, lead, open; };   // of the first token; its index in its block; every row sees all

__device__ __forceinline__ void copy4_async(const void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void mbar_arrive_after_copies(uint64_t* b) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(b)) : "memory");
}

// Page-table entry of box i of a tile, -1 where there is none.
__device__ __forceinline__ int box_page(const AttnParams& p, const Request& r, int b, int tile, int i) {
  const int entry = p.tpp ? tile / p.by_tpp : tile * p.ppt + i;
  const int slot = p.tpp ? tile % p.by_tpp * kTile : 0;
  if (p.counts ? entry >= r.len : 1ll * entry * p.P + slot >= r.len) return -1;
  return p.table[1ll * b * p.table_stride + entry];
}

// TMA warp: the pages of the CTA's tiles, one box each, K then V, as far ahead as
// the ring has room.
template <int STAGES>
__device__ __forceinline__ void walk_boxes(const AttnParams& p, Walk w, int head, const CUtensorMap& k_map,
                                           const CUtensorMap& v_map, int head_first, uint8_t* k_ring, uint8_t* v_ring,
                                           uint64_t* k_full, uint64_t* k_empty, uint64_t* v_full, uint64_t* v_empty,
                                           volatile int* stop) {
  const int lane = threadIdx.x & 31;
  const int rows = p.tpp ? kTile : p.P, boxes = p.tpp ? 1 : p.ppt;
  uint32_t g = 0;
  bool ok = true;
#pragma unroll 1
  while (w.left > 0 && ok) {
    const Request r = w.r;
    const Span span = w.span;
    const Segment seg = segment_of(w, slots_of(span));
    const int tiles = span.n == 0 ? 0 : seg.n;
    int next = -1;
    if (tiles > 0 && lane < boxes) next = box_page(p, r, w.b, span.first + seg.first, lane);
#pragma unroll 1
    for (int i = 0; i < tiles && ok; ++i, ++g) {
      const int tile = span.first + seg.first + i;
      const int page = next;
      if (i + 1 < tiles && lane < boxes) next = box_page(p, r, w.b, tile + 1, lane);
      const bool good = page >= 0 && page < p.num_pages;
      const int bytes = __popc(__ballot_sync(~0u, good)) * rows * 128;
      const int s = g % STAGES, parity = (g / STAGES & 1) ^ 1;
      const int slot = p.tpp ? tile % p.by_tpp * kTile : 0;
      const int c1 = head_first ? head : slot, c2 = head_first ? slot : head;
      const uint32_t at = s * kTcTileBytes + lane * rows * 128;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        uint64_t* full = kv ? &v_full[s] : &k_full[s];
        ok = ok && mbar_wait(kv ? &v_empty[s] : &k_empty[s], parity, stop, p.status);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        if (lane == 0) mbar_expect(full, bytes);
        __syncwarp();
        if (good) tma_box(kv ? &v_map : &k_map, smem_addr(kv ? v_ring : k_ring) + at, full, c1, c2, page);
      }
    }
    next_unit(p, seg, w);
  }
  // after a time-out: the copies still in flight land before the block's memory is given back
  if (!ok && lane == 0) {
    int never = 0;
#pragma unroll 1
    for (uint32_t i = g > STAGES ? g - STAGES : 0; i <= g; ++i) {
      mbar_wait_slow(&k_full[i % STAGES], i / STAGES & 1, &never, nullptr);
      never = 0;
      mbar_wait_slow(&v_full[i % STAGES], i / STAGES & 1, &never, nullptr);
      never = 0;
    }
  }
}

// Token-data warp; a lane has every 32nd entry of a tile.
__device__ __forceinline__ void walk_tokens(const AttnParams& p, Walk w, int head, const TokenRing& ring, TileInfo* info,
                                            uint64_t* token_full, uint64_t* token_empty, volatile int* stop) {
  const int lane = threadIdx.x & 31;
  int s = 0, phase = 0;   // of the token ring
  bool ok = true;
#pragma unroll 1
  while (w.left > 0 && ok) {
    const Request r = w.r;
    const Span span = w.span;
    const Segment seg = segment_of(w, slots_of(span));
    const int tiles = span.n == 0 ? 0 : seg.n;
    const int* table = p.table + 1ll * w.b * p.table_stride;
    const int row0 = w.qt * p.R;
    const int base_pos = r.len - r.nq;
    // every row sees the tokens at all_from .. all_to
    int all_from = 0, all_to = INT_MAX;
    if (p.causal) all_to = max(base_pos + row0 / p.by_group, -1);
    if (p.window) all_from = max(max(base_pos + (min(row0 + p.R, r.rows) - 1) / p.by_group, -1) - p.window + 1, 0);
#pragma unroll 1
    for (int i = 0; i < tiles && ok; ++i) {
      const int tile = span.first + seg.first + i;
      const int first = p.tpp ? tile / p.by_tpp : tile * p.ppt;       // page-table entry of the first token
      const int off = p.tpp ? tile % p.by_tpp * kTile : 0;            // and its slot in that page
      const int lead = off % p.by_block;
      const int here = p.tpp ? min(kTile, p.P - off) : p.ppt * p.P;   // places of the tile
      ok = mbar_wait(&token_empty[s], phase ^ 1, stop, p.status);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      // one pass unless block_tokens < 5; the table's lines are in L1 then
#pragma unroll 1
      for (int e = lane; e < ring.entries; e += 32) {
        const int t = e * p.bt - lead;   // the block's first token in the tile; below 0 only where tpp
        int limit = 0;
        if (t < here) {
          const int entry = p.tpp ? first : first + t / p.by_page, slot = p.tpp ? off + t : t % p.by_page;
          if (!p.counts) limit = static_cast<int>(min(max(r.len - 1ll * entry * p.P - slot, 0ll), static_cast<long long>(p.bt)));
          if (p.counts ? entry < r.len : limit > 0) {
            const int page = table[entry];
            if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_pages)) {
              if (p.status) atomicOr(p.status, DSD_SCALED_BAD_PAGE);
              limit = 0;
            } else {
              if (p.counts) limit = min(max(p.counts[page] - slot, 0), p.bt);
              const long long si = (1ll * page * p.Hk + head) * p.nblk + slot / p.by_block;
              float2* to = ring.scales + s * ring.entries + e;
              copy4_async(&to->x, p.ks + si);
              copy4_async(&to->y, p.vs + si);
            }
          }
        }
        ring.limit[s * ring.entries + e] = limit;
      }
      if (lane == 0) {
        const int place = p.counts ? 0 : p.tpp ? first * p.P + off : tile * p.ppt * p.P;
        info[s] = {place, lead, p.counts || (place >= all_from && place <= all_to - (kTile - 1))};
      }
      mbar_arrive_after_copies(&token_full[s]);
      mbar_arrive(&token_full[s]);
      if (++s == ring.stages) {
        s = 0;
        phase ^= 1;
      }
    }
    next_unit(p, seg, w);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Four elements of a row as they lie; aligned: one access.
__device__ __forceinline__ uint4 load_four(const uint8_t* at, int elem, bool aligned) {
  uint4 y{0, 0, 0, 0};
  if (elem == 4) {
    if (aligned) return *reinterpret_cast<const uint4*>(at);
    const uint32_t* p = reinterpret_cast<const uint32_t*>(at);
    return {p[0], p[1], p[2], p[3]};
  }
  if (aligned) {
    const uint2 z = *reinterpret_cast<const uint2*>(at);
    y.x = z.x;
    y.y = z.y;
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(at);
    y.x = p[0] | uint32_t(p[1]) << 16;
    y.y = p[2] | uint32_t(p[3]) << 16;
  }
  return y;
}
__device__ __forceinline__ float4 widen_four(uint4 y, int dtype) {
  if (dtype == DSD_TYPE_F32)
    return make_float4(__uint_as_float(y.x), __uint_as_float(y.y), __uint_as_float(y.z), __uint_as_float(y.w));
  if (dtype == DSD_TYPE_BF16)
    return make_float4(__uint_as_float(y.x << 16), __uint_as_float(y.x & 0xffff0000u), __uint_as_float(y.y << 16),
                       __uint_as_float(y.y & 0xffff0000u));
  const float2 a = __half22float2(*reinterpret_cast<__half2*>(&y.x)), b = __half22float2(*reinterpret_cast<__half2*>(&y.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

// A unit's queries in pieces.  A row is shared by as many lanes as four rows leave
// each (eight, of 16 elements), so that a group's rows are cut side by side.
template <int R>
struct QueryLanes {
  static constexpr int kRows = R < 4 ? R : 4;          // rows at a time
  static constexpr int kLanes = 32 / kRows;            // lanes of a row
  static constexpr int kQuads = 32 / kLanes;           // runs of four elements a lane
};

template <bool I8, int R, int PIECES>
__device__ __forceinline__ void cut_rows(const float4 (&x)[QueryLanes<R>::kQuads], int row, uint8_t* op, float scale_log2,
                                         float* factor) {
  constexpr int kLanes = QueryLanes<R>::kLanes, kQuads = QueryLanes<R>::kQuads;
  const int part = threadIdx.x & (kLanes - 1);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kQuads; ++i)
    top = max(top, max(max(__float_as_uint(fabsf(x[i].x)), __float_as_uint(fabsf(x[i].y))),
                       max(__float_as_uint(fabsf(x[i].z)), __float_as_uint(fabsf(x[i].w)))));
#pragma unroll
  for (int o = kLanes / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
  // the row's power of two: 2^e <= largest < 2^(e+1)
  const int e = max(static_cast<int>(top >> 23) - 127, -100);
  const float f = __uint_as_float(uint32_t((I8 ? 7 * PIECES - 2 : 7) - e + 127) << 23);
#pragma unroll
  for (int i = 0; i < kQuads; ++i) {
    uint16_t lo[PIECES], hi[PIECES];
    if constexpr (I8) {
      cut_int<PIECES>(__float2int_rn(x[i].x * f), __float2int_rn(x[i].y * f), lo);
      cut_int<PIECES>(__float2int_rn(x[i].z * f), __float2int_rn(x[i].w * f), hi);
    } else {
      cut_e4m3<PIECES>(x[i].x * f, x[i].y * f, lo);
      cut_e4m3<PIECES>(x[i].z * f, x[i].w * f, hi);
    }
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int n = j * R + row;
      *reinterpret_cast<uint32_t*>(op + n * 128 + (4 * (part * kQuads + i) ^ (n & 7) << 4)) =
          uint32_t(lo[j]) | uint32_t(hi[j]) << 16;
    }
  }
  // the first piece's unit: e4m3 2^(e - 7), int8 2^(e - 5); a row that is not finite is NaN
  const float unit = __uint_as_float(uint32_t(e - (I8 ? 5 : 7) + 127) << 23);
  if (part == 0) *factor = top >= 0x7f800000u ? NAN : scale_log2 * unit;
}

template <bool I8, int R, int PIECES>
__global__ void __launch_bounds__(kTcThreads, (TcShape<R, PIECES>::kCtas))
attn_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap k_map,
               const __grid_constant__ CUtensorMap v_map, int head_first) {
  using Shape = TcShape<R, PIECES>;
  constexpr int N = Shape::N, STAGES = Shape::kStages;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* base = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
  // the operands first: a product's padding columns read on behind its operand
  uint8_t* q_op = base;
  uint8_t* p_op = q_op + 2 * Shape::kOperand;
  uint8_t* k_ring = p_op + 2 * Shape::kOperand;
  uint8_t* v_ring = k_ring + STAGES * kTcTileBytes;
  __shared__ uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
  __shared__ uint64_t s_full[2], s_empty[2], p_full[2], o_full[2], o_empty[2], unit_full[2], unit_empty[2];
  __shared__ uint64_t token_full[kTokenStages], token_empty[kTokenStages], drained;
  __shared__ TileInfo info[kTokenStages];
  __shared__ __align__(16) uint8_t token_smem[kTokenBytes];
  __shared__ float4 red[2][R];   // a row's four warps
  __shared__ float row_factor[2][R];
  __shared__ int row_pos[2][R], row_lse[2][R];   // a row's place; its element of lse
  __shared__ long long row_out[2][R];            // its first element of out
  __shared__ UnitInfo units[2];
  __shared__ uint32_t tmem_base;
  __shared__ int stop;
  __shared__ Walk walk_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = blockIdx.x, head = cta % p.Hk;

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], 4);
      mbar_init(&unit_full[i], 1);
      mbar_init(&unit_empty[i], 5);   // the softmax warps and the MMA warp
    }
    for (int i = 0; i < kTokenStages; ++i) {
      mbar_init(&token_full[i], 64);   // every lane, and every lane's copies
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
  // the plan's scratch lies in the ring, which nothing fills before the barrier in it
  plan_walk<kTcThreads>(p, cta / p.Hk, reinterpret_cast<int*>(k_ring), &walk_s);
  Walk w = walk_s;
  if (w.left == 0) return;
  proxy_fence();   // the scratch's generic writes, before TMA writes the same bytes
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                 "r"(Shape::kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  if (warp == 4) {
    walk_boxes<STAGES>(p, w, head, k_map, v_map, head_first, k_ring, v_ring, k_full, k_empty, v_full, v_empty, &stop);
  } else if (warp == 5) {
    // ---- MMA issue: the warp waits as one, so that descriptors stay in uniform
    // registers, and one lane issues
    constexpr uint32_t s_desc = mma_desc<I8, N>(false), o_desc = mma_desc<I8, N>(true);
    const bool leader = elect_one();
    const uint64_t k_d = operand_desc(smem_addr(k_ring)), v_d = operand_desc(smem_addr(v_ring));
    const uint64_t q_d = operand_desc(smem_addr(q_op)), p_d = operand_desc(smem_addr(p_op));
    const auto all = [&](uint64_t* bar, int parity) { return __all_sync(~0u, mbar_wait(bar, parity, &stop, p.status)) != 0; };
    uint32_t g = 0;
    int ks = 0, kp = 0, vs = 0, vp = 0;   // ring stage and phase of K and of V
    bool ok = true, owed = false;         // owed: O^T of tile g - 1 is still to be issued
    const auto weigh = [&]() {
      const int t = g - 1, buf = t & 1;
      owed = false;
      ok = ok && all(&p_full[buf], t >> 1 & 1) && all(&v_full[vs], vp) && all(&o_empty[buf], (t >> 1 & 1) ^ 1);
      if (!ok) return;
      tc_fence_after();
      if (leader) {
        const uint64_t a = v_d + vs * (kTcTileBytes >> 4), b = p_d + buf * (Shape::kOperand >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) mma<I8>(tmem + 2 * N + buf * N, a + 256 * k, b + 2 * k, o_desc, k > 0);
        mma_commit(&v_empty[vs]);
        mma_commit(&o_full[buf]);
      }
      __syncwarp();
      if (++vs == STAGES) {
        vs = 0;
        vp ^= 1;
      }
    };
    int left = 0, u = 1;
    uint32_t unit = 0;
    bool end = false;
    // one step issues S^T of a tile, then O^T of the tile before it
#pragma unroll 1
    while (ok && !(end && !owed)) {
      if (left == 0 && !end) {
        // the next unit's queries are ready ahead of time, except for the first
        // units: the owed product goes before a wait for them
        const int at = unit & 1, parity = unit >> 1 & 1;
        if (owed && !__all_sync(~0u, mbar_try(&unit_full[at], parity))) {
          weigh();
          continue;
        }
        ok = all(&unit_full[at], parity);
        if (!ok) break;
        u = at;
        left = units[u].tiles;
        __syncwarp();
        if (lane == 0) mbar_arrive(&unit_empty[u]);
        ++unit;
        end = left < 0;
        continue;
      }
      const bool more = !end;
      if (more) {
        const int buf = g & 1;
        ok = all(&k_full[ks], kp) && all(&s_empty[buf], (g >> 1 & 1) ^ 1);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint64_t a = k_d + ks * (kTcTileBytes >> 4), b = q_d + u * (Shape::kOperand >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma<I8>(tmem + buf * N, a + 2 * k, b + 2 * k, s_desc, k > 0);
          mma_commit(&k_empty[ks]);
          mma_commit(&s_full[buf]);
        }
        __syncwarp();
        if (++ks == STAGES) {
          ks = 0;
          kp ^= 1;
        }
        --left;
      }
      if (owed) weigh();
      if (more) {
        owed = true;
        ++g;
      }
    }
    if (!ok) {
      // after a time-out: what was issued ends before TMEM is given back
      int never = 0;
      if (leader) mma_commit(&drained);
      mbar_wait_slow(&drained, 0, &never, nullptr);
      __syncwarp();
    }
  } else if (warp == 6) {
    walk_tokens(p, w, head, TokenRing(token_smem, p), info, token_full, token_empty, &stop);
  } else if (warp == 7) {
    // ---- queries, cut into pieces
    using Lanes = QueryLanes<R>;
    constexpr int kGroups = R / Lanes::kRows, kQuads = Lanes::kQuads;
    const int elem = p.dtype == DSD_TYPE_F32 ? 4 : 2;
    const bool aligned = reinterpret_cast<uintptr_t>(p.q) % (4 * elem) == 0 && p.qst[0] % 4 == 0 && p.qst[1] % 4 == 0;
    const int my_row = lane / Lanes::kLanes, my_elem = lane % Lanes::kLanes * 4 * kQuads;
    bool ok = true;
#pragma unroll 1
    for (uint32_t unit = 0; ok; ++unit) {
      const int u = unit & 1;
      const bool end = w.left <= 0;
      const Request r = w.r;
      const int row0 = w.qt * R;
      uint4 raw[kGroups][kQuads];
      if (!end) {
        // every address is a valid one: the loads are in flight together
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
          const int gr = min(row0 + i * Lanes::kRows + my_row, r.rows - 1);
          const long long at = 1ll * (r.q0 + gr / p.by_group) * p.qst[0] + 1ll * (head * p.G + gr % p.by_group) * p.qst[1];
#pragma unroll
          for (int j = 0; j < kQuads; ++j)
            raw[i][j] = load_four(static_cast<const uint8_t*>(p.q) + (at + (my_elem + 4 * j < p.D ? my_elem + 4 * j : 0)) * elem,
                                  elem, aligned);
        }
      }
      const Span span = w.span;
      const int slots = slots_of(span);
      const Segment seg = segment_of(w, slots);
      ok = mbar_wait(&unit_empty[u], (unit >> 1 & 1) ^ 1, &stop, p.status);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      if (!end) {
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
          const int row = i * Lanes::kRows + my_row;
          float4 x[kQuads];
#pragma unroll
          for (int j = 0; j < kQuads; ++j) {
            x[j] = widen_four(raw[i][j], p.dtype);
            if (my_elem + 4 * j >= p.D || row0 + row >= r.rows) x[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          }
          cut_rows<I8, R, PIECES>(x, row, q_op + u * Shape::kOperand, p.scale_log2, &row_factor[u][row]);
        }
        if (lane < R) {
          const int gr = min(row0 + lane, r.rows - 1), qi = gr / p.by_group, q_head = head * p.G + gr % p.by_group;
          row_pos[u][lane] = r.len - r.nq + qi;
          row_out[u][lane] = 1ll * (r.q0 + qi) * p.ost[0] + 1ll * q_head * p.ost[1];
          row_lse[u][lane] = (r.q0 + qi) * p.H + q_head;
        }
      }
      if (lane == 0) {
        UnitInfo& x = units[u];
        x.tiles = end ? -1 : span.n == 0 ? 0 : seg.n;
        x.b = w.b;
        x.qt = w.qt;
        x.rows = r.rows - row0;
        x.opens = seg.opens;
        x.ends = seg.ends;
        x.last_slot = w.at - w.slot + slots - 1;
      }
      proxy_fence();
      __syncwarp();
      if (lane == 0) mbar_arrive(&unit_full[u]);
      if (end) break;
      next_unit(p, seg, w);
    }
  } else {
    // ---- softmax
    const TokenRing ring(token_smem, p);
    const int here = p.tpp ? kTile : p.ppt * p.P;   // a tile's places (a page's last tile: entries have limit 0 behind it)
    const int my_entry = tid / p.by_block, my_place = tid % p.by_block;
    uint32_t g = 0;
    int ts_at = 0, ts_phase = 0;   // of the token ring
    bool ok = true;
    const uint32_t lanes = tmem + (uint32_t(warp * 32) << 16);
#pragma unroll 1
    for (uint32_t unit = 0; ok; ++unit) {
      const int u = unit & 1;
      ok = !softmax_sync_or(!mbar_wait(&unit_full[u], unit >> 1 & 1, &stop, p.status));
      if (!ok) break;
      const int tiles = units[u].tiles;
      if (tiles < 0) break;
      float m[R], l[R], alpha[R], acc[R];
#pragma unroll
      for (int j = 0; j < R; ++j) {
        m[j] = -INFINITY;
        l[j] = 0.0f;
        alpha[j] = 0.0f;
        acc[j] = 0.0f;
      }
      // O^T of tile t joins the sum
      const auto collect = [&](uint32_t t) {
        const int buf = t & 1;
        const bool in = mbar_wait(&o_full[buf], t >> 1 & 1, &stop, p.status);
        __syncwarp();
        tc_fence_after();
        uint32_t x[PIECES][R];
#pragma unroll
        for (int j = 0; j < PIECES; ++j) tmem_load<R>(lanes + 2 * N + buf * N + j * R, x[j]);
        tmem_load_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[buf]);
#pragma unroll
        for (int row = 0; row < R; ++row) {
          float sum = 0.0f;
#pragma unroll
          for (int j = PIECES - 1; j >= 0; --j) sum = add_pieces<I8, PIECES>(sum, x[j][row], j);
          acc[row] = fmaf(acc[row], alpha[row], sum);
        }
        return in;
      };
#pragma unroll 1
      for (int i = 0; i < tiles && ok; ++i, ++g) {
        const int buf = g & 1;
        bool in = mbar_wait(&token_full[ts_at], ts_phase, &stop, p.status);
        const TileInfo tile = info[ts_at];
        int entry = my_entry, in_block = my_place;
        if (tile.lead) {
          entry = (tile.lead + tid) / p.by_block;
          in_block = (tile.lead + tid) % p.by_block;
        }
        entry += ts_at * ring.entries;
        const int place = tile.place + tid;
        const bool open = tile.open != 0;
        const bool valid = tid < here && in_block < ring.limit[entry];
        const float2 scales = ring.scales[entry];
        const TokenScale ts = token_scale(valid ? scales.y : 0.0f);

        in = mbar_wait(&s_full[buf], g >> 1 & 1, &stop, p.status) && in;
        __syncwarp();
        if (lane == 0) mbar_arrive(&token_empty[ts_at]);
        if (++ts_at == ring.stages) {
          ts_at = 0;
          ts_phase ^= 1;
        }
        tc_fence_after();
        float s[R];
        {
          uint32_t x[PIECES][R];
#pragma unroll
          for (int j = 0; j < PIECES; ++j) tmem_load<R>(lanes + buf * N + j * R, x[j]);
          tmem_load_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[buf]);
#pragma unroll
          for (int row = 0; row < R; ++row) {
            float sum = 0.0f;
#pragma unroll
            for (int j = PIECES - 1; j >= 0; --j) sum = add_pieces<I8, PIECES>(sum, x[j][row], j);
            s[row] = valid ? fmaf(sum * scales.x, row_factor[u][row], ts.e) : -INFINITY;
          }
        }
        if (!open) {
#pragma unroll
          for (int row = 0; row < R; ++row) {
            const int pos = row_pos[u][row];
            if ((p.causal && place > pos) || (p.window && 1ll * place + p.window <= pos)) s[row] = -INFINITY;
          }
        }
#pragma unroll
        for (int row = 0; row < R; ++row) {
          const float top = warp_max(s[row]);
          if (lane == 0) reinterpret_cast<float*>(&red[buf][row])[warp] = top;
        }
        // A tile with places that a row must not see: what lies there may be NaN,
        // and 0 * NaN is NaN, so such a value row becomes zeros; rows that do see
        // it become NaN through their sum.
        bool nan_row = false;
        if constexpr (!I8) {
          if (!valid || !open) {
            in = mbar_wait(&v_full[g % STAGES], g / STAGES & 1, &stop, p.status) && in;
            uint4* row = reinterpret_cast<uint4*>(v_ring + (g % STAGES) * kTcTileBytes + tid * 128);
            nan_row = valid && row_has_nan(row, lane);
            if (!valid || nan_row) {
#pragma unroll
              for (int j = 0; j < 8; ++j) row[(j + lane) & 7] = make_uint4(0, 0, 0, 0);
            }
          }
        }
        ok = !softmax_sync_or(!in);
        if (i > 0) {
          // the last tile's product, before this tile's weights take over the factors
          const bool got = collect(g - 1);
          if (!got) stop = 1;
        }
#pragma unroll
        for (int row = 0; row < R; ++row) {
          const float4 tops = red[buf][row];
          const float top = fmaxf(fmaxf(tops.x, tops.y), fmaxf(tops.z, tops.w));
          const float now = fmaxf(m[row], top), m0 = now == -INFINITY ? 0.0f : now;
          alpha[row] = ex2(m[row] - m0);
          m[row] = now;
          float x = ex2(s[row] - m0);
          if (nan_row && s[row] != -INFINITY) x = NAN;
          l[row] = fmaf(l[row], alpha[row], s[row] == -INFINITY ? 0.0f : x * ts.inverse);
          s[row] = x * ts.factor;
        }
        uint8_t* op = p_op + buf * Shape::kOperand;
        // byte tid of row n, its 16-byte pieces swizzled within groups of 8 rows
        const auto put = [&](int n, uint32_t byte) { op[n * 128 + (tid ^ (n & 7) << 4)] = static_cast<uint8_t>(byte); };
#pragma unroll
        for (int row = 0; row < R; row += 2) {
          const float x = s[row], y = row + 1 < R ? s[row + 1] : 0.0f;
          uint16_t piece[PIECES];
          if constexpr (I8) {
            constexpr float kOne = float(1 << (7 * PIECES - 2));
            cut_int<PIECES>(__float2int_rn(x * kOne), __float2int_rn(y * kOne), piece);
          } else {
            cut_e4m3<PIECES>(x * 128.0f, y * 128.0f, piece);
          }
#pragma unroll
          for (int j = 0; j < PIECES; ++j) {
            put(j * R + row, piece[j] & 255);
            if (row + 1 < R) put(j * R + row + 1, piece[j] >> 8);
          }
        }
        proxy_fence();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf]);
      }
      if (tiles > 0 && ok) ok = collect(g - 1);

      // the row sums over the threads' tokens
#pragma unroll
      for (int row = 0; row < R; ++row) {
        float x = l[row];
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
        if (lane == 0) reinterpret_cast<float*>(&red[0][row])[warp] = x;
      }
      ok = !softmax_sync_or(!ok);
      // weight 1 is 128 (e4m3) or 2^5 in the first piece's unit (int8: 2^(7 PIECES - 2) over 2^(7 (PIECES - 1)))
      constexpr float kUnit = I8 ? 1.0f / 32 : 1.0f / 128;
      const UnitInfo x = units[u];
      const bool whole = x.opens && x.ends;
      const long long piece = (2ll * cta + x.opens) * R;
#pragma unroll
      for (int row = 0; row < R; ++row) {
        const float4 sums = red[0][row];
        const float sum = (sums.x + sums.y) + (sums.z + sums.w);
        float o = acc[row] * kUnit;
        if (whole) {
          if (row >= x.rows) continue;
          o = sum == 0.0f ? 0.0f : o / sum;
          if (tid < p.D) store_elem(p.out, row_out[u][row] + tid, p.dtype, o);
          if (tid == 0 && p.lse)
            p.lse[row_lse[u][row]] = sum == 0.0f ? -INFINITY : ((m[row] == -INFINITY ? 0.0f : m[row]) + log2f(sum)) * kLn2;
        } else {
          if (tid < p.D) p.part_o[(piece + row) * p.D + tid] = o;
          if (tid == 0) {
            p.part_ml[2 * (piece + row)] = m[row];
            p.part_ml[2 * (piece + row) + 1] = sum;
          }
        }
      }
      if (x.opens && !x.ends && tid == 0) p.meta[cta] = make_int4(x.b, x.qt, gang_of(p, x.last_slot, w.total), 0);
      // `red` is written again behind the barrier at the next unit's start
      __syncwarp();
      if (lane == 0) mbar_arrive(&unit_empty[u]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Shape::kColumns));
}

}  // namespace dsds
