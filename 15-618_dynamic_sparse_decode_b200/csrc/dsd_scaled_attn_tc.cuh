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
// Roles: warps 0-3 softmax (thread = token for S^T, = element d for O^T), warp 4
// TMA, warp 5 MMA issue.  S and O are double-buffered in TMEM: S of the next tile
// is issued before the weights of this one are ready.  O^T leaves TMEM every tile
// and adds up in registers in fp32, rescaled by the running maximum there.
#pragma once

#include <cuda.h>
#include <limits.h>

#include "dsd_scaled_common.cuh"

namespace dsds {

constexpr int kTcThreads = 192;
constexpr int kTcTileBytes = kTile * 128;

__host__ __device__ constexpr int pad16(int n) { return (n + 15) / 16 * 16; }
__host__ __device__ constexpr int pow2_at_least(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : 512; }

template <int R, int PIECES>
struct TcShape {
  static constexpr int N = pad16(R * PIECES);           // columns of S and of O
  static constexpr int kColumns = pow2_at_least(4 * N);
  static constexpr int kOperand = N * 128;              // bytes of Q' (and of one P')
  // CTAs per SM and ring stages that 512 TMEM columns and 227 KiB allow
  static constexpr int kCtas = N <= 64 ? 2 : 1;
  static constexpr int kStages = N <= 32 ? 3 : N <= 64 ? 2 : 4;
  static constexpr size_t kSmem = 1024 + size_t(kStages) * 2 * kTcTileBytes + 3 * kOperand;
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
// Bounded: gives up after about a second, or once another role has.
__device__ __noinline__ bool mbar_wait_slow(uint64_t* b, int parity, volatile int* stop, int* status) {
  const long long until = clock64() + (1ll << 31);
  while (!mbar_try(b, parity)) {
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
  static_assert(N == 1 || N == 2 || N == 4 || N == 8 || N == 16 || N == 32);
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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
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

// What a softmax thread knows of its token one tile ahead.
struct TokenAhead {
  int page, slot, held;   // held: tokens the page holds (page lists)
  long long place;
  float ks, vs;
};

// Page-table entry of token i of a tile, -1 where there is none.
__device__ __forceinline__ int entry_of(const AttnParams& p, const Request& r, int b, int tile, int i) {
  int entry, slot;
  if (p.tpp) {
    entry = tile / p.tpp;
    slot = tile % p.tpp * kTile + i;
    if (slot >= p.P) return -1;
  } else {
    if (i >= p.ppt * p.P) return -1;
    entry = tile * p.ppt + i / p.P;
    slot = i % p.P;
  }
  if (p.counts ? entry >= r.len : 1ll * entry * p.P + slot >= r.len) return -1;
  const int page = p.table[1ll * b * p.table_stride + entry];
  return page < 0 ? INT_MAX : page;
}

__device__ __forceinline__ TokenAhead resolve(const AttnParams& p, int h, int tile, int i, int page) {
  TokenAhead t{-1, 0, INT_MAX, -1, 0.0f, 0.0f};
  if (page < 0) return t;
  if (page >= p.num_pages) {
    if (p.status) atomicOr(p.status, DSD_SCALED_BAD_PAGE);
    return t;
  }
  long long entry;
  if (p.tpp) {
    entry = tile / p.tpp;
    t.slot = tile % p.tpp * kTile + i;
  } else {
    entry = 1ll * tile * p.ppt + i / p.P;
    t.slot = i % p.P;
  }
  t.page = page;
  t.place = p.counts ? 0 : entry * p.P + t.slot;
  if (p.counts) t.held = p.counts[page];
  const long long si = scale_index(p, page, h, t.slot);
  t.ks = p.ks[si];
  t.vs = p.vs[si];
  return t;
}

template <bool I8, int R, int PIECES>
__global__ void __launch_bounds__(kTcThreads, (TcShape<R, PIECES>::kCtas))
attn_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap k_map,
               const __grid_constant__ CUtensorMap v_map, int head_first) {
  using Shape = TcShape<R, PIECES>;
  constexpr int N = Shape::N, STAGES = Shape::kStages;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* base = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
  uint8_t* k_ring = base;
  uint8_t* v_ring = k_ring + STAGES * kTcTileBytes;
  uint8_t* q_op = v_ring + STAGES * kTcTileBytes;
  uint8_t* p_op = q_op + Shape::kOperand;
  __shared__ uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
  __shared__ uint64_t s_full[2], s_empty[2], p_full[2], o_full[2], o_empty[2], q_full, drained;
  __shared__ float red[2][4][R], row_factor[R];
  __shared__ uint32_t tmem_base;
  __shared__ int stop;
  __shared__ Walk walk_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = blockIdx.x;

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
    }
    mbar_init(&q_full, 4);
    mbar_init(&drained, 1);
    stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    p.meta[cta] = make_int4(0, 0, 0, -1);
  }
  // the plan's scratch lies in the ring, which nothing fills before the barrier in it
  plan_walk<kTcThreads>(p, cta, reinterpret_cast<int*>(k_ring), &walk_s);
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
  Request r = request_of(p, w.b);

  if (warp == 4) {
    // ---- TMA: the pages of a tile, one box each, K then V
    const int rows = p.tpp ? kTile : p.P, boxes = p.tpp ? 1 : p.ppt;
    uint32_t g = 0;
    bool ok = true;
    while (w.left > 0 && ok) {
      const Span span = span_of(p, r, w.qt);
      const int slots = slots_of(span);
      const Segment seg = segment_of(w, slots);
      const int tiles = span.n == 0 ? 0 : seg.n;
      for (int i = 0; i < tiles && ok; ++i, ++g) {
        const int tile = span.first + seg.first + i;
        int page = -1;
        if (lane < boxes) page = entry_of(p, r, w.b, tile, lane * p.P);
        const bool good = page >= 0 && page < p.num_pages;
        const int bytes = __popc(__ballot_sync(~0u, good)) * rows * 128;
        const int s = g % STAGES, parity = (g / STAGES & 1) ^ 1;
        const int slot = p.tpp ? tile % p.tpp * kTile : 0;
        const int c1 = head_first ? w.h : slot, c2 = head_first ? slot : w.h;
        const uint32_t at = s * kTcTileBytes + lane * rows * 128;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          uint64_t* full = kv ? &v_full[s] : &k_full[s];
          ok = ok && mbar_wait(kv ? &v_empty[s] : &k_empty[s], parity, &stop, p.status);
          ok = __all_sync(~0u, ok);
          if (!ok) break;
          if (lane == 0) mbar_expect(full, bytes);
          __syncwarp();
          if (good) tma_box(kv ? &v_map : &k_map, smem_addr(kv ? v_ring : k_ring) + at, full, c1, c2, page);
        }
      }
      w.at += seg.n;
      w.left -= seg.n;
      if (w.left > 0) next_unit(p, r, w);
    }
    // after a time-out: the copies still in flight land before the block's memory is given back
    if (!ok && lane == 0) {
      int never = 0;
      for (uint32_t i = g > STAGES ? g - STAGES : 0; i <= g; ++i) {
        mbar_wait_slow(&k_full[i % STAGES], i / STAGES & 1, &never, nullptr);
        never = 0;
        mbar_wait_slow(&v_full[i % STAGES], i / STAGES & 1, &never, nullptr);
        never = 0;
      }
    }
  } else if (warp == 5) {
    // ---- MMA issue (one lane)
    if (lane == 0) {
      constexpr uint32_t s_desc = mma_desc<I8, N>(false), o_desc = mma_desc<I8, N>(true);
      const uint64_t q_d = operand_desc(smem_addr(q_op));
      uint32_t g = 0, unit = 0;
      bool ok = true;
      const auto weigh = [&](uint32_t t) {   // O^T of tile t
        const int s = t % STAGES, buf = t & 1;
        ok = ok && mbar_wait(&p_full[buf], t >> 1 & 1, &stop, p.status) &&
             mbar_wait(&v_full[s], t / STAGES & 1, &stop, p.status) &&
             mbar_wait(&o_empty[buf], (t >> 1 & 1) ^ 1, &stop, p.status);
        if (!ok) return;
        tc_fence_after();
        const uint64_t a = operand_desc(smem_addr(v_ring + s * kTcTileBytes));
        const uint64_t b = operand_desc(smem_addr(p_op + buf * Shape::kOperand));
#pragma unroll
        for (int k = 0; k < 4; ++k) mma<I8>(tmem + 2 * N + buf * N, a + 256 * k, b + 2 * k, o_desc, k > 0);
        mma_commit(&v_empty[s]);
        mma_commit(&o_full[buf]);
      };
      while (w.left > 0 && ok) {
        const Span span = span_of(p, r, w.qt);
        const int slots = slots_of(span);
        const Segment seg = segment_of(w, slots);
        const int tiles = span.n == 0 ? 0 : seg.n;
        for (int i = 0; i < tiles && ok; ++i, ++g) {
          if (i == 0) {
            // the softmax warps write the next queries after the last unit's tiles
            if (g > 0) weigh(g - 1);
            ok = ok && mbar_wait(&q_full, unit & 1, &stop, p.status);
            ++unit;
          }
          const int s = g % STAGES, buf = g & 1;
          ok = ok && mbar_wait(&k_full[s], g / STAGES & 1, &stop, p.status) &&
               mbar_wait(&s_empty[buf], (g >> 1 & 1) ^ 1, &stop, p.status);
          if (!ok) break;
          tc_fence_after();
          const uint64_t a = operand_desc(smem_addr(k_ring + s * kTcTileBytes));
#pragma unroll
          for (int k = 0; k < 4; ++k) mma<I8>(tmem + buf * N, a + 2 * k, q_d + 2 * k, s_desc, k > 0);
          mma_commit(&k_empty[s]);
          mma_commit(&s_full[buf]);
          if (i > 0) weigh(g - 1);
        }
        w.at += seg.n;
        w.left -= seg.n;
        if (w.left > 0) next_unit(p, r, w);
      }
      if (ok && g > 0) weigh(g - 1);
      if (!ok) {
        // after a time-out: what was issued ends before TMEM is given back
        int never = 0;
        mma_commit(&drained);
        mbar_wait_slow(&drained, 0, &never, nullptr);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax
    uint32_t g = 0;
    bool ok = true;
    const uint32_t lanes = tmem + (uint32_t(warp * 32) << 16);
    while (w.left > 0 && ok) {
      const Span span = span_of(p, r, w.qt);
      const int slots = slots_of(span);
      const Segment seg = segment_of(w, slots);
      const int tiles = span.n == 0 ? 0 : seg.n;
      const int first = span.first + seg.first;
      const int row0 = w.qt * R;
      const long long base_pos = static_cast<long long>(r.len) - r.nq;

      // token data: the page-table entry two tiles ahead, the scales one
      TokenAhead ahead{-1, 0, INT_MAX, -1, 0.0f, 0.0f};
      int entry = -1;
      if (tiles > 0) ahead = resolve(p, w.h, first, tid, entry_of(p, r, w.b, first, tid));
      if (tiles > 1) entry = entry_of(p, r, w.b, first + 1, tid);

      if (tiles > 0) {
        // queries, cut into pieces; a warp takes a row, a lane four elements
        for (int row = warp; row < R; row += 4) {
          float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          const int gr = row0 + row;
          if (gr < r.rows) {
            const long long at = 1ll * (r.q0 + gr / p.G) * p.qst[0] + 1ll * (w.h * p.G + gr % p.G) * p.qst[1];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (4 * lane + j < p.D) x[j] = load_elem(p.q, at + 4 * lane + j, p.dtype);
          }
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) top = max(top, __float_as_uint(fabsf(x[j])));
          top = __reduce_max_sync(~0u, top);
          // the row's power of two: 2^e <= largest < 2^(e+1); not finite: the row is NaN
          const int e = max(static_cast<int>(top >> 23) - 127, -100);
          uint16_t lo[PIECES], hi[PIECES];
          if constexpr (I8) {
            constexpr int kBits = 7 * PIECES - 2;
            const float f = __uint_as_float(uint32_t(kBits - e + 127) << 23);
            cut_int<PIECES>(__float2int_rn(x[0] * f), __float2int_rn(x[1] * f), lo);
            cut_int<PIECES>(__float2int_rn(x[2] * f), __float2int_rn(x[3] * f), hi);
          } else {
            const float f = __uint_as_float(uint32_t(7 - e + 127) << 23);
            cut_e4m3<PIECES>(x[0] * f, x[1] * f, lo);
            cut_e4m3<PIECES>(x[2] * f, x[3] * f, hi);
          }
#pragma unroll
          for (int j = 0; j < PIECES; ++j) {
            const int n = j * R + row;
            *reinterpret_cast<uint32_t*>(q_op + n * 128 + (((lane >> 2) ^ (n & 7)) << 4) + (lane & 3) * 4) =
                uint32_t(lo[j]) | uint32_t(hi[j]) << 16;
          }
          // first piece's unit: e4m3 2^(e-7); int8 2^(e - 5)
          if (lane == 0)
            row_factor[row] = top >= 0x7f800000u ? NAN : ldexpf(p.scale_log2, I8 ? e - 5 : e - 7);
        }
        proxy_fence();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full);
      }

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
      for (int i = 0; i < tiles && ok; ++i, ++g) {
        const int buf = g & 1, tile = first + i;
        const TokenAhead t = ahead;
        if (i + 1 < tiles) ahead = resolve(p, w.h, tile + 1, tid, entry);
        if (i + 2 < tiles) entry = entry_of(p, r, w.b, tile + 2, tid);
        const bool valid = t.page >= 0 && t.slot < t.held;
        // whether every row sees every token that is there
        bool open = true;
        if (!p.counts) {
          const long long t0 = p.tpp ? 1ll * (tile / p.tpp) * p.P + tile % p.tpp * kTile : 1ll * tile * p.ppt * p.P;
          const long long last_row = min(row0 + R, r.rows) - 1;
          open = (!p.causal || t0 + kTile - 1 <= base_pos + row0 / p.G) &&
                 (!p.window || t0 > base_pos + last_row / p.G - p.window);
        }
        const TokenScale ts = token_scale(valid ? t.vs : 0.0f);

        bool in = mbar_wait(&s_full[buf], g >> 1 & 1, &stop, p.status);
        __syncwarp();
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
            s[row] = sum;
          }
        }
#pragma unroll
        for (int row = 0; row < R; ++row) {
          s[row] = valid ? fmaf(s[row] * t.ks, row_factor[row], ts.log2) : -INFINITY;
          if (!open && valid && !sees(p, r, row0 + row, t.place)) s[row] = -INFINITY;
          const float top = warp_max(s[row]);
          if (lane == 0) red[buf][warp][row] = top;
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
          const float top = fmaxf(fmaxf(red[buf][0][row], red[buf][1][row]), fmaxf(red[buf][2][row], red[buf][3][row]));
          const float now = fmaxf(m[row], top), m0 = now == -INFINITY ? 0.0f : now;
          alpha[row] = ex2(m[row] - m0);
          m[row] = now;
          float x = ex2(s[row] - m0);
          if (nan_row && s[row] != -INFINITY) x = NAN;
          l[row] = fmaf(l[row], alpha[row], s[row] == -INFINITY ? 0.0f : x * ts.inverse);
          s[row] = x * ts.factor;
        }
        uint8_t* op = p_op + buf * Shape::kOperand;
        const auto put = [&](int n, uint32_t byte) {
          op[n * 128 + (((tid >> 4) ^ (n & 7)) << 4) + (tid & 15)] = static_cast<uint8_t>(byte);
        };
#pragma unroll
        for (int row = 0; row < R; row += 2) {
          const float x = s[row], y = row + 1 < R ? s[row + 1] : 0.0f;
          uint16_t piece[PIECES];
          if constexpr (I8) {
            constexpr float kOne = float(1 << (7 * PIECES - 1));
            cut_int<PIECES>(__float2int_rn(x * kOne), __float2int_rn(y * kOne), piece);
          } else {
            cut_e4m3<PIECES>(x * 256.0f, y * 256.0f, piece);
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
        if (lane == 0) red[0][warp][row] = x;
      }
      ok = !softmax_sync_or(!ok);
      // weight 1 is 256 (e4m3) or 2^6 in the first piece's unit (int8: 2^(7 PIECES - 1) over 2^(7 (PIECES - 1)))
      constexpr float kUnit = I8 ? 1.0f / 64 : 1.0f / 256;
#pragma unroll
      for (int row = 0; row < R; ++row) {
        const float sum = (red[0][0][row] + red[0][1][row]) + (red[0][2][row] + red[0][3][row]);
        const float o = acc[row] * kUnit;
        if (seg.whole()) {
          if (row0 + row < r.rows) {
            if (tid < p.D) write_row_elem(p, r, w.h, row0 + row, tid, o, sum);
            if (tid == 0) write_row_lse(p, r, w.h, row0 + row, m[row] == -INFINITY ? 0.0f : m[row], sum);
          }
        } else {
          const long long at = (2ll * cta + seg.opens) * R + row;
          if (tid < p.D) p.part_o[at * p.D + tid] = o;
          if (tid == 0) {
            p.part_ml[2 * at] = m[row];
            p.part_ml[2 * at + 1] = sum;
          }
        }
      }
      if (!seg.whole() && seg.opens && tid == 0)
        p.meta[cta] = make_int4(w.b, w.h, w.qt, cta_of(p, w.at + slots - 1, w.total));
      // nobody writes `red` or the row factors of the next unit before all have read these
      ok = !softmax_sync_or(!ok) && ok;
      w.at += seg.n;
      w.left -= seg.n;
      if (w.left > 0) next_unit(p, r, w);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Shape::kColumns));
}

}  // namespace dsds
