// dsd_scaled_common.cuh -- what the kernels of the scaled 8-bit paged cache share:
// element conversions, the work split of the attention, its partial results and
// their join.
//
// Attention splits the KEY axis: a unit is one request, one key head and R
// consecutive query rows (row = query * group + head of the group); it walks the
// tiles of up to 128 tokens that its rows see.  All units' tiles of a head in a
// row form one axis, which is cut into equal contiguous ranges, so that one long
// request fills the machine and a ragged batch leaves no CTA idle.  A range is
// walked by a gang of CTAs at once, one for each key head: in a token-major pool
// the heads' rows of a token are neighbours in memory, and CTAs that read them at
// about the same time keep DRAM in its open pages (64 requests x 16-32k: 604 us
// with the heads one after another along the axis, 505 us with gangs).  A CTA
// derives its range from the lengths on the device (no host knowledge of them, so a
// captured graph follows them); a unit that spans ranges leaves partial results, at
// most two per CTA, which combine_kernel joins in tile order.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "dsd_b200.h"

namespace dsds {

constexpr int kTile = 128;          // tokens of a tile at most
constexpr int kMaxBatch = 4096;     // plan: one int per request in shared memory

// Division of n < 2^31 by a fixed d >= 1: with 2^(l-1) < d <= 2^l and
// m = ceil(2^(31+l) / d), floor(n m / 2^(31+l)) = floor(n / d), since the excess
// n (m d - 2^(31+l)) / (d 2^(31+l)) stays below 1 / d.  Three instructions in
// place of thirty: the walkers divide by these sizes all over.
struct Divisor {
  int d;
  uint32_t m;
  int shift;
};
inline Divisor divisor_of(int d) {
  int l = 0;
  while ((int64_t(1) << l) < d) ++l;
  return {d, static_cast<uint32_t>(((uint64_t(1) << (31 + l)) + d - 1) / d), 31 + l};
}
__device__ __forceinline__ int operator/(int n, const Divisor& v) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * v.m) >> v.shift);
}
__device__ __forceinline__ int operator%(int n, const Divisor& v) { return n - n / v * v.d; }

// Every kernel here is launched before its predecessor in the stream has ended: it
// touches memory after pdl_wait(), which waits for that end.  What the predecessor may
// have written is read with ordinary loads: the read-only path (ld.global.nc) wants
// memory that stays as it is for the kernel's whole life.  pdl_trigger() lets the
// successor's blocks be placed once all blocks of this grid have started.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

struct AttnParams {
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  long long kst[3], vst[3];
  int num_pages, P, Hk, D, bt, nblk;
  const void* q;
  void* out;
  float* lse;
  long long qst[2], ost[2];
  int dtype, batch, total_q, H, G;
  const int* q_off;
  const int* lens;
  const int* table;
  long long table_stride;
  int max_pages;
  const int* counts;
  float scale_log2;   // scale * log2(e): logits are kept in powers of two
  int causal, window;
  int* status;
  int ppt;            // pages per tile (page_size <= 128), else 0
  int tpp;            // tiles per page (page_size > 128), else 0
  int R;              // query rows of a unit
  int few;            // plan_few will do: its sums fit
  Divisor by_page, by_group, by_block, by_tpp, by_tile;   // P, G, bt, tpp, ppt * P (1 where 0)
  int token_entries, token_stages;   // of TokenRing
  int ncta, gangs;    // ncta = gangs * Hk; CTA = gang * Hk + head
  float* part_ml;     // [ncta][2][R][2]  running maximum (log2) and sum
  float* part_o;      // [ncta][2][R][D]
  int4* meta;         // [ncta]  unit a CTA leaves open: request, row tile, last gang (-1: none)
};

__device__ __forceinline__ float load_elem(const void* p, long long i, int dtype) {
  if (dtype == DSD_TYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == DSD_TYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_elem(void* p, long long i, int dtype, float x) {
  if (dtype == DSD_TYPE_F32) static_cast<float*>(p)[i] = x;
  else if (dtype == DSD_TYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

template <bool I8>
__device__ __forceinline__ float code_value(uint8_t c) {
  if constexpr (I8) return static_cast<float>(static_cast<int8_t>(c));
  __nv_fp8_e4m3 f;
  f.__x = c;
  return static_cast<float>(f);
}

// One request as the kernel sees it, every number clamped to the arrays.
struct Request {
  int q0, nq, rows;   // first query row, queries, query rows (nq * group)
  int len;            // tokens, or listed pages when page_counts is given
};

__device__ __noinline__ Request request_of(const AttnParams& p, int b) {
  Request r;
  r.q0 = b;
  r.nq = 1;
  if (p.q_off) {
    const int a = p.q_off[b], e = p.q_off[b + 1];
    r.q0 = min(max(a, 0), p.total_q);
    r.nq = min(max(e, r.q0), p.total_q) - r.q0;
  }
  r.rows = r.nq * p.G;
  const long long most = p.counts ? p.max_pages : 1ll * p.max_pages * p.P;
  r.len = static_cast<int>(min(max(static_cast<long long>(p.lens[b]), 0ll), most));
  return r;
}

// Tiles that hold `tokens` tokens of a request, and the tile of token t.
__device__ __forceinline__ int tiles_of(const AttnParams& p, int tokens) {
  if (p.tpp) return tokens / p.by_page * p.tpp + (tokens % p.by_page + kTile - 1) / kTile;
  return tokens == 0 ? 0 : (tokens - 1) / p.by_tile + 1;
}
__device__ __forceinline__ int tile_at(const AttnParams& p, int t) {
  if (p.tpp) return t / p.by_page * p.tpp + t % p.by_page / kTile;
  return t / p.by_tile;
}

// The tiles that row tile qt (R rows) sees: the first one and how many.  Out of
// line, as next_unit: several warp roles walk the units, and their code would
// otherwise fill the instruction cache (200 KiB a kernel; a unit's first pass
// through it took 15 us).
struct Span { int first, n; };

__device__ __noinline__ Span span_of(const AttnParams& p, Request r, int qt) {
  if (p.counts) return {0, p.tpp ? r.len * p.tpp : (r.len + p.ppt - 1) / p.ppt};
  const int base = r.len - r.nq, row0 = qt * p.R, row1 = min(r.rows, row0 + p.R) - 1;
  int hi = r.len, lo = 0;
  if (p.causal) hi = min(hi, max(0, base + row1 / p.by_group + 1));
  if (p.window) lo = max(0, max(base + row0 / p.by_group, -1) - p.window + 1);
  if (lo >= hi) return {0, 0};
  const int t0 = tile_at(p, lo);
  return {t0, tiles_of(p, hi) - t0};
}

// A unit without a tile still takes a slot of the axis: its rows get zeros.
__device__ __forceinline__ int slots_of(const Span& s) { return max(1, s.n); }

// Where a gang stands: unit (b, qt), slot within the unit, slots left in its range.
struct Walk {
  int b, qt, slot;
  int at, left;   // slot of the axis, slots left
  int total;
  Request r;      // of b
  Span span;      // of (b, qt)
};

// The axis in p.gangs parts that differ by one slot at most (fewer where there are
// fewer slots, so that no part between two that work is empty).
struct Cut { int each, more, parts; };   // the first `more` parts have each + 1 slots
__device__ __forceinline__ Cut cut_of(const AttnParams& p, int total) {
  const int parts = min(total, p.gangs);
  return {total / max(parts, 1), total % max(parts, 1), parts};
}
// The gang whose range holds slot s.
__device__ __forceinline__ int gang_of(const AttnParams& p, int s, int total) {
  const Cut c = cut_of(p, total);
  const int wide = c.more * (c.each + 1);
  return s < wide ? s / (c.each + 1) : c.more + (s - wide) / c.each;
}

// The status bits of a request's numbers.
__device__ __forceinline__ unsigned bad_request(const AttnParams& p, int b, const Request& r) {
  unsigned bad = 0;
  const long long most = p.counts ? p.max_pages : 1ll * p.max_pages * p.P;
  if (p.lens[b] < 0) bad |= DSD_SCALED_BAD_LENGTH;
  if (p.lens[b] > most) bad |= DSD_SCALED_BAD_PAGE;
  if (p.q_off && (p.q_off[b] != r.q0 || p.q_off[b + 1] != r.q0 + r.nq)) bad |= DSD_SCALED_BAD_LENGTH;
  return bad;
}

// plan_walk for one query each and at most 128 requests, by one warp: a lane has four
// requests in registers, and one scan finds the range.
__device__ __forceinline__ void plan_few(const AttnParams& p, int gang, Walk* w) {
  const int lane = threadIdx.x & 31;
  const int per = (p.batch + 31) / 32, first = lane * per;
  int lens[4];   // all loads before the first use
#pragma unroll
  for (int j = 0; j < 4; ++j) lens[j] = j < per && first + j < p.batch ? p.lens[first + j] : 0;
  Request r[4];
  Span span[4];
  int slots[4], mine = 0;
  unsigned bad = 0;
  const int row_tiles = (p.G + p.R - 1) / p.R;
  const long long most = p.counts ? p.max_pages : 1ll * p.max_pages * p.P;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    slots[j] = 0;
    if (j >= per || first + j >= p.batch) continue;
    r[j] = {first + j, 1, p.G, static_cast<int>(min(max(static_cast<long long>(lens[j]), 0ll), most))};
    if (lens[j] < 0) bad |= DSD_SCALED_BAD_LENGTH;
    if (lens[j] > most) bad |= DSD_SCALED_BAD_PAGE;
    span[j] = span_of(p, r[j], 0);
    slots[j] = row_tiles * slots_of(span[j]);
    mine += slots[j];
  }
  if (blockIdx.x || !p.status) bad = 0;
  if (bad) atomicOr(p.status, static_cast<int>(bad));
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, upto, o);
    if (lane >= o) upto += y;
  }
  const int total = __shfl_sync(~0u, upto, 31);
  const Cut c = cut_of(p, total);
  const int at = gang * c.each + min(gang, c.more);
  const bool works = gang < c.parts;
  if (!works && lane == 0) *w = Walk{};
  if (works && at >= upto - mine && at < upto) {   // one lane
    int rest = at - (upto - mine);
    Walk x{};
    x.total = total;
    x.at = at;
    x.left = c.each + (gang < c.more);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (rest >= 0 && rest < slots[j]) {
        const int each = slots[j] / row_tiles;
        x.b = first + j;
        x.r = r[j];
        x.span = span[j];   // the same for every row tile of one query
        x.qt = rest / each;
        x.slot = rest - x.qt * each;
        rest = -1;
      } else {
        rest -= rest >= 0 ? slots[j] : 0;
      }
    *w = x;
  }
}

// Every thread of the CTA calls it; wb has room for p.batch ints, w is shared.
template <int THREADS>
__device__ void plan_walk(const AttnParams& p, int gang, int* wb, Walk* w) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (p.few) {
    if (warp == 0) plan_few(p, gang, w);
    __syncthreads();
    return;
  }
  unsigned bad = 0;
#pragma unroll 1
  for (int b = p.q_off ? warp : tid; b < p.batch; b += p.q_off ? THREADS / 32 : THREADS) {
    const Request r = request_of(p, b);
    if (blockIdx.x == 0 && p.status && (p.q_off == nullptr || lane == 0)) bad |= bad_request(p, b, r);
    const int qts = (r.rows + p.R - 1) / p.R;
    // one query: every row tile sees the same tokens; several: the lanes share the row tiles
    long long sum = 0;
#pragma unroll 1
    for (int qt = p.q_off ? lane : 0; qt < qts; qt += 32) {
      sum += slots_of(span_of(p, r, qt));
      if (!p.q_off) {
        sum *= qts;
        break;
      }
    }
    if (p.q_off) {
#pragma unroll 1
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    }
    if (!p.q_off || lane == 0) wb[b] = static_cast<int>(min(sum, static_cast<long long>(INT_MAX)));
  }
  __syncthreads();
  if (warp == 0) {
    long long all = 0;
#pragma unroll 1
    for (int b = lane; b < p.batch; b += 32) all += wb[b];
#pragma unroll 1
    for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(~0u, all, o);
    if (all >= INT_MAX) {   // more than hours of work: refused
      bad |= DSD_SCALED_BAD_LENGTH;
      all = 0;
    }
    const int total = static_cast<int>(all);
    const Cut c = cut_of(p, total);
    Walk x{};
    x.total = total;
    if (gang < c.parts) {
      x.at = gang * c.each + min(gang, c.more);
      x.left = c.each + (gang < c.more);
      int before = 0;
#pragma unroll 1
      for (int b0 = 0; b0 < p.batch; b0 += 32) {
        const int mine = b0 + lane < p.batch ? wb[b0 + lane] : 0;
        int upto = mine;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(~0u, upto, o);
          if (lane >= o) upto += y;
        }
        const unsigned past = __ballot_sync(~0u, before + upto > x.at);
        if (past) {
          const int l = __ffs(past) - 1;
          x.b = b0 + l;
          before += __shfl_sync(~0u, upto - mine, l);
          break;
        }
        before += __shfl_sync(~0u, upto, 31);
      }
      const int rest = x.at - before;
      const Request r = x.r = request_of(p, x.b);
      const int qts = (r.rows + p.R - 1) / p.R;
      if (!p.q_off) {
        const int per = wb[x.b] / qts;
        x.qt = rest / per;
        x.slot = rest % per;
      } else {
        int sum = 0;
#pragma unroll 1
        for (int q0 = 0; q0 < qts; q0 += 32) {
          const int mine = q0 + lane < qts ? slots_of(span_of(p, r, q0 + lane)) : 0;
          int upto = mine;
#pragma unroll 1
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(~0u, upto, o);
            if (lane >= o) upto += y;
          }
          const unsigned past = __ballot_sync(~0u, sum + upto > rest);
          if (past) {
            const int l = __ffs(past) - 1;
            x.qt = q0 + l;
            x.slot = rest - sum - __shfl_sync(~0u, upto - mine, l);
            break;
          }
          sum += __shfl_sync(~0u, upto, 31);
        }
      }
    }
    if (x.left > 0) x.span = span_of(p, x.r, x.qt);
    if (lane == 0) *w = x;
  }
  if (bad && blockIdx.x == 0 && p.status) atomicOr(p.status, static_cast<int>(bad));
  __syncthreads();
}

// The part of a unit that a CTA does, and where its result goes.
struct Segment {
  int first, n;     // slots
  bool opens, ends;
  __device__ bool whole() const { return opens && ends; }
};

__device__ __forceinline__ Segment segment_of(const Walk& w, int slots) {
  Segment s;
  s.first = w.slot;
  s.n = min(w.left, slots - w.slot);
  s.opens = w.slot == 0;
  s.ends = w.slot + s.n == slots;
  return s;
}

// Past a segment, to the first slot of the next unit.
__device__ __noinline__ void next_unit(const AttnParams& p, const Segment& seg, Walk& w) {
  w.at += seg.n;
  w.left -= seg.n;
  if (w.left <= 0) return;
  w.slot = 0;
  if (++w.qt >= (w.r.rows + p.R - 1) / p.R) {
    w.qt = 0;
    do {
      ++w.b;
      if (w.b >= p.batch) return;
      w.r = request_of(p, w.b);
    } while (w.r.rows == 0);
  }
  w.span = span_of(p, w.r, w.qt);
}

// Token i (0..127) of a unit's tile: its page (-1: none), slot in the page, place in the request.
struct Token { int page, slot; long long place; };

__device__ __forceinline__ Token token_of(const AttnParams& p, const Request& r, int b, int tile, int i) {
  Token t{-1, 0, -1};
  int entry;
  if (p.tpp) {
    entry = tile / p.by_tpp;
    t.slot = tile % p.by_tpp * kTile + i;
    if (t.slot >= p.P) return t;
  } else {
    if (i >= p.ppt * p.P) return t;
    entry = tile * p.ppt + i / p.by_page;
    t.slot = i % p.by_page;
  }
  const long long place = 1ll * entry * p.P + t.slot;
  if (p.counts ? entry >= r.len : place >= r.len) return t;
  const int page = p.table[1ll * b * p.table_stride + entry];
  if (page < 0 || page >= p.num_pages) {
    if (p.status) atomicOr(p.status, DSD_SCALED_BAD_PAGE);
    return t;
  }
  if (p.counts && t.slot >= p.counts[page]) return t;
  t.page = page;
  t.place = p.counts ? 0 : place;
  return t;
}

// Whether query row `row` of the request sees the token at `place`.
__device__ __forceinline__ bool sees(const AttnParams& p, const Request& r, int row, long long place) {
  if (row >= r.rows) return false;
  const long long pos = static_cast<long long>(r.len) - r.nq + row / p.by_group;
  if (p.causal && place > pos) return false;
  return !p.window || place > pos - p.window;
}

__device__ __forceinline__ long long scale_index(const AttnParams& p, int page, int h, int slot) {
  return (1ll * page * p.Hk + h) * p.nblk + slot / p.by_block;
}

// Weights carry the value scale: with vs = f 2^e, 1 <= f < 2, and the running
// maximum m of s + e, w = 2^(s + e - m) <= 1 is the size of a token's CONTRIBUTION:
// its value codes are weighted by w f, and the softmax sum gets w 2^-e.  Cut into
// 8-bit pieces, a weight thus keeps its bits where the output needs them.  All of
// it is exact.  e stays in [-64, 100], so that the sum cannot overflow: a smaller
// scale makes f small, a zero scale adds nothing.  A scale that is not finite
// makes e NaN, and with it the logit of a row that sees the token; f stays finite
// for the rows that do not.
struct TokenScale { float e, inverse, factor; };

__device__ __forceinline__ TokenScale token_scale(float vs) {
  const int e = min(max(static_cast<int>(__float_as_uint(vs) >> 23 & 255) - 127, -64), 100);
  const float inverse = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  const float off = vs - vs;   // 0 or NaN
  return {static_cast<float>(e) + off, inverse, off == 0.0f ? vs * inverse : 1.0f};
}

constexpr float kLn2 = 0.6931471805599453f;

// One output row from its (m, l, O) state; thread-wise over elements d.
__device__ __forceinline__ void write_row_elem(const AttnParams& p, const Request& r, int h, int row,
                                               int d, float o, float l) {
  const int qi = row / p.by_group, head = h * p.G + row % p.by_group;
  const long long i = 1ll * (r.q0 + qi) * p.ost[0] + 1ll * head * p.ost[1] + d;
  store_elem(p.out, i, p.dtype, l == 0.0f ? 0.0f : o / l);
}
__device__ __forceinline__ void write_row_lse(const AttnParams& p, const Request& r, int h, int row,
                                              float m, float l) {
  if (!p.lse) return;
  const int qi = row / p.by_group, head = h * p.G + row % p.by_group;
  p.lse[1ll * (r.q0 + qi) * p.H + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Joins the partial results of the units that span ranges.  Block (c, g) looks
// after rows g, g + gridDim.y, ... of the unit CTA c leaves open: the opener's
// piece is its slot 1, the slot 0 of the same head's CTA in every following gang
// the rest, added in that order, so the result does not depend on timing.  The
// pieces' maxima come in one load a thread and their factors lie in shared memory,
// so that the sum over pieces waits for nothing but its own loads (one request of
// 120000 tokens, 37 pieces a unit: 13 us with the loads one after another).
// head_dim <= blockDim.x threads.
constexpr int kMaxPieces = 8 * 160;   // CTAs of a launch at most, checked by the host

__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ AttnParams p) {
  __shared__ float factor[kMaxPieces], part_max[8], part_sum[8];
  pdl_wait();
  pdl_trigger();
  const int c = blockIdx.x, d = threadIdx.x, lane = d & 31, warp = d >> 5, warps = blockDim.x >> 5;
  const int4 u = p.meta[c];
  if (u.z < 0) return;
  const Request r = request_of(p, u.x);
  const int head = c % p.Hk, pieces = u.z - c / p.Hk + 1;
#pragma unroll 1
  for (int row = blockIdx.y; row < p.R; row += gridDim.y) {
    const int global_row = u.y * p.R + row;
    if (global_row >= r.rows) return;
    const auto piece = [&](int i) { return (2ll * (c + i * p.Hk) + (i == 0)) * p.R + row; };
    float m = -INFINITY;
#pragma unroll 1
    for (int i = d; i < pieces; i += blockDim.x) m = fmaxf(m, factor[i] = p.part_ml[2 * piece(i)]);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (lane == 0) part_max[warp] = m;
    __syncthreads();
    for (int i = 0; i < warps; ++i) m = fmaxf(m, part_max[i]);
    const float m0 = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
#pragma unroll 1
    for (int i = d; i < pieces; i += blockDim.x) {
      const float f = exp2f(factor[i] - m0);
      factor[i] = f;
      l += f * p.part_ml[2 * piece(i) + 1];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
    if (lane == 0) part_sum[warp] = l;
    __syncthreads();
    l = 0.0f;
    for (int i = 0; i < warps; ++i) l += part_sum[i];
    float o = 0.0f;
    if (d < p.D) {
      // a piece none of whose tokens this row saw holds zeros: its factor is 0 there
#pragma unroll 8
      for (int i = 0; i < pieces; ++i) o = fmaf(factor[i], p.part_o[piece(i) * p.D + d], o);
      write_row_elem(p, r, head, global_row, d, o, l);
    }
    if (d == 0) write_row_lse(p, r, head, global_row, m0, l);
    __syncthreads();   // the next row overwrites the factors
  }
}

}  // namespace dsds
