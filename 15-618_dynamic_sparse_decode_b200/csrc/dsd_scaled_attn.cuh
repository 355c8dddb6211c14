// dsd_scaled_attn.cuh -- attention over the scaled 8-bit cache on the fp32 pipes:
// any head_dim, page size and alignment.
//
//   s_rt = scale * ks_t * (q_r . k_t),  o_r = sum_t softmax(s_r)_t vs_t v_t
//
// One pass over the tokens with the running maximum and sum.  A thread owns a
// token for the dot products (its 8-bit key row against the R query rows in
// shared memory) and one or two output elements for the weighted sum (value codes
// of a token are adjacent across the threads).
//
// Bound: byte loads, one dependent key row a thread.  64 requests of 1024-4096 tokens,
// 32 heads over 8: 2.7 ms at head_dim 256 (floor 102 us), 2.05 ms with pages of one
// token (floor 57 us); the tensor-core kernels do that batch in 79 us at head_dim 128.
#pragma once

#include "dsd_scaled_common.cuh"

namespace dsds {

constexpr int kSimpleThreads = 128;

inline size_t simple_smem(int R, int D, int batch) {
  return size_t(4) * (R * D + R * kTile + 4 * kTile + 3 * R + batch) + 64;
}

template <bool I8, int R>
__global__ void __launch_bounds__(kSimpleThreads) attn_simple_kernel(const __grid_constant__ AttnParams p) {
  extern __shared__ float smem[];
  float* q_s = smem;                       // [R][D]
  float* w_s = q_s + R * p.D;              // [R][128] logits, then weights
  float* inv_s = w_s + R * kTile;          // [128] 2^-e and f of the value scales
  float* fac_s = inv_s + kTile;            // [128]
  int* page_s = reinterpret_cast<int*>(fac_s + kTile);   // [128]
  int* slot_s = page_s + kTile;            // [128]
  float* m_s = reinterpret_cast<float*>(slot_s + kTile); // [R]
  float* l_s = m_s + R;
  float* a_s = l_s + R;
  int* wb = reinterpret_cast<int*>(a_s + R);
  __shared__ Walk walk_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cta = blockIdx.x;

  const int head = cta % p.Hk;
  pdl_wait();
  pdl_trigger();
  plan_walk<kSimpleThreads>(p, cta / p.Hk, wb, &walk_s);
  Walk w = walk_s;
  if (tid == 0) p.meta[cta] = make_int4(0, 0, -1, 0);
  if (w.left == 0) return;
  while (w.left > 0) {
    const Request r = w.r;
    const Span span = w.span;
    const int slots = slots_of(span);
    const Segment seg = segment_of(w, slots);
    const int row0 = w.qt * R;
    for (int i = tid; i < R * p.D; i += kSimpleThreads) {
      const int row = row0 + i / p.D, d = i % p.D;
      float x = 0.0f;
      if (row < r.rows)
        x = load_elem(p.q, 1ll * (r.q0 + row / p.by_group) * p.qst[0] + 1ll * (head * p.G + row % p.by_group) * p.qst[1] + d, p.dtype);
      q_s[i] = x;
    }
    if (tid < R) {
      m_s[tid] = -INFINITY;
      l_s[tid] = 0.0f;
    }
    float acc[R][2] = {};
    __syncthreads();
    const int tiles = span.n == 0 ? 0 : seg.n;
    for (int i = 0; i < tiles; ++i) {
      const Token t = token_of(p, r, w.b, span.first + seg.first + i, tid);
      float s[R];
#pragma unroll
      for (int j = 0; j < R; ++j) s[j] = 0.0f;
      TokenScale ts{0.0f, 0.0f, 0.0f};
      if (t.page >= 0) {
        const long long si = scale_index(p, t.page, head, t.slot);
        ts = token_scale(p.vs[si]);
        const float ks = p.ks[si];
        const uint8_t* row = p.k + t.page * p.kst[0] + t.slot * p.kst[1] + head * p.kst[2];
        for (int d = 0; d < p.D; ++d) {
          const float x = code_value<I8>(row[d]);
#pragma unroll
          for (int j = 0; j < R; ++j) s[j] = fmaf(x, q_s[j * p.D + d], s[j]);
        }
#pragma unroll
        for (int j = 0; j < R; ++j)
          s[j] = sees(p, r, row0 + j, t.place) ? fmaf(s[j] * ks, p.scale_log2, ts.e) : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < R; ++j) w_s[j * kTile + tid] = t.page >= 0 ? s[j] : -INFINITY;
      page_s[tid] = t.page;
      slot_s[tid] = t.slot;
      inv_s[tid] = ts.inverse;
      fac_s[tid] = ts.factor;
      __syncthreads();
      for (int j = warp; j < R; j += 4) {
        float x[4], top = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) top = fmaxf(top, x[k] = w_s[j * kTile + 32 * k + lane]);
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        const float m = fmaxf(m_s[j], top), m0 = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int at = 32 * k + lane;
          const float wt = exp2f(x[k] - m0);
          if (x[k] != -INFINITY) sum = fmaf(wt, inv_s[at], sum);
          w_s[j * kTile + at] = wt * fac_s[at];
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (lane == 0) {
          const float a = exp2f(m_s[j] - m0);
          a_s[j] = a;
          l_s[j] = fmaf(l_s[j], a, sum);
          m_s[j] = m;
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < R; ++j) {
        acc[j][0] *= a_s[j];
        acc[j][1] *= a_s[j];
      }
      for (int k = 0; k < kTile; ++k) {
        const int page = page_s[k];
        if (page < 0) continue;
        const uint8_t* row = p.v + page * p.vst[0] + slot_s[k] * p.vst[1] + head * p.vst[2];
        const float x0 = tid < p.D ? code_value<I8>(row[tid]) : 0.0f;
        const float x1 = tid + kSimpleThreads < p.D ? code_value<I8>(row[tid + kSimpleThreads]) : 0.0f;
#pragma unroll
        for (int j = 0; j < R; ++j) {
          const float wt = w_s[j * kTile + k];
          if (wt != 0.0f) {   // a token the row does not see may hold anything
            acc[j][0] = fmaf(wt, x0, acc[j][0]);
            acc[j][1] = fmaf(wt, x1, acc[j][1]);
          }
        }
      }
      __syncthreads();
    }
    if (seg.whole()) {
      for (int j = 0; j < R && row0 + j < r.rows; ++j) {
        const float l = l_s[j];
        if (tid == 0) write_row_lse(p, r, head, row0 + j, m_s[j], l);
      }
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (row0 + j < r.rows) {
          if (tid < p.D) write_row_elem(p, r, head, row0 + j, tid, acc[j][0], l_s[j]);
          if (tid + kSimpleThreads < p.D)
            write_row_elem(p, r, head, row0 + j, tid + kSimpleThreads, acc[j][1], l_s[j]);
        }
    } else {
      const long long at = (2ll * cta + seg.opens) * R;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (tid < p.D) p.part_o[(at + j) * p.D + tid] = acc[j][0];
        if (tid + kSimpleThreads < p.D) p.part_o[(at + j) * p.D + tid + kSimpleThreads] = acc[j][1];
        if (tid == 0) {
          p.part_ml[2 * (at + j)] = m_s[j];
          p.part_ml[2 * (at + j) + 1] = l_s[j];
        }
      }
      if (seg.opens && tid == 0)
        p.meta[cta] = make_int4(w.b, w.qt, gang_of(p, w.at + slots - 1, w.total), 0);
    }
    next_unit(p, seg, w);
    __syncthreads();
  }
}

}  // namespace dsds
