// dsd_scaled_append.cuh -- keys and values of new tokens into the scaled 8-bit
// cache, keys (and queries) rotated by their position on the way.
//
//   (a, b) -> (a c - b s, b c + a s),  code = rn(y / scale),  scale = amax / qmax
//
// The unit of work is one request's block of block_tokens tokens: its scale needs
// the largest of all its new values, so one team of warps holds a (block, head)
// whole.  Units are numbered without a prefix sum over the batch: request b's
// begin at offsets[b] / block_tokens + 2 b, which leaves room for the partly filled
// blocks at both ends, and a warp-wide search finds b again.
//
// Bound: HBM bytes (read both rows once, write a byte an element); a row stays in
// registers, as it lies, between the maximum and the rounding.  56000 tokens of
// fp16, 32 + 2 x 8 heads of 128, half of each rotated, e4m3 in blocks of 64: 0.27 ms,
// 5.0 TB/s of the measured 6.56 (queries alone 5.7, keys and values alone 3.5, where
// the rounding's instructions still show).  With keys, values and queries as rounds
// of one loop it took 0.61 ms.
#pragma once

#include <type_traits>

#include "dsd_scaled_common.cuh"

namespace dsds {

constexpr int kAppendThreads = 256;
constexpr int kAppendKeep = 2;   // slots (of 2*VE values) a lane keeps in registers
constexpr int kAppendHeads = 4;  // query heads a lane has in flight

struct AppendParams {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  long long kst[3], vst[3];
  int num_pages, P, Hk, D, bt, nblk;
  const void* kin;
  const void* vin;
  const void* qin;
  void* qout;
  long long kin_st[2], vin_st[2], qin_st[2], qout_st[2];
  int batch, total, max_pages, Hq;
  const int* off;
  const int* lens;
  const int* table;
  long long table_stride;
  const float* cos;
  const float* sin;
  const int* positions;
  int rot_positions, rd, interleaved;
  int* counts;
  int* status;
  int slots;   // slots of a row
  int team;    // warps per (block, head)
  int y_kv;    // blockIdx.y below: keys and values; from there on: queries
};

template <bool I8>
__device__ __forceinline__ uint8_t encode(float x) {
  if constexpr (I8) {
    return static_cast<uint8_t>(static_cast<int8_t>(min(127, max(-127, __float2int_rn(x)))));
  }
  return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

template <typename T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(x);
  else return __half2float(x);
}
template <typename T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(x);
  else return __float2half_rn(x);
}

// VE adjacent elements; 16-byte accesses when VE == 8 (the host checked alignment).
template <typename T, int VE>
__device__ __forceinline__ void load_vec(const T* p, float* x) {
  if constexpr (VE == 1) {
    x[0] = to_float(*p);
  } else {
    constexpr int kVecs = VE * sizeof(T) / 16;
    __align__(16) T raw[VE];
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
    for (int i = 0; i < VE; ++i) x[i] = to_float(raw[i]);
  }
}
template <typename T, int VE>
__device__ __forceinline__ void store_vec(T* p, const float* x) {
  if constexpr (VE == 1) {
    *p = from_float<T>(x[0]);
  } else {
    constexpr int kVecs = VE * sizeof(T) / 16;
    __align__(16) T raw[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) raw[i] = from_float<T>(x[i]);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<uint4*>(raw)[i];
  }
}
template <int N>
__device__ __forceinline__ void load_table(const float* p, float* x) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 y = reinterpret_cast<const float4*>(p)[i];
      x[4 * i] = y.x; x[4 * i + 1] = y.y; x[4 * i + 2] = y.z; x[4 * i + 3] = y.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = p[i];
  }
}
template <bool I8, int VE>
__device__ __forceinline__ void store_codes(uint8_t* p, const float* x, float inv) {
  if constexpr (VE == 1) {
    *p = encode<I8>(x[0] * inv);
  } else {
    __align__(8) uint8_t raw[VE];
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < VE; ++i) raw[i] = encode<true>(x[i] * inv);
    } else {
#pragma unroll
      for (int i = 0; i < VE; i += 2)
        reinterpret_cast<__nv_fp8x2_storage_t*>(raw)[i / 2] =
            __nv_cvt_float2_to_fp8x2(make_float2(x[i] * inv, x[i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    }
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(raw);
  }
}

// A slot is two runs of VE elements of a row: the halves of rotated pairs
// (i, i + rd/2), or neighbours.
template <int VE>
struct Slot { int e0, e1; bool two, turned; int angle; };

template <int VE>
__device__ __forceinline__ Slot<VE> slot_of(const AppendParams& p, int s) {
  Slot<VE> r;
  const int pairs = p.rd / (2 * VE);   // slots with rotated pairs
  if (p.interleaved || s >= pairs) {
    r.e0 = 2 * VE * s;                 // half: rd + 2 VE (s - pairs), the same number
    r.e1 = r.e0 + VE;
    r.turned = p.interleaved && r.e0 < p.rd;
    r.angle = r.e0 / 2;
  } else {
    r.e0 = VE * s;
    r.e1 = p.rd / 2 + VE * s;
    r.turned = true;
    r.angle = VE * s;
  }
  r.two = r.e1 < p.D;
  return r;
}

template <typename T, int VE>
__device__ __forceinline__ void load_pair(const T* row, const Slot<VE>& s, float (&x)[2 * VE]) {
  load_vec<T, VE>(row + s.e0, x);
  if (s.two) load_vec<T, VE>(row + s.e1, x + VE);
  else
#pragma unroll
    for (int i = 0; i < VE; ++i) x[VE + i] = 0.0f;
}

// A slot as it lies in memory.
template <typename T, int VE>
struct RawSlot {
  __align__(16) T v[2 * VE];

  __device__ __forceinline__ void load(const T* row, const Slot<VE>& s) {
    if constexpr (VE == 1) {
      v[0] = row[s.e0];
      v[1] = s.two ? row[s.e1] : T(0.0f);
    } else {
      constexpr int kVecs = VE * sizeof(T) / 16;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(row + s.e0)[i];
        reinterpret_cast<uint4*>(v)[kVecs + i] =
            s.two ? reinterpret_cast<const uint4*>(row + s.e1)[i] : make_uint4(0, 0, 0, 0);
      }
    }
  }
  __device__ __forceinline__ void widen(float (&x)[2 * VE]) const {
#pragma unroll
    for (int i = 0; i < 2 * VE; ++i) x[i] = to_float(v[i]);
  }
};

template <int VE>
__device__ __forceinline__ void load_angles(const AppendParams& p, const Slot<VE>& s, int pos, float (&c)[VE], float (&n)[VE]) {
  const long long at = 1ll * pos * (p.rd / 2) + s.angle;
  load_table<VE>(p.cos + at, c);
  load_table<VE>(p.sin + at, n);
}

template <int VE>
__device__ __forceinline__ void turn_slot(const AppendParams& p, const float (&c)[VE], const float (&n)[VE], float (&x)[2 * VE]) {
  // unfused: the same bits as a product, a product and their sum in fp32
  const auto turn_pair = [](float& a, float& b, float c, float n) {
    const float y = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, n));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, n));
    a = y;
  };
  if (p.interleaved) {
#pragma unroll
    for (int i = 0; i < VE; ++i) turn_pair(x[2 * i], x[2 * i + 1], c[i], n[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) turn_pair(x[i], x[VE + i], c[i], n[i]);
  }
}

template <typename T, int VE>
__device__ __forceinline__ void load_slot(const AppendParams& p, const T* row, const Slot<VE>& s, int pos,
                                          bool turn, float (&x)[2 * VE]) {
  load_pair<T, VE>(row, s, x);
  if (!turn || !s.turned) return;
  float c[VE], n[VE];
  load_angles<VE>(p, s, pos, c, n);
  turn_slot<VE>(p, c, n, x);
}

// Older codes of a block under its new scale.
template <bool I8, int VE>
__device__ __noinline__ void requantise(const AppendParams& p, uint8_t* codes, long long token_stride, int held, int rank,
                                        int width, float ratio) {
  const int vecs = p.D / VE;
  for (int at = rank; at < held * vecs; at += width) {
    uint8_t* c = codes + at / vecs * token_stride + at % vecs * VE;
    float x[VE];
    if constexpr (VE == 1) {
      x[0] = code_value<I8>(*c);
    } else {
      const uint2 raw = *reinterpret_cast<const uint2*>(c);
#pragma unroll
      for (int j = 0; j < VE; ++j) x[j] = code_value<I8>(reinterpret_cast<const uint8_t*>(&raw)[j]);
    }
    store_codes<I8, VE>(c, x, ratio);
  }
}

// 1 / scale.  A block of scale 0 has finite values below 2^-100 only, which 2^-126 rounds
// to 0 as 0 would, but infinities stay infinite and saturate.
__device__ __forceinline__ float inverse_of(float scale) { return scale > 0.0f ? 1.0f / scale : 1.17549435e-38f; }

// Largest magnitude, NaN aside; may be infinite.
template <int VE>
__device__ __forceinline__ float largest(const float (&x)[2 * VE], float m) {
#pragma unroll
  for (int i = 0; i < 2 * VE; ++i) m = fmaxf(m, fabsf(x[i]));
  return m;
}
template <int VE>
__device__ __forceinline__ float finite_max(const float (&x)[2 * VE], float m) {
#pragma unroll
  for (int i = 0; i < 2 * VE; ++i) {
    const float a = fabsf(x[i]);
    m = fmaxf(m, a < INFINITY ? a : 0.0f);
  }
  return m;
}

// J > 0: a team's lanes hold the block whole, J slots each, and take a head's keys and
// values in one round: all loads in flight, one barrier for both maxima, the slots'
// places and (J <= 2, 16-bit rows) angles kept from head to head (7400 tokens, blocks of
// 16: 37.8 us with the angles kept, 38.7 without, long prompts 270 and 280; fp32 rows 58
// and 59; blocks of 128, J = 4, 47.7 and 40.7: no registers are left there).  J = 0: any
// block, its rows read again for the rounding.
template <typename T, bool I8, int VE, int J>
__global__ void __launch_bounds__(kAppendThreads, J ? 2 : 3) append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ float team_max[2][2][kAppendThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int u = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  int b = u, row0 = u, end = u + 1;
  if (p.off) {
    // a request whose offsets descend has no unit: the last block, mostly an idle one, looks
    if (p.status && blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) {
      bool bad = false;
      for (int at = threadIdx.x; at < p.batch; at += kAppendThreads) bad = bad || p.off[at + 1] < p.off[at];
      if (bad) atomicOr(p.status, DSD_SCALED_BAD_LENGTH);
    }
    // the last request whose first unit is not behind u
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
      const bool past = at >= hi || p.off[at] / p.bt > u - 2 * at;
      lo += step * __popc(__ballot_sync(~0u, !past));
      hi = min(hi, lo + step);
    }
    b = lo;
    row0 = p.off[b];
    end = p.off[b + 1];
  }
  if (end <= row0) return;
  const int len = p.lens[b];
  const bool lead = threadIdx.x == 0 && blockIdx.y == 0;
  if (row0 < 0 || end > p.total || len < end - row0) {
    if (lead && p.status) atomicOr(p.status, DSD_SCALED_BAD_LENGTH);
    return;
  }
  const int start = len - (end - row0), i = p.off ? u - 2 * b - row0 / p.bt : 0;
  const long long blk = 1ll * (start / p.bt) + i;
  const long long from = max(static_cast<long long>(start), blk * p.bt);
  const long long to = min(static_cast<long long>(len), (blk + 1) * p.bt);
  if (i < 0 || from >= to) return;
  const int ntok = static_cast<int>(to - from);
  const int held = static_cast<int>(from - blk * p.bt);
  const int row = row0 + static_cast<int>(from - start);       // of the block's first new token
  const long long entry = blk * p.bt / p.P;
  const int first = static_cast<int>(blk * p.bt % p.P);        // the block's first slot in its page
  const int page = entry < p.max_pages ? p.table[b * p.table_stride + entry] : -1;
  const bool good = page >= 0 && page < p.num_pages;
  if (lead) {
    if (!good && p.status) atomicOr(p.status, DSD_SCALED_BAD_PAGE);
    if (good && p.counts)
      p.counts[page] = static_cast<int>(min(static_cast<long long>(p.P), len - entry * p.P));
  }

  const int teams = kAppendThreads / 32 / p.team;
  const int team = warp / p.team, rank = warp % p.team * 32 + lane, width = p.team * 32;
  const int items = 2 * p.Hk;
  const int work = ntok * p.slots;
  const auto position = [&](int t) {
    return p.positions ? p.positions[row + t] : static_cast<int>(from) + t;
  };
  const auto in_table = [&](int pos) { return !p.cos || (pos >= 0 && pos < p.rot_positions); };
  if (blockIdx.y >= p.y_kv) {
    // ---- queries: a lane keeps its slot's angles and takes the heads in turn
    constexpr int kHeads = sizeof(T) == 4 ? 2 : kAppendHeads;
    const int groups = max(1, kAppendThreads / work);   // lanes that share a slot
    const int q_parts = gridDim.y - p.y_kv, q_part = blockIdx.y - p.y_kv;
    const int stride = groups * q_parts;
    for (int at = threadIdx.x; at < work * groups; at += kAppendThreads) {
      const int slot = at % work, t = slot / p.slots, pos = position(t);
      if (!in_table(pos)) {
        if (p.status) atomicOr(p.status, DSD_SCALED_BAD_POSITION);
        continue;
      }
      const Slot<VE> s = slot_of<VE>(p, slot % p.slots);
      const bool turn = p.cos && s.turned;
      float c[VE], n[VE];
      if (turn) load_angles<VE>(p, s, pos, c, n);
      const T* in = static_cast<const T*>(p.qin) + (row + t) * p.qin_st[0];
      T* out = static_cast<T*>(p.qout) + (row + t) * p.qout_st[0];
      for (int h0 = at / work * q_parts + q_part; h0 < p.Hq; h0 += kHeads * stride) {
        RawSlot<T, VE> raw[kHeads];   // as they lie: half the registers of 16-bit rows
#pragma unroll
        for (int j = 0; j < kHeads; ++j)
          if (h0 + j * stride < p.Hq) raw[j].load(in + (h0 + j * stride) * p.qin_st[1], s);
#pragma unroll
        for (int j = 0; j < kHeads; ++j)
          if (h0 + j * stride < p.Hq) {
            float x[2 * VE];
            raw[j].widen(x);
            if (turn) turn_slot<VE>(p, c, n, x);
            T* o = out + (h0 + j * stride) * p.qout_st[1];
            store_vec<T, VE>(o + s.e0, x);
            if (s.two) store_vec<T, VE>(o + s.e1, x + VE);
          }
      }
    }
    return;
  }
  int flip = 0;
  if constexpr (J > 0) {
    constexpr bool kKeepAngles = J <= 2 && sizeof(T) == 2;
    constexpr float kQmax = I8 ? 127.0f : 448.0f;
    bool live[J];
    int t[J], pos[J];
    Slot<VE> slot[J];
    float c[kKeepAngles ? J : 1][VE], n[kKeepAngles ? J : 1][VE];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int at = j * width + rank;
      t[j] = at < work ? at / p.slots : 0;
      slot[j] = slot_of<VE>(p, at - t[j] * p.slots);
      pos[j] = position(t[j]);
      live[j] = good && at < work;
      if (live[j] && !in_table(pos[j])) {
        live[j] = false;
        if (p.status) atomicOr(p.status, DSD_SCALED_BAD_POSITION);
      }
      if constexpr (kKeepAngles)
        if (live[j] && p.cos && slot[j].turned) load_angles<VE>(p, slot[j], pos[j], c[j], n[j]);
    }
    const auto key = [&](int j, const RawSlot<T, VE>& raw, float (&x)[2 * VE]) {
      raw.widen(x);
      if (!p.cos || !slot[j].turned) return;
      if constexpr (kKeepAngles) {
        turn_slot<VE>(p, c[j], n[j], x);
      } else {
        load_angles<VE>(p, slot[j], pos[j], c[0], n[0]);
        turn_slot<VE>(p, c[0], n[0], x);
      }
    };
    for (int base = blockIdx.y * teams; base < p.Hk; base += p.y_kv * teams) {
      const int head = base + team;
      const bool on = head < p.Hk && good;
      const long long si = (1ll * page * p.Hk + head) * p.nblk + first / p.bt;
      const float old_k = on && held ? p.ks[si] : 0.0f, old_v = on && held ? p.vs[si] : 0.0f;
      const T* kin = static_cast<const T*>(p.kin) + row * p.kin_st[0] + head * p.kin_st[1];
      const T* vin = static_cast<const T*>(p.vin) + row * p.vin_st[0] + head * p.vin_st[1];
      RawSlot<T, VE> k[J], v[J];
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (on && live[j]) {
          k[j].load(kin + t[j] * p.kin_st[0], slot[j]);
          v[j].load(vin + t[j] * p.vin_st[0], slot[j]);
        }
      float mk = 0.0f, mv = 0.0f;
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (on && live[j]) {
          float x[2 * VE];
          key(j, k[j], x);
          mk = largest<VE>(x, mk);
          v[j].widen(x);
          mv = largest<VE>(x, mv);
        }
      if (mk == INFINITY || mv == INFINITY) {   // seldom: infinities stay out of the scale
        mk = mv = 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (on && live[j]) {
            float x[2 * VE];
            key(j, k[j], x);
            mk = finite_max<VE>(x, mk);
            v[j].widen(x);
            mv = finite_max<VE>(x, mv);
          }
      }
      // non-negative floats order like their bits
      mk = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(mk)));
      mv = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(mv)));
      if (p.team > 1) {
        // two arrays in turn: one is read while the next round's is written
        if (lane == 0) {
          team_max[flip][0][warp] = mk;
          team_max[flip][1][warp] = mv;
        }
        __syncthreads();
        for (int j = 0; j < p.team; ++j) {
          mk = fmaxf(mk, team_max[flip][0][team * p.team + j]);
          mv = fmaxf(mv, team_max[flip][1][team * p.team + j]);
        }
        flip ^= 1;
      }
      if (!on) continue;
      const auto finish = [&](bool is_v, float m, float old) {
        const float fresh = m < 7.888609052210118e-31f ? 0.0f : m * (1.0f / kQmax);   // 2^-100
        const float scale = held ? fmaxf(old, fresh) : fresh;
        const float inv = inverse_of(scale);
        const long long* st = is_v ? p.vst : p.kst;
        uint8_t* codes = (is_v ? p.v : p.k) + page * st[0] + first * st[1] + head * st[2];
        if (held && scale > old) requantise<I8, VE>(p, codes, st[1], held, rank, width, old * inv);
        // every lane of the team has read `old` before the maximum's exchange
        if (rank == 0) (is_v ? p.vs : p.ks)[si] = scale;
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (live[j]) {
            float x[2 * VE];
            if (is_v) v[j].widen(x);
            else key(j, k[j], x);
            uint8_t* to = codes + (held + t[j]) * st[1];
            store_codes<I8, VE>(to + slot[j].e0, x, inv);
            if (slot[j].two) store_codes<I8, VE>(to + slot[j].e1, x + VE, inv);
          }
      };
      finish(false, mk, old_k);
      finish(true, mv, old_v);
    }
  } else {
    for (int base = blockIdx.y * teams; base < items; base += p.y_kv * teams) {
      const int item = base + team;
      const bool is_v = item >= p.Hk;
      const int head = is_v ? item - p.Hk : item;
      const bool turn = p.cos && !is_v;
      const bool on = item < items && good;
      const long long* in_st = is_v ? p.vin_st : p.kin_st;
      const T* in = static_cast<const T*>(is_v ? p.vin : p.kin) + row * in_st[0] + head * in_st[1];
      const long long si = (1ll * page * p.Hk + head) * p.nblk + first / p.bt;
      float* scales = is_v ? p.vs : p.ks;
      const float old = on && held ? scales[si] : 0.0f;

      float keep[kAppendKeep][2 * VE];
      bool live[kAppendKeep];
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < kAppendKeep; ++j) {
        const int at = j * width + rank;
        live[j] = on && at < work;
        if (live[j]) {
          const int t = at / p.slots, pos = position(t);
          live[j] = in_table(pos);
          if (live[j]) {
            load_slot<T, VE>(p, in + t * in_st[0], slot_of<VE>(p, at % p.slots), pos, turn, keep[j]);
            m = finite_max<VE>(keep[j], m);
          } else if (p.status) {
            atomicOr(p.status, DSD_SCALED_BAD_POSITION);
          }
        }
      }
      if (on)
        for (int at = kAppendKeep * width + rank; at < work; at += width) {
          const int t = at / p.slots, pos = position(t);
          if (!in_table(pos)) {
            if (p.status) atomicOr(p.status, DSD_SCALED_BAD_POSITION);
            continue;
          }
          float x[2 * VE];
          load_slot<T, VE>(p, in + t * in_st[0], slot_of<VE>(p, at % p.slots), pos, turn, x);
          m = finite_max<VE>(x, m);
        }
      // non-negative floats order like their bits
      m = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(m)));
      if (p.team > 1) {
        // two arrays in turn: one is read while the next round's is written
        if (lane == 0) team_max[flip][0][warp] = m;
        __syncthreads();
        for (int j = 0; j < p.team; ++j) m = fmaxf(m, team_max[flip][0][team * p.team + j]);
        flip ^= 1;
      }
      if (!on) continue;

      constexpr float kQmax = I8 ? 127.0f : 448.0f;
      const float fresh = m < 7.888609052210118e-31f ? 0.0f : m * (1.0f / kQmax);   // 2^-100
      const float scale = held ? fmaxf(old, fresh) : fresh;
      const float inv = inverse_of(scale);
      const long long* st = is_v ? p.vst : p.kst;
      uint8_t* codes = (is_v ? p.v : p.k) + page * st[0] + first * st[1] + head * st[2];
      if (held && scale > old) requantise<I8, VE>(p, codes, st[1], held, rank, width, old * inv);
      // every lane of the team has read `old` before the maximum's exchange
      if (rank == 0) scales[si] = scale;
      const auto put = [&](int at, const float (&x)[2 * VE]) {
        const Slot<VE> s = slot_of<VE>(p, at % p.slots);
        uint8_t* c = codes + (held + at / p.slots) * st[1];
        store_codes<I8, VE>(c + s.e0, x, inv);
        if (s.two) store_codes<I8, VE>(c + s.e1, x + VE, inv);
      };
#pragma unroll
      for (int j = 0; j < kAppendKeep; ++j)
        if (live[j]) put(j * width + rank, keep[j]);
      for (int at = kAppendKeep * width + rank; at < work; at += width) {
        const int t = at / p.slots, pos = position(t);
        if (!in_table(pos)) continue;
        float x[2 * VE];
        load_slot<T, VE>(p, in + t * in_st[0], slot_of<VE>(p, at % p.slots), pos, turn, x);
        put(at, x);
      }
    }
  }
}

}  // namespace dsds
