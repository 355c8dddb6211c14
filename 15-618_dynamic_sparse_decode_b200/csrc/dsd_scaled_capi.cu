// dsd_scaled_capi.cu -- C ABI of the scaled 8-bit paged cache (include/dsd_b200.h):
// argument checks, the choice of kernel and the launches.  Stateless apart from
// per-device attributes that are looked up once.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <mutex>
#include <string>
#include <utility>

#include "dsd_b200.h"
#include "dsd_internal.h"
#include "dsd_scaled_append.cuh"
#include "dsd_scaled_attn.cuh"
#include "dsd_scaled_attn_tc.cuh"
#include "dsd_scaled_attn_wide.cuh"

namespace {

using namespace dsd_internal;
using dsds::AppendParams;
using dsds::AttnParams;

constexpr int kMaxDevices = 64;

// What a launch needs to know of a device, looked up on its first call.
struct Device {
  bool ready = false;
  int sms = 0;
};
std::mutex g_mutex;
Device g_devices[kMaxDevices];

void SetAttentionAttributes(int device);

const Device& DeviceOf(int device) {
  if (device < 0 || device >= kMaxDevices) Fail(DSD_EINVAL, "device index out of range");
  std::lock_guard<std::mutex> lock(g_mutex);
  Device& d = g_devices[device];
  if (!d.ready) {
    int major = 0;
    Check(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device), "device");
    if (major != 10) Fail(DSD_EUNAVAILABLE, "no sm_100 GPU at this device index");
    Check(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, device), "SM count");
    SetAttentionAttributes(device);
    d.ready = true;
  }
  return d;
}

bool Aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
int ElemBytes(int dtype) { return dtype == DSD_TYPE_F32 ? 4 : 2; }

void CheckCache(const dsd_scaled_cache* c) {
  if (!c) Fail(DSD_EINVAL, "null cache");
  if (c->kv_format != DSD_KV_FP8_SCALED && c->kv_format != DSD_KV_I8_SCALED)
    Fail(DSD_EINVAL, "kv_format must be DSD_KV_FP8_SCALED or DSD_KV_I8_SCALED");
  if (c->num_pages <= 0) Fail(DSD_EINVAL, "num_pages must be positive");
  if (c->page_size < 1 || c->page_size > 4096) Fail(DSD_EINVAL, "page_size must be in [1, 4096]");
  if (c->num_kv_heads < 1 || c->num_kv_heads > 128) Fail(DSD_EINVAL, "num_kv_heads must be in [1, 128]");
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8)
    Fail(DSD_EINVAL, "head_dim must be a multiple of 8 in [8, 256]");
  if (c->block_tokens < 1 || c->block_tokens > 256 || c->page_size % c->block_tokens)
    Fail(DSD_EINVAL, "block_tokens must divide page_size and be at most 256");
  for (int i = 0; i < 3; ++i)
    if (c->k_stride[i] <= 0 || c->v_stride[i] <= 0) Fail(DSD_EINVAL, "cache strides must be positive");
}

void CheckCachePointers(const dsd_scaled_cache* c) {
  if (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales) Fail(DSD_EINVAL, "null cache array");
  if (!Aligned(c->k_scales, 4) || !Aligned(c->v_scales, 4)) Fail(DSD_EINVAL, "scales must be 4-byte aligned");
}

// int32 arrays on the device; null where the call has none
template <typename... T>
void CheckInts(const T*... p) {
  if (!(Aligned(p, 4) && ...)) Fail(DSD_EINVAL, "int32 device arrays must be 4-byte aligned");
}

// Rows of head_dim elements that a call writes: where two of them certainly share
// memory (a stride below a row's length, or two dimensions of one stride), the blocks
// that write them would race.
void CheckWritten(int head_dim, std::initializer_list<std::pair<int64_t, int64_t>> dims, const char* what) {
  for (auto a = dims.begin(); a != dims.end(); ++a)
    for (auto b = dims.begin(); b != dims.end(); ++b)
      if (a->first > 1 && (a->second < head_dim || (a != b && b->first > 1 && a->second == b->second)))
        Fail(DSD_EINVAL, std::string("the rows of ") + what + " overlap");
}

void CheckType(int dtype) {
  if (dtype != DSD_TYPE_F32 && dtype != DSD_TYPE_BF16 && dtype != DSD_TYPE_F16)
    Fail(DSD_EINVAL, "dtype must be DSD_TYPE_F32, DSD_TYPE_BF16 or DSD_TYPE_F16");
}

// Launches a kernel that may be placed before its predecessor in the stream has
// ended (it waits on the device before it touches memory): the launch's latency
// disappears behind the predecessor's last blocks.
template <typename... P, typename... A>
void Launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  Check(cudaLaunchKernelEx(&cfg, kernel, args...), "kernel launch");
}

// ------------------------------------------------------------------ append

template <typename T, bool I8>
void LaunchAppendAs(const AppendParams& p, int ve, int j, dim3 grid, cudaStream_t s) {
  using namespace dsds;
  if (ve == 1) Launch(append_kernel<T, I8, 1, 0>, grid, kAppendThreads, 0, s, p);
  else if (j == 1) Launch(append_kernel<T, I8, 8, 1>, grid, kAppendThreads, 0, s, p);
  else if (j == 2) Launch(append_kernel<T, I8, 8, 2>, grid, kAppendThreads, 0, s, p);
  else if (j == 4) Launch(append_kernel<T, I8, 8, 4>, grid, kAppendThreads, 0, s, p);
  else Launch(append_kernel<T, I8, 8, 0>, grid, kAppendThreads, 0, s, p);
}

template <typename T>
void LaunchAppend(const AppendParams& p, bool i8, int ve, int j, dim3 grid, cudaStream_t s) {
  if (i8) LaunchAppendAs<T, true>(p, ve, j, grid, s);
  else LaunchAppendAs<T, false>(p, ve, j, grid, s);
}

void Append(int device, const dsd_scaled_cache* c, const dsd_scaled_append_args* a, cudaStream_t s) {
  NvtxRange nvtx("dsd_scaled_append");
  CheckCache(c);
  if (!a) Fail(DSD_EINVAL, "null arguments");
  CheckType(a->dtype);
  if (a->batch < 0 || a->total_tokens < 0) Fail(DSD_EINVAL, "batch and total_tokens must not be negative");
  if (!a->token_offsets && a->total_tokens != a->batch)
    Fail(DSD_EINVAL, "without token_offsets every request has one token: total_tokens must equal batch");
  if (a->num_q_heads < 0 || a->num_q_heads > 4096) Fail(DSD_EINVAL, "num_q_heads must be in [0, 4096]");
  if (a->max_pages_per_request < 0 || a->page_table_stride < 0)
    Fail(DSD_EINVAL, "page-table sizes must not be negative");
  if ((a->cos == nullptr) != (a->sin == nullptr)) Fail(DSD_EINVAL, "cos and sin come together");
  if (a->cos) {
    if (a->rotary_dim < 2 || a->rotary_dim % 2 || a->rotary_dim > c->head_dim)
      Fail(DSD_EINVAL, "rotary_dim must be even, in [2, head_dim]");
    if (a->rotary_positions <= 0) Fail(DSD_EINVAL, "rotary_positions must be positive");
    if (!Aligned(a->cos, 4) || !Aligned(a->sin, 4)) Fail(DSD_EINVAL, "cos and sin must be 4-byte aligned");
  }
  if (a->batch == 0 || a->total_tokens == 0) return;
  CheckCachePointers(c);
  if (!a->k || !a->v || !a->seq_lens || (!a->page_table && a->max_pages_per_request > 0))
    Fail(DSD_EINVAL, "null device array");
  if (a->num_q_heads && (!a->q || !a->q_out)) Fail(DSD_EINVAL, "num_q_heads > 0 needs q and q_out");
  CheckInts(a->token_offsets, a->seq_lens, a->page_table, a->positions, a->token_counts, a->status);
  const int eb = ElemBytes(a->dtype);
  const void* rows[] = {a->k, a->v, a->num_q_heads ? a->q : a->k, a->num_q_heads ? a->q_out : a->k};
  const int64_t* strides[] = {a->k_stride, a->v_stride, a->num_q_heads ? a->q_stride : a->k_stride,
                              a->num_q_heads ? a->q_out_stride : a->k_stride};
  for (int i = 0; i < 4; ++i) {
    if (!Aligned(rows[i], eb)) Fail(DSD_EINVAL, "k, v, q and q_out must be aligned to their type");
    if (strides[i][0] < 0 || strides[i][1] < 0) Fail(DSD_EINVAL, "row strides must not be negative");
  }
  for (const int64_t* st : {c->k_stride, c->v_stride})
    CheckWritten(c->head_dim, {{c->num_pages, st[0]}, {c->page_size, st[1]}, {c->num_kv_heads, st[2]}}, "the cache");
  if (a->num_q_heads)
    CheckWritten(c->head_dim, {{a->total_tokens, a->q_out_stride[0]}, {a->num_q_heads, a->q_out_stride[1]}}, "q_out");

  // 8-element accesses where every row, and each half of its rotated part, starts on
  // their boundary, else single elements (7400 tokens of bf16, 32 + 2 x 8 heads of 96:
  // rotary_dim 32 23 us, rotary_dim 24 96 us)
  const int rd = a->cos ? a->rotary_dim : 0;
  bool wide = rd % 16 == 0;
  for (int i = 0; i < 4; ++i)
    wide = wide && Aligned(rows[i], 16) && strides[i][0] % 8 == 0 && strides[i][1] % 8 == 0;
  if (a->cos) wide = wide && Aligned(a->cos, 16) && Aligned(a->sin, 16);
  wide = wide && Aligned(c->k_codes, 8) && Aligned(c->v_codes, 8);
  for (int i = 0; i < 3; ++i) wide = wide && c->k_stride[i] % 8 == 0 && c->v_stride[i] % 8 == 0;
  const int ve = wide ? 8 : 1;

  DeviceGuard guard(device);
  const Device& dev = DeviceOf(device);
  AppendParams p{};
  p.k = static_cast<uint8_t*>(c->k_codes);
  p.v = static_cast<uint8_t*>(c->v_codes);
  p.ks = c->k_scales;
  p.vs = c->v_scales;
  for (int i = 0; i < 3; ++i) {
    p.kst[i] = c->k_stride[i];
    p.vst[i] = c->v_stride[i];
  }
  p.num_pages = c->num_pages;
  p.P = c->page_size;
  p.Hk = c->num_kv_heads;
  p.D = c->head_dim;
  p.bt = c->block_tokens;
  p.nblk = c->page_size / c->block_tokens;
  p.kin = a->k;
  p.vin = a->v;
  p.qin = a->q;
  p.qout = a->q_out;
  for (int i = 0; i < 2; ++i) {
    p.kin_st[i] = a->k_stride[i];
    p.vin_st[i] = a->v_stride[i];
    p.qin_st[i] = a->q_stride[i];
    p.qout_st[i] = a->q_out_stride[i];
  }
  p.batch = a->batch;
  p.total = a->total_tokens;
  p.max_pages = a->max_pages_per_request;
  p.Hq = a->num_q_heads;
  p.off = a->token_offsets;
  p.lens = a->seq_lens;
  p.table = a->page_table;
  p.table_stride = a->page_table_stride;
  p.cos = a->cos;
  p.sin = a->sin;
  p.positions = a->positions;
  p.rot_positions = a->rotary_positions;
  p.rd = rd;
  p.interleaved = a->interleaved != 0;
  p.counts = a->token_counts;
  p.status = a->status;
  p.slots = (p.D + 2 * ve - 1) / (2 * ve);
  const int64_t units = p.off ? int64_t(p.total) / p.bt + 2 * int64_t(p.batch) : p.batch;
  if (units > INT32_MAX) Fail(DSD_EINVAL, "too many tokens for one call");
  // A team of warps holds a head's block whole, one slot a lane where a warp can (a
  // decode step), else two, four in the largest teams; blocks beyond that are read twice.
  const int block_slots = (p.off ? std::min(p.bt, p.total) : 1) * p.slots;
  const int largest = dsds::kAppendThreads * 4;
  const int j = ve == 1 || block_slots > largest ? 0 : block_slots <= 32 ? 1 : block_slots <= largest / 2 ? 2 : 4;
  p.team = 1;
  while (p.team < 8 && p.team * 32 * (j ? j : dsds::kAppendKeep) < block_slots) p.team *= 2;
  // blockIdx.y: CTAs of one block of tokens, keys and values first, then queries; as
  // many as give every SM one when there are few blocks, else up to eight rounds (of
  // heads) to a CTA: its first loads wait for one another (offsets, lengths, pages), so
  // fewer and longer CTAs win (7400 tokens of int8: 45 us, with eight CTAs per SM and
  // four rounds 52 us).
  const int teams = dsds::kAppendThreads / 32 / p.team;
  const auto parts = [&](int rounds) {
    const int64_t want = (dev.sms + units - 1) / units;
    return int(std::min<int64_t>(rounds, std::max<int64_t>(want, (rounds + 7) / 8)));
  };
  p.y_kv = parts(((j ? 1 : 2) * p.Hk + teams - 1) / teams);
  const int y_q = p.Hq ? parts((p.Hq + 4 * dsds::kAppendHeads - 1) / (4 * dsds::kAppendHeads)) : 0;
  const dim3 grid{static_cast<unsigned>(units), static_cast<unsigned>(p.y_kv + y_q), 1};
  const bool i8 = c->kv_format == DSD_KV_I8_SCALED;
  if (a->dtype == DSD_TYPE_F32) LaunchAppend<float>(p, i8, ve, j, grid, s);
  else if (a->dtype == DSD_TYPE_BF16) LaunchAppend<__nv_bfloat16>(p, i8, ve, j, grid, s);
  else LaunchAppend<__half>(p, i8, ve, j, grid, s);
}

// --------------------------------------------------------------- attention

constexpr int kSimpleMaxSmem = 4 * (8 * 256 + 8 * dsds::kTile + 4 * dsds::kTile + 24 + dsds::kMaxBatch) + 64;

template <bool I8, int R>
void SetSimple() {
  Check(cudaFuncSetAttribute(dsds::attn_simple_kernel<I8, R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kSimpleMaxSmem), "shared memory attribute");
}

// f(kernel, shape) for the tensor-core kernel of R query rows
template <typename T>
struct Tag { using type = T; };
template <bool I8, int PIECES, int R, typename F>
void WithTcRows(F&& f) { f(dsds::attn_tc_kernel<I8, R, PIECES>, Tag<dsds::TcShape<R, PIECES>>{}); }
template <bool I8, int PIECES, typename F>
void WithTc(int R, F&& f) {
  switch (R) {
    case 1: return WithTcRows<I8, PIECES, 1>(f);
    case 2: return WithTcRows<I8, PIECES, 2>(f);
    case 4: return WithTcRows<I8, PIECES, 4>(f);
    default: return WithTcRows<I8, PIECES, 8>(f);
  }
}
template <typename F>
void WithTc(bool i8, bool fp32, int R, F&& f) {
  if (i8 && fp32) return WithTc<true, 4>(R, f);
  if (i8) return WithTc<true, 3>(R, f);
  if (fp32) return WithTc<false, 6>(R, f);
  return WithTc<false, 3>(R, f);
}
constexpr int kTcMaxRows = 8;   // query rows of a narrow unit

// More query rows of a request than this, on average, go to the wide kernel (never
// fp32, see there).  The narrow one reads the cache once for every 8 rows, the wide
// one widens each tile once whatever the rows.  64 requests of 1024-4096 tokens, 4 key
// heads, bf16, narrow / wide: 12 rows 88 / 115 us, 16 rows 90 / 115, 20 rows 129 / 124,
// 24 rows 127 / 117, 28 rows 163 / 128, 48 rows 237 / 131; int8 at 16 rows 88 / 119, at
// 24 124 / 137, at 28 153 / 137; fp16 98 / 146, 130 / 141 and 167 / 151.  Between 16 and
// 24 the two are near one another, unless a chunk stands among single tokens: with 63
// of those, one of 100 queries (12 rows) 174 / 243, one of 320 (24 rows) 325 / 268.
constexpr int kNarrowMaxRows = 16;

template <typename F>
void WithWide(bool i8, int dtype, F&& f) {
  const bool two = dtype == DSD_TYPE_F16;
  if (i8 && two) f(dsds::attn_wide_kernel<true, 2>, Tag<dsds::WideShape<2>>{});
  else if (i8) f(dsds::attn_wide_kernel<true, 1>, Tag<dsds::WideShape<1>>{});
  else if (two) f(dsds::attn_wide_kernel<false, 2>, Tag<dsds::WideShape<2>>{});
  else f(dsds::attn_wide_kernel<false, 1>, Tag<dsds::WideShape<1>>{});
}

void SetAttentionAttributes(int device) {
  SetSimple<false, 1>(); SetSimple<false, 2>(); SetSimple<false, 4>(); SetSimple<false, 8>();
  SetSimple<true, 1>(); SetSimple<true, 2>(); SetSimple<true, 4>(); SetSimple<true, 8>();
  int reserve = 0, shared = 0, registers = 0;   // of a block; of an SM
  Check(cudaDeviceGetAttribute(&reserve, cudaDevAttrReservedSharedMemoryPerBlock, device), "device");
  Check(cudaDeviceGetAttribute(&shared, cudaDevAttrMaxSharedMemoryPerMultiprocessor, device), "device");
  Check(cudaDeviceGetAttribute(&registers, cudaDevAttrMaxRegistersPerMultiprocessor, device), "device");
  for (int i8 = 0; i8 < 2; ++i8)
    for (int fp32 = 0; fp32 < 2; ++fp32) {
      // The plan cuts the work for this many CTAs per SM.  (The occupancy call answers one
      // for every kernel that allocates tensor memory, also where two run.)
      const auto set = [&](auto kernel, auto tag, int threads, int ctas) {
        using Shape = typename decltype(tag)::type;
        Check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Shape::kSmem)),
              "shared memory attribute");
        cudaFuncAttributes fa;
        Check(cudaFuncGetAttributes(&fa, kernel), "function attributes");
        const size_t bytes = (fa.sharedSizeBytes + Shape::kSmem + reserve + 127) / 128 * 128;
        if (bytes * ctas > size_t(shared) || (fa.numRegs + 7) / 8 * 8 * threads * ctas > registers)
          Fail(DSD_EUNAVAILABLE, "an SM has no room for " + std::to_string(ctas) + " attention blocks of " +
                                     std::to_string(bytes) + " bytes and " + std::to_string(fa.numRegs) + " registers");
      };
      const auto set_narrow = [&](auto kernel, auto tag) {
        set(kernel, tag, dsds::kTcThreads, decltype(tag)::type::kCtas);
      };
      const auto set_wide = [&](auto kernel, auto tag) { set(kernel, tag, dsds::kWideThreads, 1); };
      for (int R = 1; R <= kTcMaxRows; R *= 2) WithTc(i8, fp32, R, set_narrow);
      WithWide(i8, fp32 ? DSD_TYPE_F16 : DSD_TYPE_BF16, set_wide);
    }
}

template <bool I8>
void LaunchSimple(const AttnParams& p, cudaStream_t s) {
  const size_t smem = dsds::simple_smem(p.R, p.D, p.batch);
  switch (p.R) {
    case 1: Launch(dsds::attn_simple_kernel<I8, 1>, dim3(p.ncta), dsds::kSimpleThreads, smem, s, p); break;
    case 2: Launch(dsds::attn_simple_kernel<I8, 2>, dim3(p.ncta), dsds::kSimpleThreads, smem, s, p); break;
    case 4: Launch(dsds::attn_simple_kernel<I8, 4>, dim3(p.ncta), dsds::kSimpleThreads, smem, s, p); break;
    default: Launch(dsds::attn_simple_kernel<I8, 8>, dim3(p.ncta), dsds::kSimpleThreads, smem, s, p); break;
  }
}

// TMA's view of one code array: elements, then tokens and heads by their stride,
// then pages.  Only such orders can be encoded: every stride a multiple of 16
// bytes and of the one before it.
struct CodeOrder {
  bool ok = false, head_first = false;
  int64_t stride[3];   // of dimensions 1, 2, 3
};

CodeOrder OrderOf(const dsd_scaled_cache* c, const void* codes, const int64_t* st, bool head_first) {
  CodeOrder o;
  o.head_first = head_first;
  const int64_t sizes[3] = {head_first ? c->num_kv_heads : c->page_size, head_first ? c->page_size : c->num_kv_heads,
                            c->num_pages};
  const int64_t given[3] = {head_first ? st[2] : st[1], head_first ? st[1] : st[2], st[0]};
  // a dimension of one may have any stride: it takes the least that fits
  int64_t before = 16, span = (c->head_dim + 15) / 16 * 16;
  for (int i = 0; i < 3; ++i) {
    o.stride[i] = sizes[i] > 1 ? given[i] : span;
    if (o.stride[i] % before || o.stride[i] < c->head_dim || o.stride[i] >= (int64_t(1) << 40)) return o;
    before = o.stride[i];
    span = std::max(span, o.stride[i] * sizes[i]);
  }
  o.ok = Aligned(codes, 16);
  return o;
}

struct TcMaps { CodeOrder k, v; };

// The rule of the tensor-core path: rows of 16 to 128 bytes in 16-byte steps (one
// 128-byte operand row, the rest of it zero-filled by TMA), pages of whole
// 8-row swizzle groups, and strides that TMA takes.  Everything else runs on the
// fp32 pipes.
bool TensorCores(const dsd_scaled_cache* c, TcMaps* maps) {
  if (c->head_dim % 16 || c->head_dim > 128 || c->page_size % 8) return false;
  for (const bool head_first : {true, false}) {
    maps->k = OrderOf(c, c->k_codes, c->k_stride, head_first);
    maps->v = OrderOf(c, c->v_codes, c->v_stride, head_first);
    if (maps->k.ok && maps->v.ok) return true;
  }
  return false;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled Encoder() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  if (!fn) Fail(DSD_ECUDA, "the driver has no cuTensorMapEncodeTiled");
  return fn;
}

CUtensorMap MapOf(const dsd_scaled_cache* c, const void* codes, const CodeOrder& o) {
  const cuuint32_t rows = cuuint32_t(std::min(c->page_size, dsds::kTile));
  const cuuint64_t tokens = cuuint64_t(c->page_size), heads = cuuint64_t(c->num_kv_heads);
  const cuuint64_t dims[4] = {cuuint64_t(c->head_dim), o.head_first ? heads : tokens, o.head_first ? tokens : heads,
                              cuuint64_t(c->num_pages)};
  const cuuint64_t strides[3] = {cuuint64_t(o.stride[0]), cuuint64_t(o.stride[1]), cuuint64_t(o.stride[2])};
  const cuuint32_t box[4] = {128, o.head_first ? 1 : rows, o.head_first ? rows : 1, 1};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  CUtensorMap map;
  const CUresult r = Encoder()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(codes), dims, strides, box,
                               ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) Fail(DSD_ECUDA, "cuTensorMapEncodeTiled failed (" + std::to_string(int(r)) + ")");
  return map;
}

struct AttnPlan {
  bool tc = false, wide = false;
  TcMaps maps;
  int R = 1, ncta = 0, gangs = 0;
  int64_t ml_at = 0, o_at = 0, bytes = 0;   // workspace: meta, then ml, then O
};

AttnPlan PlanAttention(const Device& dev, const dsd_scaled_cache* c, const dsd_scaled_attention_args* a) {
  AttnPlan pl;
  const int group = a->num_q_heads / c->num_kv_heads;
  const bool i8 = c->kv_format == DSD_KV_I8_SCALED, fp32 = a->dtype == DSD_TYPE_F32;
  pl.tc = TensorCores(c, &pl.maps);
  // query rows of a request: exact for one query each, the average otherwise
  const int64_t queries = a->q_offsets ? (int64_t(a->total_queries) + a->batch - 1) / a->batch : 1;
  const int64_t rows = queries * group;
  pl.wide = pl.tc && !fp32 && rows > kNarrowMaxRows;
  if (pl.wide) pl.R = dsds::kWideRows;
  while (pl.R < kTcMaxRows && pl.R < rows) pl.R *= 2;
  int per_sm = pl.wide ? 1 : 8;
  if (pl.tc && !pl.wide)
    WithTc(i8, fp32, pl.R, [&](auto, auto tag) { per_sm = decltype(tag)::type::kCtas; });
  pl.gangs = std::max(1, per_sm * dev.sms / c->num_kv_heads);
  pl.ncta = pl.gangs * c->num_kv_heads;
  if (pl.gangs > dsds::kMaxPieces) Fail(DSD_EUNAVAILABLE, "more SMs than the join is laid out for");
  pl.ml_at = (int64_t(pl.ncta) * 16 + 255) / 256 * 256;
  pl.o_at = pl.ml_at + (int64_t(pl.ncta) * 2 * pl.R * 8 + 255) / 256 * 256;
  pl.bytes = pl.o_at + int64_t(pl.ncta) * 2 * pl.R * c->head_dim * 4;
  return pl;
}

void CheckAttention(const dsd_scaled_cache* c, const dsd_scaled_attention_args* a) {
  CheckCache(c);
  if (!a) Fail(DSD_EINVAL, "null arguments");
  CheckType(a->dtype);
  if (a->batch < 0 || a->batch > dsds::kMaxBatch) Fail(DSD_EINVAL, "batch must be in [0, 4096]");
  if (a->total_queries < 0) Fail(DSD_EINVAL, "total_queries must not be negative");
  if (!a->q_offsets && a->total_queries != a->batch)
    Fail(DSD_EINVAL, "without q_offsets every request has one query: total_queries must equal batch");
  if (a->num_q_heads < 1 || a->num_q_heads > 4096 || a->num_q_heads % c->num_kv_heads)
    Fail(DSD_EINVAL, "num_q_heads must be a multiple of num_kv_heads, at most 4096");
  if (int64_t(a->total_queries) * a->num_q_heads > INT32_MAX - 4096)
    Fail(DSD_EINVAL, "too many query rows for one call");
  if (a->max_pages_per_request < 0 || a->page_table_stride < 0)
    Fail(DSD_EINVAL, "page-table sizes must not be negative");
  if (a->window < 0) Fail(DSD_EINVAL, "window must not be negative");
  if (a->page_counts && (a->causal || a->window))
    Fail(DSD_EINVAL, "a page list has no order: causal and window must be 0 with page_counts");
  if (a->page_counts && int64_t(a->max_pages_per_request) * (c->page_size / dsds::kTile + 1) > INT32_MAX)
    Fail(DSD_EINVAL, "the page lists are too long for one call");
  if (!std::isfinite(a->scale)) Fail(DSD_EINVAL, "scale must be finite");
}

void Attention(int device, const dsd_scaled_cache* c, const dsd_scaled_attention_args* a, cudaStream_t s) {
  NvtxRange nvtx("dsd_scaled_attention");
  CheckAttention(c, a);
  if (a->batch == 0 || a->total_queries == 0) return;
  CheckCachePointers(c);
  if (!a->q || !a->out || !a->lens || (!a->page_table && a->max_pages_per_request > 0))
    Fail(DSD_EINVAL, "null device array");
  CheckInts(a->q_offsets, a->lens, a->page_table, a->page_counts, a->status);
  const int eb = ElemBytes(a->dtype);
  if (!Aligned(a->q, eb) || !Aligned(a->out, eb) || !Aligned(a->lse, 4))
    Fail(DSD_EINVAL, "q, out and lse must be aligned to their type");
  for (int i = 0; i < 2; ++i)
    if (a->q_stride[i] < 0 || a->out_stride[i] < 0) Fail(DSD_EINVAL, "row strides must not be negative");
  CheckWritten(c->head_dim, {{a->total_queries, a->out_stride[0]}, {a->num_q_heads, a->out_stride[1]}}, "out");
  DeviceGuard guard(device);
  const Device& dev = DeviceOf(device);
  const AttnPlan pl = PlanAttention(dev, c, a);
  if (!a->workspace || !Aligned(a->workspace, 16) || a->workspace_bytes < pl.bytes)
    Fail(DSD_EINVAL, "workspace must be 16-byte aligned with at least " + std::to_string(pl.bytes) + " bytes");

  AttnParams p{};
  p.k = static_cast<const uint8_t*>(c->k_codes);
  p.v = static_cast<const uint8_t*>(c->v_codes);
  p.ks = c->k_scales;
  p.vs = c->v_scales;
  for (int i = 0; i < 3; ++i) {
    p.kst[i] = c->k_stride[i];
    p.vst[i] = c->v_stride[i];
  }
  p.num_pages = c->num_pages;
  p.P = c->page_size;
  p.Hk = c->num_kv_heads;
  p.D = c->head_dim;
  p.bt = c->block_tokens;
  p.nblk = c->page_size / c->block_tokens;
  p.q = a->q;
  p.out = a->out;
  p.lse = a->lse;
  for (int i = 0; i < 2; ++i) {
    p.qst[i] = a->q_stride[i];
    p.ost[i] = a->out_stride[i];
  }
  p.dtype = a->dtype;
  p.batch = a->batch;
  p.total_q = a->total_queries;
  p.H = a->num_q_heads;
  p.G = a->num_q_heads / c->num_kv_heads;
  p.q_off = a->q_offsets;
  p.lens = a->lens;
  p.table = a->page_table;
  p.table_stride = a->page_table_stride;
  p.max_pages = a->max_pages_per_request;
  p.counts = a->page_counts;
  p.scale_log2 = static_cast<float>(double(a->scale) * 1.4426950408889634);
  p.causal = a->causal != 0;
  // a window of all places is none
  p.window = a->window >= 1ll * a->max_pages_per_request * c->page_size ? 0 : a->window;
  p.status = a->status;
  p.ppt = p.P <= dsds::kTile ? dsds::kTile / p.P : 0;
  p.tpp = p.P <= dsds::kTile ? 0 : (p.P + dsds::kTile - 1) / dsds::kTile;
  p.R = pl.R;
  // one query each, at most 128 requests, and no sum of tiles beyond an int
  const int64_t tiles = p.counts ? int64_t(p.max_pages) * std::max(1, p.tpp)
                                 : (int64_t(p.max_pages) * p.P + 7) / 8 + p.max_pages;
  p.few = !p.q_off && p.batch <= 128 && tiles * ((p.G + p.R - 1) / p.R) * p.batch < INT32_MAX;
  p.by_page = dsds::divisor_of(p.P);
  p.by_group = dsds::divisor_of(p.G);
  p.by_block = dsds::divisor_of(p.bt);
  p.by_tpp = dsds::divisor_of(std::max(1, p.tpp));
  p.by_tile = dsds::divisor_of(std::max(1, p.ppt * p.P));
  p.token_entries = (dsds::kTile + p.bt - 1) / p.bt + 1;
  p.token_stages = std::min(dsds::kTokenStages, dsds::kTokenBytes / (12 * p.token_entries));
  p.ncta = pl.ncta;
  p.gangs = pl.gangs;
  char* ws = static_cast<char*>(a->workspace);
  p.meta = reinterpret_cast<int4*>(ws);
  p.part_ml = reinterpret_cast<float*>(ws + pl.ml_at);
  p.part_o = reinterpret_cast<float*>(ws + pl.o_at);

  const bool i8 = c->kv_format == DSD_KV_I8_SCALED;
  if (pl.tc) {
    const CUtensorMap k_map = MapOf(c, c->k_codes, pl.maps.k), v_map = MapOf(c, c->v_codes, pl.maps.v);
    const bool fp32 = a->dtype == DSD_TYPE_F32;
    const auto launch = [&](auto kernel, auto tag) {
      Launch(kernel, dim3(p.ncta), pl.wide ? dsds::kWideThreads : dsds::kTcThreads, decltype(tag)::type::kSmem, s, p,
             k_map, v_map, int(pl.maps.k.head_first));
    };
    if (pl.wide) WithWide(i8, a->dtype, launch);
    else WithTc(i8, fp32, p.R, launch);
  } else if (i8) {
    LaunchSimple<true>(p, s);
  } else {
    LaunchSimple<false>(p, s);
  }
  Launch(dsds::combine_kernel, dim3(unsigned(p.ncta), unsigned(std::min(p.R, 32))), p.D <= 128 ? 128 : 256, 0, s, p);
}

__global__ void take_status_kernel(int* status, int* bits) {
  dsds::pdl_wait();
  *bits = atomicExch(status, 0);
}

void TakeStatus(int device, int32_t* status, int32_t* bits, cudaStream_t s) {
  if (!status || !bits || !Aligned(status, 4) || !Aligned(bits, 4))
    Fail(DSD_EINVAL, "status and bits must be 4-byte aligned device words");
  DeviceGuard guard(device);
  DeviceOf(device);
  Launch(take_status_kernel, dim3(1), 1, 0, s, status, bits);
}

}  // namespace

extern "C" {

int dsd_scaled_append(int device, const dsd_scaled_cache* cache, const dsd_scaled_append_args* args,
                      void* stream) {
  return Guard([&]() { Append(device, cache, args, static_cast<cudaStream_t>(stream)); });
}

int dsd_scaled_attention_workspace(int device, const dsd_scaled_cache* cache,
                                   const dsd_scaled_attention_args* args, int64_t* bytes) {
  return Guard([&]() {
    CheckAttention(cache, args);
    if (!bytes) Fail(DSD_EINVAL, "null result");
    *bytes = 0;
    if (args->batch == 0 || args->total_queries == 0) return;
    DeviceGuard guard(device);
    *bytes = PlanAttention(DeviceOf(device), cache, args).bytes;
  });
}

int dsd_scaled_attention(int device, const dsd_scaled_cache* cache, const dsd_scaled_attention_args* args,
                         void* stream) {
  return Guard([&]() { Attention(device, cache, args, static_cast<cudaStream_t>(stream)); });
}

int dsd_scaled_take_status(int device, int32_t* status, int32_t* bits, void* stream) {
  return Guard([&]() { TakeStatus(device, status, bits, static_cast<cudaStream_t>(stream)); });
}

}  // extern "C"
