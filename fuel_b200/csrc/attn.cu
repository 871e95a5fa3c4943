// C ABI of the paged-cache and prompt attention (include/fuelq.h, "Attention for batches of sequences"), in a translation unit
// of its own beside fuelq.cu.
#include "../../include/fuelq.h"

#include <cmath>
#include <type_traits>

#include "attn.cuh"
#include "launch.cuh"
#include "paged_decode.cuh"
#include "prompt_attn.cuh"
#include "prompt_attn_f32.cuh"

namespace fq {
namespace {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int type_bytes(int t) { return t == kF32 ? 4 : t == kF16 || t == kBF16 ? 2 : 0; }
inline bool type_pair(int act, int cache) { return type_bytes(act) && type_bytes(cache) && (act == kF32 || act == cache); }
// page_size as a shift, -1 if it is none of the sizes
inline int page_shift_of(int page_size) {
  for (int s = 0; s <= 10; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}
// a row stride in elements: whole 16-byte words, and rows that do not overlap
inline bool stride_ok(int64_t stride, int heads, int head_dim, int act) {
  return stride >= (int64_t)heads * head_dim && stride * type_bytes(act) % 16 == 0;
}
// the kernels take scale log2(e), which has to be a number too
inline bool scale_ok(float scale) { return scale >= 0x1p-100f && scale <= 0x1p127f; }
constexpr int64_t kMaxRows = 0x7fffffff, kMaxPromptRows = (1 << 30) - 256;  // prompts: twice as many are a coordinate of a copy
constexpr int64_t kMaxSlots = 1 << 26;  // empty sequences times heads, which a warp looks through while the others' waits run
constexpr int kMaxHeads = 16383;  // q, k and v heads together are a grid dimension

// f(activation type, cache type, head size) for one of the pairs the entries take
template <typename A, typename C, typename F>
int32_t with_head(int head_dim, F f) {
  if (head_dim == 128) return f(A(), C(), std::integral_constant<int, 128>());
  return f(A(), C(), std::integral_constant<int, 64>());
}
template <typename F>
int32_t with_types(int act, int cache, int head_dim, F f) {
  if (act == kF16) return with_head<__half, __half>(head_dim, f);
  if (act == kBF16) return with_head<__nv_bfloat16, __nv_bfloat16>(head_dim, f);
  if (cache == kF16) return with_head<float, __half>(head_dim, f);
  if (cache == kBF16) return with_head<float, __nv_bfloat16>(head_dim, f);
  return with_head<float, float>(head_dim, f);
}
// the current device's number of SMs, 0 on failure
int sm_count() {
  static int count[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (count[dev] == 0 && cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return count[dev];
}
// once for each kernel and device: more dynamic shared memory than a launch gets by default
template <typename K>
bool allow_smem(K kernel, int bytes, bool (&set)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (!set[dev]) set[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
  return set[dev];
}

// heads of an item of the decode kernel, in eights: one for groups up to eight heads, two beyond (in pieces of sixteen)
inline int decode_tiles_of_heads(int group) { return group <= 8 ? 1 : 2; }
constexpr size_t kDecodeMetaBytes = (size_t)kDecodeMaxBlocks * 2 * sizeof(int4);

template <typename A, typename C, int kHd, int kNT>
int32_t launch_decode(DecodeParams& p, cudaStream_t stream) {
  using Cfg = DecodeCfg<A, C, kHd, kNT>;
  static bool set[64] = {};
  const int sms = sm_count();
  auto kernel = paged_decode_kernel<A, C, kHd, kNT>;
  if (sms == 0 || !allow_smem(kernel, Cfg::kSmem, set)) return kLaunchFailure;
  p.chunks = (p.group + Cfg::kHeads - 1) / Cfg::kHeads;
  const int blocks = sms * Cfg::kPerSm < kDecodeMaxBlocks ? sms * Cfg::kPerSm : kDecodeMaxBlocks;
  cudaError_t e = launch(kernel, dim3((unsigned)blocks), dim3(32 * kDecodeWarps), Cfg::kSmem, stream, p);
  if (e == cudaSuccess)
    e = launch(paged_join_kernel<A, C, kHd, kNT>, dim3((unsigned)blocks, (unsigned)(p.group < Cfg::kHeads ? p.group : Cfg::kHeads)),
               dim3(kHd), 0, stream, p);
  return e == cudaSuccess ? kOk : kLaunchFailure;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// tensor map of 16-bit rows [rows][heads][head_dim], `stride` elements apart: boxes of 128 bytes of one head x box_rows rows, 128-byte
// swizzle, zeros behind the last row
bool make_rows_map(const void* x, int64_t rows, int heads, int head_dim, int64_t stride, int box_rows, CUtensorMap* map) {
  static EncodeTiledFn encode = nullptr;
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess || !fn)
      return false;
    encode = (EncodeTiledFn)fn;
  }
  const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)head_dim * 2, (cuuint64_t)stride * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows}, ones[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(x), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct PromptArgs {
  const void *q, *k, *v;
  void* out;
  const int* cu;
  int64_t q_stride, k_stride, v_stride, n_rows;
  int n_seqs, n_heads, n_kv;
  float c;
  uint8_t* workspace;
};
template <typename T, int kHd>
int32_t launch_prompt(const PromptArgs& r, cudaStream_t stream) {
  using Cfg = PromptCfg<T, kHd>;
  static bool set[64] = {};
  const int sms = sm_count();
  auto kernel = prompt_attn_kernel<T, kHd>;
  if (sms == 0 || !allow_smem(kernel, Cfg::kSmem, set)) return kLaunchFailure;
  PromptParams p = {};
  p.out = r.out, p.v = r.v, p.v_stride = r.v_stride, p.cu = r.cu, p.n_rows = r.n_rows;
  p.n_items = prompt_slots(r.n_rows, r.n_seqs, kPaRows) * r.n_heads;
  p.n_seqs = r.n_seqs, p.n_heads = r.n_heads, p.group = r.n_heads / r.n_kv, p.c = r.c;
  CUtensorMap qmap, kmap, vmap;
  if (!make_rows_map(r.q, r.n_rows, r.n_heads, kHd, r.q_stride, kPaTile, &qmap) ||
      !make_rows_map(r.k, r.n_rows, r.n_kv, kHd, r.k_stride, kPaTile, &kmap) ||
      !make_rows_map(r.v, r.n_rows, r.n_kv, kHd, r.v_stride, kPaTile, &vmap))
    return kLaunchFailure;
  const dim3 grid((unsigned)(p.n_items < sms ? p.n_items : sms));
  return launch(kernel, grid, dim3(kPaThreads), Cfg::kSmem, stream, p, qmap, kmap, vmap) == cudaSuccess ? kOk : kLaunchFailure;
}

// Workspace of the 32-bit form: the parts and powers of q, k and v; where each begins, and the whole
struct PromptF32Workspace {
  size_t q, k, v, q_up, kv_up, marked, bytes;
};
PromptF32Workspace prompt_f32_workspace(int64_t rows, int heads, int kv, int head_dim) {
  PromptF32Workspace w;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t begin = at;
    at += align_up(n, 256);
    return begin;
  };
  w.q = take((size_t)rows * heads * head_dim * 4);
  w.k = take((size_t)rows * kv * head_dim * 4);
  w.v = take((size_t)rows * kv * head_dim * 4);
  w.q_up = take((size_t)rows * heads * sizeof(float));
  w.kv_up = take((size_t)rows * kv * sizeof(float2));
  w.marked = take((size_t)rows * kv * sizeof(int2));
  w.bytes = at;
  return w;
}
template <int kHd>
int32_t launch_prompt_f32(const PromptArgs& r, cudaStream_t stream) {
  using Cfg = PromptF32Cfg<kHd>;
  static bool set[64] = {};
  const int sms = sm_count();
  auto kernel = prompt_attn_f32_kernel<kHd>;
  if (sms == 0 || !allow_smem(kernel, Cfg::kSmem, set)) return kLaunchFailure;
  const PromptF32Workspace w = prompt_f32_workspace(r.n_rows, r.n_heads, r.n_kv, kHd);
  const int64_t slots = prompt_slots(r.n_rows, r.n_seqs, kPaTile);
  PromptF32Params p = {};
  p.q = (const float*)r.q, p.k = (const float*)r.k, p.v = (const float*)r.v, p.out = (float*)r.out;
  p.q_stride = r.q_stride, p.k_stride = r.k_stride, p.v_stride = r.v_stride, p.cu = r.cu, p.n_rows = r.n_rows;
  p.n_items = slots * r.n_heads, p.n_seqs = r.n_seqs, p.n_heads = r.n_heads, p.n_kv = r.n_kv, p.group = r.n_heads / r.n_kv, p.c = r.c;
  p.qp = (__half*)(r.workspace + w.q), p.kp = (__half*)(r.workspace + w.k), p.vp = (__half*)(r.workspace + w.v);
  p.q_up = (float*)(r.workspace + w.q_up), p.kv_up = (float2*)(r.workspace + w.kv_up), p.marked = (int2*)(r.workspace + w.marked);
  CUtensorMap qmap, kmap, vmap;  // both parts in one map, the second behind the first
  if (!make_rows_map(p.qp, 2 * r.n_rows, r.n_heads, kHd, (int64_t)r.n_heads * kHd, kPaTile, &qmap) ||
      !make_rows_map(p.kp, 2 * r.n_rows, r.n_kv, kHd, (int64_t)r.n_kv * kHd, kPaTile, &kmap) ||
      !make_rows_map(p.vp, 2 * r.n_rows, r.n_kv, kHd, (int64_t)r.n_kv * kHd, Cfg::kUnitKeys, &vmap))
    return kLaunchFailure;
  cudaError_t e = launch(prompt_split_kernel<kHd>, dim3((unsigned)slots, (unsigned)(r.n_heads + 2 * r.n_kv)), dim3(32 * kSplitWarps), 0,
                         stream, p);
  if (e != cudaSuccess) return kLaunchFailure;
  const dim3 grid((unsigned)(p.n_items < sms ? p.n_items : sms));
  return launch(kernel, grid, dim3(kPfaThreads), Cfg::kSmem, stream, p, qmap, kmap, vmap) == cudaSuccess ? kOk : kLaunchFailure;
}

inline int32_t status_of(cudaError_t e) { return e == cudaSuccess ? kOk : kLaunchFailure; }

}  // namespace

cudaError_t attn_device_error(int* code, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_fq_dev_error, sizeof(int));
  if (e == cudaSuccess && clear && *code) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_fq_dev_error, &zero, sizeof(int));
  }
  return e;
}

}  // namespace fq

using namespace fq;

extern "C" {

int32_t fuelq_paged_append(int32_t act_type, int32_t cache_type, const void* k, int64_t k_stride, const void* v,
                           int64_t v_stride, const void* q, int64_t q_stride, void* q_out, void* k_out, void* kcache,
                           void* vcache, const int32_t* page_table, const int32_t* seq_ids, const int32_t* positions,
                           const float* cos_table, const float* sin_table, int64_t n_rows, int32_t n_seqs, int32_t n_heads,
                           int32_t n_kv, int32_t head_dim, int32_t page_size, int32_t n_pages, int32_t max_pages,
                           int32_t max_pos, void* stream) {
  if (!type_pair(act_type, cache_type) || (head_dim != 64 && head_dim != 128)) return kNotSupported;
  const int shift = page_shift_of(page_size);
  if (shift < 0) return kNotSupported;
  if (n_rows < 0 || n_rows > kMaxRows || n_seqs < 0 || n_kv <= 0 || n_pages < 0 || max_pages < 0 || max_pos < 0) return kInvalidProblem;
  if (q && (n_heads <= 0 || n_heads % n_kv)) return kInvalidProblem;
  if (n_rows == 0) return kOk;
  // a cache without pages, a table without columns, angles of no positions: nothing is read of them
  if (!k || !v || !positions || (q && !q_out) || (n_pages && (!kcache || !vcache)) || (max_pages && n_seqs && !page_table) ||
      (max_pos && (!cos_table || !sin_table)))
    return kInvalidProblem;
  if (!stride_ok(k_stride, n_kv, head_dim, act_type) || !stride_ok(v_stride, n_kv, head_dim, act_type)) return kInvalidProblem;
  if (q && !stride_ok(q_stride, n_heads, head_dim, act_type)) return kInvalidProblem;
  if (!seq_ids && n_rows > n_seqs) return kInvalidProblem;
  // in place only where a row is written where it was read
  if ((q && q_out == q && q_stride != (int64_t)n_heads * head_dim) || (k_out == k && k_stride != (int64_t)n_kv * head_dim))
    return kInvalidProblem;
  if (!aligned16(k) || !aligned16(v) || !aligned16(kcache) || !aligned16(vcache) || !aligned16(cos_table) || !aligned16(sin_table) ||
      (q && (!aligned16(q) || !aligned16(q_out))) || !aligned16(k_out))
    return kMisaligned;
  AppendParams p = {};
  p.k = k, p.v = v, p.q = q, p.q_out = q_out, p.k_out = k_out, p.kc = kcache, p.vc = vcache;
  p.k_stride = k_stride, p.v_stride = v_stride, p.q_stride = q ? q_stride : 0;
  p.table = page_table, p.seq_ids = seq_ids, p.positions = positions, p.cos_table = cos_table, p.sin_table = sin_table;
  p.n_seqs = n_seqs, p.n_heads = q ? n_heads : 0, p.n_kv = n_kv;
  p.page_shift = shift, p.n_pages = n_pages, p.max_pages = max_pages, p.max_pos = max_pos;
  // few rows: a block for every 16 (head_dim 64: 32) lines, so that all loads of the call are in flight at once
  const int lines = p.n_heads + 2 * n_kv, slots = kAppendThreads / (head_dim / 16);
  const int pieces = (lines + slots - 1) / slots;
  const bool few = n_rows * pieces <= 1024;
  p.lines_per_block = few ? slots : lines;
  const dim3 grid((unsigned)n_rows, (unsigned)(few ? pieces : 1));
  return with_types(act_type, cache_type, head_dim, [&](auto a, auto c, auto hd) {
    return status_of(launch(paged_append_kernel<decltype(a), decltype(c), decltype(hd)::value>, grid, dim3(kAppendThreads), 0,
                            (cudaStream_t)stream, p));
  });
}

size_t fuelq_paged_attn_workspace_bytes(int32_t n_seqs, int32_t n_heads, int32_t n_kv, int32_t head_dim) {
  if (n_seqs <= 0 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv || (head_dim != 64 && head_dim != 128)) return 0;
  const size_t slot = (size_t)decode_tiles_of_heads(n_heads / n_kv) * 8 * (head_dim + 2) * sizeof(float);
  return kDecodeMetaBytes + 2 * kDecodeMaxBlocks * slot;
}

int32_t fuelq_paged_attn_decode(int32_t act_type, int32_t cache_type, const void* q, int64_t q_stride, const void* kcache,
                                const void* vcache, void* out, const int32_t* page_table, const int32_t* seq_lens,
                                int32_t n_seqs, int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t page_size,
                                int32_t n_pages, int32_t max_pages, float scale, void* workspace, size_t workspace_bytes,
                                void* stream) {
  if (!type_pair(act_type, cache_type) || (head_dim != 64 && head_dim != 128)) return kNotSupported;
  const int shift = page_shift_of(page_size);
  if (shift < 0) return kNotSupported;
  if (n_seqs < 0 || n_kv <= 0 || n_heads <= 0 || n_heads > kMaxHeads || n_heads % n_kv || !scale_ok(scale) || n_pages < 0 || max_pages < 0)
    return kInvalidProblem;
  if (n_seqs == 0) return kOk;
  if (!q || (n_pages && (!kcache || !vcache)) || !out || (max_pages && !page_table) || !seq_lens) return kInvalidProblem;
  if (!stride_ok(q_stride, n_heads, head_dim, act_type)) return kInvalidProblem;
  const size_t need = fuelq_paged_attn_workspace_bytes(n_seqs, n_heads, n_kv, head_dim);
  if (need && (!workspace || workspace_bytes < need)) return kWorkspace;
  if (!aligned16(q) || !aligned16(kcache) || !aligned16(vcache) || !aligned16(out) || !aligned16(workspace)) return kMisaligned;
  DecodeParams p = {};
  p.q = q, p.k = kcache, p.v = vcache, p.out = out, p.q_stride = q_stride, p.table = page_table, p.lens = seq_lens;
  p.n_seqs = n_seqs, p.n_heads = n_heads, p.n_kv = n_kv, p.group = n_heads / n_kv;
  p.page_shift = shift, p.n_pages = n_pages, p.max_pages = max_pages, p.scale = scale;
  p.meta = (int4*)workspace, p.slots = (float*)((uint8_t*)workspace + kDecodeMetaBytes);
  return with_types(act_type, cache_type, head_dim, [&](auto a, auto c, auto hd) {
    using Act = decltype(a);
    using Cache = decltype(c);
    constexpr int kHd = decltype(hd)::value;
    return decode_tiles_of_heads(p.group) == 1 ? launch_decode<Act, Cache, kHd, 1>(p, (cudaStream_t)stream)
                                               : launch_decode<Act, Cache, kHd, 2>(p, (cudaStream_t)stream);
  });
}

size_t fuelq_prompt_attn_workspace_bytes(int32_t act_type, int64_t n_rows, int32_t n_heads, int32_t n_kv, int32_t head_dim) {
  if (!type_bytes(act_type) || n_rows <= 0 || n_rows > kMaxPromptRows || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  return act_type == kF32 ? prompt_f32_workspace(n_rows, n_heads, n_kv, head_dim).bytes : 0;
}

int32_t fuelq_prompt_attn(int32_t act_type, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                          int64_t v_stride, void* out, const int32_t* cu_seqlens, int32_t n_seqs, int64_t n_rows,
                          int32_t n_heads, int32_t n_kv, int32_t head_dim, float scale, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (!type_bytes(act_type) || (head_dim != 64 && head_dim != 128)) return kNotSupported;
  if (n_seqs < 0 || n_rows < 0 || n_rows > kMaxPromptRows || n_kv <= 0 || n_heads <= 0 || n_heads > kMaxHeads || n_heads % n_kv ||
      !scale_ok(scale))
    return kInvalidProblem;
  if ((int64_t)n_seqs * n_heads > kMaxSlots) return kNotSupported;
  if (n_seqs == 0 || n_rows == 0) return kOk;
  if (!q || !k || !v || !out || !cu_seqlens) return kInvalidProblem;
  if (!stride_ok(q_stride, n_heads, head_dim, act_type) || !stride_ok(k_stride, n_kv, head_dim, act_type) ||
      !stride_ok(v_stride, n_kv, head_dim, act_type))
    return kInvalidProblem;
  const size_t need = fuelq_prompt_attn_workspace_bytes(act_type, n_rows, n_heads, n_kv, head_dim);
  if (need && (!workspace || workspace_bytes < need)) return kWorkspace;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(workspace)) return kMisaligned;
  PromptArgs a = {};
  a.q = q, a.k = k, a.v = v, a.out = out, a.cu = cu_seqlens, a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
  a.n_rows = n_rows, a.n_seqs = n_seqs, a.n_heads = n_heads, a.n_kv = n_kv, a.c = scale * 1.4426950408889634f;
  a.workspace = (uint8_t*)workspace;
  cudaStream_t st = (cudaStream_t)stream;
  if (act_type == kF16) return head_dim == 128 ? launch_prompt<__half, 128>(a, st) : launch_prompt<__half, 64>(a, st);
  if (act_type == kBF16) return head_dim == 128 ? launch_prompt<__nv_bfloat16, 128>(a, st) : launch_prompt<__nv_bfloat16, 64>(a, st);
  return head_dim == 128 ? launch_prompt_f32<128>(a, st) : launch_prompt_f32<64>(a, st);
}

}  // extern "C"
