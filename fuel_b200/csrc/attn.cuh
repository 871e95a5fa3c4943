// Attention for batches of sequences: keys and values appended to a paged cache, one new token per sequence over its pages,
// whole packed prompts. Entries in attn.cu, contract in include/fuelq.h.
#pragma once
#include <cuda_bf16.h>

#include "fq_common.cuh"

namespace fq {

cudaError_t attn_device_error(int* code, bool clear);  // the error word of these kernels (attn.cu)

// ---- values of the three types
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 2^x; below 2^-126: zero
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// eight consecutive values, held as they are in memory
template <typename T>
struct Vec8 {
  static constexpr int kWords = sizeof(T) / 2;  // 16-byte words
  uint4 w[kWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32(reinterpret_cast<const T*>(w)[i]);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(w)[i] = from_f32<T>(f[i]);
  }
};

// ---- append -------------------------------------------------------------------------------------
//   lo' = lo * cos - hi * sin,  hi' = hi * cos + lo * sin   with lo, hi the halves of a head, in f32, rounded once into the
//   output's type; the same operations in the same order as rope_store_kernel, so the same bits.
// Bound by HBM for prompts and by latency for single tokens. A thread block takes one row of the batch: its position, page and
// angles are read once per thread and serve all the heads ("lines": query heads, key heads, value heads) the thread walks.
// A thread holds eight elements of the lower half of a line and the eight that they turn with: 16-byte accesses for every type.
struct AppendParams {
  const void *k, *v, *q;
  void *q_out, *k_out, *kc, *vc;
  int64_t k_stride, v_stride, q_stride;
  const int *table, *seq_ids, *positions;
  const float *cos_table, *sin_table;
  int n_seqs, n_heads, n_kv;  // n_heads: 0 without q
  int page_shift, n_pages, max_pages, max_pos;
  int lines_per_block;
};
constexpr int kAppendThreads = 128;

// 64 registers, so that eight blocks an SM keep enough rows in flight. 13009 rows, 32/8 heads of 128: bf16 56.7 us, 5.6 TB/s of rows and
// cache (with more registers and fewer blocks 75.5), f32 98.4, 6.5 TB/s (106.5), f32 over f16 89.3, 6.6 TB/s (99.6). 1023 rows: 5.7 (7.4),
// 10.9 (10.5), 9.8 (9.7)
template <typename A, typename C, int kHd>
__global__ void __launch_bounds__(kAppendThreads, 8) paged_append_kernel(const AppendParams p) {
  constexpr int kHalf = kHd / 2, kChunks = kHalf / 8, kSlots = kAppendThreads / kChunks;
  constexpr int kBatch = 2;  // lines a thread has in flight
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.x;
  const int pos = p.positions[row];
  const int64_t seq = p.seq_ids ? (int64_t)p.seq_ids[row] : row;
  if (pos < 0 || seq < 0) return;  // padding
  const int page_at = pos >> p.page_shift;
  const bool in_table = seq < p.n_seqs && page_at < p.max_pages && pos < p.max_pos;
  const int page = in_table ? p.table[seq * p.max_pages + page_at] : -1;
  if (page < 0 || page >= p.n_pages) {
    if (threadIdx.x == 0) record_dev_error(kErrIndex);
    return;
  }
  const int c = threadIdx.x % kChunks;
  float cs[8], sn[8];
  Vec8<float> t;
  t.load(p.cos_table + (int64_t)pos * kHd + 8 * c);
  t.get(cs);
  t.load(p.sin_table + (int64_t)pos * kHd + 8 * c);
  t.get(sn);
  const int first = blockIdx.y * p.lines_per_block;
  const int last = min(first + p.lines_per_block, p.n_heads + 2 * p.n_kv);
  const int64_t in_page = pos & ((1 << p.page_shift) - 1);
  const A* q = reinterpret_cast<const A*>(p.q) + row * p.q_stride;
  const A* k = reinterpret_cast<const A*>(p.k) + row * p.k_stride;
  const A* v = reinterpret_cast<const A*>(p.v) + row * p.v_stride;
  for (int l0 = first + threadIdx.x / kChunks; l0 < last; l0 += kBatch * kSlots) {
    Vec8<A> lo[kBatch], hi[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int l = l0 + b * kSlots;
      if (l >= last) break;
      const A* src = l < p.n_heads ? q + l * kHd : l < p.n_heads + p.n_kv ? k + (l - p.n_heads) * kHd : v + (l - p.n_heads - p.n_kv) * kHd;
      lo[b].load(src + 8 * c);
      hi[b].load(src + kHalf + 8 * c);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int l = l0 + b * kSlots;
      if (l >= last) break;
      float x[8], y[8];
      lo[b].get(x);
      hi[b].get(y);
      const bool value = l >= p.n_heads + p.n_kv;
      if (!value) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a = x[i], z = y[i];
          x[i] = __fsub_rn(__fmul_rn(a, cs[i]), __fmul_rn(z, sn[i]));
          y[i] = __fadd_rn(__fmul_rn(z, cs[i]), __fmul_rn(a, sn[i]));
        }
      }
      A* out = nullptr;  // the contiguous result beside the cache
      if (l < p.n_heads)
        out = reinterpret_cast<A*>(p.q_out) + (row * p.n_heads + l) * kHd;
      else if (!value && p.k_out)
        out = reinterpret_cast<A*>(p.k_out) + (row * p.n_kv + (l - p.n_heads)) * kHd;
      if (out) {
        Vec8<A> o;
        o.set(x);
        o.store(out + 8 * c);
        o.set(y);
        o.store(out + kHalf + 8 * c);
      }
      if (l >= p.n_heads) {
        const int head = value ? l - p.n_heads - p.n_kv : l - p.n_heads;
        C* dst = reinterpret_cast<C*>(value ? p.vc : p.kc) + ((((int64_t)page * p.n_kv + head) << p.page_shift) + in_page) * kHd;
        Vec8<C> o;
        o.set(x);
        o.store(dst + 8 * c);
        o.set(y);
        o.store(dst + kHalf + 8 * c);
      }
    }
  }
}

}  // namespace fq
