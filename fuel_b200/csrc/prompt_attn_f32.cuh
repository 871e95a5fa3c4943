// Causal attention inside packed prompts (fuelq_prompt_attn) for 32-bit activations, to 32-bit accuracy on the f16 tensor cores.
//
// Every factor is a power of two times two f16 parts, x = 2^e (hi + lo), 22 bits, and a product is three of theirs, summed in
// f32: hi hi + lo hi + hi lo (lo lo is below 2^-22). f16 at three products is twice as fast as bf16 at the six that it would
// take for as many bits, or tf32 at its half rate; what f16 lacks in range the powers of two give:
//   q, k   one for each row and head: S = (Q' K'^T)_ij 2^(eq_i + ek_j)
//   v      one for each row and head, put into the weight: with f_j the row's power, w_ij = 2^(s_ij + f_j - m_i), m the maximum of
//          s + f in the key tile, so that w V' has f16's range whatever the rows' magnitudes. sum_j w_ij 2^-f_j is the softmax's
//          sum in the same unit as O = sum_j w_ij V'_j, so the result is their quotient
// A score is added to a whole power there, which loses nothing while the score is below 2^23 or so, and scores at f32's ends leave it.
// Rows whose largest is beyond 2^22 (in units of the exponent) are computed once more at the end, with sums in 64 bits
// (weigh_again), and so are rows that see values of more than 2^100 apart, whose sums would need more than f32's range. The powers
// of v stay above 2^-80 and, in a tile, within 2^100 of the largest before them: no row loses bits to a larger one behind it.
// prompt_split_kernel writes the parts and powers (bound by HBM: 4 bytes in, 4 out); values that are not finite are taken out of v
// there, and the tiles that had some are marked: the few rows that see one add it again from the original at the end.
// The tensor cores' f32 sums round towards zero, which over a long row adds up (1.6e-5 of it at 4000 keys). So they sum one
// key tile at a time, and the tiles' results are added in registers, rounded to nearest, each with its maximum: the softmax of a
// tile needs nothing from the tile before, and two warpgroups take the tiles in turn.
// Bound by the tensor cores: three times the 16-bit kernel's products. One tile of 128 query rows per thread block; S of the next
// key tile is in tensor memory before the weights of this one are needed, so softmax and sums run beside the products. K and
// V come in units of 16 KB through a ring each, a tile long, and a product frees its units one by one: there is no room
// for a second tile.
//   warps 0-3, 4-7  softmax of every other key tile: a thread per row
//   warps 8-11      O: a thread per row adds the tiles' products, finishes and stores it
//   warps 12, 15    copies: the parts of Q and K, of V
//   warp 13         issues the MMAs
//   warp 14         finds the block's items and brings the powers of each key tile
// Measured, 32/8 heads of 128: 512 tokens 34.7 us (the split some 8 of them), 4096 tokens 525 us: 262 TFLOP/s of the scores that are
// seen, 786 of f16 products; heads of 64 410 us. An issuing warp that waits for ten units and flags a key tile bounds it now, some 300
// cycles each. Of 4096 rows of four heads, 125 us, one infinite column of the values makes 0.37 ms, scores beyond 2^22 in every row 21 ms.
#pragma once
#include "prompt_attn.cuh"

namespace fq {

struct PromptF32Params {
  const float *q, *k, *v;
  float* out;
  int64_t q_stride, k_stride, v_stride;
  const int* cu;
  int64_t n_rows, n_items;
  int n_seqs, n_heads, n_kv, group;
  float c;
  // workspace
  __half *qp, *kp, *vp;  // parts: [2][n_rows][heads][hd]
  float* q_up;           // [heads][n_rows]    c 2^eq
  float2* kv_up;         // [n_kv][n_rows]     2^ek, f
  int2* marked;          // [n_kv][n_rows]     at the first row of a tile: does it hold a value that is not finite (bit 0), 128 + its
                         //                    largest f (bits 8 to 15) and its least (16 to 23); its largest ek
};

// one tile of 128 rows of one head; 64 registers, so that two blocks an SM have 64 KB each in flight (512 rows, 96 heads: one block of 256
// threads an SM took 26 us)
constexpr int kSplitWarps = 16;
template <int kHd>
__global__ void __launch_bounds__(32 * kSplitWarps, 2) prompt_split_kernel(const PromptF32Params p) {
  constexpr int kPer = kHd / 32;
  pdl_launch_dependents();
  pdl_wait();
  const PromptBlock b = prompt_block(p.cu, p.n_seqs, p.n_rows, blockIdx.x, kPaTile);
  if (b.row >= b.len) {
    if (b.len < 0 && blockIdx.y == 0 && threadIdx.x == 0) record_dev_error(kErrIndex);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kind = (int)blockIdx.y < p.n_heads ? 0 : (int)blockIdx.y < p.n_heads + p.n_kv ? 1 : 2;
  const int head = (int)blockIdx.y - (kind == 0 ? 0 : kind == 1 ? p.n_heads : p.n_heads + p.n_kv), heads = kind == 0 ? p.n_heads : p.n_kv;
  const float* src = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
  const int64_t stride = kind == 0 ? p.q_stride : kind == 1 ? p.k_stride : p.v_stride;
  __half* dst = kind == 0 ? p.qp : kind == 1 ? p.kp : p.vp;
  const int64_t plane = p.n_rows * heads * kHd;
  const int rows = min(kPaTile, b.len - b.row);
  constexpr int kMine = kPaTile / kSplitWarps;  // rows of a warp
  alignas(16) float x[kMine][kPer];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const float* in = src + (b.first + b.row + warp + kSplitWarps * i) * stride + head * kHd + lane * kPer;
    if (warp + kSplitWarps * i >= rows) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[i][e] = 0.f;
    } else if constexpr (kPer == 4) {
      *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(in);
    } else {
      *reinterpret_cast<float2*>(x[i]) = *reinterpret_cast<const float2*>(in);
    }
  }
  bool odd = false;
  int power[kMine];  // the largest value of a row comes to [2^14, 2^15)
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const bool fin = isfinite(x[i][e]);
      if (fin) top = fmaxf(top, fabsf(x[i][e]));
      if (kind == 2 && !fin) odd = true, x[i][e] = 0.f;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    power[i] = top > 0.f ? ilogbf(top) - 14 : -1000;
  }
  // k, v: the largest power of a row and those before it in the tile. Lane l finds it for row 4 l + the last two bits of this warp's rows
  __shared__ alignas(16) int power_s[kPaTile];
  __shared__ int least_s;
  int before = 0, most = 0, least = 1000;
  if (kind != 0) {
    if (threadIdx.x == 0) least_s = 1000;
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      if (lane == 0) power_s[warp + kSplitWarps * i] = power[i];
    __syncthreads();
    const int4 q = reinterpret_cast<const int4*>(power_s)[lane];
    const int of[4] = {q.x, max(q.x, q.y), max(max(q.x, q.y), q.z), max(max(q.x, q.y), max(q.z, q.w))};
    int upto = of[3];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto = max(upto, o);
    }
    const int lower = __shfl_up_sync(0xffffffffu, upto, 1), own = warp & 2 ? (warp & 1 ? of[3] : of[2]) : (warp & 1 ? of[1] : of[0]);
    before = lane ? max(lower, own) : own;
    most = __shfl_sync(0xffffffffu, upto, 31);
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int largest = __shfl_sync(0xffffffffu, before, (warp + kSplitWarps * i) >> 2);
    if (warp + kSplitWarps * i >= rows) break;
    const int64_t row = b.first + b.row + warp + kSplitWarps * i;
    // q, k: a row of zeros or nothing but denormals keeps a power in f32's range
    const int e0 = kind == 2 ? max(power[i], max(largest - 100, -80)) : max(power[i], -112);
    least = min(least, e0);
    const float down = exp2f((float)-e0);
    alignas(8) __half hi[kPer], lo[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float y = x[i][e] * down;
      hi[e] = __float2half_rn(y);
      lo[e] = isfinite(y) ? __float2half_rn(y - __half2float(hi[e])) : __ushort_as_half(0);
    }
    __half* o = dst + (row * heads + head) * kHd + lane * kPer;
    if constexpr (kPer == 4) {
      *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(hi);
      *reinterpret_cast<uint2*>(o + plane) = *reinterpret_cast<const uint2*>(lo);
    } else {
      *reinterpret_cast<uint32_t*>(o) = *reinterpret_cast<const uint32_t*>(hi);
      *reinterpret_cast<uint32_t*>(o + plane) = *reinterpret_cast<const uint32_t*>(lo);
    }
    if (lane == 0) {
      const int64_t at = (int64_t)head * p.n_rows + row;
      if (kind == 0) p.q_up[at] = fminf(exp2f((float)e0) * p.c, 3.402823466e38f);  // at f32's end any score but 0 takes all or nothing
      else if (kind == 1) p.kv_up[at].x = exp2f((float)e0);
      else p.kv_up[at].y = (float)e0;
    }
  }
  int2* mark = &p.marked[(int64_t)head * p.n_rows + b.first + b.row];
  if (kind == 1 && threadIdx.x == 0) mark->y = max(most, -112);
  if (kind == 2) {
    if (lane == 0) atomicMin(&least_s, least);
    const int any = __syncthreads_or(odd);
    if (threadIdx.x == 0) mark->x = (any ? 1 : 0) | (128 + max(most, -80)) << 8 | (128 + least_s) << 16;
  }
}

constexpr int kPfaThreads = 512;
// registers of a softmax thread, of one that holds a row of O, of the others: 128 x (2 x 120 + 192 + 80) of the launch's 512 x 128
// (heads of 128: 8 bytes of a thread on its stack). Nothing is called that is not inlined: a function of its own would know nothing
// of these splits
constexpr int kPfaSoftmaxRegs = 120, kPfaSumRegs = 192, kPfaOtherRegs = 80;
constexpr int kPfaAhead = 4;  // key tiles that the softmax may be ahead of the sums (two, for the tensor memory), and their own

constexpr int kPfaRing = 4;  // units of K, and of V

struct PromptF32Ctl {
  float2 stats[kPfaAhead][kPaTile];    // of a row: the maximum of s + f, the sum of w 2^-f
  float4 up[2][kPaTile / 2];           // of two keys: 2^ek, 2^ek, f, f
  float2 down[2][kPaTile / 2];         // 2^-f, 2^-f
  uint64_t q_full, q_empty, s_full[2], p_full[2], pv_full, pv_empty, up_full[2], up_empty[2];
  ItemRing items;
  uint64_t k_full[kPfaRing], k_empty[kPfaRing], v_full[kPfaRing], v_empty[kPfaRing];
  uint32_t tmem_base;
  int abort_flag;
  int busy[4];  // a warp that holds rows of O is computing some again: the others' waits may take longer
};

template <int kHd>
struct PromptF32Cfg {
  static constexpr int kTileBytes = kPaTile * kHd * 2;  // one part of a tile
  static constexpr int kUnitBytes = kPaTile * 128;      // of K: 64 columns of a part; of V: kUnitKeys rows of a part
  static constexpr int kUnits = kTileBytes / kUnitBytes, kUnitKeys = kPaTile / kUnits;
  static constexpr int kSmem = 1024 + 2 * kTileBytes + 2 * kPfaRing * kUnitBytes + 4 * kStageBytes + (int)sizeof(PromptF32Ctl) + 16;
};

// Whether the values that row `row0 + lane` of a sequence of `len` rows sees lie more than 2^100 apart; up: of its first row
__device__ __forceinline__ bool sees_far_apart(const float2* up, int row0, int len, int lane) {
  float above = -INFINITY, below = INFINITY;
  for (int key = lane; key < row0; key += 32) above = fmaxf(above, up[key].y), below = fminf(below, up[key].y);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    above = fmaxf(above, __shfl_xor_sync(0xffffffffu, above, off));
    below = fminf(below, __shfl_xor_sync(0xffffffffu, below, off));
  }
  if (row0 + lane < len) above = fmaxf(above, up[row0 + lane].y), below = fminf(below, up[row0 + lane].y);
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const float a = __shfl_up_sync(0xffffffffu, above, off), b = __shfl_up_sync(0xffffffffu, below, off);
    if (lane >= off) above = fmaxf(above, a), below = fminf(below, b);
  }
  return above - below > 100.f;
}

// Rows of a warp (the bits of `which`) once more, by the definition with sums in 64 bits: four keys at a time, the lanes over the columns.
// Values that are not finite are left to add_not_finite. q: the first parts of the warp's first row, the second ones `parts` behind them
// (the queries themselves may lie under the result); k, v: of the sequence's first; row: the first's number; up: c 2^eq of the
// lane's row
template <int kHd>
__device__ __forceinline__ void weigh_again(const __half* q, int64_t q_stride, int64_t parts, float up, const float* k, int64_t k_stride,
                                         const float* v, int64_t v_stride, int row, uint32_t which, float* dst, int64_t dst_stride,
                                         int lane) {
  constexpr int kMine = kHd / 32, kKeys = 4;
  for (; which; which &= which - 1) {
    const int r = __ffs(which) - 1;
    double x[kMine], o[kMine] = {}, top = -(double)INFINITY, sum = 0.0;
    const double times = (double)__shfl_sync(0xffffffffu, up, r);
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
      const __half* at = q + r * q_stride + lane + 32 * e;
      x[e] = (double)(__half2float(at[0]) + __half2float(at[parts])) * times;
    }
    for (int64_t key = 0; key <= row + r; key += kKeys) {
      double s[kKeys], most = top;
      float y[kKeys][kMine];
#pragma unroll
      for (int i = 0; i < kKeys; ++i) {
        const int64_t at = min(key + i, (int64_t)(row + r));
        s[i] = 0.0;
#pragma unroll
        for (int e = 0; e < kMine; ++e) {
          s[i] = fma(x[e], (double)k[at * k_stride + lane + 32 * e], s[i]);
          y[i][e] = v[at * v_stride + lane + 32 * e];
        }
      }
#pragma unroll
      for (int i = 0; i < kKeys; ++i) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], off);
        if (key + i > row + r) s[i] = -(double)INFINITY;
        most = fmax(most, s[i]);
      }
      if (most > top) {
        const double keep = exp2f((float)(top - most));
        sum *= keep;
#pragma unroll
        for (int e = 0; e < kMine; ++e) o[e] *= keep;
        top = most;
      }
#pragma unroll
      for (int i = 0; i < kKeys; ++i) {
        const double w = s[i] == -(double)INFINITY ? 0.0 : exp2f((float)(s[i] - top));  // +inf and NaN: NaN
        sum += w;
#pragma unroll
        for (int e = 0; e < kMine; ++e) o[e] = fma(w, isfinite(y[i][e]) ? (double)y[i][e] : 0.0, o[e]);
      }
    }
    const double inv = sum == 0.0 ? 0.0 : 1.0 / sum;
#pragma unroll
    for (int e = 0; e < kMine; ++e) dst[r * dst_stride + lane + 32 * e] = (float)(o[e] * inv);
  }
}

// The rows of a warp whose key tiles hold values that are not finite: adds those that each row sees, the lanes' columns side by side: the
// first key with +inf, -inf, NaN of every column, looked for once for all rows. (A lane by itself for its row, column after column,
// takes seconds where a long prompt's values are infinite throughout, and the block's other warps wait two.) v: the head's values of the
// sequence's first row; marked: the marks of its tiles; row: the warp's first; dst: its result
template <int kHd>
__device__ __forceinline__ void add_not_finite(const float* v, int64_t v_stride, const int2* marked, int row, int rows, float* dst,
                                            int64_t dst_stride, int lane) {
  constexpr int kMine = kHd / 32, kNone = 0x7fffffff;
  int first[3][kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) first[0][i] = first[1][i] = first[2][i] = kNone;
  const int end = row + rows;
  for (int64_t from = 0; from < end; from += 32 * kPaTile) {
    const int64_t mine = from + lane * kPaTile;
    uint32_t tiles = __ballot_sync(0xffffffffu, mine < end && (marked[mine].x & 1));
    for (; tiles; tiles &= tiles - 1) {
      const int key0 = (int)from + (__ffs(tiles) - 1) * kPaTile;
#pragma unroll 8
      for (int n = 0; n < kPaTile; ++n)
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const int key = min(key0 + n, end - 1);
          const float f = v[key * v_stride + lane + 32 * i];
          first[0][i] = f == INFINITY ? min(first[0][i], key) : first[0][i];
          first[1][i] = f == -INFINITY ? min(first[1][i], key) : first[1][i];
          first[2][i] = f != f ? min(first[2][i], key) : first[2][i];
        }
    }
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    if (min(first[0][i], min(first[1][i], first[2][i])) >= end) continue;
#pragma unroll 4
    for (int r = 0; r < rows; ++r) {
      float sum = dst[r * dst_stride + lane + 32 * i];
      if (first[0][i] <= row + r) sum += INFINITY;
      if (first[1][i] <= row + r) sum -= INFINITY;
      if (first[2][i] <= row + r) sum += __int_as_float(0x7fc00000);
      dst[r * dst_stride + lane + 32 * i] = sum;
    }
  }
}

template <int kHd>
__global__ void __launch_bounds__(kPfaThreads, 1) prompt_attn_f32_kernel(const PromptF32Params p, const __grid_constant__ CUtensorMap qmap,
                                                                         const __grid_constant__ CUtensorMap kmap,
                                                                         const __grid_constant__ CUtensorMap vmap) {
  using Cfg = PromptF32Cfg<kHd>;
  constexpr int kTileBytes = Cfg::kTileBytes, kUnitBytes = Cfg::kUnitBytes, kUnits = Cfg::kUnits, kUnitKeys = Cfg::kUnitKeys;
  extern __shared__ __align__(1024) uint8_t pfa_smem[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pfa_smem) + 1023) & ~(uintptr_t)1023);
  uint8_t* v_ring = base + 2 * kTileBytes + kPfaRing * kUnitBytes;
  const uint32_t q_addr = smem_u32(base), k_addr = q_addr + 2 * kTileBytes, v_addr = smem_u32(v_ring);
  uint8_t* stages = v_ring + kPfaRing * kUnitBytes;  // of the rows on their way out, a warp each
  auto* ctl = reinterpret_cast<PromptF32Ctl*>(stages + 4 * kStageBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&ctl->q_full, 1), mbar_init(&ctl->q_empty, 1), mbar_init(&ctl->pv_full, 1), mbar_init(&ctl->pv_empty, 128);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->s_full[i], 1), mbar_init(&ctl->p_full[i], 128);
      mbar_init(&ctl->up_full[i], 1), mbar_init(&ctl->up_empty[i], 128);
    }
    for (int s = 0; s < kItemRing; ++s) mbar_init(&ctl->items.full[s], 1), mbar_init(&ctl->items.empty[s], 16);  // every warp
    for (int s = 0; s < kPfaRing; ++s) {
      mbar_init(&ctl->k_full[s], 1), mbar_init(&ctl->k_empty[s], 1);
      mbar_init(&ctl->v_full[s], 1), mbar_init(&ctl->v_empty[s], 1);
    }
    ctl->abort_flag = 0;
    for (int i = 0; i < 4; ++i) ctl->busy[i] = 0;
    mbar_init_fence();
  }
  if (warp == 13) tmem_alloc(&ctl->tmem_base, 512);  // two S (the weights' upper parts over each), their lower parts, O of a tile
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&ctl->tmem_base);
  volatile int* abort_flag = &ctl->abort_flag;
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (mbar_poll_bounded(bar, parity & 1u)) return true;
    const volatile int* busy = ctl->busy;
    for (int more = 0; more < 1000 && !*abort_flag && (busy[0] | busy[1] | busy[2] | busy[3]); ++more)
      if (mbar_poll_bounded(bar, parity & 1u)) return true;
    if (!*abort_flag) record_dev_error(code);
    *abort_flag = 1;
    return false;
  };
  const uint32_t p_low = tmem + 256, pv_acc = tmem + 384;

  if (warp >= 12) set_regs_down<kPfaOtherRegs>();
  if (warp == 12 || warp == 15) {
    // ---------------- copies: Q and K, V. Units of a tile: lower part, upper part
    if (lane == 0) {
      const bool values = warp == 15;
      uint64_t* full = values ? ctl->v_full : ctl->k_full;
      uint64_t* empty = values ? ctl->v_empty : ctl->k_empty;
      uint32_t unit = 0, items = 0;
      bool ok = true;
      PromptItem it;
      for (; ok && !*abort_flag && get_item<false>(ctl->items, items, it, wait); ++items) {
        const int kvh = it.head / p.group;
        if (!values) {
          if (items && !(ok = wait(&ctl->q_empty, items - 1, kErrEmptyWait))) break;
          mbar_arrive_expect_tx(&ctl->q_full, 2 * kTileBytes);
          for (int part = 0; part < 2; ++part)
            for (int b = 0; b < kUnits; ++b)
              tma_load_3d(q_addr + part * kTileBytes + b * kUnitBytes, &qmap, 64 * b, it.head, (int)(part * p.n_rows + it.first + it.row),
                          &ctl->q_full);
        }
        for (int j = 0; j < it.n && ok && !*abort_flag; ++j)
          for (int u = 0; u < 2 * kUnits && ok; ++u, ++unit) {
            const uint32_t s = unit % kPfaRing;
            if (unit >= kPfaRing && !(ok = wait(&empty[s], unit / kPfaRing - 1, kErrEmptyWait))) break;
            mbar_arrive_expect_tx(&full[s], kUnitBytes);
            const int row = (int)((1 - u / kUnits) * p.n_rows + it.first + j * kPaTile), piece = u % kUnits;
            if (!values) {
              tma_load_3d(k_addr + s * kUnitBytes, &kmap, 64 * piece, kvh, row, &full[s]);
            } else {
              for (int b = 0; b < kHd / 64; ++b)
                tma_load_3d(v_addr + s * kUnitBytes + b * kUnitKeys * 128, &vmap, 64 * b, kvh, row + piece * kUnitKeys, &full[s]);
            }
          }
      }
      pdl_launch_dependents();
      if (*abort_flag) {  // leaving early: let the copies already requested land first
        for (uint32_t u = unit > kPfaRing ? unit - kPfaRing : 0; u < unit; ++u)
          if (!mbar_wait_bounded(&full[u % kPfaRing], (u / kPfaRing) & 1)) record_dev_error(kErrDrainWait);
        if (!values && items && !mbar_wait_bounded(&ctl->q_full, (items - 1) & 1)) record_dev_error(kErrDrainWait);
      }
    }
  } else if (warp == 13) {
    // ---------------- MMA issue
    constexpr uint32_t s_desc = umma_idesc_f16(kPaTile, kPaTile), o_desc = umma_idesc_f16(kPaTile, kHd) | kIdescBColumns;
    const uint32_t acc = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t q_desc = umma_desc_sw128(q_addr), k_desc = umma_desc_sw128(k_addr), v_desc = umma_desc_sw128_mn(v_addr, kUnitKeys * 128);
    const bool leader = elect_one();
    auto ready = [&](uint64_t* bar, uint32_t parity, int code) { return (bool)__all_sync(0xffffffffu, wait(bar, parity, code)); };
    uint32_t items = 0, steps = 0;
    bool ok = true;
    PromptItem it;
    for (; ok && get_item<true>(ctl->items, items, it, wait); ++items) {
      // S of key tile j into its half of tensor memory. The small products come first, hi lo of each unit of the lower part, lo hi of
      // the upper part's, then hi hi: sums that round towards zero do so eight times at their full size, not 24
      auto scores = [&](int j) {
        const uint32_t d = acc + ((steps + j) & 1) * kPaTile;
#pragma unroll
        for (int u = 0; u < 3 * kUnits; ++u) {
          const int piece = u % kUnits;
          const uint32_t n = (steps + j) * 2 * kUnits + (u < 2 * kUnits ? u : u - kUnits), st = n % kPfaRing;
          if (u < 2 * kUnits && !ready(&ctl->k_full[st], n / kPfaRing, kErrFullWait)) return false;
          const uint64_t a = q_desc + (uint64_t)(((u / kUnits == 1 ? kTileBytes : 0) + piece * kUnitBytes) >> 4);
          const uint64_t b = k_desc + (uint64_t)(st * kUnitBytes >> 4);
          if (leader) {
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_bf16(d, a + 2 * k, b + 2 * k, s_desc, (u | k) != 0);
            if (u / kUnits != 1) umma_commit(&ctl->k_empty[st]);
          }
        }
        if (leader) {
          if (j + 1 == it.n) umma_commit(&ctl->q_empty);
          umma_commit(&ctl->s_full[(steps + j) & 1]);
        }
        return true;
      };
      if (!(ok = ready(&ctl->q_full, items, kErrFullWait))) break;
      ok = scores(0);
      for (int j = 0; j < it.n && ok; ++j) {
        if (j + 1 < it.n && !(ok = scores(j + 1))) break;
        const uint32_t step = steps + j, hi = acc + (step & 1) * kPaTile, lo = acc + 256 + (step & 1) * 64, d = acc + 384;
        if (!(ok = ready(&ctl->p_full[step & 1], step / 2, kErrMmaWait))) break;
        if (step && !(ok = ready(&ctl->pv_empty, step - 1, kErrTmemWait))) break;
#pragma unroll
        for (int u = 0; u < 3 * kUnits; ++u) {  // in the same order
          const int piece = u % kUnits;
          const uint32_t n = step * 2 * kUnits + (u < 2 * kUnits ? u : u - kUnits), st = n % kPfaRing;
          if (ok && u < 2 * kUnits) ok = ready(&ctl->v_full[st], n / kPfaRing, kErrFullWait);
          const uint32_t a = (u / kUnits == 1 ? lo : hi) + piece * (kUnitKeys / 2);
          const uint64_t b = v_desc + (uint64_t)(st * kUnitBytes >> 4);
          if (ok && leader) {
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < kUnitKeys / 16; ++k) umma_f16_ts(d, a + k * 8, b + (uint64_t)(k * 2048 >> 4), o_desc, (u | k) != 0);
            if (u / kUnits != 1) umma_commit(&ctl->v_empty[st]);
          }
        }
        if (ok && leader) umma_commit(&ctl->pv_full);
      }
      steps += it.n;
    }
  } else if (warp == 14) {
    // ---------------- the items, one ahead, and the powers of each key tile
    uint32_t steps = 0, items = 0;
    int64_t x = blockIdx.x;
    auto next = [&]() { return find_item(p.cu, p.n_seqs, p.n_rows, p.n_heads, p.n_items, kPaTile, x, lane); };
    PromptItem ahead = next(), it;
    bool ok = put_item(ctl->items, 0, ahead, lane, wait);
    for (; ok && get_item<true>(ctl->items, items, it, wait); ++items) {
      ahead = next();
      if (!(ok = put_item(ctl->items, items + 1, ahead, lane, wait))) break;
      const float2* src = p.kv_up + (int64_t)(it.head / p.group) * p.n_rows + it.first;
      for (int j = 0; j < it.n && ok; ++j, ++steps) {
        if (steps >= 2 && !(ok = __all_sync(0xffffffffu, wait(&ctl->up_empty[steps & 1], steps / 2 - 1, kErrEmptyWait)))) break;
        float* up = reinterpret_cast<float*>(ctl->up[steps & 1]);
        float* down = reinterpret_cast<float*>(ctl->down[steps & 1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = i * 32 + lane, key = j * kPaTile + at;
          const float2 u = key < it.len ? src[key] : make_float2(0.f, 0.f);
          up[at / 2 * 4 + (at & 1)] = u.x, up[at / 2 * 4 + 2 + (at & 1)] = u.y;
          down[at] = exp2f(-u.y);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->up_full[steps & 1]);
      }
    }
  } else if (warp < 8) {
    // ---------------- softmax: a thread per row of every other key tile
    set_regs_down<kPfaSoftmaxRegs>();
    const uint32_t half = warp >> 2;
    const int r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + half * kPaTile, lo_addr = p_low + lanes + half * 64;
    const uint32_t up = smem_u32(ctl->up[half]), down = smem_u32(ctl->down[half]);
    uint32_t steps = 0;
    bool ok = true;
    PromptItem it;
    for (uint32_t items = 0; ok && get_item<true>(ctl->items, items, it, wait); ++items) {
      const int row = it.row + r;
      const float cq = row < it.len ? p.q_up[(int64_t)it.head * p.n_rows + it.first + row] : 0.f;
      const uint64_t cq2 = pair(cq, cq);
      for (int j = (steps ^ half) & 1; j < it.n; j += 2) {
        const uint32_t step = steps + j;
        ok = wait(&ctl->up_full[half], step / 2, kErrFullWait) && wait(&ctl->s_full[half], step / 2, kErrMmaWait);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
        const bool last = j + 1 == it.n;
        // the maximum, and again from tensor memory the weights, in short loops with the next columns on their way (code that is run
        // through once per key tile comes at some four cycles an instruction)
        float top[2] = {-INFINITY, -INFINITY};
        auto look = [&](auto masked) {
          uint32_t s[2][16];
          tmem_ld16_nowait(s_addr, s[0]);
#pragma unroll 1
          for (int c0 = 0; c0 < 8; c0 += 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = c0 + h;
              tmem_wait_ld16(s[h]);
              if (c < 7) tmem_ld16_nowait(s_addr + 16 * (c + 1), s[h ^ 1]);
              const int seen = r - 16 * c;  // the last of the sixteen keys that this row sees
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                const float4 w = lds_f4(up + (8 * c + i / 2) * 16);
                float a, b;
                unpair(fma2(pair(__uint_as_float(s[h][i]), __uint_as_float(s[h][i + 1])), mul2(pair(w.x, w.y), cq2), pair(w.z, w.w)), a, b);
                if (decltype(masked)::value && i > seen) a = -INFINITY;
                if (decltype(masked)::value && i + 1 > seen) b = -INFINITY;
                top[i / 2 & 1] = max3(top[i / 2 & 1], a, b);
              }
            }
          }
        };
        if (last) look(std::true_type());
        else look(std::false_type());
        const float ref = fmaxf(top[0], top[1]), rr = 14.f - (ref == -INFINITY ? 0.f : ref);  // weights up to 2^14
        const uint64_t rr2 = pair(rr, rr);
        uint64_t sum2 = pair(0.f, 0.f);
        auto weigh = [&](auto masked) {
          uint32_t s[2][8];
          tmem_ld8_nowait(s_addr, s[0]);
#pragma unroll 1
          for (int c0 = 0; c0 < 16; c0 += 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = c0 + h;
              tmem_wait_ld8(s[h]);
              if (c < 15) tmem_ld8_nowait(s_addr + 8 * (c + 1), s[h ^ 1]);
              const int seen = r - 8 * c;
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int i = 0; i < 8; i += 2) {
                const float4 w = lds_f4(up + (4 * c + i / 2) * 16);
                float a, b;
                const uint64_t s2 = pair(__uint_as_float(s[h][i]), __uint_as_float(s[h][i + 1]));
                unpair(fma2(s2, mul2(pair(w.x, w.y), cq2), add2(pair(w.z, w.w), rr2)), a, b);
                if (decltype(masked)::value && i > seen) a = -INFINITY;
                if (decltype(masked)::value && i + 1 > seen) b = -INFINITY;
                a = exp2_approx(a), b = exp2_approx(b);
                sum2 = fma2(pair(a, b), lds_pair(down + (4 * c + i / 2) * 8), sum2);
                hi[i / 2] = cvt2<__half>(a, b);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[i / 2]));
                lo[i / 2] = cvt2<__half>(a - f.x, b - f.y);
              }
              // over columns of S that have been read: in front of the ones in flight
              tmem_st4(s_addr + 4 * c, hi);
              tmem_st4(lo_addr + 4 * c, lo);
            }
          }
        };
        if (last) weigh(std::true_type());
        else weigh(std::false_type());
        float a, b;
        unpair(sum2, a, b);
        ctl->stats[step % kPfaAhead][r] = make_float2(ref, a + b);
        mbar_arrive(&ctl->up_empty[half]);
        if (last && it.row + kPaTile > it.len) {
          // the tile goes on behind the sequence: whatever stands there, 0 times it has to be 0. The products of the tile
          // before are waited for first: then that tile's values had landed, and the parity below can only mean this one's
          if (j && !(ok = __all_sync(0xffffffffu, wait(&ctl->pv_full, step - 1, kErrMmaWait)))) break;
          const int from = it.len - it.row;  // rows of the sequence in the tile
#pragma unroll 1
          for (int u = 0; u < 2 * kUnits && ok; ++u) {
            const uint32_t n = step * 2 * kUnits + u, st = n % kPfaRing;
            if (!(ok = __all_sync(0xffffffffu, wait(&ctl->v_full[st], n / kPfaRing, kErrFullWait)))) break;
            uint8_t* v = v_ring + st * kUnitBytes;
            for (int i = max(from - (u % kUnits) * kUnitKeys, 0) * 8 + r; i < kUnitKeys * 8; i += 128)
              for (int box = 0; box < kHd / 64; ++box)
                *reinterpret_cast<uint4*>(v + box * kUnitKeys * 128 + i * 16) = make_uint4(0, 0, 0, 0);
          }
          if (!ok) break;
          fence_proxy_async();
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ctl->p_full[half]);
      }
      steps += it.n;
    }
  } else if (warp < 12) {
    // ---------------- O: a thread per row
    set_regs_up<kPfaSumRegs>();
    const int r = threadIdx.x & 127;
    const uint32_t addr = pv_acc + ((uint32_t)((warp & 3) * 32) << 16);
    uint32_t steps = 0;
    bool ok = true;
    PromptItem it;
    for (uint32_t items = 0; ok && get_item<true>(ctl->items, items, it, wait); ++items) {
      const int row = it.row + r, row0 = row - lane;  // row0: of the warp
      const int64_t rows_at = (int64_t)(it.head / p.group) * p.n_rows + it.first;
      // the marks of its key tiles, read while the first of them is computed
      bool odd = false;
      int up = -1000, above = 0, below = 255;
      for (int j = lane; j < it.n; j += 32) {
        const int2 mark = p.marked[rows_at + (int64_t)j * kPaTile];
        odd |= mark.x & 1, up = max(up, mark.y);
        above = max(above, mark.x >> 8 & 255), below = min(below, mark.x >> 16);
      }
      const float q_up = row < it.len ? p.q_up[(int64_t)it.head * p.n_rows + it.first + row] : 0.f;
      odd = __any_sync(0xffffffffu, odd);
      const float reach = q_up * exp2f((float)__reduce_max_sync(0xffffffffu, up));
      const bool apart = __reduce_max_sync(0xffffffffu, above) - __reduce_min_sync(0xffffffffu, below) > 100;
      float o[kHd], ref = -INFINITY, sum = 0.f;
#pragma unroll
      for (int e = 0; e < kHd; ++e) o[e] = 0.f;
      for (int j = 0; j < it.n; ++j, ++steps) {
        if (!(ok = __all_sync(0xffffffffu, wait(&ctl->pv_full, steps, kErrMmaWait)))) break;
        tc_fence_after();
        const float2 st = ctl->stats[steps % kPfaAhead][r];
        const float to = fmaxf(ref, st.x), keep = ref == to ? 1.f : exp2f(ref - to), take = st.x == to ? 1.f : exp2f(st.x - to);
        ref = to;
        sum = sum * keep + st.y * take;
#pragma unroll
        for (int i = 0; i < kHd / 16; ++i) {
          uint32_t v[16];
          tmem_ld16(addr + 16 * i, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[16 * i + e] = fmaf(o[16 * i + e], keep, __uint_as_float(v[e]) * take);
        }
        tc_fence_before();
        mbar_arrive(&ctl->pv_empty);
      }
      if (!ok) break;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      // rows to be computed again: their maximum is beyond 2^22 or has left f32, where the powers of their factors allow it (a product of
      // two parts is below 2^37; otherwise an infinity in q or k has made it); the powers' product may leave f32 where the score
      // itself is of any size; the values lie too far apart
      bool far = (reach > 0x1p-15f && !(fabsf(ref) <= 0x1p22f)) || !(reach <= 0x1p120f);
      if (apart) far |= sees_far_apart(p.kv_up + rows_at, row0, it.len, lane);
      const uint32_t again = __ballot_sync(0xffffffffu, far && row < it.len);
      float* dst = p.out + ((it.first + row0) * p.n_heads + it.head) * kHd;
#pragma unroll
      for (int i = 0; i < kHd / 16; ++i) {
        uint4 v[4];
        float* w = reinterpret_cast<float*>(v);
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = o[16 * i + e] * inv;
        store_rows64(smem_u32(stages) + (warp & 3) * kStageBytes, lane, v, reinterpret_cast<uint8_t*>(dst + 16 * i),
                     (int64_t)p.n_heads * kHd * 4, it.len - row0);
      }
      if (again) {
        ctl->busy[warp & 3] = 1;
        __syncwarp();  // the rows are written
        const int kvh = it.head / p.group;
        weigh_again<kHd>(p.qp + ((it.first + row0) * p.n_heads + it.head) * kHd, (int64_t)p.n_heads * kHd, p.n_rows * p.n_heads * kHd, q_up,
                         p.k + it.first * p.k_stride + kvh * kHd, p.k_stride, p.v + it.first * p.v_stride + kvh * kHd, p.v_stride, row0,
                         again, dst, (int64_t)p.n_heads * kHd, lane);
        __syncwarp();
        ctl->busy[warp & 3] = 0;
      }
      if (odd && row0 < it.len) {
        ctl->busy[warp & 3] = 1;
        __syncwarp();  // the rows are written
        add_not_finite<kHd>(p.v + it.first * p.v_stride + (it.head / p.group) * kHd, p.v_stride, p.marked + rows_at, row0,
                            min(32, it.len - row0), dst, (int64_t)p.n_heads * kHd, lane);
        __syncwarp();
        ctl->busy[warp & 3] = 0;
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 13) tmem_dealloc(tmem, 512);
}

}  // namespace fq
