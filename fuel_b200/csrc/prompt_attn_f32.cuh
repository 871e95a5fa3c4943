// Causal attention inside packed prompts (fuelq_prompt_attn) for 32-bit activations, to 32-bit accuracy on the f16 tensor cores.
//
// Every factor is a power of two times two f16 parts, x = 2^e (hi + lo), 22 bits, and a product is three of theirs, summed in
// f32: hi hi + lo hi + hi lo (lo lo is below 2^-22). f16 at three products is twice as fast as bf16 at the six that it would
// take for as many bits, or tf32 at its half rate; what f16 lacks in range the powers of two give:
//   q, k   one for each row and head: S = (Q' K'^T)_ij 2^(eq_i + ek_j)
//   v      one for each row and head, put into the weight: with f_j the row's power, w_ij = 2^(s_ij + f_j - m'_i), m' the running
//          maximum of s + f, so that w V' has f16's range whatever the rows' magnitudes; the sum of the softmax keeps p_ij =
//          2^(s_ij - m_i) and its own running maximum, and out = (O / l) 2^(m' - m)
// so no row loses bits to a larger one, in front of it or behind it. prompt_split_kernel writes the parts and powers (bound by
// HBM: 4 bytes in, 4 out); values that are not finite are taken out of v there, and the tiles that had some are marked: the few
// rows that see one add it again from the original at the end.
// The tensor cores' f32 sums round towards zero, which over a long row adds up (1.6e-5 of it at 4000 keys). So they sum one
// key tile at a time, and the tiles' results are added in registers, rounded to nearest.
// Bound by the tensor cores: three times the 16-bit kernel's products. One tile of 128 query rows per thread block; S of the next
// key tile is in tensor memory before the weights of this one are needed, so the softmax (two exponentials a score) and the
// sums run beside the products.
//   warps 0-3  softmax: a thread per row        warps 4-7  O: a thread per row adds the tiles' products, finishes and stores it
//   warp 8     copies: the parts of Q, K and V, 32 KB each, through one ring
//   warp 9     issues the MMAs                  warp 10    brings the powers of each key tile
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
  int* marked;           // [n_kv][n_rows]     at the first row of a tile: does it hold a value that is not finite?
};

template <int kHd>
__global__ void __launch_bounds__(256) prompt_split_kernel(const PromptF32Params p) {
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
  bool odd = false;
#pragma unroll 4
  for (int i = warp; i < rows; i += 8) {
    const int64_t row = b.first + b.row + i;
    alignas(16) float x[kPer];
    const float* in = src + row * stride + head * kHd + lane * kPer;
    if constexpr (kPer == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(in);
    else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(in);
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const bool fin = isfinite(x[e]);
      if (fin) top = fmaxf(top, fabsf(x[e]));
      if (kind == 2 && !fin) odd = true, x[e] = 0.f;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    // the largest value comes to [2^14, 2^15); rows of nothing but denormals keep their lower bits out of f16's reach
    const int e0 = top > 0.f ? max(ilogbf(top) - 14, -112) : 0;
    const float down = exp2f((float)-e0);
    alignas(8) __half hi[kPer], lo[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float y = x[e] * down;
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
      if (kind == 0) p.q_up[at] = exp2f((float)e0) * p.c;
      else if (kind == 1) p.kv_up[at].x = exp2f((float)e0);
      else p.kv_up[at].y = top > 0.f ? (float)e0 : -1e30f;  // a row of zeros weighs nothing in O
    }
  }
  if (kind == 2) {
    const int any = __syncthreads_or(odd);
    if (threadIdx.x == 0) p.marked[(int64_t)head * p.n_rows + b.first + b.row] = any;
  }
}

constexpr int kPfaThreads = 384;
// registers: 128 threads of each, 128 x (240 + 176 + 88) of the launch's 384 x 168
constexpr int kPfaSoftmaxRegs = 240, kPfaSumRegs = 176, kPfaOtherRegs = 88;
constexpr int kPfaAhead = 4;  // steps and items that the softmax may be ahead of the sums (two, for the tensor memory; and their own)

template <int kStages>
struct PromptF32Ctl {
  uint64_t q_full, q_empty, s_full[2], p_full, pv_full[2], pv_empty[2], up_full[2], up_empty[2];
  uint64_t kv_full[kStages], kv_empty[kStages];
  float keep[kPfaAhead][kPaTile];    // by step: what the row's reference has moved by
  float2 finish[kPfaAhead][kPaTile]; // by item: what the row's O is multiplied by at the end
  uint32_t tmem_base;
  int abort_flag;
};

template <int kHd>
struct PromptF32Cfg {
  static constexpr int kStages = kHd == 128 ? 4 : 8;
  static constexpr int kTileBytes = kPaTile * kHd * 2;  // one part of a tile
  static constexpr int kUpBytes = 2 * kPaTile * 8;
  static constexpr int kSmem = 1024 + (2 + kStages) * kTileBytes + kUpBytes + (int)sizeof(PromptF32Ctl<kStages>) + 16;
};

// A row of the result whose key tiles hold values that are not finite: adds those that the row sees
template <int kHd>
__device__ __noinline__ void add_not_finite(const PromptF32Params& p, int64_t first, int row, int head, float* dst) {
  const int kvh = head / p.group;
  const int* marked = p.marked + (int64_t)kvh * p.n_rows + first;
  for (int d = 0; d < kHd; ++d) {
    float sum = dst[d];
    for (int tile = 0; tile <= row && !isnan(sum); tile += kPaTile) {
      if (!marked[tile]) continue;
      for (int key = tile; key < tile + kPaTile && key <= row; ++key) {
        const float f = p.v[(first + key) * p.v_stride + kvh * kHd + d];
        if (!isfinite(f)) sum += f;
      }
    }
    dst[d] = sum;
  }
}

template <int kHd>
__global__ void __launch_bounds__(kPfaThreads, 1) prompt_attn_f32_kernel(const PromptF32Params p, const __grid_constant__ CUtensorMap qmap,
                                                                         const __grid_constant__ CUtensorMap kmap,
                                                                         const __grid_constant__ CUtensorMap vmap) {
  using Cfg = PromptF32Cfg<kHd>;
  constexpr int kStages = Cfg::kStages, kTileBytes = Cfg::kTileBytes, kBoxes = kHd / 64, kBoxBytes = kPaTile * 128;
  extern __shared__ __align__(1024) uint8_t pfa_smem[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pfa_smem) + 1023) & ~(uintptr_t)1023);
  const uint32_t q_addr = smem_u32(base), kv_addr = q_addr + 2 * kTileBytes;
  float4* up_s = reinterpret_cast<float4*>(base + (2 + kStages) * kTileBytes);  // [2][64] pairs of keys: 2^ek, f of each
  auto* ctl = reinterpret_cast<PromptF32Ctl<kStages>*>(base + (2 + kStages) * kTileBytes + Cfg::kUpBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&ctl->q_full, 1), mbar_init(&ctl->q_empty, 1), mbar_init(&ctl->p_full, 128);
    for (int i = 0; i < 2; ++i) mbar_init(&ctl->pv_full[i], 1), mbar_init(&ctl->pv_empty[i], 128);
    for (int i = 0; i < 2; ++i) mbar_init(&ctl->s_full[i], 1), mbar_init(&ctl->up_full[i], 1), mbar_init(&ctl->up_empty[i], 128);
    for (int s = 0; s < kStages; ++s) mbar_init(&ctl->kv_full[s], 1), mbar_init(&ctl->kv_empty[s], 1);
    ctl->abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 9) tmem_alloc(&ctl->tmem_base, 512);  // two S (the weights' two parts over each), two products
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&ctl->tmem_base);
  volatile int* abort_flag = &ctl->abort_flag;
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (mbar_poll_bounded(bar, parity & 1u)) return true;
    if (!*abort_flag) record_dev_error(code);
    *abort_flag = 1;
    return false;
  };
  struct Item {
    int64_t first;
    int len, row, head, n;
  };
  auto item = [&](int64_t x, Item& it) {
    const int64_t slot = x / p.n_heads;
    const PromptBlock b = prompt_block(p.cu, p.n_seqs, p.n_rows, slot, kPaTile);
    if (b.row >= b.len) return false;
    it.first = b.first, it.len = b.len, it.row = b.row, it.head = (int)(x - slot * p.n_heads), it.n = b.row / kPaTile + 1;
    return true;
  };

  if (warp >= 8) set_regs_down<kPfaOtherRegs>();
  if (warp == 8) {
    // ---------------- copies
    if (lane == 0) {
      uint32_t unit = 0, items = 0;  // a unit: one part of a key or value tile
      bool ok = true;
      for (int64_t x = blockIdx.x; x < p.n_items && ok && !*abort_flag; x += gridDim.x) {
        Item it;
        if (!item(x, it)) continue;
        const int kvh = it.head / p.group;
        if (items && !(ok = wait(&ctl->q_empty, items - 1, kErrEmptyWait))) break;
        mbar_arrive_expect_tx(&ctl->q_full, 2 * kTileBytes);
        for (int part = 0; part < 2; ++part)
          for (int b = 0; b < kBoxes; ++b)
            tma_load_3d(q_addr + part * kTileBytes + b * kBoxBytes, &qmap, 64 * b, it.head, (int)(part * p.n_rows + it.first + it.row), &ctl->q_full);
        ++items;
        for (int j = 0; j < it.n && ok && !*abort_flag; ++j)
          for (int u = 0; u < 4 && ok; ++u) {  // K hi, K lo, V hi, V lo
            const uint32_t s = unit % kStages;
            if (unit >= kStages && !(ok = wait(&ctl->kv_empty[s], unit / kStages - 1, kErrEmptyWait))) break;
            mbar_arrive_expect_tx(&ctl->kv_full[s], kTileBytes);
            for (int b = 0; b < kBoxes; ++b)
              tma_load_3d(kv_addr + s * kTileBytes + b * kBoxBytes, u < 2 ? &kmap : &vmap, 64 * b, kvh,
                          (int)((u & 1) * p.n_rows + it.first + j * kPaTile), &ctl->kv_full[s]);
            ++unit;
          }
      }
      pdl_launch_dependents();
      if (*abort_flag) {  // leaving early: let the copies already requested land first
        for (uint32_t u = unit > kStages ? unit - kStages : 0; u < unit; ++u)
          if (!mbar_wait_bounded(&ctl->kv_full[u % kStages], (u / kStages) & 1)) record_dev_error(kErrDrainWait);
        if (items && !mbar_wait_bounded(&ctl->q_full, (items - 1) & 1)) record_dev_error(kErrDrainWait);
      }
    }
  } else if (warp == 9) {
    // ---------------- MMA issue: one thread
    if (lane == 0) {
      const uint32_t s_desc = umma_idesc_f16(kPaTile, kPaTile), o_desc = umma_idesc_f16(kPaTile, kHd) | kIdescBColumns;
      uint32_t unit = 0, items = 0, steps = 0;
      bool ok = true;
      for (int64_t x = blockIdx.x; x < p.n_items && ok && !*abort_flag; x += gridDim.x) {
        Item it;
        if (!item(x, it)) continue;
        auto ready = [&](uint32_t u) { return wait(&ctl->kv_full[u % kStages], u / kStages, kErrFullWait); };
        // S of key tile j into its half of tensor memory: hi hi, lo hi, hi lo
        auto scores = [&](int j) {
          const uint32_t u = unit + 4 * j, d = tmem + ((steps + j) & 1) * kPaTile;
          if (!ready(u)) return false;
          tc_fence_after();
#pragma unroll
          for (int part = 0; part < 3; ++part) {
            if (part == 2 && !ready(u + 1)) return false;
            if (part == 2) tc_fence_after();
            const uint32_t a = q_addr + (part == 1 ? kTileBytes : 0), b = kv_addr + ((u + (part == 2)) % kStages) * kTileBytes;
#pragma unroll
            for (int k = 0; k < kHd / 16; ++k) {
              const uint32_t off = (k / 4) * kBoxBytes + (k % 4) * 32;
              umma_bf16(d, umma_desc_sw128(a + off), umma_desc_sw128(b + off), s_desc, (part | k) != 0);
            }
            if (part) umma_commit(&ctl->kv_empty[(u + part - 1) % kStages]);
          }
          if (j + 1 == it.n) umma_commit(&ctl->q_empty);
          umma_commit(&ctl->s_full[(steps + j) & 1]);
          return true;
        };
        if (!(ok = wait(&ctl->q_full, items++, kErrFullWait))) break;
        ok = scores(0);
        for (int j = 0; j < it.n && ok; ++j) {
          if (j + 1 < it.n && !(ok = scores(j + 1))) break;
          const uint32_t step = steps + j, d = tmem + 256 + (step & 1) * 128;
          if (!(ok = wait(&ctl->p_full, step, kErrMmaWait))) break;
          if (step >= 2 && !(ok = wait(&ctl->pv_empty[step & 1], step / 2 - 1, kErrTmemWait))) break;
          const uint32_t u = unit + 4 * j + 2, w = tmem + ((steps + j) & 1) * kPaTile;
#pragma unroll
          for (int part = 0; part < 3; ++part) {
            if (part != 1 && !(ok = ready(u + part / 2))) break;
            tc_fence_after();
            const uint32_t b = kv_addr + ((u + part / 2) % kStages) * kTileBytes;
#pragma unroll
            for (int k = 0; k < kPaTile / 16; ++k)
              umma_f16_ts(d, w + (part == 1 ? 64 : 0) + k * 8, umma_desc_sw128_mn(b + k * 2048, kBoxBytes), o_desc, (part | k) != 0);
            if (part) umma_commit(&ctl->kv_empty[(u + part - 1) % kStages]);
          }
          if (ok) umma_commit(&ctl->pv_full[step & 1]);
        }
        unit += 4 * it.n, steps += it.n;
      }
    }
  } else if (warp == 10) {
    // ---------------- the powers of each key tile
    uint32_t steps = 0;
    bool ok = true;
    for (int64_t x = blockIdx.x; x < p.n_items && ok && !*abort_flag; x += gridDim.x) {
      Item it;
      if (!item(x, it)) continue;
      const float2* src = p.kv_up + (int64_t)(it.head / p.group) * p.n_rows + it.first;
      for (int j = 0; j < it.n && ok; ++j, ++steps) {
        if (steps >= 2 && !(ok = __all_sync(0xffffffffu, wait(&ctl->up_empty[steps & 1], steps / 2 - 1, kErrEmptyWait)))) break;
        float2* dst = reinterpret_cast<float2*>(up_s) + (steps & 1) * kPaTile;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = j * kPaTile + i * 32 + lane;
          dst[i * 32 + lane] = key < it.len ? src[key] : make_float2(0.f, 0.f);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->up_full[steps & 1]);
      }
    }
  } else if (warp < 4) {
    // ---------------- softmax: a thread per row
    set_regs_up<kPfaSoftmaxRegs>();
    const int r = threadIdx.x;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    uint32_t unit = 0, steps = 0, items = 0;
    bool ok = true;
    for (int64_t x = blockIdx.x; x < p.n_items && ok; x += gridDim.x) {
      Item it;
      if (!item(x, it)) continue;
      const int row = it.row + r;
      const float cq = row < it.len ? p.q_up[(int64_t)it.head * p.n_rows + it.first + row] : 0.f;
      float m = -INFINITY, ref = -INFINITY, sum = 0.f;  // running maxima of s and of s + f
      for (int j = 0; j < it.n; ++j, ++steps) {
        const uint32_t s_addr = tmem + lanes + (steps & 1) * kPaTile;
        const float4* up = up_s + (steps & 1) * (kPaTile / 2);
        ok = wait(&ctl->up_full[steps & 1], steps / 2, kErrFullWait) && wait(&ctl->s_full[steps & 1], steps / 2, kErrMmaWait);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
        uint32_t s[kPaTile];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32_nowait(s_addr + 32 * i, s + 32 * i);
        tmem_wait_ld();
        const bool last = j + 1 == it.n;
        float top[2] = {-INFINITY, -INFINITY}, topf[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kPaTile; i += 2) {
          const float4 u = up[i / 2];
          float a = __uint_as_float(s[i]) * u.x * cq, b = __uint_as_float(s[i + 1]) * u.z * cq;
          if (last && i > r) a = -INFINITY;
          if (last && i + 1 > r) b = -INFINITY;
          top[0] = fmaxf(top[0], a), top[1] = fmaxf(top[1], b);
          topf[0] = fmaxf(topf[0], a + u.y), topf[1] = fmaxf(topf[1], b + u.w);
          s[i] = __float_as_uint(a), s[i + 1] = __float_as_uint(b);
        }
        const float most = fmaxf(m, fmaxf(top[0], top[1])), mostf = fmaxf(ref, fmaxf(topf[0], topf[1]));
        if (most != m) {
          sum *= exp2f(m - most);
          m = most;
        }
        ctl->keep[steps % kPfaAhead][r] = mostf == ref ? 1.f : exp2f(ref - mostf);
        ref = mostf;
        const float mm = m == -INFINITY ? 0.f : m, rr = (ref == -INFINITY ? 0.f : ref) - 14.f;  // weights up to 2^14
        float part[2] = {0.f, 0.f};
        uint32_t whi[32], wlo[32];
#pragma unroll
        for (int i = 0; i < kPaTile; i += 2) {
          const float4 u = up[i / 2];
          const float a = __uint_as_float(s[i]), b = __uint_as_float(s[i + 1]);
          part[0] += exp2_approx(a - mm), part[1] += exp2_approx(b - mm);
          const float wa = exp2_approx((a + u.y) - rr), wb = exp2_approx((b + u.w) - rr);
          const uint32_t hi = cvt2<__half>(wa, wb);
          const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          whi[(i / 2) & 31] = hi;
          wlo[(i / 2) & 31] = cvt2<__half>(wa - h.x, wb - h.y);
          if (i % 64 == 62) {
            tmem_st32(s_addr + (i / 64) * 32, whi);
            tmem_st32(s_addr + 64 + (i / 64) * 32, wlo);
          }
        }
        sum += part[0] + part[1];
        mbar_arrive(&ctl->up_empty[steps & 1]);
        if (last) {
          // out = (O / l) 2^(m' - m); the weights had 2^14 more. In two steps, so that no power leaves f32's range before the
          // product
          const float f1 = exp2f(0.5f * ((ref == -INFINITY ? 0.f : ref) - mm - 14.f));
          ctl->finish[items % kPfaAhead][r] = make_float2(f1, sum == 0.f ? 0.f : f1 / sum);
          if (it.row + kPaTile > it.len) {
            // the tile goes on behind the sequence: whatever stands there, 0 times it has to be 0. The products of the tile
            // before are waited for first: then that tile's values had landed, and the parity below can only mean this one's
            if (j && !(ok = __all_sync(0xffffffffu, wait(&ctl->pv_full[(steps - 1) & 1], (steps - 1) / 2, kErrMmaWait)))) break;
            const int from = it.len - it.row;  // rows of the sequence in the tile
#pragma unroll 1
            for (int part_i = 0; part_i < 2 && ok; ++part_i) {
              const uint32_t u = unit + 4 * j + 2 + part_i;
              if (!(ok = __all_sync(0xffffffffu, wait(&ctl->kv_full[u % kStages], u / kStages, kErrFullWait)))) break;
              uint8_t* v = base + (2 + u % kStages) * kTileBytes;
              for (int i = from * 8 + r; i < kPaTile * 8; i += 128)
                for (int b = 0; b < kBoxes; ++b) *reinterpret_cast<uint4*>(v + b * kBoxBytes + i * 16) = make_uint4(0, 0, 0, 0);
            }
            if (!ok) break;
            fence_proxy_async();
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ctl->p_full);
      }
      unit += 4 * it.n;
      ++items;
    }
  } else if (warp < 8) {
    // ---------------- O: a thread per row
    set_regs_up<kPfaSumRegs>();
    const int r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t steps = 0, items = 0;
    bool ok = true;
    for (int64_t x = blockIdx.x; x < p.n_items && ok; x += gridDim.x) {
      Item it;
      if (!item(x, it)) continue;
      float o[kHd];
#pragma unroll
      for (int e = 0; e < kHd; ++e) o[e] = 0.f;
      for (int j = 0; j < it.n; ++j, ++steps) {
        if (!(ok = __all_sync(0xffffffffu, wait(&ctl->pv_full[steps & 1], steps / 2, kErrMmaWait)))) break;
        tc_fence_after();
        const float keep = ctl->keep[steps % kPfaAhead][r];
        const uint32_t addr = tmem + lanes + 256 + (steps & 1) * 128;
#pragma unroll
        for (int i = 0; i < kHd / 16; ++i) {
          uint32_t v[16];
          tmem_ld16(addr + 16 * i, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[16 * i + e] = fmaf(o[16 * i + e], keep, __uint_as_float(v[e]));
        }
        tc_fence_before();
        mbar_arrive(&ctl->pv_empty[steps & 1]);
      }
      if (!ok) break;
      const int row = it.row + r;
      const int64_t rows_at = (int64_t)(it.head / p.group) * p.n_rows + it.first;
      const float2 f = ctl->finish[items % kPfaAhead][r];
      bool odd = false;
      for (int j = lane; j < it.n; j += 32) odd |= p.marked[rows_at + (int64_t)j * kPaTile] != 0;
      odd = __any_sync(0xffffffffu, odd);
      if (row < it.len) {
        float* dst = p.out + ((it.first + row) * p.n_heads + it.head) * kHd;
#pragma unroll
        for (int e = 0; e < kHd; e += 4)
          *reinterpret_cast<float4*>(dst + e) = make_float4(o[e] * f.x * f.y, o[e + 1] * f.x * f.y, o[e + 2] * f.x * f.y, o[e + 3] * f.x * f.y);
        if (odd) add_not_finite<kHd>(p, it.first, row, it.head, dst);
      }
      __syncwarp();
      ++items;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

}  // namespace fq
