// Causal attention inside packed prompts on the 5th-generation tensor cores (fuelq_prompt_attn), 16-bit types.
//
//   S = Q K^T,  P = exp2(c S - c m),  O += P V,  out = O / sum(P),   c = scale log2(e)
//
// with m a reference that follows the running maximum of the row: it moves only when the maximum has passed it by 2^8, so that
// O, which stays in tensor memory, is hardly ever rescaled (P then reaches 2^8 at most; sums and products are f32).
// Bound by the tensor cores and, at head_dim 64 above all, by the 16 exponentials a clock and SM.
// A persistent thread block per SM takes blocks of 256 query rows of one head, the longest of a sequence first, as two tiles of
// 128 rows that take turns: while the tensor cores multiply for one tile, the other one's softmax runs.
//   warps 0-3, 4-7  softmax of tile 0, 1: one thread per row. Reads S from tensor memory, writes P over it in the inputs' type,
//                   which the second product reads from there; at the end divides and stores its rows
//   warp 8          copies (TMA): Q tiles, and K and V tiles of 128 keys through one ring
//   warp 9          issues the MMAs: S of the next key tile goes out behind the product of the last, so the tensor cores have
//                   work whenever one of the tiles is ready; 10 and 11 only make up the group of four that gives registers away
// Keys behind a row: the scores of the last key tile are masked. A value of NaN or infinity there would still reach earlier rows
// as 0 x NaN, so the softmax warps take such values out of the last tile in shared memory and add them to the rows they
// belong to at the end. Rows of the next sequence, or of nobody, that the last tile touches are taken out the same way.
#pragma once
#include <type_traits>

#include "attn.cuh"
#include "attn_plan.h"
#include "umma.cuh"

namespace fq {

struct PromptParams {
  void* out;
  const int* cu;
  int64_t n_rows, n_items;
  int n_seqs, n_heads, group;
  float c;
};
constexpr int kPaThreads = 384, kPaTile = 128, kPaRows = 2 * kPaTile;
// registers of a softmax thread (its row of S is 128 of them) and of the others: 256 x 208 + 128 x 80 of the launch's 384 x 168
constexpr int kPaSoftmaxRegs = 208, kPaOtherRegs = 80;

// ---- PTX wrappers
__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                   smem_dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
               : "memory");
}
// the first operand from tensor memory
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// a tile [k rows][64 columns of 128 bytes] whose columns are the operand's rows (N), 128-byte swizzle: groups of 64 columns
// `group_bytes` apart, groups of eight k rows 1024 bytes apart
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(uint32_t smem_addr, uint32_t group_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3ffffu) >> 4);
  d |= (uint64_t)(group_bytes >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
constexpr uint32_t kIdescBColumns = 1u << 16;  // the second operand is stored by columns (N contiguous)

__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// waits for the loads before it; their registers pass through the instruction, so that nothing that reads them can move in front
__device__ __forceinline__ void tmem_wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), 
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), 
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), 
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), 
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), 
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
               "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t lds_pair(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two f32 at a time
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t cvt2(float a, float b);
template <>
__device__ __forceinline__ uint32_t cvt2<__half>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <>
__device__ __forceinline__ uint32_t cvt2<__nv_bfloat16>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// one lane of the warp, in a form that lets the compiler keep what the MMAs take (descriptors, addresses) in uniform registers: the
// whole warp runs the issuing role and only the instructions themselves are this lane's. With the role in a branch of one
// lane an MMA took 125 cycles to issue, twice what it runs
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}
template <int kRegs>
__device__ __forceinline__ void set_regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void set_regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }
// is one of the two 16-bit values an infinity or NaN?
template <typename T>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  const uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

// Values taken out of a tile of values, by column: the first of its rows that holds +inf, -inf, NaN. Records carry the number of
// their item, in a form that a later item's replaces an earlier one's under atomicMin, so that they are never cleared.
template <int kHd>
struct TakenOut {
  uint32_t last;  // 1 + the last item with a record
  uint32_t row[3][kHd];
};
__device__ __forceinline__ uint32_t taken_word(uint32_t item, int row) { return ((0xffffffu - item) << 8) | (uint32_t)row; }
// the row of a record, or a row behind all others if it is not of this item
__device__ __forceinline__ int taken_row(uint32_t word, uint32_t item) { return word >> 8 == 0xffffffu - item ? (int)(word & 0xff) : 0x100; }

template <int kHd, int kStages>
struct PromptCtl {
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2];
  uint64_t kv_full[kStages], kv_empty[kStages];
  uint64_t taken_free;  // tile 1 has read the record of tile 0 (once per item with a tile 1)
  TakenOut<kHd> taken[2];
  uint32_t tmem_base;
  int abort_flag;
};

// What an item holds for the two tiles
struct PromptItem {
  int64_t first;  // first row of the sequence
  int len, row, head;
  int n0, n1;  // key tiles of each tile of rows; 0: it has no rows
};
__device__ __forceinline__ bool prompt_item(const PromptParams& p, int64_t x, PromptItem& it, bool& bad) {
  const int64_t slot = x / p.n_heads;
  it.head = (int)(x - slot * p.n_heads);
  const PromptBlock b = prompt_block(p.cu, p.n_seqs, p.n_rows, slot, kPaRows);
  bad = b.len < 0;
  if (b.row >= b.len) return false;
  it.first = b.first, it.len = b.len, it.row = b.row;
  it.n0 = b.row / kPaTile + 1;
  it.n1 = b.row + kPaTile < b.len ? it.n0 + 1 : 0;
  return true;
}

template <typename T, int kHd>
struct PromptCfg {
  static constexpr int kStages = kHd == 128 ? 4 : 8;
  static constexpr int kTileBytes = kPaTile * kHd * 2;
  static constexpr int kSmem = 1024 + (2 + kStages) * kTileBytes + (int)sizeof(PromptCtl<kHd, kStages>) + 16;
};

template <typename T, int kHd>
__global__ void __launch_bounds__(kPaThreads, 1) prompt_attn_kernel(const PromptParams p, const __grid_constant__ CUtensorMap qmap,
                                                                    const __grid_constant__ CUtensorMap kmap,
                                                                    const __grid_constant__ CUtensorMap vmap) {
  using Cfg = PromptCfg<T, kHd>;
  constexpr int kStages = Cfg::kStages, kTileBytes = Cfg::kTileBytes, kBoxes = kHd / 64, kBoxBytes = kPaTile * 128;
  extern __shared__ __align__(1024) uint8_t pa_smem[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pa_smem) + 1023) & ~(uintptr_t)1023);
  const uint32_t q_addr = smem_u32(base), kv_addr = q_addr + 2 * kTileBytes;
  auto* ctl = reinterpret_cast<PromptCtl<kHd, kStages>*>(base + (2 + kStages) * kTileBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(&ctl->q_full[x], 1), mbar_init(&ctl->q_empty[x], 1);
      mbar_init(&ctl->s_full[x], 1), mbar_init(&ctl->p_full[x], 128), mbar_init(&ctl->o_full[x], 1);
      ctl->taken[x].last = 0;
    }
    for (int s = 0; s < kStages; ++s) mbar_init(&ctl->kv_full[s], 1), mbar_init(&ctl->kv_empty[s], 1);
    mbar_init(&ctl->taken_free, 128);
    ctl->abort_flag = 0;
    mbar_init_fence();
  }
  for (int i = threadIdx.x; i < 3 * kHd; i += kPaThreads) ctl->taken[0].row[0][i] = ctl->taken[1].row[0][i] = 0xffffffffu;
  if (warp == 9) tmem_alloc(&ctl->tmem_base, 512);  // S of both tiles (P over it), O of both tiles
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&ctl->tmem_base);
  volatile int* abort_flag = &ctl->abort_flag;
  // every wait is bounded; the first that runs out ends the block's work in all roles
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (mbar_poll_bounded(bar, parity & 1u)) return true;
    if (!*abort_flag) record_dev_error(code);
    *abort_flag = 1;
    return false;
  };

  if (warp >= 8) set_regs_down<kPaOtherRegs>();
  if (warp == 8) {
    // ---------------- copies
    if (lane == 0) {
      uint32_t unit = 0, tiles[2] = {0, 0};  // key and value tiles requested; items of each row tile
      bool ok = true;
      for (int64_t x = blockIdx.x; x < p.n_items && ok && !*abort_flag; x += gridDim.x) {
        PromptItem it;
        bool bad;
        if (!prompt_item(p, x, it, bad)) {
          if (bad) record_dev_error(kErrIndex);
          continue;
        }
        const int kvh = it.head / p.group, row0 = (int)it.first + it.row;
        auto load_q = [&](int t) {
          if (tiles[t] && !wait(&ctl->q_empty[t], tiles[t] - 1, kErrEmptyWait)) return false;
          mbar_arrive_expect_tx(&ctl->q_full[t], kTileBytes);
          for (int b = 0; b < kBoxes; ++b)
            tma_load_3d(q_addr + t * kTileBytes + b * kBoxBytes, &qmap, 64 * b, it.head, row0 + t * kPaTile, &ctl->q_full[t]);
          ++tiles[t];
          return true;
        };
        auto load_kv = [&](const CUtensorMap* map, int j) {
          const uint32_t s = unit % kStages;
          if (unit >= kStages && !wait(&ctl->kv_empty[s], unit / kStages - 1, kErrEmptyWait)) return false;
          mbar_arrive_expect_tx(&ctl->kv_full[s], kTileBytes);
          for (int b = 0; b < kBoxes; ++b)
            tma_load_3d(kv_addr + s * kTileBytes + b * kBoxBytes, map, 64 * b, kvh, (int)it.first + j * kPaTile, &ctl->kv_full[s]);
          ++unit;
          return true;
        };
        ok = load_q(0);
        const int n = it.n1 ? it.n1 : it.n0;
        for (int j = 0; j < n && ok && !*abort_flag; ++j) {
          ok = load_kv(&kmap, j);
          if (ok && j == 0 && it.n1) ok = load_q(1);
          if (ok) ok = load_kv(&vmap, j);
        }
      }
      pdl_launch_dependents();
      if (*abort_flag) {  // leaving early: let the copies already requested land first
        for (uint32_t u = unit > kStages ? unit - kStages : 0; u < unit; ++u)
          if (!mbar_wait_bounded(&ctl->kv_full[u % kStages], (u / kStages) & 1)) record_dev_error(kErrDrainWait);
        for (int t = 0; t < 2; ++t)
          if (tiles[t] && !mbar_wait_bounded(&ctl->q_full[t], (tiles[t] - 1) & 1)) record_dev_error(kErrDrainWait);
      }
    }
  } else if (warp == 9) {
    // ---------------- MMA issue
    constexpr bool kF16 = std::is_same<T, __half>::value;
    constexpr uint32_t s_desc = kF16 ? umma_idesc_f16(kPaTile, kPaTile) : umma_idesc_bf16(kPaTile, kPaTile);
    constexpr uint32_t o_desc = (kF16 ? umma_idesc_f16(kPaTile, kHd) : umma_idesc_bf16(kPaTile, kHd)) | kIdescBColumns;
    const uint32_t acc = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t q_desc = umma_desc_sw128(q_addr), k_desc = umma_desc_sw128(kv_addr), v_desc = umma_desc_sw128_mn(kv_addr, kBoxBytes);
    const bool leader = elect_one();
    auto ready = [&](uint64_t* bar, uint32_t parity, int code) { return (bool)__all_sync(0xffffffffu, wait(bar, parity, code)); };
    uint32_t unit = 0, tiles[2] = {0, 0}, steps[2] = {0, 0};  // steps: key tiles of each row tile so far
    bool ok = true;
    for (int64_t x = blockIdx.x; x < p.n_items && ok; x += gridDim.x) {
      PromptItem it;
      bool bad;
      if (!prompt_item(p, x, it, bad)) continue;
      const int n = it.n1 ? it.n1 : it.n0, nt[2] = {it.n0, it.n1};
      auto stage = [&](int j, bool value) { return (unit + 2 * j + value) % kStages; };
      auto kv_ready = [&](int j, bool value) { return ready(&ctl->kv_full[stage(j, value)], (unit + 2 * j + value) / kStages, kErrFullWait); };
      auto scores = [&](int t, int j) {
        const uint64_t a = q_desc + (uint64_t)(t * kTileBytes >> 4), b = k_desc + (uint64_t)(stage(j, false) * kTileBytes >> 4);
        if (leader) {
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < kHd / 16; ++k) {
            const uint64_t off = ((k / 4) * kBoxBytes + (k % 4) * 32) >> 4;
            umma_bf16(acc + t * kPaTile, a + off, b + off, s_desc, k != 0);
          }
          umma_commit(&ctl->s_full[t]);
          if (j + 1 == nt[t]) umma_commit(&ctl->q_empty[t]);
        }
      };
      ok = kv_ready(0, false);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!ok || !nt[t]) continue;
        ok = ready(&ctl->q_full[t], tiles[t]++, kErrFullWait);
        if (ok) scores(t, 0);
      }
      if (ok && leader) umma_commit(&ctl->kv_empty[stage(0, false)]);
      for (int j = 0; j < n && ok; ++j) {
        if (!(ok = kv_ready(j, true))) break;
        if (j + 1 < n && !(ok = kv_ready(j + 1, false))) break;
        const uint64_t b = v_desc + (uint64_t)(stage(j, true) * kTileBytes >> 4);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || j >= nt[t]) continue;
          if (!(ok = ready(&ctl->p_full[t], steps[t]++, kErrMmaWait))) continue;
          if (leader) {
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < kPaTile / 16; ++k)
              umma_f16_ts(acc + 256 + t * 128, acc + t * kPaTile + k * 8, b + (uint64_t)(k * 2048 >> 4), o_desc, (j | k) != 0);
          }
          if (j + 1 < nt[t]) scores(t, j + 1);
          else if (j + 1 < n && leader) umma_commit(&ctl->o_full[t]);
        }
        if (ok && leader) {
          umma_commit(&ctl->kv_empty[stage(j, true)]);
          if (j + 1 < n) umma_commit(&ctl->kv_empty[stage(j + 1, false)]);
          else umma_commit(&ctl->o_full[it.n1 ? 1 : 0]);  // last of all: nothing of this block arrives after its results are read
        }
      }
      unit += 2 * n;
    }
  } else if (warp < 8) {
    // ---------------- softmax: a thread per row of tile t
    set_regs_up<kPaSoftmaxRegs>();
    const int t = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + t * kPaTile, o_addr = tmem + lanes + 256 + t * 128;
    uint32_t unit = 0, steps = 0, done = 0, done1 = 0;  // items so far; those with a tile 1
    bool ok = true;
    for (int64_t x = blockIdx.x; x < p.n_items && ok; x += gridDim.x) {
      PromptItem it;
      bool bad;
      if (!prompt_item(p, x, it, bad)) continue;
      const int n = it.n1 ? it.n1 : it.n0, mine = t ? it.n1 : it.n0;
      float ref = -INFINITY, mc = 0.f;  // the reference; c times it
      uint64_t sum2[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
      for (int j = 0; j < mine && ok; ++j) {
        if (!(ok = __all_sync(0xffffffffu, wait(&ctl->s_full[t], steps++, kErrMmaWait)))) break;
        tc_fence_after();
        uint32_t s[kPaTile];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32_nowait(s_addr + 32 * i, s + 32 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_wait_ld(s + 32 * i);
        const bool last = j + 1 == mine;
        if (last) {  // keys behind the row
#pragma unroll
          for (int i = 0; i < kPaTile; ++i)
            if (i > r) s[i] = 0xff800000u;
        }
        float top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i] = __uint_as_float(s[i]);
#pragma unroll
        for (int i = 4; i < kPaTile; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(s[i]));
        const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        if (j == 0) {
          ref = most;
          mc = ref == -INFINITY ? 0.f : ref * p.c;
        } else {
          const bool move = (most - ref) * p.c > 8.f;
          if (__any_sync(0xffffffffu, move)) {  // O is complete up to the tile before: S of this one came after it
            // each row by its own scores alone: its bits do not depend on what else is in the warp
            const float keep = move ? exp2_approx((ref - most) * p.c) : 1.f;
            if (move) ref = most;
            mc = ref == -INFINITY ? 0.f : ref * p.c;
#pragma unroll
            for (int i = 0; i < kHd / 32; ++i) {
              uint32_t o[32];
              tmem_ld32_nowait(o_addr + 32 * i, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
              tmem_st32(o_addr + 32 * i, o);
            }
            float a, b;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              unpair(sum2[i], a, b);
              sum2[i] = pair(a * keep, b * keep);
            }
          }
        }
        const uint64_t c2 = pair(p.c, p.c), m2 = pair(-mc, -mc);
        uint32_t w[kPaTile / 2];
#pragma unroll
        for (int i = 0; i < kPaTile; i += 2) {
          float a, b;
          unpair(fma2(pair(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), c2, m2), a, b);
          a = exp2_approx(a), b = exp2_approx(b);
          sum2[(i >> 1) & 1] = add2(sum2[(i >> 1) & 1], pair(a, b));
          w[i >> 1] = cvt2<T>(a, b);
          if (i % 64 == 62) tmem_st32(s_addr + (i / 64) * 32, w + (i / 64) * 32);
        }
        if (last) {
          // values of the last key tile that are not finite: out of the tile, into the record
          const uint32_t u = unit + 2 * j + 1, st = u % kStages;
          if (!(ok = __all_sync(0xffffffffu, wait(&ctl->kv_full[st], u / kStages, kErrFullWait)))) break;
          uint8_t* v = base + (2 + st) * kTileBytes;
          TakenOut<kHd>* rec = &ctl->taken[t];
          bool found = false;
#pragma unroll 4
          for (int i = 0; i < kTileBytes / 16 / 128; ++i) {
            const int at = (i * 128 + r) * 16;
            const uint4 q = *reinterpret_cast<const uint4*>(v + at);
            if (!(not_finite2<T>(q.x) || not_finite2<T>(q.y) || not_finite2<T>(q.z) || not_finite2<T>(q.w))) continue;
            // tile 0's record is read by tile 1 too, perhaps still for the last item that had one
            if (t == 0 && !found && done1 && !wait(&ctl->taken_free, done1 - 1, kErrMmaWait)) break;
            found = true;
            const int box = at / kBoxBytes, key = (at % kBoxBytes) / 128, chunk = ((at % 128) / 16) ^ (key & 7);
            T* e = reinterpret_cast<T*>(v + at);
            for (int k = 0; k < 8; ++k) {
              const float f = to_f32(e[k]);
              if (isfinite(f)) continue;
              atomicMin(&rec->row[f != f ? 2 : f < 0.f ? 1 : 0][box * 64 + chunk * 8 + k], taken_word(done, key));
              e[k] = from_f32<T>(0.f);
            }
          }
          if (found) {
            rec->last = done + 1;
            fence_proxy_async();
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ctl->p_full[t]);
      }
      if (ok && mine) {
        if (!(ok = __all_sync(0xffffffffu, wait(&ctl->o_full[t], t ? done1 : done, kErrMmaWait)))) break;
        tc_fence_after();
        float a, b, a1, b1;
        unpair(sum2[0], a, b), unpair(sum2[1], a1, b1);
        const float total = (a + b) + (a1 + b1), inv = total == 0.f ? 0.f : 1.f / total;
        const int row = it.row + t * kPaTile + r;
        const bool rec0 = ctl->taken[0].last == done + 1, rec1 = t && ctl->taken[1].last == done + 1;
        T* dst = reinterpret_cast<T*>(p.out) + ((it.first + row) * p.n_heads + it.head) * kHd;
#pragma unroll
        for (int i = 0; i < kHd / 32; ++i) {
          uint32_t o[32];
          tmem_ld32_nowait(o_addr + 32 * i, o);
          tmem_wait_ld(o);
          if (row < it.len) {
            if (rec0 || rec1) {
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                float f = __uint_as_float(o[e]);
#pragma unroll 1
                for (int k = 0; k < 1 + t; ++k) {
                  if (!(k ? rec1 : rec0)) continue;
                  const int upto = k == t ? r : kPaTile - 1;  // tile 1 sees all of tile 0's keys
                  const volatile uint32_t* q = &ctl->taken[k].row[0][32 * i + e];
                  if (taken_row(q[0], done) <= upto) f += INFINITY;
                  if (taken_row(q[kHd], done) <= upto) f -= INFINITY;
                  if (taken_row(q[2 * kHd], done) <= upto) f += __int_as_float(0x7fc00000);
                }
                o[e] = __float_as_uint(f);
              }
            }
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 q;
              q.x = cvt2<T>(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
              q.y = cvt2<T>(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
              q.z = cvt2<T>(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
              q.w = cvt2<T>(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
              *reinterpret_cast<uint4*>(dst + 32 * i + e) = q;
            }
          }
          __syncwarp();
        }
        tc_fence_before();
        if (t) mbar_arrive(&ctl->taken_free);
      }
      unit += 2 * n;
      ++done;
      done1 += it.n1 != 0;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

}  // namespace fq
