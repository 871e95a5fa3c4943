// Causal attention inside packed prompts on the 5th-generation tensor cores (fuelq_prompt_attn), 16-bit types.
//
//   S = Q K^T,  P = exp2(c S - c m),  O += P V,  out = O / sum(P),   c = scale log2(e)
//
// with m a reference that follows the running maximum of the row: it moves only when the maximum has passed it by 2^8, so that
// O, which stays in tensor memory, is hardly ever rescaled (P then reaches 2^8 at most, times 2^7 in f16, to keep clear of its lower end,
// and times 2^-24 in bf16, to keep O clear of f32's upper end; sums and products are f32). P is rounded once to the inputs' type: half a
// step of each weight, in f16 2^-32 of the largest at least. P in two parts would be half as many products again.
// Bound by the tensor cores and, at head_dim 64 above all, by the 16 exponentials a clock and SM.
// A persistent thread block per SM takes blocks of 256 query rows of one head, the longest of a sequence first, as two tiles of
// 128 rows that take turns: while the tensor cores multiply for one tile, the other one's softmax runs.
//   warps 0-3, 4-7  softmax of tile 0, 1: one thread per row. Reads S from tensor memory, writes P over it in the inputs' type,
//                   which the second product reads from there; at the end divides and stores its rows
//   warp 8          copies (TMA): Q tiles, and K and V tiles of 128 keys through one ring
//   warp 9          issues the MMAs: S of the next key tile goes out behind the product of the last, so the tensor cores have
//                   work whenever one of the tiles is ready
//   warp 10         finds the block's items ahead of the others (11 only makes up the group of four that gives registers away)
// Keys behind a row: the scores of the last key tile are masked. A value of NaN or infinity there would still reach earlier rows
// as 0 x NaN, so the softmax warps take such values out of the last tile in shared memory and add them to the rows they
// belong to at the end. Rows of the next sequence, or of nobody, that the last tile touches are taken out the same way.
// Measured, 32/8 heads of 128: one prompt of 16384 tokens, f16, 1.90 to 2.26 ms by card (970 to 1160 TFLOP/s of the scores that are
// seen, the card under its power limit), 4096 tokens 160 us; 24 prompts up to 2048, bf16, 331 to 343 us (513 to 532). A row tile's
// softmax (ld 250, maximum 450, exponentials 1370 cycles) and its own products (1380 from the last weight to the next scores) follow
// one another, so with two tiles in turn the tensor cores wait a quarter of the time. Tensor memory has no room for a third; the
// products could begin on half of the weights, which is not done. Blocks of rows are dealt round the thread blocks whatever they
// cost: in the 24 prompts the fullest has 157 key tiles and item ends where the average is 115, in one prompt of 4096 80 of 62.
#pragma once
#include <type_traits>

#include "attn.cuh"
#include "attn_plan.h"
#include "umma.cuh"

namespace fq {

struct PromptParams {
  void* out;
  const void* v;
  int64_t v_stride;
  const int* cu;
  int64_t n_rows, n_items;
  int n_seqs, n_heads, group;
  float c;
};
constexpr int kPaThreads = 384, kPaTile = 128, kPaRows = 2 * kPaTile;
// registers of a softmax thread (its row of S is 128 of them) and of the others: 256 x 208 + 128 x 80 of the launch's 384 x 168. (The
// form for heads of 64 keeps 48 bytes of a thread on its stack all the same, that for 128 nothing)
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
__device__ __forceinline__ void tmem_ld8_nowait(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld8(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%4], {%0,%1,%2,%3};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
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
// the largest of three, NaN if one is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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
// 2^x of two values on the multiply-add pipes: x = n + f with n the nearest integer, found by adding 1.5 2^23, 2^f by a polynomial of
// degree four (fitted to the least relative error over [-1/2, 1/2], its constant held at 1: 2.9e-6), n added to its exponent. From
// -127 down, -inf among them, the exponent comes to nothing and the result is zero itself: a masked key's weight, which the largest
// bf16 value behind the row must not show through. NaN does not pass
__device__ __forceinline__ void exp2_poly2(uint64_t x, float& a, float& b) {
  unpair(x, a, b);
  x = pair(fmaxf(a, -127.f), fmaxf(b, -127.f));
  const uint64_t magic = pair(12582912.f, 12582912.f), t = add2(x, magic);
  const uint64_t f = fma2(add2(t, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), x);
  uint64_t y = fma2(f, pair(0x1.3a1804p-7f, 0x1.3a1804p-7f), pair(0x1.c9fcb2p-5f, 0x1.c9fcb2p-5f));
  y = fma2(y, f, pair(0x1.ec0326p-3f, 0x1.ec0326p-3f));
  y = fma2(y, f, pair(0x1.62e12cp-1f, 0x1.62e12cp-1f));
  y = fma2(y, f, pair(1.f, 1.f));
  float ta, tb;
  unpair(t, ta, tb);
  unpair(y, a, b);
  a = __uint_as_float(__float_as_uint(a) + (__float_as_uint(ta) << 23));
  b = __uint_as_float(__float_as_uint(b) + (__float_as_uint(tb) << 23));
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
// whole warp runs the issuing role and only the instructions themselves are this lane's (4096 tokens of f16: 176 us, with the role in
// a branch of one lane 194)
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}
template <int kRegs>
__device__ __forceinline__ void set_regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void set_regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }
// bit 15 or 31 of the result: the value below it is an infinity or NaN (its exponent, all ones, overflows by one more)
template <typename T>
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
  return (w & 0x7fff7fffu) + (std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u);
}
__device__ __forceinline__ uint4 lds_u4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts_u4(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A warp's 32 rows, 64 bytes of each in its lane's registers, to memory: turned round in shared memory so that four lanes write a
// row's 64 bytes together (a lane by itself would touch 32 lines with every store: the epilogue was 6000 cycles long). rows: how
// many of them there are
constexpr int kStageRow = 80, kStageBytes = 32 * kStageRow;  // 80: eight rows in eight different 16-byte columns of the banks
__device__ __forceinline__ void store_rows64(uint32_t stage, int lane, const uint4 (&v)[4], uint8_t* dst, int64_t row_bytes, int rows) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) sts_u4(stage + lane * kStageRow + 16 * i, v[i]);
  __syncwarp();
  dst += (lane >> 2) * row_bytes + 16 * (lane & 3);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 8 * i + (lane >> 2);
    const uint4 q = lds_u4(stage + row * kStageRow + 16 * (lane & 3));
    if (row < rows) *reinterpret_cast<uint4*>(dst + 8 * i * row_bytes) = q;
  }
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

// The items of a thread block are found by a warp of their own and handed to the others through a ring: the search (dependent loads,
// a division) is 2700 cycles long, which every role had between two items before
struct PromptItem {
  int64_t first;  // first row of the sequence
  int len;        // its rows; -1: there are no more items
  int row, head;  // first row of the block within the sequence
  int n;          // key tiles of the block's first 128 rows
};
constexpr int kItemRing = 4;
struct ItemRing {
  uint64_t full[kItemRing], empty[kItemRing];
  PromptItem item[kItemRing];
};
// The next item from x on (in steps of the grid) whose block has rows; the whole warp looks
__device__ __forceinline__ PromptItem find_item(const int* cu, int n_seqs, int64_t n_rows, int n_heads, int64_t n_items, int rows,
                                                int64_t& x, int lane) {
  PromptItem it;
  for (; x < n_items; x += gridDim.x) {
    const int64_t slot = x / n_heads;
    int lo = 0, hi = n_seqs;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, at = lo + lane * step;
      const uint32_t before = __ballot_sync(0xffffffffu, at < hi && prompt_slot(cu[at], at, rows) <= slot);
      lo += max(__popc(before) - 1, 0) * step;
      hi = min(lo + step, hi);
    }
    const PromptBlock b = prompt_block_of(cu, lo, n_rows, slot, rows);
    if (b.len < 0 && lane == 0) record_dev_error(kErrIndex);
    if (b.row >= b.len) continue;
    it.first = b.first, it.len = b.len, it.row = b.row, it.head = (int)(x - slot * n_heads), it.n = b.row / kPaTile + 1;
    x += gridDim.x;
    return it;
  }
  it.first = 0, it.len = -1, it.row = it.head = it.n = 0;
  return it;
}
// the n-th item into the ring; false if its place was not free in time
template <typename Wait>
__device__ __forceinline__ bool put_item(ItemRing& ring, uint32_t n, const PromptItem& it, int lane, Wait& wait) {
  const uint32_t s = n % kItemRing;
  if (n >= kItemRing && !__all_sync(0xffffffffu, wait(&ring.empty[s], n / kItemRing - 1, kErrEmptyWait))) return false;
  if (lane == 0) {
    ring.item[s] = it;
    mbar_arrive(&ring.full[s]);
  }
  return true;
}
// the n-th item, for the whole warp or for the one lane that runs a role; false if there is none, or none in time
template <bool kWarp, typename Wait>
__device__ __forceinline__ bool get_item(ItemRing& ring, uint32_t n, PromptItem& it, Wait& wait) {
  const uint32_t s = n % kItemRing;
  bool ok = wait(&ring.full[s], n / kItemRing, kErrFullWait);
  if constexpr (kWarp) ok = __all_sync(0xffffffffu, ok);
  if (!ok) return false;
  it = ring.item[s];
  if constexpr (kWarp) __syncwarp();
  if (!kWarp || (threadIdx.x & 31) == 0) mbar_arrive(&ring.empty[s]);
  return it.len >= 0;
}

// Rows of a warp (the bits of `which`) with NaN in their result beside a finite sum of weights: an infinite value whose weight has rounded to
// zero. Each column becomes what it holds that is not finite, the lanes over the columns: the first key with +inf, -inf, NaN of
// every column, looked for once for all rows. v: the head's values of the sequence's first row; row: the warp's first; dst: its result
template <typename T, int kHd>
__device__ __forceinline__ void put_not_finite(const T* v, int64_t v_stride, int row, uint32_t which, T* dst, int64_t dst_stride, int lane) {
  constexpr int kMine = kHd / 32, kNone = 0x7fffffff;
  int first[3][kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) first[0][i] = first[1][i] = first[2][i] = kNone;
  const int last = row + 31 - __clz(which);  // of the rows in question
  for (int key0 = 0; key0 <= last; key0 += 8) {
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int key = min(key0 + n, last);
        const float f = to_f32(v[key * v_stride + lane + 32 * i]);
        first[0][i] = f == INFINITY ? min(first[0][i], key) : first[0][i];
        first[1][i] = f == -INFINITY ? min(first[1][i], key) : first[1][i];
        first[2][i] = f != f ? min(first[2][i], key) : first[2][i];
      }
  }
  for (; which; which &= which - 1) {
    const int r = __ffs(which) - 1;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      float sum = 0.f;
      if (first[0][i] <= row + r) sum += INFINITY;
      if (first[1][i] <= row + r) sum -= INFINITY;
      if (first[2][i] <= row + r) sum += __int_as_float(0x7fc00000);
      if (sum != 0.f) dst[r * dst_stride + lane + 32 * i] = from_f32<T>(sum);
    }
  }
}

template <int kHd, int kStages>
struct PromptCtl {
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2];
  uint64_t kv_full[kStages], kv_empty[kStages];
  uint64_t taken_free[2];  // the threads of a tile have read the records of an item (tile 1 reads both)
  TakenOut<kHd> taken[2];
  ItemRing items;
  uint32_t tmem_base;
  int abort_flag;
};

// key tiles of the second 128 rows of a block, 0 if it has none
__device__ __forceinline__ int second_tiles(const PromptItem& it) { return it.row + kPaTile < it.len ? it.n + 1 : 0; }

// What a row's scores are multiplied by, c, and what is added, `up` - ref c (up: see PromptCfg). The sum is rounded, and its error is in all
// of the row's weights alike: nothing while it is small. f16 has room for weights that are smaller, not larger: one more is taken off
// where the error is above a half. From 2^28 on (bf16: 2^30), where the weights of scores that differ are 2^-16 of one another or
// less, and where ref c leaves f32, the factor is a power of two, whose product is not rounded: the nearest to c that keeps ref's in range
template <typename T>
__device__ __forceinline__ void scale_row(float ref, float c, float up, float& row_c, float& add) {
  constexpr bool kF16 = std::is_same<T, __half>::value;
  row_c = c;
  float product = ref == -INFINITY ? 0.f : ref * c;
  if (fabsf(ref) < INFINITY && !(fabsf(product) <= (kF16 ? 0x1p28f : 0x1p30f))) {
    const uint32_t exponent = (__float_as_uint(ref) >> 23) & 255u, room = min(380u - exponent, 254u);  // ref 2^k below 2^127
    row_c = fminf(__uint_as_float(__float_as_uint(c * 1.41421356f) & 0x7f800000u), __uint_as_float(room << 23));
    product = ref * row_c;
  }
  add = up - product;
  if (kF16 && fmaf(ref, row_c, add) > up + 0.5f) add = __int_as_float(__float_as_int(add) + (add > 0.f ? -1 : 1));
}

template <typename T, int kHd>
struct PromptCfg {
  static constexpr int kStages = kHd == 128 ? 4 : 8;
  // one pair of scores in so many has its exponentials on the multiply-add pipes (the exponential unit does 16 a clock and SM).
  // 24 prompts up to 2048, head_dim 128: none 374, one in eight 335, six 340, five 341 us; one prompt of 256: 13.5, 11.8, 11.8, 11.8.
  // 8192 tokens, head_dim 64, where half the products meet as many exponentials: none 484, one in six 501, five 465, four 483 us
  static constexpr int kPolyEvery = kHd == 128 ? 6 : 4;
  // f16 ends at 2^-24: its weights are 2^7 times larger, up to 2^15; bf16's 2^24 times smaller, so that values at f32's ends can be
  // summed
  static constexpr float kUp = std::is_same<T, __half>::value ? 7.f : -24.f;
  static constexpr int kTileBytes = kPaTile * kHd * 2;
  static constexpr int kSmem = 1024 + (2 + kStages) * kTileBytes + 8 * kStageBytes + (int)sizeof(PromptCtl<kHd, kStages>) + 16;
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
  uint8_t* stages = base + (2 + kStages) * kTileBytes;  // of the rows on their way out, a warp each
  auto* ctl = reinterpret_cast<PromptCtl<kHd, kStages>*>(stages + 8 * kStageBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(&ctl->q_full[x], 1), mbar_init(&ctl->q_empty[x], 1);
      mbar_init(&ctl->s_full[x], 1), mbar_init(&ctl->p_full[x], 128), mbar_init(&ctl->o_full[x], 1);
      ctl->taken[x].last = 0;
    }
    for (int s = 0; s < kStages; ++s) mbar_init(&ctl->kv_full[s], 1), mbar_init(&ctl->kv_empty[s], 1);
    mbar_init(&ctl->taken_free[0], 128), mbar_init(&ctl->taken_free[1], 128);
    for (int s = 0; s < kItemRing; ++s) mbar_init(&ctl->items.full[s], 1), mbar_init(&ctl->items.empty[s], 10);  // warps 0 to 9
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
      PromptItem it;
      for (uint32_t items = 0; ok && !*abort_flag && get_item<false>(ctl->items, items, it, wait); ++items) {
        const int n1 = second_tiles(it), kvh = it.head / p.group, row0 = (int)it.first + it.row;
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
        const int n = n1 ? n1 : it.n;
        for (int j = 0; j < n && ok && !*abort_flag; ++j) {
          ok = load_kv(&kmap, j);
          if (ok && j == 0 && n1) ok = load_q(1);
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
    PromptItem it;
    for (uint32_t items = 0; ok && get_item<true>(ctl->items, items, it, wait); ++items) {
      const int n1 = second_tiles(it), n = n1 ? n1 : it.n, nt[2] = {it.n, n1};
      auto stage = [&](int j, bool value) { return (unit + 2 * j + value) % kStages; };
      auto kv_ready = [&](int j, bool value) {
        return ready(&ctl->kv_full[stage(j, value)], (unit + 2 * j + value) / kStages, kErrFullWait);
      };
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
          else umma_commit(&ctl->o_full[n1 ? 1 : 0]);  // last of all: nothing of this block arrives after its results are read
        }
      }
      unit += 2 * n;
    }
  } else if (warp == 10) {
    // ---------------- the items
    int64_t x = blockIdx.x;
    PromptItem it;
    uint32_t items = 0;
    do {
      it = find_item(p.cu, p.n_seqs, p.n_rows, p.n_heads, p.n_items, kPaRows, x, lane);
    } while (put_item(ctl->items, items++, it, lane, wait) && it.len >= 0);
  } else if (warp < 8) {
    // ---------------- softmax: a thread per row of tile t
    set_regs_up<kPaSoftmaxRegs>();
    const int t = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + t * kPaTile, o_addr = tmem + lanes + 256 + t * 128;
    uint32_t unit = 0, steps = 0, done = 0, done1 = 0;  // items so far; those with a tile 1
    bool ok = true;
    PromptItem it;
    for (; ok && get_item<true>(ctl->items, done, it, wait);) {
      const int n1 = second_tiles(it), n = n1 ? n1 : it.n, mine = t ? n1 : it.n;
      float ref = -INFINITY, row_c = p.c, add = 0.f;  // the reference; what scores are multiplied by; what is added then
      uint64_t sum2[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
      for (int j = 0; j < mine && ok; ++j) {
        if (!(ok = __all_sync(0xffffffffu, wait(&ctl->s_full[t], steps++, kErrMmaWait)))) break;
        tc_fence_after();
        const bool last = j + 1 == mine;
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // NaN where a visible score is: then the whole row is
        uint64_t c2, m2;
        // the row's reference, once its maximum is in top[]
        auto refer = [&]() {
          float most = max3_nan(top[0], top[1], max3_nan(top[2], top[3], top[3]));
          if (most == INFINITY) most = __int_as_float(0x7fc00000);  // inf - inf is in this row's softmax
          if (j == 0) {
            ref = most;
            scale_row<T>(ref, p.c, Cfg::kUp, row_c, add);
          } else {
            const bool move = !((most - ref) * row_c <= 8.f);
            if (__any_sync(0xffffffffu, move)) {  // O is complete up to the tile before: S of this one came after it
              // each row by its own scores alone: its bits do not depend on what else is in the warp
              float keep = 1.f;
              if (move && most != ref) {  // (equal: both -inf, nothing of weight yet)
                const float before = ref, c0 = row_c, add0 = add;
                ref = most;
                scale_row<T>(ref, p.c, Cfg::kUp, row_c, add);
                keep = before == -INFINITY ? 0.f : exp2_approx(row_c == c0 ? add - add0 : (before - most) * p.c);
                if (most != most) keep = most;
              }
#pragma unroll 1
              for (int i = 0; i < kHd / 16; ++i) {
                uint32_t o[16];
                tmem_ld16(o_addr + 16 * i, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                tmem_st16(o_addr + 16 * i, o);
              }
              float a, b;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                unpair(sum2[i], a, b);
                sum2[i] = pair(a * keep, b * keep);
              }
            }
          }
          c2 = pair(row_c, row_c), m2 = pair(add, add);
        };
        auto weight2 = [&](int i, uint32_t s0, uint32_t s1) {  // of pair i of the tile
          float a, b;
          const uint64_t x = fma2(pair(__uint_as_float(s0), __uint_as_float(s1)), c2, m2);
          if (i % Cfg::kPolyEvery == Cfg::kPolyEvery - 1) {
            exp2_poly2(x, a, b);
          } else {
            unpair(x, a, b);
            a = exp2_approx(a), b = exp2_approx(b);
          }
          sum2[i & 1] = add2(sum2[i & 1], pair(a, b));
          return cvt2<T>(a, b);
        };
        if (!last) {
          uint32_t s[kPaTile];
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_ld32_nowait(s_addr + 32 * i, s + 32 * i);
#pragma unroll
          for (int i = 0; i < 4; ++i) tmem_wait_ld(s + 32 * i);
#pragma unroll
          for (int i = 0; i < kPaTile; i += 2)
            top[(i >> 1) & 3] = max3_nan(top[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          refer();
          uint32_t w[kPaTile / 2];
#pragma unroll
          for (int i = 0; i < kPaTile / 2; ++i) {
            w[i] = weight2(i, s[2 * i], s[2 * i + 1]);
            if (i % 32 == 31) tmem_st32(s_addr + i - 31, w + i - 31);
          }
        } else {
          // The last tile of an item, with keys behind the row: short loops that read the scores from tensor memory twice. Code that is
          // run through once comes at some four cycles an instruction, and this is run once an item: 64 prompts of 256 tokens take
          // 116 us this way, 143 with the lines above; 4096 tokens 181 us if every tile is taken this way, 158 otherwise
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t s[32];
            tmem_ld32_nowait(s_addr + 32 * c, s);
            tmem_wait_ld(s);
            const int seen = r - 32 * c;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i > seen) s[i] = 0xff800000u;
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              top[(i >> 1) & 3] = max3_nan(top[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          }
          refer();
          uint32_t s[2][16];
          tmem_ld16_nowait(s_addr, s[0]);
#pragma unroll 1
          for (int c0 = 0; c0 < 8; c0 += 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = c0 + h, seen = r - 16 * c;
              tmem_wait_ld16(s[h]);
              if (c < 7) tmem_ld16_nowait(s_addr + 16 * (c + 1), s[h ^ 1]);
              uint32_t w[8];
#pragma unroll
              for (int i = 0; i < 8; ++i)
                w[i] = weight2(i, 2 * i > seen ? 0xff800000u : s[h][2 * i], 2 * i + 1 > seen ? 0xff800000u : s[h][2 * i + 1]);
              tmem_st8(s_addr + 8 * c, w);  // over scores that have been read: in front of the ones in flight
            }
          }
        }
        if (last) {
          // values of the last key tile that are not finite: out of the tile, into the record
          const uint32_t u = unit + 2 * j + 1, st = u % kStages;
          if (!(ok = __all_sync(0xffffffffu, wait(&ctl->kv_full[st], u / kStages, kErrFullWait)))) break;
          uint8_t* v = base + (2 + st) * kTileBytes;
          TakenOut<kHd>* rec = &ctl->taken[t];
          const uint32_t v_mine = smem_u32(v) + r * 16;
          uint32_t odd = 0;
#pragma unroll 4
          for (int i = 0; i < kTileBytes / 16 / 128; ++i) {
            const uint4 q = lds_u4(v_mine + i * 2048);
            odd |= not_finite2<T>(q.x) | not_finite2<T>(q.y) | not_finite2<T>(q.z) | not_finite2<T>(q.w);
          }
          const bool found = (odd & 0x80008000u) != 0;
          // the record may still be read for the item before: by a slower warp of this tile, and tile 0's by tile 1, whose last item may
          // lie further back
          if (found && (t || !done || wait(&ctl->taken_free[0], done - 1, kErrMmaWait)) &&
              (!done1 || wait(&ctl->taken_free[1], done1 - 1, kErrMmaWait))) {
#pragma unroll 1
            for (int i = 0; i < kTileBytes / 16 / 128; ++i) {
              const int at = (i * 128 + r) * 16, box = at / kBoxBytes, key = (at % kBoxBytes) / 128, chunk = ((at % 128) / 16) ^ (key & 7);
              T* e = reinterpret_cast<T*>(v + at);
              for (int k = 0; k < 8; ++k) {
                const float f = to_f32(e[k]);
                if (isfinite(f)) continue;
                atomicMin(&rec->row[f != f ? 2 : f < 0.f ? 1 : 0][box * 64 + chunk * 8 + k], taken_word(done, key));
                e[k] = from_f32<T>(0.f);
              }
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
        const int row0 = row - lane;  // of the warp
        uint8_t* dst = reinterpret_cast<uint8_t*>(reinterpret_cast<T*>(p.out) + ((it.first + row0) * p.n_heads + it.head) * kHd);
        const int64_t row_bytes = (int64_t)p.n_heads * kHd * sizeof(T);
        float most = 0.f;  // NaN if one of the row's sums is
#pragma unroll 1
        for (int i = 0; i < kHd / 32; ++i) {
          uint32_t o[32];
          tmem_ld32_nowait(o_addr + 32 * i, o);
          tmem_wait_ld(o);
#pragma unroll
          for (int e = 0; e < 32; e += 2) most = max3_nan(most, __uint_as_float(o[e]), __uint_as_float(o[e + 1]));
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
          uint4 v[4];
          uint32_t* w = reinterpret_cast<uint32_t*>(v);
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = cvt2<T>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
          store_rows64(smem_u32(stages) + warp * kStageBytes, lane, v, dst + 64 * i, row_bytes, it.len - row0);
        }
        const uint32_t odd = __ballot_sync(0xffffffffu, most != most && total == total && row < it.len);
        if (odd) {
          __syncwarp();  // the rows are written
          put_not_finite<T, kHd>(reinterpret_cast<const T*>(p.v) + it.first * p.v_stride + it.head / p.group * kHd, p.v_stride, row0,
                                 odd, reinterpret_cast<T*>(dst), (int64_t)p.n_heads * kHd, lane);
        }
        tc_fence_before();
        mbar_arrive(&ctl->taken_free[t]);
      }
      unit += 2 * n;
      ++done;
      done1 += n1 != 0;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

}  // namespace fq
