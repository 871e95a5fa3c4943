// Attention of one new token per sequence over a paged cache (fuelq_paged_attn_decode).
//
//   out[h] = sum_j p_j V[j] / sum_j p_j,   p_j = exp2(c (q[h] . K[j]) - m),   c = scale log2(e)
//
// Bound by HBM: every key and value is read once, for all the heads that share it, and used for 2 x heads multiply-adds.
// Layout of the products: the KEYS are the 16-row operand of the warp-wide matrix instruction and up to eight query heads of
// one kv head are its 8 columns, so that grouped heads cost nothing more and no row is wasted on padding:
//   S^T [16 keys x 8 heads] = K [16 x hd] . Q^T,     O^T [hd x 8 heads] += V^T [hd x 16 keys] . P^T
// The 5th-generation instruction has no use here: its 128-row tile would hold 8 of 128 rows of work.
// Accuracy: 32-bit activations are split into parts that the cache's type holds exactly and multiplied part by part into one
// f32 sum: f16 caches take q and p as two f16 parts (22 bits; q scaled by a power of two into range), bf16 caches as three bf16
// parts (24 bits), f32 caches everything as two tf32 parts (22 bits). The instruction's f32 sums round towards zero, which shows
// over a long row, so they are kept short and joined by additions that round to nearest. 16-bit activations are their own single
// part; p is then rounded once to their type. f16 ends at 2^-24, and one key of e^12 times the others' weight is common: relative to
// the running maximum their weights had six bits left. So f16 weights are relative to the largest of their own tile's 16 or 32 keys,
// 2^14 for it, and second parts are 2^11 times too large, in a sum of their own: 22 bits for weights down to 2^-27 of the tile's
// largest, 11 in a single part down to 2^-28.
// Work: tiles of kTile keys of all (sequence, kv head) items, laid end to end and dealt out evenly (attn_plan.h), so that one
// long sequence, many short ones and any mixture fill the device alike. A warp owns 16 (head_dim 64: 32) keys of each
// tile and runs by itself: its own ring of cp.async copies that runs on across items, its own running maximum and sums; the
// block's four warps join their results in shared memory at the end of an item, a quarter of the columns each, pieces of an item
// in other blocks by paged_join_kernel in a fixed order.
// Measured: 100003 keys, 32/8 heads of 128, f32 activations over f16 71 to 79 us by card (5.2 to 5.8 TB/s), over bf16 75; 64 sequences
// up to 8192, bf16, 91 to 94 us (5.6 to 5.8 TB/s); 32 of 2000, f32 98 us; 256 up to 2047, 32/4 heads of 64, f16, 37 to 39 us (3.6 to
// 3.8 TB/s: two or three short items a block, whose beginnings and ends are latency; without places for them in the split 64 us);
// 64 of 2000, 32/2 heads of 128, bf16 36 us; 513 keys, 32 heads, f32, 15 us: one tile a block, its join and the second launch.
// Weights of 16-bit activations in two parts would leave only the result's own rounding (bf16 2.2e-3 -> 1.7e-3 of the result): 256
// sequences 36.8 -> 38.8 us, 64 of 2000 with 16 heads a kv head 36.2 -> 38.0.
#pragma once
#include <type_traits>

#include "attn.cuh"
#include "attn_plan.h"

namespace fq {

struct DecodeParams {
  const void *q, *k, *v;
  void* out;
  int64_t q_stride;
  const int *table, *lens;
  int n_seqs, n_heads, n_kv, group, chunks;  // group: heads of a kv head; chunks: pieces of a group, of up to 8 * kNT heads
  int page_shift, n_pages, max_pages;
  float scale;
  int4* meta;    // [blocks] the item whose first piece is this block's last: sequence or -1, head chunk, its tiles (first, count)
  float* slots;  // [2 * blocks] pieces
};
constexpr int kDecodeWarps = 4;
constexpr int kDecodeMaxBlocks = 320;  // two on each of a B200's 148 SMs, rounded up

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two tf32 parts of a float: the upper 10 mantissa bits, and what they leave (exact in f32) rounded to as many: half of the last
// place that the instruction reads is added, and it ignores the rest
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = x & 0xffffe000u;
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi)) + 0x1000u;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const T v[2] = {from_f32<T>(a), from_f32<T>(b)};
  return *reinterpret_cast<const uint32_t*>(v);
}
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
  a = to_f32(reinterpret_cast<const T*>(&w)[0]), b = to_f32(reinterpret_cast<const T*>(&w)[1]);
}

template <typename A, typename C, int kHd_, int kNT_>
struct DecodeCfg {
  static constexpr int kHd = kHd_, kNT = kNT_, kHeads = 8 * kNT;  // heads of an item
  static constexpr bool kF32 = sizeof(C) == 4, kWideAct = sizeof(A) == 4;
  static constexpr int kSub = kHd == 64 ? 2 : 1, kKeys = 16 * kSub;  // keys of a warp per tile
  static constexpr int kTile = kDecodeWarps * kKeys;
  static constexpr int kRow = kHd * (int)sizeof(C), kUnit = kKeys * kRow;  // bytes of a row; of a warp's keys (or values) of a tile
  static constexpr int kParts = !kWideAct ? 1 : kF32 ? 2 : sizeof(C) == 2 && std::is_same<C, __nv_bfloat16>::value ? 3 : 2;
  // weights meet the values times this: for f16's range, and elsewhere so that values at f32's ends can be summed
  static constexpr float kWeightTop = std::is_same<C, __half>::value ? 0x1p14f : 0x1p-24f;
  static constexpr int kKs = kF32 ? kHd / 8 : kHd / 16, kMt = kHd / 16;
  static constexpr int kQBytes = kNT * kParts * kKs * 256;             // q in the order of the instruction's operand
  // at the end of an item: a warp's statistics, and three quarters of its sums, for the other warps to join
  static constexpr int kStatBytes = 32 * kNT * 16, kQuarter = kMt / kDecodeWarps, kQuarterBytes = 32 * kNT * kQuarter * 16;
  static constexpr int kMergeBytes = kDecodeWarps * (kStatBytes + 3 * kQuarterBytes);
  static constexpr int kShared = kQBytes > kMergeBytes ? kQBytes : kMergeBytes;
  // two thread blocks an SM need 113 KB each at most; the widest form runs alone with a deeper ring
  static constexpr int kRing = kF32 ? (kNT == 2 ? 6 : 3) : (kNT == 2 ? 5 : 6);
  static constexpr int kPerSm = kF32 && kNT == 2 ? 1 : 2;
  static constexpr int kSmem = kDecodeWarps * kRing * kUnit + kShared + kHeads * 4 + kDecodeWarps * 8 * 4 + 64;
  static constexpr int kSlot = kHeads * (kHd + 2);  // floats of a piece: [heads][hd], then maxima, then sums
};

// A tile in the list
struct TilePos {
  int64_t x;                           // its place
  int seq, chunk, tile, tiles, keys;  // chunk: kv head and piece of its group; tiles, keys: of the sequence
};

template <typename Cfg>
__device__ __forceinline__ void next_tile(TilePos& t, const DecodeParams& p) {
  ++t.x;
  if (++t.tile < t.tiles) return;
  t.x += kItemUnits;
  t.tile = 0;
  if (++t.chunk < p.n_kv * p.chunks) return;
  t.chunk = 0;
  do {
    if (++t.seq >= p.n_seqs) {  // behind the last item: nobody's tile
      t.seq = p.n_seqs - 1;
      t.tiles = t.keys = 0;
      return;
    }
    t.keys = seq_keys(p.lens[t.seq], p.max_pages, p.page_shift);
    t.tiles = (t.keys + Cfg::kTile - 1) / Cfg::kTile;
  } while (t.tiles == 0);
}

template <typename A, typename C, int kHd, int kNT>
__global__ void __launch_bounds__(32 * kDecodeWarps) paged_decode_kernel(const DecodeParams p) {
  using Cfg = DecodeCfg<A, C, kHd, kNT>;
  constexpr int kKeys = Cfg::kKeys, kSub = Cfg::kSub, kRow = Cfg::kRow, kUnit = Cfg::kUnit, kRing = Cfg::kRing, kKs = Cfg::kKs,
                kMt = Cfg::kMt, kParts = Cfg::kParts, kHeads = Cfg::kHeads;
  constexpr bool kF32 = Cfg::kF32, kF16 = std::is_same<C, __half>::value;
  constexpr float kMost = 3.402823466e38f;
  constexpr float kWeightTop = Cfg::kWeightTop, kPartStep = 2048.f;
  extern __shared__ __align__(128) uint8_t dec_smem[];
  __shared__ int64_t start_s[3];
  __shared__ int64_t scan_s[kDecodeWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  uint8_t* ring = dec_smem + warp * kRing * kUnit;
  uint8_t* shared = dec_smem + kDecodeWarps * kRing * kUnit;  // q, and between items the warps' results
  float* factor_s = reinterpret_cast<float*>(shared + Cfg::kShared);
  uint32_t* seen_s = reinterpret_cast<uint32_t*>(factor_s + kHeads) + warp * 8;  // which keys of a warp's next tiles exist
  pdl_launch_dependents();
  pdl_wait();

  // ---- the run of this block: total number of tiles, where its first one lies
  const int items = p.n_kv * p.chunks;
  const int per = (p.n_seqs + 32 * kDecodeWarps - 1) / (32 * kDecodeWarps);
  const int s0 = min((int)threadIdx.x * per, p.n_seqs), s1 = min(s0 + per, p.n_seqs);
  const int64_t mine = seq_units(p.lens, s0, s1, p.max_pages, p.page_shift, Cfg::kTile);
  int64_t incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += o;
  }
  if (lane == 31) scan_s[warp] = incl;
  __syncthreads();
  int64_t total1 = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kDecodeWarps; ++w) {
    if (w < warp) before += scan_s[w];
    total1 += scan_s[w];
  }
  const int64_t total = total1 * items;
  const int blocks = total < (int64_t)gridDim.x ? (int)total : (int)gridDim.x;
  const bool active = (int)blockIdx.x < blocks;
  const int64_t x0 = active ? split_begin(total, blocks, blockIdx.x) : 0, x1 = active ? split_begin(total, blocks, blockIdx.x + 1) : 0;
  {
    int64_t at = (before + incl - mine) * items;  // first tile of this thread's sequences
    if (active && at <= x0 && x0 < at + mine * items) {
      int s = s0;
      for (;; ++s) {
        const int64_t n = (int64_t)item_units(seq_tiles(p.lens[s], p.max_pages, p.page_shift, Cfg::kTile)) * items;
        if (x0 < at + n) break;
        at += n;
      }
      start_s[0] = s, start_s[1] = at;
    }
  }
  // free slots of the batch: rows of zeros
  for (int s = blockIdx.x; s < p.n_seqs; s += gridDim.x) {
    const int len = p.lens[s];
    if (len > ((int64_t)p.max_pages << p.page_shift) && threadIdx.x == 0) record_dev_error(kErrIndex);
    if (seq_keys(len, p.max_pages, p.page_shift) == 0) {
      uint32_t* o = reinterpret_cast<uint32_t*>(reinterpret_cast<A*>(p.out) + (int64_t)s * p.n_heads * kHd);
      for (int i = threadIdx.x; i < p.n_heads * kHd * (int)sizeof(A) / 4; i += 32 * kDecodeWarps) o[i] = 0;
    }
  }
  __syncthreads();
  TilePos use;
  use.x = x1;
  if (active) {
    use.seq = (int)start_s[0];
    use.keys = seq_keys(p.lens[use.seq], p.max_pages, p.page_shift);
    use.tiles = (use.keys + Cfg::kTile - 1) / Cfg::kTile;
    const int64_t rest = x0 - start_s[1];
    use.chunk = (int)quotient(rest, item_units(use.tiles));
    use.tile = (int)(rest - (int64_t)use.chunk * item_units(use.tiles));
    use.x = x0;
    if (use.tile >= use.tiles) {  // the run begins with places behind an item
      use.x = x0 - use.tile + use.tiles - 1;
      use.tile = use.tiles - 1;
      next_tile<Cfg>(use, p);
    }
  }
  if (use.x >= x1) {
    if (threadIdx.x == 0) p.meta[2 * blockIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }
  TilePos get = use;

  // ---- copies. Lane r holds the place of key r of the tile to be fetched: its row in the cache, or -1
  const uint8_t* kc = reinterpret_cast<const uint8_t*>(p.k);
  const uint8_t* vc = reinterpret_cast<const uint8_t*>(p.v);
  constexpr int kLanesPerRow = kRow / 16, kRowsPerCopy = 32 / kLanesPerRow, kCopies = kKeys / kRowsPerCopy;
  uint32_t fetched = 0;   // tiles whose keys have been requested
  bool values_due = false;
  int64_t place = -1;     // of this lane's key, of the tile being fetched
  int next_page = -1;     // page of this lane's key in the tile after it, looked up ahead of its use
  auto look_up = [&](const TilePos& t) {
    const int key = t.tile * Cfg::kTile + warp * kKeys + (lane & (kKeys - 1));
    if (key >= t.keys) return -1;
    const int page = p.table[(int64_t)t.seq * p.max_pages + (key >> p.page_shift)];
    if (page < 0 || page >= p.n_pages) {
      record_dev_error(kErrIndex);
      return -1;
    }
    return page;
  };
  auto copy_unit = [&](const uint8_t* base, int slot, bool value) {
    const uint32_t dst = smem_u32(ring + slot * kUnit);
    const int c = lane % kLanesPerRow;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int r = i * kRowsPerCopy + lane / kLanesPerRow;
      const int64_t at = __shfl_sync(0xffffffffu, place, r);
      const int sw = kF32 && value ? c ^ ((r & 3) << 1) : c ^ (r & 7);
      cp_async16(dst + r * kRow + sw * 16, base + (at < 0 ? 0 : at * kRow + c * 16), at >= 0);
    }
    cp_async_commit();
  };
  auto fetch_keys = [&](int slot) {
    values_due = get.x < x1;
    if (values_due) {
      const int key = get.tile * Cfg::kTile + warp * kKeys + (lane & (kKeys - 1));
      place = next_page < 0 ? -1
                            : (((int64_t)next_page * p.n_kv + get.chunk / p.chunks) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
      const uint32_t seen = __ballot_sync(0xffffffffu, place >= 0);
      if (lane == 0) seen_s[fetched & 7] = seen;
      ++fetched;
      next_tile<Cfg>(get, p);
      next_page = get.x < x1 ? look_up(get) : -1;
      copy_unit(kc, slot, false);
    } else {
      cp_async_commit();
    }
  };
  auto fetch_values = [&](int slot) {  // of the tile whose keys were fetched last
    if (values_due) copy_unit(vc, slot, true);
    else cp_async_commit();
  };
  next_page = look_up(get);
  int in = 0, out_slot = 0;  // ring slots of the next unit to request, of the next to use
  bool keys_next = true;
  auto request = [&]() {
    if (keys_next) fetch_keys(in);
    else fetch_values(in);
    keys_next = !keys_next;
    in = in + 1 == kRing ? 0 : in + 1;
  };

  // ---- one item after the other
  float m[kNT][2], l[kNT][2], o[kNT][kMt][4];
  float factor[kNT][2];
  int nh = 0;
  int64_t item_first = use.x - use.tile;  // first place of the item in the list
  // the query heads of an item, two (or four) for each warp: read ahead, put into the order of the instruction's operand later
  constexpr int kPer = kHd / 32, kMine = kHeads / kDecodeWarps;
  float qx[kMine][kPer];
  auto load_q = [&]() {
    const int kvh = use.chunk / p.chunks, part = use.chunk - kvh * p.chunks;
    nh = min(kHeads, p.group - part * kHeads);
    const A* q = reinterpret_cast<const A*>(p.q) + use.seq * p.q_stride + (int64_t)(kvh * p.group + part * kHeads) * kHd + lane * kPer;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int h = warp + j * kDecodeWarps;
#pragma unroll
      for (int i = 0; i < kPer; ++i) qx[j][i] = h < nh ? to_f32(q[h * kHd + i]) : 0.f;
    }
  };
  auto begin_item = [&]() {
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int h = warp + j * kDecodeWarps;
      float(&x)[kPer] = qx[j];
      float f = p.scale * 1.4426950408889634f;
      if constexpr (Cfg::kWideAct && std::is_same<C, __half>::value) {  // a power of two that brings the row into f16's range
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) top = fmaxf(top, isinf(x[i]) ? 0.f : fabsf(x[i]));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const int e = min(max(top > 0.f ? ilogbf(top) : 0, -100), 127);
        const float up = exp2f((float)(13 - e));
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] *= up;
        f = fminf(f * exp2f((float)(e - 13)), kMost);  // at f32's end any score but 0 takes all or nothing
      }
      const int nt = h >> 3, n = h & 7;
#pragma unroll
      for (int i = 0; i < kPer; i += 2) {
        const int d = lane * kPer + i;
        uint32_t* w = reinterpret_cast<uint32_t*>(shared);
        if constexpr (kF32) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int dd = d + k, at = ((nt * kParts * kKs + dd / 8) * 32 + n * 4 + (dd & 3)) * 2 + ((dd >> 2) & 1);
            uint32_t hi, lo;
            split_tf32(__float_as_uint(x[i + k]), hi, lo);
            w[at] = hi;
            w[at + kKs * 64] = lo;
          }
        } else {
          const int at = ((nt * kParts * kKs + d / 16) * 32 + n * 4 + ((d & 7) >> 1)) * 2 + ((d >> 3) & 1);
          float a = x[i], b = x[i + 1];
#pragma unroll
          for (int part_i = 0; part_i < kParts; ++part_i) {
            const uint32_t u = pack2<C>(a, b);
            w[at + part_i * kKs * 64] = u;
            float ra, rb;
            unpack2<C>(u, ra, rb);
            a -= ra, b -= rb;
          }
        }
      }
      if (lane == 0) factor_s[h] = f;
    }
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) m[nt][j] = -INFINITY, l[nt][j] = 0.f;
#pragma unroll
      for (int t = 0; t < kMt; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][t][i] = 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) factor[nt][0] = factor_s[nt * 8 + 2 * tq], factor[nt][1] = factor_s[nt * 8 + 2 * tq + 1];
  };

  // The four warps' results joined, each warp a quarter of the columns; whole items are finished, pieces are left for
  // paged_join_kernel. done: the item ends here; last: so does this block's run
  auto end_item = [&](const TilePos& at, int heads, bool done, bool last) {
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], off);
    __syncthreads();  // nobody reads q any more
    constexpr int kQ = Cfg::kQuarter;
    float4* stats = reinterpret_cast<float4*>(shared) + lane;                                 // [warp][nt][lane]
    float4* box = reinterpret_cast<float4*>(shared + kDecodeWarps * Cfg::kStatBytes) + lane;  // [to][from][nt][tile of the quarter][lane]
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      stats[(warp * kNT + nt) * 32] = make_float4(m[nt][0], m[nt][1], l[nt][0], l[nt][1]);
#pragma unroll
      for (int t = 0; t < kMt; ++t) {
        const int to = t / kQ, from = warp - (warp > to ? 1 : 0);
        const float(&x)[4] = o[nt][t];
        if (to != warp) box[(((to * 3 + from) * kNT + nt) * kQ + t % kQ) * 32] = make_float4(x[0], x[1], x[2], x[3]);
      }
    }
    __syncthreads();
    const int kvh = at.chunk / p.chunks, part = at.chunk - kvh * p.chunks;
    const bool whole = done && item_first >= x0;
    float* slot = p.slots + (int64_t)split_slot(total, blocks, blockIdx.x, item_first) * Cfg::kSlot;
    A* dst = reinterpret_cast<A*>(p.out) + ((int64_t)at.seq * p.n_heads + kvh * p.group + part * kHeads) * kHd;
    // results that are not finite while the sum of their weights is: bit 4 (nt kQ + q) + i
    uint32_t odd = 0;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      float4 st[kDecodeWarps];
      float top[2] = {-INFINITY, -INFINITY}, f[kDecodeWarps][2], sum[2] = {0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kDecodeWarps; ++w) {
        st[w] = stats[(w * kNT + nt) * 32];
        top[0] = fmaxf(top[0], st[w].x), top[1] = fmaxf(top[1], st[w].y);
      }
      const float ref[2] = {top[0] == -INFINITY ? 0.f : top[0], top[1] == -INFINITY ? 0.f : top[1]};
#pragma unroll
      for (int w = 0; w < kDecodeWarps; ++w) {
        f[w][0] = exp2f(st[w].x - ref[0]), f[w][1] = exp2f(st[w].y - ref[1]);
        sum[0] += st[w].z * f[w][0], sum[1] += st[w].w * f[w][1];
      }
      const float inv[2] = {sum[0] == 0.f ? 0.f : 1.f / kWeightTop / sum[0], sum[1] == 0.f ? 0.f : 1.f / kWeightTop / sum[1]};
      const float own[2] = {exp2f(m[nt][0] - ref[0]), exp2f(m[nt][1] - ref[1])};
#pragma unroll
      for (int q = 0; q < kQ; ++q) {
        float r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float lower = warp & 1 ? o[nt][kQ + q][i] : o[nt][q][i], upper = warp & 1 ? o[nt][3 * kQ + q][i] : o[nt][2 * kQ + q][i];
          r[i] = (warp & 2 ? upper : lower) * own[i & 1];
        }
#pragma unroll
        for (int w = 0; w < kDecodeWarps; ++w) {
          if (w == warp) continue;
          const float4 b = box[(((warp * 3 + w - (w > warp ? 1 : 0)) * kNT + nt) * kQ + q) * 32];
          r[0] += b.x * f[w][0], r[1] += b.y * f[w][1], r[2] += b.z * f[w][0], r[3] += b.w * f[w][1];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int h = nt * 8 + 2 * tq + (i & 1), d = 16 * (warp * kQ + q) + g + 8 * (i >> 1);
          if (h < heads) {
            if (!isfinite(r[i]) && isfinite(sum[i & 1])) odd |= 1u << (4 * (nt * kQ + q) + i);
            if (whole) dst[h * kHd + d] = from_f32<A>(r[i] * inv[i & 1]);
            else slot[h * kHd + d] = r[i];
          }
        }
      }
      if (!whole && warp == 0 && g == 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int h = nt * 8 + 2 * tq + j;
          slot[kHeads * kHd + h] = top[j], slot[kHeads * (kHd + 1) + h] = sum[j];
        }
      }
    }
    if (__any_sync(0xffffffffu, odd != 0)) {
      // An infinite value is infinite in the result whatever its weight, but its product with a part of the weight that is negative or
      // zero is not. So what the piece's values hold that is not finite is summed up here, the lanes over the warp's columns, and takes
      // the place of such a result. (An infinity in the cache costs its batch time, finite values nothing. The whole warp takes this way
      // together, and nothing in it is a call)
      const int from = (int)max(x0 - item_first, (int64_t)0) * Cfg::kTile;
      const int to = (int)min((int64_t)(at.tile + 1) * Cfg::kTile, (int64_t)at.keys);
      const int* pages = p.table + (int64_t)at.seq * p.max_pages;
      const C* column = reinterpret_cast<const C*>(p.v) + ((int64_t)kvh * kHd << p.page_shift) + 16 * warp * kQ + lane % (16 * kQ);
      const int64_t page_stride = (int64_t)p.n_kv * kHd << p.page_shift;
      float found = 0.f;
#pragma unroll 8
      for (int key = from; key < to; ++key) {
        const int page = pages[key >> p.page_shift];
        const bool is = page >= 0 && page < p.n_pages;
        const float x = is ? to_f32(column[page * page_stride + (int64_t)(key & ((1 << p.page_shift) - 1)) * kHd]) : 0.f;
        found += isfinite(x) ? 0.f : x;
      }
#pragma unroll 1
      for (int b = 0; b < 4 * kNT * kQ; ++b) {
        const int i = b & 3, q = (b >> 2) % kQ, h = 8 * (b / (4 * kQ)) + 2 * tq + (i & 1), in_warp = 16 * q + g + 8 * (i >> 1);
        const float f = __shfl_sync(0xffffffffu, found, in_warp);
        if (((odd >> b) & 1) && f != 0.f) {
          if (whole) dst[h * kHd + 16 * warp * kQ + in_warp] = from_f32<A>(f);
          else slot[h * kHd + 16 * warp * kQ + in_warp] = f;
        }
      }
    }
    if (last && threadIdx.x == 0) {  // the end of this block's run: does an item go on from here that began here?
      const bool first_piece = !done && item_first >= x0;
      p.meta[2 * blockIdx.x] = make_int4(first_piece ? at.seq : -1, at.chunk, at.tiles, blocks);
      p.meta[2 * blockIdx.x + 1] =
          make_int4((int)(item_first & 0xffffffff), (int)(item_first >> 32), (int)(total & 0xffffffff), (int)(total >> 32));
    }
    __syncthreads();
  };

  load_q();
#pragma unroll 1
  for (int i = 0; i < kRing; ++i) request();
  begin_item();
  for (uint32_t i = 0;; ++i) {
    // scores
    cp_async_wait<kRing - 1>();
    __syncwarp();
    const uint32_t kbase = smem_u32(ring + out_slot * kUnit);
    float s[kSub][kNT][4];
#pragma unroll
    for (int sub = 0; sub < kSub; ++sub) {
      float acc[4][kNT][4] = {};  // the instruction's sums round towards zero: four short ones, low parts before high ones
      const int row = sub * 16 + (lane & 15);
#pragma unroll
      for (int ks = 0; ks < kKs; ++ks) {
        uint32_t a[4];
        ldsm4(kbase + row * kRow + (((ks * 2 + (lane >> 4)) ^ (row & 7)) * 16), a);
        if constexpr (kF32) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) split_tf32(a[j], hi[j], lo[j]);
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
            const uint2 qh = reinterpret_cast<const uint2*>(shared)[(nt * 2 * kKs + ks) * 32 + lane];
            const uint2 ql = reinterpret_cast<const uint2*>(shared)[((nt * 2 + 1) * kKs + ks) * 32 + lane];
            mma8_tf32(acc[ks & 3][nt], lo, ql.x, ql.y);
            mma8_tf32(acc[ks & 3][nt], lo, qh.x, qh.y);
            mma8_tf32(acc[ks & 3][nt], hi, ql.x, ql.y);
            mma8_tf32(acc[ks & 3][nt], hi, qh.x, qh.y);
          }
        } else {
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
            for (int part = kParts - 1; part >= 0; --part) {
              const uint2 b = reinterpret_cast<const uint2*>(shared)[((nt * kParts + part) * kKs + ks) * 32 + lane];
              mma16(acc[ks & 3][nt], a, b.x, b.y, C());
            }
        }
      }
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[sub][nt][j] = (acc[0][nt][j] + acc[1][nt][j]) + (acc[2][nt][j] + acc[3][nt][j]);
    }
    const uint32_t seen = seen_s[i & 7];
    __syncwarp();  // the slot and the word above are free
    request();
    out_slot = out_slot + 1 == kRing ? 0 : out_slot + 1;

    // weights: relative to the running maximum, which moves only when a score passes it by 2^8, so that it is looked for across lanes
    // rarely; f16 caches: to the largest score of the tile, for f16's range (`take` brings the tile's sums to the maximum)
    bool up = false, far = false;
    float x[kSub][kNT][4];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int sub = 0; sub < kSub; ++sub)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[sub][nt][j] = s[sub][nt][j] * factor[nt][j & 1];
          far |= fabsf(x[sub][nt][j]) > kMost;
        }
    if (__any_sync(0xffffffffu, far)) {
      // finite products stay finite when they are scaled. A product of -inf is a weight of zero, one of +inf makes the row NaN as inf - inf
      // does. (f32 caches: infinite factors have made NaN of it in their second parts, and an infinite product is one at f32's end)
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int sub = 0; sub < kSub; ++sub)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float& y = x[sub][nt][j];
            if (!(fabsf(y) > kMost)) continue;
            if (kF32 || fabsf(s[sub][nt][j]) <= kMost) y = copysignf(kMost, y);
            else if (y > 0.f) y = __int_as_float(0x7fc00000);
          }
    }
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int sub = 0; sub < kSub; ++sub)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (!((seen >> (sub * 16 + g + 8 * (j >> 1))) & 1)) x[sub][nt][j] = -INFINITY;
          s[sub][nt][j] = x[sub][nt][j];
          up |= x[sub][nt][j] > m[nt][j & 1] + 8.f;
        }
    float top[kNT][2], take[kNT][2];
    auto find_top = [&]() {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[nt][j] = -INFINITY;
#pragma unroll
          for (int sub = 0; sub < kSub; ++sub) top[nt][j] = fmaxf(top[nt][j], fmaxf(s[sub][nt][j], s[sub][nt][j + 2]));
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) top[nt][j] = fmaxf(top[nt][j], __shfl_xor_sync(0xffffffffu, top[nt][j], off));
        }
    };
    if constexpr (kF16) find_top();
    if (__any_sync(0xffffffffu, up)) {
      if constexpr (!kF16) find_top();
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bool move = top[nt][j] > m[nt][j] + 8.f;  // by this head's scores alone: its bits do not depend on the others'
          const float keep = move ? exp2f(m[nt][j] - top[nt][j]) : 1.f;
          if (move) m[nt][j] = top[nt][j];
          l[nt][j] *= keep;
#pragma unroll
          for (int t = 0; t < kMt; ++t) o[nt][t][j] *= keep, o[nt][t][j + 2] *= keep;
        }
    }
    uint32_t pf[kSub][kNT][kParts][kF32 ? 4 : 2];  // p as the second operand of the products with V
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      float ref[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float to = kF16 ? top[nt][j] : m[nt][j];
        ref[j] = to == -INFINITY ? 0.f : to;
        take[nt][j] = !kF16 ? 1.f : to == -INFINITY ? 0.f : exp2f(to - m[nt][j]);
      }
#pragma unroll
      for (int sub = 0; sub < kSub; ++sub) {
        float e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          e[j] = exp2_approx(s[sub][nt][j] - ref[j & 1]);
          if constexpr (kF16) l[nt][j & 1] = fmaf(e[j], take[nt][j & 1], l[nt][j & 1]);
          else l[nt][j & 1] += e[j];
          e[j] *= kWeightTop;
        }
        if constexpr (kF32) {
          // this lane wants keys tq, tq + 4, tq + 8, tq + 12 of head g; lane 4 * key + g / 2 has them for keys below 8 in e[g & 1]
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int src = 4 * (tq + 4 * (j & 1)) + (g >> 1);
            const float a = __shfl_sync(0xffffffffu, e[2 * (j >> 1)], src), b = __shfl_sync(0xffffffffu, e[2 * (j >> 1) + 1], src);
            split_tf32(__float_as_uint(g & 1 ? b : a), pf[sub][nt][0][j], pf[sub][nt][1][j]);
          }
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float a = e[2 * half], b = e[2 * half + 1];
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              const uint32_t u = pack2<C>(a, b);
              float ra, rb;
              unpack2<C>(u, ra, rb);
              a -= ra, b -= rb;
              if constexpr (kF16) a *= kPartStep, b *= kPartStep;
              pf[sub][nt][part][half] = transpose8(u);
            }
          }
        }
      }
    }

    // weighted values
    cp_async_wait<kRing - 1>();
    __syncwarp();
    uint8_t* vunit = ring + out_slot * kUnit;
    const uint32_t vbase = smem_u32(vunit);
    // a tile's products by themselves, then added to O with a sum that rounds to nearest
#pragma unroll
    for (int t = 0; t < kMt; ++t) {
      float tile[kNT][4] = {}, low[kNT][4] = {};  // low: the second parts of f16 weights, kPartStep times too large
#pragma unroll
      for (int sub = 0; sub < kSub; ++sub) {
        if constexpr (kF32) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {  // keys 8 * half ..
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int key = sub * 16 + 8 * half + tq + 4 * (j >> 1), d = 16 * t + g + 8 * (j & 1);
              const uint8_t* at = vunit + key * kRow + (((d >> 2) ^ ((key & 3) << 1)) * 16) + (d & 3) * 4;
              const uint32_t x = *reinterpret_cast<const uint32_t*>(at);
              split_tf32(x, hi[j], lo[j]);
            }
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) {
              mma8_tf32(tile[nt], lo, pf[sub][nt][1][2 * half], pf[sub][nt][1][2 * half + 1]);
              mma8_tf32(tile[nt], lo, pf[sub][nt][0][2 * half], pf[sub][nt][0][2 * half + 1]);
              mma8_tf32(tile[nt], hi, pf[sub][nt][1][2 * half], pf[sub][nt][1][2 * half + 1]);
              mma8_tf32(tile[nt], hi, pf[sub][nt][0][2 * half], pf[sub][nt][0][2 * half + 1]);
            }
          }
        } else {
          const int row = sub * 16 + (lane & 7) + ((lane >> 4) & 1) * 8;
          uint32_t a[4];
          ldsm4_t(vbase + row * kRow + (((t * 2 + ((lane >> 3) & 1)) ^ (row & 7)) * 16), a);
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
            for (int part = kParts - 1; part >= 0; --part)
              mma16(kF16 && part ? low[nt] : tile[nt], a, pf[sub][nt][part][0], pf[sub][nt][part][1], C());
        }
      }
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (kF16) {
            const float all = kParts > 1 ? fmaf(low[nt][i], 1.f / kPartStep, tile[nt][i]) : tile[nt][i];
            o[nt][t][i] = fmaf(all, take[nt][i & 1], o[nt][t][i]);
          } else {
            o[nt][t][i] += tile[nt][i];
          }
        }
    }
    __syncwarp();
    request();
    out_slot = out_slot + 1 == kRing ? 0 : out_slot + 1;

    // the end of the item, or of this block's run
    const bool done = use.tile + 1 == use.tiles;
    const TilePos at = use;
    next_tile<Cfg>(use, p);
    if (done || use.x >= x1) {
      const bool last = use.x >= x1;
      const int heads = nh;
      if (!last) load_q();
      end_item(at, heads, done, last);
      if (last) break;
      item_first = use.x;
      begin_item();
    }
  }
  cp_async_wait<0>();
}

// The pieces of an item that lies in several blocks' runs, in the order of the blocks. One block per (run, head of the item): it
// looks whether an item goes on from its run that began there.
template <typename A, typename C, int kHd, int kNT>
__global__ void __launch_bounds__(kHd) paged_join_kernel(const DecodeParams p) {
  using Cfg = DecodeCfg<A, C, kHd, kNT>;
  __shared__ float weight_s[kDecodeMaxBlocks];
  __shared__ float red_s[2][kHd / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int4 a = p.meta[2 * blockIdx.x];
  if (a.x < 0) return;
  const int part = a.y % p.chunks, h = blockIdx.y;
  if (h >= min(Cfg::kHeads, p.group - part * Cfg::kHeads)) return;
  const int4 b = p.meta[2 * blockIdx.x + 1];
  const int64_t first = (int64_t)(((uint64_t)(uint32_t)b.y << 32) | (uint32_t)b.x);
  const int64_t total = (int64_t)(((uint64_t)(uint32_t)b.w << 32) | (uint32_t)b.z);
  const int blocks = a.w, b0 = blockIdx.x, n = split_block(total, blocks, first + a.z - 1) - b0 + 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // pieces behind the first begin with their blocks' runs: slot 2 b
  const float* first_slot = p.slots + (int64_t)split_slot(total, blocks, b0, first) * Cfg::kSlot;
  auto slot = [&](int i) { return i == 0 ? first_slot : p.slots + (int64_t)(2 * (b0 + i)) * Cfg::kSlot; };
  float top = -INFINITY;
  for (int i = threadIdx.x; i < n; i += kHd) top = fmaxf(top, slot(i)[Cfg::kHeads * kHd + h]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (lane == 0) red_s[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kHd / 32; ++w) top = fmaxf(top, red_s[0][w]);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int i = threadIdx.x; i < n; i += kHd) {
    const float w = exp2f(slot(i)[Cfg::kHeads * kHd + h] - ref);
    weight_s[i] = w;
    sum += w * slot(i)[Cfg::kHeads * (kHd + 1) + h];
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane == 0) red_s[1][warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kHd / 32; ++w) sum += red_s[1][w];
  float acc = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float x = slot(i)[h * kHd + threadIdx.x];
    acc += isinf(x) ? x : weight_s[i] * x;  // infinite also where the piece's weight has come to nothing
  }
  const int kvh = a.y / p.chunks;
  reinterpret_cast<A*>(p.out)[((int64_t)a.x * p.n_heads + kvh * p.group + part * Cfg::kHeads + h) * kHd + threadIdx.x] =
      from_f32<A>(sum == 0.f ? 0.f : acc * (1.f / Cfg::kWeightTop / sum));
}

}  // namespace fq
