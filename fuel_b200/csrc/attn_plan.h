// How the attention kernels deal their work out: index arithmetic alone, the same on the host, so that it can be tested there.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define FQ_HD __host__ __device__ __forceinline__
#else
#define FQ_HD inline
#endif

namespace fq {

// ---- decode. The keys of a sequence are cut into tiles, a unit of work ("item") is one sequence and one kv head. The tiles of
// all items, laid end to end with kItemUnits places behind each item for what an item costs besides its tiles, are dealt out in
// equal runs to the thread blocks: block b has places [split_begin(b), split_begin(b + 1)). An item whose tiles lie in several
// runs is joined from its pieces.
constexpr int kItemUnits = 2;
// quotients of numbers that hardly ever pass 32 bits, where the long division is a hundred instructions
FQ_HD int64_t quotient(int64_t a, int64_t b) { return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b; }
FQ_HD int64_t split_begin(int64_t total, int blocks, int b) { return quotient(total * b, blocks); }
// the block whose run holds place x: the largest b with split_begin(b) <= x
FQ_HD int split_block(int64_t total, int blocks, int64_t x) { return (int)quotient((x + 1) * blocks - 1, total); }
// where block b leaves its piece of an item that begins at place `first`: its first slot if the piece begins with its run
FQ_HD int split_slot(int64_t total, int blocks, int b, int64_t first) { return 2 * b + (split_begin(total, blocks, b) < first ? 1 : 0); }
// tiles of a sequence: lengths below zero count as zero, lengths behind the end of its page table row as that end
FQ_HD int seq_keys(int len, int max_pages, int page_shift) {
  const int64_t room = (int64_t)max_pages << page_shift;
  return len < 0 ? 0 : len > room ? (int)room : len;
}
FQ_HD int seq_tiles(int len, int max_pages, int page_shift, int tile) {
  return (int)(((int64_t)seq_keys(len, max_pages, page_shift) + tile - 1) / tile);
}

FQ_HD int item_units(int tiles) { return tiles ? tiles + kItemUnits : 0; }
// places of one kv head of sequences [from, to): more than 32 bits count where long sequences share their pages
FQ_HD int64_t seq_units(const int* lens, int from, int to, int max_pages, int page_shift, int tile) {
  int64_t sum = 0;
  for (int s = from; s < to; ++s) sum += item_units(seq_tiles(lens[s], max_pages, page_shift, tile));
  return sum;
}

// ---- prompts. An item is a block of `rows` rows of one sequence and one query head. Sequence s has the block numbers ("slots")
// from prompt_slot(cu[s], s) up to the next sequence's: at least as many as it has blocks, without any sum over the
// sequences before it; the few that are left over are empty.
FQ_HD int64_t prompt_slot(int64_t first_row, int seq, int rows) { return (first_row < 0 ? 0 : first_row / rows) + seq; }
FQ_HD int64_t prompt_slots(int64_t n_rows, int n_seqs, int rows) { return n_rows / rows + n_seqs; }
struct PromptBlock {
  int64_t first;  // first row of the sequence
  int len;        // its rows; -1: its boundaries are none
  int row;        // first row of the block within the sequence; >= len: empty
};
// The block of a slot that is one of sequence s. The blocks of a sequence come in descending order, the longest first.
FQ_HD PromptBlock prompt_block_of(const int* cu, int s, int64_t n_rows, int64_t slot, int rows) {
  PromptBlock b;
  b.first = cu[s];
  const int64_t end = cu[s + 1];
  if (b.first < 0 || end < b.first || end > n_rows) {
    b.len = -1, b.row = 0;
    return b;
  }
  b.len = (int)(end - b.first);
  const int64_t back = prompt_slot(end, s + 1, rows) - 1 - slot;  // 0 for the last slot of the sequence
  const int64_t row = back * rows;
  b.row = back < 0 || row >= b.len ? b.len : (int)row;
  return b;
}
// The same, the sequence (the last whose slots begin at or before this one) looked for
FQ_HD PromptBlock prompt_block(const int* cu, int n_seqs, int64_t n_rows, int64_t slot, int rows) {
  int lo = 0, hi = n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prompt_slot(cu[mid], mid, rows) <= slot) lo = mid; else hi = mid;
  }
  return prompt_block_of(cu, lo, n_rows, slot, rows);
}

}  // namespace fq
