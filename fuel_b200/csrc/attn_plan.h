// How the attention kernels deal their work out: index arithmetic alone, the same on the host, so that it can be tested there.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define FQ_HD __host__ __device__ __forceinline__
#else
#define FQ_HD inline
#endif

namespace fq {

// ---- decode. The keys of a sequence are cut into tiles, a unit of work ("item") is one sequence and one kv head, and the
// tiles of all items, laid end to end, are dealt out in equal runs to the thread blocks: block b has tiles
// [split_begin(b), split_begin(b + 1)). An item that lies in several runs is joined from its pieces.
FQ_HD int64_t split_begin(int64_t total, int blocks, int b) { return total * b / blocks; }
// the block whose run holds `tile`: the largest b with split_begin(b) <= tile
FQ_HD int split_block(int64_t total, int blocks, int64_t tile) { return (int)(((tile + 1) * blocks - 1) / total); }
// where block b leaves its piece of an item that begins at tile `first`: its first slot if the piece begins with its run
FQ_HD int split_slot(int64_t total, int blocks, int b, int64_t first) { return 2 * b + (split_begin(total, blocks, b) < first ? 1 : 0); }
// tiles of a sequence: lengths below zero count as zero, lengths behind the end of its page table row as that end
FQ_HD int seq_keys(int len, int max_pages, int page_shift) {
  const int64_t room = (int64_t)max_pages << page_shift;
  return len < 0 ? 0 : len > room ? (int)room : len;
}
FQ_HD int seq_tiles(int len, int max_pages, int page_shift, int tile) { return (int)(((int64_t)seq_keys(len, max_pages, page_shift) + tile - 1) / tile); }

}  // namespace fq
