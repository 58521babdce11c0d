// Decode attention against the paged cache on the tensor cores (paged_decode.cu), called by the dispatch in decode.cu.
#pragma once
#include "scores.cuh"

namespace tk {

struct PagedDecode {
  const void *q, *kc, *vc;        // [B, hq, D], [blocks, block_size, hkv, D] bf16
  const int *tables, *seq_lens;   // [B, max_blocks], [B]
  void* out;                      // [B, hq, D]
  const void* sinks;              // [hq] (nullptr: none)
  OutGate gate;
  int hq, hkv, G, block_size, max_blocks, window, chunk;
  float scale_log2;
};

// What a decode over shared prefixes found there (paged_shared.cu), to be joined with a sequence's own pages.
struct PagedJoin {
  const int* rows;                // [B][4]: tokens of the prefix, first slot, slots, row of the sequence's first head in them
  const float* part;              // [slots, hkv, 128, D] unscaled outputs
  const float2* stat;             // [slots, hkv, 128] maximum (log2 units), sum
  int slots, num_blocks;
  int* err;
};

// False when the shape is not one of this kernel's.
bool paged_decode_mma(const PagedDecode& p, int B, int d, int e, cudaStream_t stream);
// The sequence's own pages and the join: any group of query heads, rows of 64 or 128.  Starts beside the kernel before it on the stream and waits for its results.
void paged_decode_join(const PagedDecode& p, const PagedJoin& join, int B, int d, cudaStream_t stream);

}  // namespace tk
