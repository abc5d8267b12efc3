// Launches of the chunk attention's kernels, without the join.  Those of each type of
// the cache are compiled by themselves (chunk_kernels_bf16.hip, chunk_kernels_f8.hip).
#pragma once
#include "chunk_prefill.h"
#include "chunk_stream.h"

namespace cvsa {

// Rows of a sequence and KV head that the stream kernel takes at most: two
// tiles of a wave (one at D = 256, whose two tiles' outputs alone would fill a
// wave's registers).
template <int D>
constexpr int chunk_few_rows() {
  return D == 256 ? 32 : 64;
}

template <int D, bool F8>
void launch_chunk_prefill(const ChunkArgs &a, const ChunkClass &c, unsigned grid, hipStream_t s);
template <int D, bool F8>
void launch_chunk_stream(const ChunkArgs &a, const ChunkClass &c, hipStream_t s);

}  // namespace cvsa
