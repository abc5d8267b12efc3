// The launches of chunk_launch.h for one type of the cache (CVSA_CHUNK_F8).
#include "chunk_launch.h"

namespace cvsa {

template <int D, bool F8>
void launch_chunk_prefill(const ChunkArgs &a, const ChunkClass &c, unsigned grid, hipStream_t s) {
  if constexpr (D == 64 || D == 128) {
    if (c.tile_rows == 256)
      hipLaunchKernelGGL((chunk_prefill_kernel<D, 8, F8>), dim3(grid), dim3(512), 0, s, a, c);
  }
  if constexpr (D != 128) {
    if (c.tile_rows == 128)
      hipLaunchKernelGGL((chunk_prefill_kernel<D, 4, F8>), dim3(grid), dim3(256), 0, s, a, c);
  }
}

template <int D, bool F8>
void launch_chunk_stream(const ChunkArgs &a, const ChunkClass &c, hipStream_t s) {
  const unsigned wgs = (unsigned)(c.splits * a.H_kv);
  const dim3 block(chunk_stream_waves<D, F8>() * 64);
  if constexpr (F8) {
    hipLaunchKernelGGL((chunk_stream_kernel<D, 1, F8>), dim3(wgs, c.tile_rows / 32), block, 0, s,
                       a, c);
  } else {
    if constexpr (chunk_few_rows<D>() > 32) {
      if (c.tile_rows > 32)
        hipLaunchKernelGGL((chunk_stream_kernel<D, 2, F8>), dim3(wgs), block, 0, s, a, c);
    }
    if (c.tile_rows <= 32)
      hipLaunchKernelGGL((chunk_stream_kernel<D, 1, F8>), dim3(wgs), block, 0, s, a, c);
  }
}

#define CVSA_CHUNK_LAUNCHES(D)                                                             \
  template void launch_chunk_prefill<D, CVSA_CHUNK_F8>(const ChunkArgs &, const ChunkClass &, \
                                                       unsigned, hipStream_t);             \
  template void launch_chunk_stream<D, CVSA_CHUNK_F8>(const ChunkArgs &, const ChunkClass &,  \
                                                      hipStream_t);
CVSA_CHUNK_LAUNCHES(32)
CVSA_CHUNK_LAUNCHES(64)
CVSA_CHUNK_LAUNCHES(128)
CVSA_CHUNK_LAUNCHES(256)

}  // namespace cvsa
