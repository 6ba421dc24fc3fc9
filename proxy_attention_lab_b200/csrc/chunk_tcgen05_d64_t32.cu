// chunk_tcgen05_kernel for head_dim = 64, tokens_per_page = 32 (a translation unit per shape keeps the build parallel).
#include "chunk_tcgen05.cuh"

namespace pal {

int launch_chunk_d64_t32(const ChunkArgs& a, cudaStream_t stream) { return launch_chunk_shape<64, 32>(a, stream); }

}  // namespace pal
