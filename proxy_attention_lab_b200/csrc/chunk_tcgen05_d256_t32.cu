// chunk_tcgen05_kernel for head_dim = 256, tokens_per_page = 32 (a translation unit per shape keeps the build parallel).
#include "chunk_tcgen05.cuh"

namespace pal {

int launch_chunk_d256_t32(const ChunkArgs& a, cudaStream_t stream) { return launch_chunk_shape<256, 32>(a, stream); }

}  // namespace pal
