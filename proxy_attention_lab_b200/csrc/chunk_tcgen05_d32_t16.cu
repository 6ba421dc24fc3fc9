// chunk_tcgen05_kernel for head_dim = 32, tokens_per_page = 16 (a translation unit per shape keeps the build parallel).
#include "chunk_tcgen05.cuh"

namespace pal {

int launch_chunk_d32_t16(const ChunkArgs& a, cudaStream_t stream) { return launch_chunk_shape<32, 16>(a, stream); }

}  // namespace pal
