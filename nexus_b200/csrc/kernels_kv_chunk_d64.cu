// kernels_kv_chunk_d64.cu -- chunk attention over the paged cache, head_dim 64.
#include "kernels_kv_chunk.cuh"

namespace nx {
cudaError_t launch_kv_chunk_d64(const KvAttnParams &p, cudaStream_t st) { return kvc::launch_chunk_dim<64>(p, st); }
}  // namespace nx
