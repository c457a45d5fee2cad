// kernels_kv_chunk_d128.cu -- chunk attention over the paged cache, head_dim 128.
#include "kernels_kv_chunk.cuh"

namespace nx {
cudaError_t launch_kv_chunk_d128(const KvAttnParams &p, cudaStream_t st) { return kvc::launch_chunk_dim<128>(p, st); }
}  // namespace nx
