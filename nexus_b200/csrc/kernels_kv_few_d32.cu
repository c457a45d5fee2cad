// kernels_kv_few_d32.cu -- few-row attention over the paged cache, head_dim 32.
#include "kernels_kv_few.cuh"

namespace nx {
cudaError_t launch_kv_few_d32(const KvAttnParams &p, cudaStream_t st) { return kvf::launch_few_dim<32>(p, st); }
}  // namespace nx
