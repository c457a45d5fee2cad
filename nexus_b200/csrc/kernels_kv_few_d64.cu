// kernels_kv_few_d64.cu -- few-row attention over the paged cache, head_dim 64.
#include "kernels_kv_few.cuh"

namespace nx {
cudaError_t launch_kv_few_d64(const KvAttnParams &p, cudaStream_t st) { return kvf::launch_few_dim<64>(p, st); }
}  // namespace nx
