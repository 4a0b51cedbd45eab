// dfs_attn_selftest.cu -- what the attention kernels do when a wait of theirs runs out, which no call of the operators
// can bring about: the same device functions in a block of their own.
#include "dfs_attn_tc.cuh"

namespace dfs {
namespace {

__global__ void __launch_bounds__(256) wait_kernel(int32_t* status) {
  __shared__ uint64_t bar;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (!tc_wait(&bar, 0)) report_timeout(status);
}

}  // namespace
}  // namespace dfs

extern "C" int dfs_selftest_wait(int which, int32_t* status, void* stream) {
  if (which != 0 || !status) return DFS_ERR_INVALID_ARGUMENT;
  dfs::wait_kernel<<<1, 256, 0, static_cast<cudaStream_t>(stream)>>>(status);
  return cudaGetLastError() == cudaSuccess ? DFS_OK : DFS_ERR_CUDA;
}
