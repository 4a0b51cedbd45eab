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

// A block that gives up while copies are on their way: after land_copies every word of them is in shared memory.
constexpr int kRing = 3, kPieces = 512;  // of 16 bytes, a copy
__device__ uint4 g_source[kRing * kPieces];

__global__ void __launch_bounds__(256) land_kernel(int32_t* missing) {
  __shared__ uint64_t full[kRing];
  __shared__ uint4 staged[kRing * kPieces];
  const int tid = threadIdx.x, warp = warp_index();
  for (int x = tid; x < kRing * kPieces; x += 256) {
    g_source[x] = make_uint4(x + 1, ~x, 3 * x + 1, x + 7);
    staged[x] = make_uint4(0, 0, 0, 0);
  }
  if (tid == 0) {
    for (int s = 0; s < kRing; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
  }
  asm volatile("fence.proxy.async;" ::: "memory");  // the copies read and write after the stores above
  __syncthreads();
  if (warp == 0) {
    if (tid == 0)
      for (int s = 0; s < kRing; ++s) {
        const uint32_t bar = smem_u32(&full[s]);
        mbar_arrive_expect_tx(bar, kPieces * 16);
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                smem_u32(&staged[s * kPieces])),
            "l"(__cvta_generic_to_global(&g_source[s * kPieces])), "r"(kPieces * 16), "r"(bar)
            : "memory");
      }
    __syncwarp();
    land_copies<kRing>(full, kRing);
  }
  __syncthreads();
  for (int x = tid; x < kRing * kPieces; x += 256) {
    const uint4 v = staged[x];
    if (v.x != x + 1u || v.y != ~static_cast<uint32_t>(x) || v.z != 3u * x + 1 || v.w != x + 7u) atomicAdd(missing, 1);
  }
}

}  // namespace
}  // namespace dfs

extern "C" int dfs_selftest_wait(int which, int32_t* status, void* stream) {
  if (which < 0 || which > 1 || !status) return DFS_ERR_INVALID_ARGUMENT;
  const auto kernel = which == 0 ? dfs::wait_kernel : dfs::land_kernel;
  kernel<<<1, 256, 0, static_cast<cudaStream_t>(stream)>>>(status);
  return cudaGetLastError() == cudaSuccess ? DFS_OK : DFS_ERR_CUDA;
}
