// dfs_relbias.cu -- learned relative position bias by buckets: the dense bias,
// its gradient, and the sums by bucket that the fused attention backward ends with.
//
//   bias[h, i, j] = w[h, b(i + q_start - j)],  dw[h, c] = sum over b(delta) = c of
//   the diagonal delta of dbias[h].
#include <climits>

#include "dfs_attn.cuh"

namespace dfs {

// Sums by bucket of `parts` rows of sums by distance, in a fixed order: thread
// columns walk the distances, thread rows the parts; the rows are added in
// order, then a warp per bucket adds that bucket's distances.
template <typename T>
__global__ void __launch_bounds__(kBucketThreads) bucket_sums_kernel(const float* part, int parts, int D,
                                                                     const int32_t* lut, int nb, T* out) {
  extern __shared__ float sm[];
  const int W = 2 * D + 1, h = blockIdx.x, tid = threadIdx.x;
  float* acc = sm;                                   // W
  float* rows = sm + W;                              // kBucketThreads
  const float* src = part + static_cast<size_t>(h) * parts * W;
  constexpr int kCols = 64, kRows = kBucketThreads / kCols;
  const int cx = tid % kCols, ry = tid / kCols;
  for (int x0 = 0; x0 < W; x0 += kCols) {
    const int x = x0 + cx;
    float s = 0.0f;
    if (x < W)
      for (int r = ry; r < parts; r += kRows) s += src[static_cast<size_t>(r) * W + x];
    rows[ry * kCols + cx] = s;
    __syncthreads();
    if (ry == 0 && x < W) {
      float t = 0.0f;
#pragma unroll
      for (int r = 0; r < kRows; ++r) t += rows[r * kCols + cx];
      acc[x] = t;
    }
    __syncthreads();
  }
  for (int b = tid / 32; b < nb; b += kBucketThreads / 32) {
    float s = 0.0f;
    for (int x = tid & 31; x < W; x += 32) s += lut[x] == b ? acc[x] : 0.0f;
    s = warp_sum(s);
    if ((tid & 31) == 0) out[static_cast<size_t>(h) * nb + b] = from_f32<T>(s);
  }
}

cudaError_t launch_bucket_sums(const float* part, int H, int parts, int D, const int32_t* lut, int nb, int dtype,
                               void* out, cudaStream_t st) {
  const size_t sm = (2 * D + 1 + kBucketThreads) * sizeof(float);
  if (dtype == DFS_F32)
    bucket_sums_kernel<float><<<H, kBucketThreads, sm, st>>>(part, parts, D, lut, nb, static_cast<float*>(out));
  else if (dtype == DFS_BF16)
    bucket_sums_kernel<__nv_bfloat16><<<H, kBucketThreads, sm, st>>>(part, parts, D, lut, nb,
                                                                    static_cast<__nv_bfloat16*>(out));
  else
    bucket_sums_kernel<__half><<<H, kBucketThreads, sm, st>>>(part, parts, D, lut, nb, static_cast<__half*>(out));
  return cudaGetLastError();
}

namespace {

constexpr int kRowsPerTile = 32;  // rows of one CTA's tile
constexpr int kThreads = 256;

struct RelParams {
  const void* w;
  const int32_t* lut;
  int nb, D, H, nq, nk, qs;
};

template <typename T>
DFS_DEV T load_t(const void* p, size_t i) { return static_cast<const T*>(p)[i]; }

// One CTA writes kRowsPerTile rows of one head, a thread per column in turn.
template <typename T>
__global__ void __launch_bounds__(kThreads) relbias_fwd_kernel(RelParams P, T* out) {
  extern __shared__ unsigned char raw[];
  T* tab = reinterpret_cast<T*>(raw);
  const int h = blockIdx.y;
  for (int x = threadIdx.x; x < 2 * P.D + 1; x += kThreads)
    tab[x] = load_t<T>(P.w, static_cast<size_t>(h) * P.nb + min(max(P.lut[x], 0), P.nb - 1));
  __syncthreads();
  const int i1 = min(P.nq, static_cast<int>(blockIdx.x + 1) * kRowsPerTile);
  for (int i = blockIdx.x * kRowsPerTile; i < i1; ++i) {
    T* row = out + (static_cast<size_t>(h) * P.nq + i) * P.nk;
    for (int j = threadIdx.x; j < P.nk; j += kThreads) row[j] = tab[min(max(i + P.qs - j, -P.D), P.D) + P.D];
  }
}

// One CTA sums by distance over kRowsPerTile rows of one head.  A thread owns
// one diagonal at a time (fixed order, no atomics); the diagonals beyond the
// table are summed per thread and joined at the end.
template <typename T>
__global__ void __launch_bounds__(kThreads) relbias_bwd_kernel(RelParams P, const T* dB, float* part) {
  extern __shared__ float acc[];
  __shared__ float ends[2][kThreads / 32];
  const int h = blockIdx.y, D = P.D, W = 2 * D + 1, tid = threadIdx.x;
  for (int x = tid; x < W; x += kThreads) acc[x] = 0.0f;
  __syncthreads();
  const int i0 = blockIdx.x * kRowsPerTile, i1 = min(P.nq, i0 + kRowsPerTile);
  const T* base = dB + static_cast<size_t>(h) * P.nq * P.nk;
  float lo = 0.0f, hi = 0.0f;
  // diagonals e = i - j, from i0 - (nk - 1) to i1 - 1
  for (int e = i0 - (P.nk - 1) + tid; e < i1; e += kThreads) {
    float s = 0.0f;
    for (int i = i0; i < i1; ++i) {
      const int j = i - e;
      if (j >= 0 && j < P.nk) s += to_f32<T>(base[static_cast<size_t>(i) * P.nk + j]);
    }
    const int delta = e + P.qs;
    if (delta <= -D) lo += s;
    else if (delta >= D) hi += s;
    else acc[delta + D] = s;
  }
  if (D == 0) hi += lo, lo = 0.0f;  // one entry stands for every distance
  lo = warp_sum(lo);
  hi = warp_sum(hi);
  if ((tid & 31) == 0) ends[0][tid / 32] = lo, ends[1][tid / 32] = hi;
  __syncthreads();
  if (tid < 2) {
    float s = 0.0f;
    for (int w = 0; w < kThreads / 32; ++w) s += ends[tid][w];
    if (D > 0 || tid == 1) acc[tid == 0 ? 0 : 2 * D] = s;
  }
  __syncthreads();
  float* dst = part + (static_cast<size_t>(h) * gridDim.x + blockIdx.x) * W;
  for (int x = tid; x < W; x += kThreads) dst[x] = acc[x];
}

int row_tiles(int nq) { return (nq + kRowsPerTile - 1) / kRowsPerTile; }

bool bias_ok(const dfs_relbias* b) {
  return b && b->lut && b->num_buckets > 0 && b->max_distance >= 0 && b->max_distance <= DFS_MAX_BUCKET_DISTANCE &&
         (b->dtype == DFS_BF16 || b->dtype == DFS_F16 || b->dtype == DFS_F32);
}
// positions and distances stay inside 32 bits
bool sizes_ok(int H, int nq, int nk, int qs) {
  return H >= 0 && nq >= 0 && nk >= 0 && nq <= (1 << 28) && nk <= (1 << 28) && qs >= -(1 << 28) && qs <= (1 << 28);
}

}  // namespace
}  // namespace dfs

using namespace dfs;

extern "C" int dfs_relbias_fwd(int H, int n_q, int n_k, int q_start, const dfs_relbias* b, void* out, void* stream) {
  if (!bias_ok(b) || !sizes_ok(H, n_q, n_k, q_start)) return DFS_ERR_INVALID_ARGUMENT;
  if (H == 0 || n_q == 0 || n_k == 0) return DFS_OK;
  if (!b->weight || !out) return DFS_ERR_INVALID_ARGUMENT;
  if (H > 65535) return DFS_ERR_UNSUPPORTED;
  const RelParams P{b->weight, b->lut, b->num_buckets, b->max_distance, H, n_q, n_k, q_start};
  const dim3 grid(row_tiles(n_q), H);
  const size_t sm = (2 * P.D + 1) * (b->dtype == DFS_F32 ? 4 : 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (b->dtype == DFS_F32)
    relbias_fwd_kernel<float><<<grid, kThreads, sm, st>>>(P, static_cast<float*>(out));
  else if (b->dtype == DFS_BF16)
    relbias_fwd_kernel<__nv_bfloat16><<<grid, kThreads, sm, st>>>(P, static_cast<__nv_bfloat16*>(out));
  else
    relbias_fwd_kernel<__half><<<grid, kThreads, sm, st>>>(P, static_cast<__half*>(out));
  return cudaGetLastError() == cudaSuccess ? DFS_OK : DFS_ERR_CUDA;
}

extern "C" size_t dfs_relbias_bwd_work(int H, int n_q, int n_k, const dfs_relbias* b) {
  if (!bias_ok(b) || !sizes_ok(H, n_q, n_k, 0)) return 0;
  return static_cast<size_t>(H) * row_tiles(n_q) * (2 * b->max_distance + 1) * sizeof(float);
}

extern "C" int dfs_relbias_bwd(int H, int n_q, int n_k, int q_start, const dfs_relbias* b, const void* d_bias,
                               void* d_weight, void* work, size_t work_bytes, void* stream) {
  if (!bias_ok(b) || !sizes_ok(H, n_q, n_k, q_start)) return DFS_ERR_INVALID_ARGUMENT;
  if (H == 0) return DFS_OK;
  if (!d_weight || (n_q > 0 && n_k > 0 && (!d_bias || !work))) return DFS_ERR_INVALID_ARGUMENT;
  if (H > 65535) return DFS_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int parts = 0;
  if (n_q > 0 && n_k > 0) {
    if (work_bytes < dfs_relbias_bwd_work(H, n_q, n_k, b)) return DFS_ERR_WORKSPACE;
    parts = row_tiles(n_q);
    const RelParams P{b->weight, b->lut, b->num_buckets, b->max_distance, H, n_q, n_k, q_start};
    const dim3 grid(parts, H);
    const size_t sm = (2 * P.D + 1) * sizeof(float);
    float* part = static_cast<float*>(work);
    if (b->dtype == DFS_F32)
      relbias_bwd_kernel<float><<<grid, kThreads, sm, st>>>(P, static_cast<const float*>(d_bias), part);
    else if (b->dtype == DFS_BF16)
      relbias_bwd_kernel<__nv_bfloat16><<<grid, kThreads, sm, st>>>(P, static_cast<const __nv_bfloat16*>(d_bias),
                                                                    part);
    else
      relbias_bwd_kernel<__half><<<grid, kThreads, sm, st>>>(P, static_cast<const __half*>(d_bias), part);
    if (cudaGetLastError() != cudaSuccess) return DFS_ERR_CUDA;
  }
  return launch_bucket_sums(static_cast<const float*>(work), H, parts, b->max_distance, b->lut, b->num_buckets,
                            b->dtype, d_weight, st) == cudaSuccess
             ? DFS_OK
             : DFS_ERR_CUDA;
}
