// dfs_relbias.cu -- learned relative position bias by buckets: the dense bias,
// its gradient, and the sums by bucket that the fused attention backward ends with.
//
//   bias[h, i, j] = w[h, b(i + q_start - j)],  dw[h, c] = sum over b(delta) = c of
//   the diagonal delta of dbias[h].
//
// Both are bound by memory: H n_q n_k elements written, or read.  Measured at 16 x
// 8192 x 8192 bfloat16: both directions in 660 us, 6.5 TB/s, 99 % of a plain copy's
// rate; at 4 x 1000 x 1537 fp32, whose rows start off 16-byte boundaries, 7.6 us
// forward and 18.7 + 5.5 us for the gradient and its sums.
#include <climits>
#include <type_traits>

#include "dfs_attn.cuh"
#include "dfs_tma.cuh"

namespace dfs {
namespace {

// Sums by bucket of `parts` rows of sums by distance, in a fixed order.  A cluster
// of 8 CTAs serves a head: each takes every 8th group of 32 distances, 16 rows of
// threads walk the parts and are added in order; the first CTA gathers the sums by
// distance and a warp per bucket adds that bucket's.
constexpr int kBucketThreads = 512, kBucketCtas = 8;

template <typename T>
__global__ void __cluster_dims__(kBucketCtas) __launch_bounds__(kBucketThreads)
    bucket_sums_kernel(const float* part, int parts, int D, const int32_t* lut, int nb, T* out) {
  extern __shared__ float acc[];  // 2 D + 1, complete in the cluster's first CTA
  __shared__ float rows[16][32];
  const int W = 2 * D + 1, h = blockIdx.x / kBucketCtas, rank = blockIdx.x % kBucketCtas, tid = threadIdx.x;
  const int cx = tid % 32, ry = tid / 32;
  const float* src = part + static_cast<size_t>(h) * parts * W;
  const uint32_t first = dsmem_addr(smem_u32(acc), 0);
  cluster_sync();  // the first CTA's memory exists
  allow_next();
  wait_previous();
  for (int x0 = rank * 32; x0 < W; x0 += kBucketCtas * 32) {
    const int x = x0 + cx;
    float s = 0.0f;
    if (x < W) {
#pragma unroll 8
      for (int r = ry; r < parts; r += 16) s += src[static_cast<size_t>(r) * W + x];
    }
    rows[ry][cx] = s;
    __syncthreads();
    if (ry == 0 && x < W) {
      float t = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) t += rows[r][cx];
      dsmem_st(first + 4 * x, t);
    }
    __syncthreads();
  }
  cluster_sync();
  if (rank != 0) return;
  for (int b = ry; b < nb; b += kBucketThreads / 32) {
    float s = 0.0f;
    for (int x = cx; x < W; x += 32) s += lut[x] == b ? acc[x] : 0.0f;
    s = warp_sum(s);
    if (cx == 0) out[static_cast<size_t>(h) * nb + b] = from_f32<T>(s);
  }
}

}  // namespace

cudaError_t launch_bucket_sums(const float* part, int H, int parts, int D, const int32_t* lut, int nb, int dtype,
                               void* out, cudaStream_t st) {
  const size_t sm = (2 * D + 1) * sizeof(float);
  const int grid = H * kBucketCtas;
  if (dtype == DFS_F32)
    return launch_dependent(bucket_sums_kernel<float>, grid, kBucketThreads, sm, st, part, parts, D, lut, nb,
                            static_cast<float*>(out));
  if (dtype == DFS_BF16)
    return launch_dependent(bucket_sums_kernel<__nv_bfloat16>, grid, kBucketThreads, sm, st, part, parts, D, lut, nb,
                            static_cast<__nv_bfloat16*>(out));
  return launch_dependent(bucket_sums_kernel<__half>, grid, kBucketThreads, sm, st, part, parts, D, lut, nb,
                          static_cast<__half*>(out));
}

namespace {

constexpr int kRelThreads = 256;
constexpr int kRelWarps = kRelThreads / 32;

struct RelParams {
  const void* w;
  const int32_t* lut;
  int nb, D, H, nq, nk, qs;
  int rows;       // rows of a CTA's tile
  int row_tiles, col_tiles;
};

// Forward.  A thread writes 16 bytes of a row at a time, on 16-byte boundaries of
// memory whatever the row's start; the pieces that stick out at a row's ends are
// written element by element.  A piece whose distances lie beyond the table is one
// value; others are looked up in the head's table in shared memory.
// X threads side by side, 256 / X rows at once; grid (row tiles x column tiles, H).
template <typename U>
__global__ void __launch_bounds__(kRelThreads) relbias_fwd_kernel(RelParams P, U* out, int log2x) {
  extern __shared__ unsigned char raw[];
  constexpr int V = 16 / sizeof(U);
  U* tab = reinterpret_cast<U*>(raw);
  const int h = blockIdx.y, tid = threadIdx.x;
  allow_next();
  wait_previous();
  const U* w = static_cast<const U*>(P.w) + static_cast<size_t>(h) * P.nb;
  for (int x = tid; x < 2 * P.D + 1; x += kRelThreads) tab[x] = w[min(max(P.lut[x], 0), P.nb - 1)];
  __syncthreads();
  const int c = ((blockIdx.x % P.col_tiles) << log2x) + (tid & ((1 << log2x) - 1));
  const int i1 = min(P.nq, static_cast<int>(blockIdx.x / P.col_tiles + 1) * P.rows);
  const U ends[2] = {tab[0], tab[2 * P.D]};
  for (int i = blockIdx.x / P.col_tiles * P.rows + (tid >> log2x); i < i1; i += kRelThreads >> log2x) {
    U* row = out + (static_cast<size_t>(h) * P.nq + i) * P.nk;
    const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(row) / sizeof(U) % V);
    const int64_t j64 = static_cast<int64_t>(c) * V - mis;  // the piece's first column
    if (j64 >= P.nk) continue;
    const int j = static_cast<int>(j64), delta = i + P.qs - j;  // of the first column; the last has delta - V + 1
    union { uint4 q; U e[V]; } v;
    if (delta - (V - 1) >= P.D || delta <= -P.D) {
      const U x = ends[delta > 0 || (delta == 0 && P.D == 0)];
#pragma unroll
      for (int e = 0; e < V; ++e) v.e[e] = x;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v.e[e] = tab[min(max(delta - e, -P.D), P.D) + P.D];
    }
    if (j >= 0 && j + V <= P.nk) {
      *reinterpret_cast<uint4*>(row + j) = v.q;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (j + e >= 0 && j + e < P.nk) row[j + e] = v.e[e];
    }
  }
}

// 16 bytes that start `a` elements into a warp's run of 16-byte pieces (next: the
// piece after this lane's), by selects on the run's common a.
template <int V>
DFS_DEV uint4 realign(uint4 own, uint4 next, int a) {
  uint32_t v[8] = {own.x, own.y, own.z, own.w, next.x, next.y, next.z, next.w};
  const int words = V == 8 ? a >> 1 : a;
  if (words & 2) {
#pragma unroll
    for (int k = 0; k < 6; ++k) v[k] = v[k + 2];
  }
  if (words & 1) {
#pragma unroll
    for (int k = 0; k < 7; ++k) v[k] = v[k + 1];
  }
  if (V == 8 && (a & 1)) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __funnelshift_r(v[k], v[k + 1], 16);
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename T>
DFS_DEV void unpack(uint4 q, float (&x)[16 / sizeof(T)]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (sizeof(T) == 4) {
      x[k] = __uint_as_float(w[k]);
    } else if (std::is_same<T, __nv_bfloat16>::value) {
      x[2 * k] = __uint_as_float(w[k] << 16);
      x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      x[2 * k] = f.x;
      x[2 * k + 1] = f.y;
    }
  }
}

// Backward.  A warp walks down a strip of 32 V columns, V of them per lane, with
// one running sum per column: the sum of the diagonal that passes through it.
// After each row the sums move one column on (one shuffle a row), so a diagonal
// is summed in the order of its rows, without atomics; the sum that leaves the
// strip's last column is complete.  Strips beyond the table's ends need no
// diagonals, one sum serves.  grid (row tiles x column tiles, H).
template <typename T>
__global__ void __launch_bounds__(kRelThreads) relbias_bwd_kernel(RelParams P, const T* dB, float* part) {
  constexpr int V = 16 / sizeof(T), C = 32 * V;
  extern __shared__ float sm[];
  const int D = P.D, W = 2 * D + 1, tid = threadIdx.x, warp = tid / 32, lane = tid % 32, h = blockIdx.y;
  float* acc = sm;                       // W
  float* strips = sm + W;                // [kRelWarps][rows + C - 1]: a strip's diagonals
  __shared__ float ends[2][kRelWarps];
  __shared__ int is_near[kRelWarps];
  const int len = P.rows + C - 1;
  const int i0 = blockIdx.x / P.col_tiles * P.rows, i1 = min(P.nq, i0 + P.rows);
  const int J0 = blockIdx.x % P.col_tiles * (kRelWarps * C), s0 = J0 + warp * C, j = s0 + lane * V;
  const T* head = dB + static_cast<size_t>(h) * P.nq * P.nk;
  const T* end = dB + static_cast<size_t>(P.H) * P.nq * P.nk;
  for (int x = tid; x < W; x += kRelThreads) acc[x] = 0.0f;
  allow_next();
  wait_previous();

  // V elements of row i from column j on, zeros outside the row
  auto fetch = [&](int i) -> uint4 {
    const T* at = head + static_cast<size_t>(i) * P.nk + j;
    const int a = static_cast<int>(reinterpret_cast<uintptr_t>(at) / sizeof(T) % V);  // the same for the whole warp
    auto piece = [&](const T* q) -> uint4 {
      if (q >= dB && q + V <= end) return __ldcs(reinterpret_cast<const uint4*>(q));
      union { uint4 q; T e[V]; } v;
      v.q = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (q + e >= dB && q + e < end) v.e[e] = q[e];
      return v.q;
    };
    uint4 x = make_uint4(0, 0, 0, 0);
    if (j - a < P.nk) x = piece(at - a);
    if (a != 0) {
      uint4 n;
      n.x = __shfl_down_sync(0xffffffffu, x.x, 1);
      n.y = __shfl_down_sync(0xffffffffu, x.y, 1);
      n.z = __shfl_down_sync(0xffffffffu, x.z, 1);
      n.w = __shfl_down_sync(0xffffffffu, x.w, 1);
      if (lane == 31) n = j - a + V < P.nk ? piece(at - a + V) : make_uint4(0, 0, 0, 0);
      x = realign<V>(x, n, a);
    }
    if (j + V > P.nk) {
      union { uint4 q; T e[V]; } v;
      v.q = x;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (j + e >= P.nk) v.e[e] = from_f32<T>(0.0f);
      x = v.q;
    }
    return x;
  };

  float lo = 0.0f, hi = 0.0f;
  const bool some = s0 < P.nk;
  const int d_lo = i0 + P.qs - (s0 + C - 1), d_hi = i1 - 1 + P.qs - s0;  // the strip's distances
  const bool far = d_lo >= D || d_hi <= -D;
  if (lane == 0) is_near[warp] = some && !far;
  if (some) {
    float2 run[V / 2];
#pragma unroll
    for (int e = 0; e < V / 2; ++e) run[e] = make_float2(0.0f, 0.0f);
    float* out = strips + warp * len;
    auto add_row = [&](uint4 x) {
      float v[V];
      unpack<T>(x, v);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) run[e] = __fadd2_rn(run[e], make_float2(v[2 * e], v[2 * e + 1]));
    };
    // the sums of a near strip move on by one column between two rows
    auto move_on = [&]() {
      const float in = __shfl_up_sync(0xffffffffu, run[V / 2 - 1].y, 1);
#pragma unroll
      for (int e = V / 2 - 1; e > 0; --e) run[e] = make_float2(run[e - 1].y, run[e].x);
      run[0] = make_float2(lane == 0 ? 0.0f : in, run[0].x);
    };
    // rows that need no care: whole in columns, and on 16-byte boundaries like their neighbours
    const bool easy = s0 + C <= P.nk && P.nk % V == 0 && (reinterpret_cast<uintptr_t>(dB) & 15u) == 0;
    int i = i0;
    if (easy) {
      const T* at = head + static_cast<size_t>(i0) * P.nk + j;
      const size_t pitch = static_cast<size_t>(P.nk);
      for (; i + 8 <= i1; i += 8, at += 8 * pitch) {
        uint4 x[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) x[r] = __ldcs(reinterpret_cast<const uint4*>(at + r * pitch));
        if (far) {
#pragma unroll
          for (int r = 0; r < 8; ++r) add_row(x[r]);
        } else {
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            if (i + r > i0) move_on();
            add_row(x[r]);
            if (lane == 31) out[i + r - i0] = run[V / 2 - 1].y;  // slot s: diagonal i0 - (s0 + C - 1) + s
          }
        }
      }
    }
    for (; i < i1; i += 4) {
      uint4 x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = i + r < i1 ? fetch(i + r) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (i + r >= i1) break;
        if (!far && i + r > i0) move_on();
        add_row(x[r]);
        if (!far && lane == 31) out[i + r - i0] = run[V / 2 - 1].y;
      }
    }
    if (far) {
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < V / 2; ++e) s += run[e].x + run[e].y;
      (d_lo >= D ? hi : lo) = s;
    } else {
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        float* last = out + (i1 - 1 - i0 + C - 1 - lane * V - 2 * e);
        last[0] = run[e].x;
        last[-1] = run[e].y;
      }
    }
  }
  __syncthreads();
  // the near strips' diagonals, by distance: one thread each, the strips in order
  const int e0 = i0 - (J0 + kRelWarps * C - 1);
  for (int e = e0 + tid; e <= i1 - 1 - J0; e += kRelThreads) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kRelWarps; ++w) {
      const int slot = e - (i0 - (J0 + w * C + C - 1));
      if (is_near[w] && slot >= 0 && slot < i1 - i0 + C - 1) s += strips[w * len + slot];
    }
    const int delta = e + P.qs;
    if (delta <= -D) lo += s;
    else if (delta >= D) hi += s;
    else acc[delta + D] = s;
  }
  if (D == 0) hi += lo, lo = 0.0f;  // one entry stands for every distance
  lo = warp_sum(lo);
  hi = warp_sum(hi);
  if (lane == 0) ends[0][warp] = lo, ends[1][warp] = hi;
  __syncthreads();
  if (tid < 2 && (D > 0 || tid == 1)) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kRelWarps; ++w) s += ends[tid][w];
    acc[tid == 0 ? 0 : 2 * D] = s;
  }
  __syncthreads();
  float* dst = part + (static_cast<size_t>(h) * gridDim.x + blockIdx.x) * W;
  for (int x = tid; x < W; x += kRelThreads) dst[x] = acc[x];
}

bool bias_ok(const dfs_relbias* b) {
  return b && b->lut && b->num_buckets > 0 && b->max_distance >= 0 && b->max_distance <= DFS_MAX_BUCKET_DISTANCE &&
         (b->dtype == DFS_BF16 || b->dtype == DFS_F16 || b->dtype == DFS_F32);
}
// positions and distances stay inside 32 bits
bool sizes_ok(int H, int nq, int nk, int qs) {
  return H >= 0 && nq >= 0 && nk >= 0 && nq <= (1 << 28) && nk <= (1 << 28) && qs >= -(1 << 28) && qs <= (1 << 28);
}
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int elem_size(int dtype) { return dtype == DFS_F32 ? 4 : 2; }

// Backward tiles: 8 strips of 512 bytes of columns; as many rows (a multiple of 32 up to 256, so that partial
// sums stay a small part of what is read) as leave about four CTAs an SM.
void bwd_tiles(int H, int nq, int nk, int dtype, RelParams& P) {
  P.col_tiles = static_cast<int>(ceil_div(nk, kRelWarps * 512 / elem_size(dtype)));
  P.rows = 256;
  while (P.rows > 32 && H * ceil_div(nq, P.rows) * P.col_tiles < 4 * 148) P.rows /= 2;
  P.row_tiles = static_cast<int>(ceil_div(nq, P.rows));
}

}  // namespace
}  // namespace dfs

using namespace dfs;

extern "C" int dfs_relbias_fwd(int H, int n_q, int n_k, int q_start, const dfs_relbias* b, void* out, void* stream) {
  if (!bias_ok(b) || !sizes_ok(H, n_q, n_k, q_start)) return DFS_ERR_INVALID_ARGUMENT;
  if (H == 0 || n_q == 0 || n_k == 0) return DFS_OK;
  if (!b->weight || !out) return DFS_ERR_INVALID_ARGUMENT;
  const int size = elem_size(b->dtype), V = 16 / size;
  RelParams P{b->weight, b->lut, b->num_buckets, b->max_distance, H, n_q, n_k, q_start, 0, 0, 0};
  const int64_t pieces = ceil_div(n_k, V) + 1;  // of a row that starts between two 16-byte boundaries
  int log2x = 3;
  while (log2x < 8 && (int64_t{1} << log2x) < pieces) ++log2x;
  P.col_tiles = static_cast<int>(ceil_div(pieces, int64_t{1} << log2x));
  // rows of a CTA: 32 passes of its threads at most, fewer while there are not eight CTAs an SM
  P.rows = 32 * (kRelThreads >> log2x);
  while (P.rows > (kRelThreads >> log2x) && H * ceil_div(n_q, P.rows) * P.col_tiles < 8 * 148) P.rows /= 2;
  P.row_tiles = static_cast<int>(ceil_div(n_q, P.rows));
  if (H > 65535 || static_cast<int64_t>(P.row_tiles) * P.col_tiles > INT_MAX) return DFS_ERR_UNSUPPORTED;
  const dim3 grid(P.row_tiles * P.col_tiles, H);
  const size_t sm = (2 * P.D + 1) * size;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (size == 4)
    relbias_fwd_kernel<uint32_t><<<grid, kRelThreads, sm, st>>>(P, static_cast<uint32_t*>(out), log2x);
  else
    relbias_fwd_kernel<uint16_t><<<grid, kRelThreads, sm, st>>>(P, static_cast<uint16_t*>(out), log2x);
  return cudaGetLastError() == cudaSuccess ? DFS_OK : DFS_ERR_CUDA;
}

extern "C" size_t dfs_relbias_bwd_work(int H, int n_q, int n_k, const dfs_relbias* b) {
  if (!bias_ok(b) || !sizes_ok(H, n_q, n_k, 0)) return 0;
  RelParams P{};
  bwd_tiles(H, n_q, n_k, b->dtype, P);
  return static_cast<size_t>(H) * P.row_tiles * P.col_tiles * (2 * b->max_distance + 1) * sizeof(float);
}

extern "C" int dfs_relbias_bwd(int H, int n_q, int n_k, int q_start, const dfs_relbias* b, const void* d_bias,
                               void* d_weight, void* work, size_t work_bytes, void* stream) {
  if (!bias_ok(b) || !sizes_ok(H, n_q, n_k, q_start)) return DFS_ERR_INVALID_ARGUMENT;
  if (H == 0) return DFS_OK;
  if (!d_weight || (n_q > 0 && n_k > 0 && (!d_bias || !work))) return DFS_ERR_INVALID_ARGUMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  RelParams P{b->weight, b->lut, b->num_buckets, b->max_distance, H, n_q, n_k, q_start, 0, 0, 0};
  bwd_tiles(H, n_q, n_k, b->dtype, P);
  const int64_t parts = static_cast<int64_t>(P.row_tiles) * P.col_tiles;
  if (H > 65535 || parts > INT_MAX) return DFS_ERR_UNSUPPORTED;
  if (parts > 0) {
    if (work_bytes < dfs_relbias_bwd_work(H, n_q, n_k, b)) return DFS_ERR_WORKSPACE;
    const dim3 grid(static_cast<unsigned>(parts), H);
    const size_t sm = (2 * P.D + 1 + kRelWarps * (P.rows + 512 / elem_size(b->dtype) - 1)) * sizeof(float);
    float* part = static_cast<float*>(work);
    if (b->dtype == DFS_F32)
      relbias_bwd_kernel<float><<<grid, kRelThreads, sm, st>>>(P, static_cast<const float*>(d_bias), part);
    else if (b->dtype == DFS_BF16)
      relbias_bwd_kernel<__nv_bfloat16><<<grid, kRelThreads, sm, st>>>(P, static_cast<const __nv_bfloat16*>(d_bias),
                                                                    part);
    else
      relbias_bwd_kernel<__half><<<grid, kRelThreads, sm, st>>>(P, static_cast<const __half*>(d_bias), part);
    if (cudaGetLastError() != cudaSuccess) return DFS_ERR_CUDA;
  }
  return launch_bucket_sums(static_cast<const float*>(work), H, static_cast<int>(parts), b->max_distance, b->lut,
                            b->num_buckets, b->dtype, d_weight, st) == cudaSuccess
             ? DFS_OK
             : DFS_ERR_CUDA;
}
