// dfs_attn.cuh -- what the local-attention kernels share: launch parameters, the
// rule of which key a query sees, element types, and the expanded bias table.
#pragma once

#include <atomic>
#include <cfloat>

#include "dfs_device.cuh"

namespace dfs {

struct Strided {
  char* p;              // element (b, h, n, c) at p + (b sb + h sh + n sn + c) * size
  int64_t sb, sh, sn;   // in elements; 64 bits: a long cache passes 2^31 elements
};

struct AttnParams {
  Strided q, k, v, o, d_o, d_q, d_k, d_v;
  char* o_lo;           // laid out as o: o's rounding error, or null
  float* lse;           // (B,H,n_q) log2 units, +inf for a row that sees nothing
  float* dsum;          // (B,H,n_q) D_i = sum_j p_ij dP_ij (backward workspace)
  const uint8_t* mask;  // (B,n_k) or null
  const void* w;        // (H, nb) bias weights of type wdtype, or null
  const int32_t* lut;   // (2 D + 1)
  float* dw_part;       // (H, parts, 2 D + 1) sums of dS by distance, or null
  float* sink_part;     // fp32 parts of the sink keys' gradients, or null
  float* near_part;     // fp32 parts of key tiles' gradients, or null
  int sink_tiles, far_segs, far_len;  // key tiles that hold sinks; segments of queries beyond the window, steps of each
  int near_segs;        // segments of every key tile's other steps
  int32_t* status;
  const void* lengths;  // decode: (B,) int32, or int64 if wide_lengths
  int wide_lengths;
  int nb, D, wdtype;
  int parts;            // rows of dw_part per head: key tiles (and far segments) of all batch elements
  int B, H, Hkv, G, nq, nk, d;
  int causal, window, sinks, qs;
  float scale, scale2;  // scale; scale * log2(e)
};

// Programmatic dependent launches: a kernel's blocks may be set up while the one before it ends.  Nothing of
// global memory is read or written before wait_previous(); allow_next() comes after a block's TMEM allocation, so
// that the next kernel's blocks, which wait for this one to end, cannot hold the columns that it still needs.
DFS_DEV void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
DFS_DEV void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Visible apart from the mask.  A window of "all" is INT_MAX/2 by the host.
DFS_DEV bool key_near(int delta, int j, int causal, int window, int sinks) {
  if (causal ? delta < 0 : false) return false;
  return (delta < window && -delta < window) || j < sinks;
}

// Keys of sequence b's cache that hold a token, [0, n_k].
DFS_DEV int seq_length(const AttnParams& P, int b) {
  const int64_t n = P.wide_lengths ? static_cast<const int64_t*>(P.lengths)[b]
                                   : static_cast<const int32_t*>(P.lengths)[b];
  return static_cast<int>(min(max(n, int64_t{0}), static_cast<int64_t>(P.nk)));
}

// Keys [lo, hi) that positions p0..p1 may see through the window (sinks apart).
DFS_DEV void near_keys(const AttnParams& P, int p0, int p1, int& lo, int& hi) {
  lo = max(0, p0 - P.window + 1);
  hi = P.causal ? min(P.nk, p1 + 1) : min(P.nk, p1 + P.window);
  hi = max(hi, 0);
  lo = min(lo, hi);
}
// Sink keys [0, n) that the last position p1 may see.
DFS_DEV int sink_keys(const AttnParams& P, int p1) {
  const int n = P.causal ? min(P.sinks, p1 + 1) : P.sinks;
  return max(0, min(n, P.nk));
}

template <typename T>
DFS_DEV float to_f32(T x);
template <>
DFS_DEV float to_f32<float>(float x) { return x; }
template <>
DFS_DEV float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
DFS_DEV float to_f32<__half>(__half x) { return __half2float(x); }
template <typename T>
DFS_DEV T from_f32(float x);
template <>
DFS_DEV float from_f32<float>(float x) { return x; }
template <>
DFS_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16(x); }
template <>
DFS_DEV __half from_f32<__half>(float x) { return __float2half(x); }

template <typename T>
DFS_DEV T* row_ptr(const Strided& s, int b, int h, int64_t n) {
  return reinterpret_cast<T*>(s.p) + b * s.sb + h * s.sh + n * s.sn;
}

// A bias weight in log2 units, the finite ones within +-32000.  A type's lowest value, with which a table may hide
// distances, would overflow to -inf here, and a row that sees such keys only would count as one that sees none; and
// with -1e9 such a row's log-sum m + log2(l) would no longer hold log2(l), so that the backward's p were l times too
// large.  At 32000 logits and log-sums keep steps of 2^-9, so those rows are right to 2^-10; beside any other key such a
// key's p is 0 all the same.
constexpr float kBiasLimit = 32000.0f;
DFS_DEV float bias_log2(float w) {
  const float x = w * kLog2e;
  return fabsf(w) <= FLT_MAX ? fminf(fmaxf(x, -kBiasLimit), kBiasLimit) : x;  // infinities and NaN as they are
}
// Weight of head h's bucket b.
DFS_DEV float bias_weight(const AttnParams& P, int h, int b) {
  return bias_log2(load_as_f32<void>(P.w, static_cast<size_t>(h) * P.nb + min(max(b, 0), P.nb - 1), P.wdtype));
}

// tab[delta + D] = weight[h, lut[delta + D]] in log2 units for the whole table (a block's threads).
DFS_DEV void load_bias_table(float* tab, const AttnParams& P, int h, int tid, int nthreads) {
  for (int x = tid; x < 2 * P.D + 1; x += nthreads) tab[x] = bias_weight(P, h, P.lut[x]);
}

// Raises kernel K's limit of dynamic shared memory to `most`, what it needs with the largest bias table (D =
// DFS_MAX_BUCKET_DISTANCE): once per device, for the call costs host time, and to the same value in every call, so
// that no host thread can lower it between another's check and its launch.  And, where the kernel splits its
// registers, checks that the shares fit what it is launched with (an increase that the block's own registers cannot
// serve would wait forever).
template <auto K>
cudaError_t prepare_kernel(size_t most, int threads = 0, int share = 0) {
  constexpr int kMaxDevices = 64;
  static std::atomic<bool> ready[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < kMaxDevices && ready[dev].load(std::memory_order_acquire)) return cudaSuccess;
  if (share > 0) {
    cudaFuncAttributes at;
    if ((e = cudaFuncGetAttributes(&at, K)) != cudaSuccess) return e;
    if ((at.numRegs + 7) / 8 * 8 * threads < share) return cudaErrorInvalidConfiguration;
  }
  e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
  if (e == cudaSuccess && dev < kMaxDevices) ready[dev].store(true, std::memory_order_release);
  return e;
}

// launchers (host)
cudaError_t launch_bucket_sums(const float* part, int H, int parts, int D, const int32_t* lut, int nb, int dtype,
                               void* out, cudaStream_t st);
// vec: fp32 rows on 16-byte boundaries
cudaError_t launch_attn_simt_fwd(const AttnParams& P, int dtype, bool vec, cudaStream_t st);
cudaError_t launch_attn_simt_bwd(const AttnParams& P, int dtype, bool vec, cudaStream_t st);
cudaError_t launch_decode_mma(const AttnParams& P, int dtype, cudaStream_t st);  // 16-bit, staged by TMA
cudaError_t launch_decode_any(const AttnParams& P, int dtype, bool vec, cudaStream_t st);

}  // namespace dfs
