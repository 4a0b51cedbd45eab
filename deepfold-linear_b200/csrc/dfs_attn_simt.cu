// dfs_attn_simt.cu -- local attention on the fp32 pipes: every type, any strides.
//
// The exact-product path: fp32 operands run here because a tensor-core product
// of fp32 operands keeps 11 bits of each.  16-bit operands whose addresses or
// strides are not multiples of 16 bytes run here too.
//
// One CTA owns 64 queries (forward, dQ) or 64 keys (dK, dV) of one head and
// walks the tiles of 64 that its rows see; 256 threads hold 4 x 4 pairs each,
// with both operands of every product read from shared memory as rows of the
// contraction index, so 16 FMAs cost two 16-byte reads.  The forward keeps the
// running maximum and sum of each row; the backward recomputes p from the saved
// log-sum, so its passes need no reductions across threads.
#include <climits>

#include "dfs_attn.cuh"

namespace dfs {
namespace {

constexpr int kT = 64;        // tile edge, and the padded head dim
constexpr int kLd = kT + 4;   // row pitch: 16-byte aligned, rows on different banks
constexpr int kNT = 256;
constexpr int kTile = kT * kLd;

// acc[r][c] += sum over k < K of A[k][4 ty + r] * B[k][4 tx + c]
DFS_DEV void tile_product(const float* A, const float* B, int K, int ty, int tx, float (&acc)[4][4]) {
#pragma unroll 4
  for (int k = 0; k < K; ++k) {
    const float4 a = *reinterpret_cast<const float4*>(A + k * kLd + 4 * ty);
    const float4 b = *reinterpret_cast<const float4*>(B + k * kLd + 4 * tx);
    const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[r][c] = fmaf(av[r], bv[c], acc[r][c]);
  }
}

DFS_DEV void zero(float (&a)[4][4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) a[r][c] = 0.0f;
}

// Rows [n0, n0 + 64) of (b, h) into T[c][row] and / or R[row][c] (either may be
// null), zeros beyond n, beyond d and where the mask hides the row.
template <typename E>
DFS_DEV void load_tile(const Strided& s, int b, int h, int n0, int n, int d, const uint8_t* mask, float* T, float* R,
                       int tid) {
  for (int x = tid; x < kT * kT; x += kNT) {
    const int r = x / kT, c = x % kT, row = n0 + r;
    float v = 0.0f;
    if (row < n && c < d && (mask == nullptr || mask[row] != 0)) v = to_f32<E>(row_ptr<E>(s, b, h, row)[c]);
    if (T) T[c * kLd + r] = v;
    if (R) R[r * kLd + c] = v;
  }
}

// The logit of a pair in log2 units, -inf where the key is hidden.
DFS_DEV float logit2(const AttnParams& P, const float* tab, const uint8_t* mask, float qk, int i, int j) {
  const int delta = i + P.qs - j;
  if (i >= P.nq || j >= P.nk || (mask != nullptr && mask[j] == 0) ||
      !key_near(delta, j, P.causal, P.window, P.sinks))
    return -INFINITY;
  const float bias = tab ? tab[min(max(delta, -P.D), P.D) + P.D] : 0.0f;
  return fmaf(qk, P.scale2, bias);
}

// Key tiles of 64 seen by positions p0..p1: the sink tiles [0, ns), then the window's [t0, t1).
struct KeyTiles {
  int ns, t0, t1;
  DFS_DEV KeyTiles(const AttnParams& P, int p0, int p1) {
    int lo, hi;
    near_keys(P, p0, p1, lo, hi);
    t0 = lo / kT;
    t1 = hi > lo ? (hi + kT - 1) / kT : t0;
    ns = min((sink_keys(P, p1) + kT - 1) / kT, hi > lo ? t0 : INT_MAX);
  }
  DFS_DEV int count() const { return ns + (t1 - t0); }
  DFS_DEV int operator[](int x) const { return x < ns ? x : t0 + (x - ns); }
};

template <typename E>
__global__ void __launch_bounds__(kNT) simt_fwd_kernel(AttnParams P) {
  extern __shared__ __align__(16) float sm[];
  float *Qt = sm, *Kt = Qt + kTile, *Vr = Kt + kTile, *Pt = Vr + kTile, *tab = nullptr;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / P.G, tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int i0 = blockIdx.x * kT;
  if (P.w) {
    tab = Pt + kTile;
    load_bias_table(tab, P.w, P.lut, P.D, P.nb, P.wdtype, h, kLog2e, tid, kNT);
  }
  const uint8_t* mask = P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr;
  load_tile<E>(P.q, b, h, i0, P.nq, P.d, nullptr, Qt, nullptr, tid);
  const KeyTiles tiles(P, i0 + P.qs, min(i0 + kT, P.nq) - 1 + P.qs);
  float o[4][4], m[4], l[4];
  zero(o);
#pragma unroll
  for (int r = 0; r < 4; ++r) m[r] = -INFINITY, l[r] = 0.0f;
  for (int x = 0; x < tiles.count(); ++x) {
    const int j0 = tiles[x] * kT;
    __syncthreads();
    load_tile<E>(P.k, b, hk, j0, P.nk, P.d, mask, Kt, nullptr, tid);
    load_tile<E>(P.v, b, hk, j0, P.nk, P.d, mask, nullptr, Vr, tid);
    __syncthreads();
    float s[4][4];
    zero(s);
    tile_product(Qt, Kt, P.d, ty, tx, s);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = i0 + 4 * ty + r;
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = logit2(P, tab, mask, s[r][c], i, j0 + 4 * tx + c);
        top = fmaxf(top, s[r][c]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float mn = fmaxf(m[r], top), ref = mn == -INFINITY ? 0.0f : mn;
      const float shrink = exp2f(m[r] - ref);
      float sum = 0.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = exp2f(s[r][c] - ref);
        sum += s[r][c];
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      l[r] = l[r] * shrink + sum;
      m[r] = mn;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        o[r][c] *= shrink;
        Pt[(4 * tx + c) * kLd + 4 * ty + r] = s[r][c];
      }
    }
    __syncthreads();
    tile_product(Pt, Vr, kT, ty, tx, o);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + 4 * ty + r;
    if (i >= P.nq) continue;
    const float inv = l[r] > 0.0f ? 1.0f / l[r] : 0.0f;
    E* row = row_ptr<E>(P.o, b, h, i);
    E* rest = P.o_lo ? reinterpret_cast<E*>(P.o_lo) + (row - reinterpret_cast<E*>(P.o.p)) : nullptr;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (4 * tx + c < P.d) {
        const float v = o[r][c] * inv;
        row[4 * tx + c] = from_f32<E>(v);
        if (rest) rest[4 * tx + c] = from_f32<E>(v - to_f32<E>(from_f32<E>(v)));
      }
    if (P.lse && tx == 0)
      P.lse[(static_cast<size_t>(b) * P.H + h) * P.nq + i] = l[r] > 0.0f ? m[r] + log2f(l[r]) : INFINITY;
  }
}

// dQ of 64 queries, and D_i for the key pass.  Here D_i = sum_c dO_ic O_ic comes
// from O (with what its rounding took, where the forward kept that); the key pass
// gets D_i + sum_j dS_ij, which is sum_j p_ij dP_ij in fp32 (sum_j p_ij = 1).  The
// sums of dS by bucket need that: they cancel within a row, and from a bfloat16 O
// alone they were 4e-3 off.
template <typename E>
__global__ void __launch_bounds__(kNT) simt_dq_kernel(AttnParams P) {
  extern __shared__ __align__(16) float sm[];
  float *Qt = sm, *dOt = Qt + kTile, *Kt = dOt + kTile, *Kr = Kt + kTile, *Vt = Kr + kTile, *dSt = Vt + kTile;
  float* tab = dSt + kTile;                 // 2 D + 1
  __shared__ float Drow[kT];
  const int h = blockIdx.y, b = blockIdx.z, hk = h / P.G, tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int i0 = blockIdx.x * kT;
  if (P.w) load_bias_table(tab, P.w, P.lut, P.D, P.nb, P.wdtype, h, kLog2e, tid, kNT);
  const uint8_t* mask = P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr;
  load_tile<E>(P.q, b, h, i0, P.nq, P.d, nullptr, Qt, nullptr, tid);
  load_tile<E>(P.d_o, b, h, i0, P.nq, P.d, nullptr, dOt, nullptr, tid);
  __syncthreads();
  if (tid < kT) {
    float s = 0.0f;
    const int i = i0 + tid;
    if (i < P.nq) {
      const E* orow = row_ptr<E>(P.o, b, h, i);
      const E* rest = nullptr;
      if (P.o_lo) rest = reinterpret_cast<const E*>(P.o_lo) + (orow - reinterpret_cast<const E*>(P.o.p));
      for (int c = 0; c < P.d; ++c)
        s = fmaf(dOt[c * kLd + tid], to_f32<E>(orow[c]) + (rest ? to_f32<E>(rest[c]) : 0.0f), s);
    }
    Drow[tid] = s;
  }
  __syncthreads();
  float lse[4], Di[4], rest[4], dq[4][4];
  zero(dq);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = i0 + 4 * ty + r;
    lse[r] = i < P.nq ? P.lse[(static_cast<size_t>(b) * P.H + h) * P.nq + i] : INFINITY;
    Di[r] = Drow[4 * ty + r];
    rest[r] = 0.0f;
  }
  const KeyTiles tiles(P, i0 + P.qs, min(i0 + kT, P.nq) - 1 + P.qs);
  for (int x = 0; x < tiles.count(); ++x) {
    const int j0 = tiles[x] * kT;
    __syncthreads();
    load_tile<E>(P.k, b, hk, j0, P.nk, P.d, mask, Kt, Kr, tid);
    load_tile<E>(P.v, b, hk, j0, P.nk, P.d, mask, Vt, nullptr, tid);
    __syncthreads();
    float s[4][4], dp[4][4];
    zero(s);
    zero(dp);
    tile_product(Qt, Kt, P.d, ty, tx, s);
    tile_product(dOt, Vt, P.d, ty, tx, dp);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int i = i0 + 4 * ty + r, j = j0 + 4 * tx + c;
        const float p = exp2f(logit2(P, P.w ? tab : nullptr, mask, s[r][c], i, j) - lse[r]);
        const float ds = p * (dp[r][c] - Di[r]);
        rest[r] += ds;
        dSt[(4 * tx + c) * kLd + 4 * ty + r] = ds;
      }
    __syncthreads();
    tile_product(dSt, Kr, kT, ty, tx, dq);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) rest[r] += __shfl_xor_sync(0xffffffffu, rest[r], w);
    const int i = i0 + 4 * ty + r;
    if (i >= P.nq) continue;
    if (tx == 0) P.dsum[(static_cast<size_t>(b) * P.H + h) * P.nq + i] = Di[r] + rest[r];
    E* row = row_ptr<E>(P.d_q, b, h, i);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (4 * tx + c < P.d) row[4 * tx + c] = from_f32<E>(dq[r][c] * P.scale);
  }
}

// dK and dV of 64 keys: the queries of every head of the group that see them;
// and, per head, the sums of dS by distance (a thread per diagonal of a tile, so
// every sum has one order).
template <typename E>
__global__ void __launch_bounds__(kNT) simt_dkv_kernel(AttnParams P) {
  extern __shared__ __align__(16) float sm[];
  float *Kt = sm, *Vt = Kt + kTile, *Qt = Vt + kTile, *Qr = Qt + kTile, *dOt = Qr + kTile, *dOr = dOt + kTile;
  float *Pt = dOr + kTile, *dSt = Pt + kTile, *tab = dSt + kTile;
  const int W = 2 * P.D + 1;
  float* acc = tab + (P.w ? W : 0);  // 2 D + 1
  __shared__ float ends[2][4];
  const bool dw = P.dw_part != nullptr;
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int j0 = blockIdx.x * kT, j1 = min(j0 + kT, P.nk);
  const uint8_t* mask = P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr;
  load_tile<E>(P.k, b, hk, j0, P.nk, P.d, mask, Kt, nullptr, tid);
  load_tile<E>(P.v, b, hk, j0, P.nk, P.d, mask, Vt, nullptr, tid);
  // queries that see some key of the tile: [i_lo, i_hi)
  int i_lo = P.causal ? j0 - P.qs : j0 - P.window + 1 - P.qs, i_hi = j1 - 1 + P.window - P.qs;
  if (j0 < P.sinks) {
    i_hi = P.nq;
    if (!P.causal) i_lo = 0;
  }
  i_lo = max(i_lo, 0);
  i_hi = min(i_hi, P.nq);
  float dk[4][4], dv[4][4];
  zero(dk);
  zero(dv);
  for (int g = 0; g < P.G; ++g) {
    const int h = hk * P.G + g;
    if (P.w) {
      __syncthreads();
      load_bias_table(tab, P.w, P.lut, P.D, P.nb, P.wdtype, h, kLog2e, tid, kNT);
    }
    if (dw)
      for (int x = tid; x < W; x += kNT) acc[x] = 0.0f;
    float lo = 0.0f, hi = 0.0f;  // this thread's sums of the distances beyond the table's ends
    const float* lse = P.lse + (static_cast<size_t>(b) * P.H + h) * P.nq;
    const float* Dv = P.dsum + (static_cast<size_t>(b) * P.H + h) * P.nq;
    for (int i0 = i_lo / kT * kT; i0 < i_hi; i0 += kT) {
      __syncthreads();
      load_tile<E>(P.q, b, h, i0, P.nq, P.d, nullptr, Qt, Qr, tid);
      load_tile<E>(P.d_o, b, h, i0, P.nq, P.d, nullptr, dOt, dOr, tid);
      __syncthreads();
      float s[4][4], dp[4][4];
      zero(s);
      zero(dp);
      tile_product(Kt, Qt, P.d, ty, tx, s);
      tile_product(Vt, dOt, P.d, ty, tx, dp);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int i = i0 + 4 * tx + c;
        const float ls = i < P.nq ? lse[i] : INFINITY, Di = i < P.nq ? Dv[i] : 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = exp2f(logit2(P, P.w ? tab : nullptr, mask, s[r][c], i, j0 + 4 * ty + r) - ls);
          Pt[(4 * tx + c) * kLd + 4 * ty + r] = p;
          dSt[(4 * tx + c) * kLd + 4 * ty + r] = p * (dp[r][c] - Di);
        }
      }
      __syncthreads();
      tile_product(Pt, dOr, kT, ty, tx, dv);
      tile_product(dSt, Qr, kT, ty, tx, dk);
      if (dw && tid < 2 * kT - 1) {  // thread tid owns the tile's diagonal e = query - key
        const int e = tid - (kT - 1);
        float t = 0.0f;
        for (int i = max(0, e); i < min(kT, kT + e); ++i) t += dSt[i * kLd + i - e];
        const int delta = i0 + P.qs - j0 + e;
        if (delta <= -P.D) lo += t;
        else if (delta >= P.D) hi += t;
        else acc[delta + P.D] += t;
      }
    }
    if (dw) {
      if (P.D == 0) hi += lo, lo = 0.0f;
      lo = warp_sum(lo);
      hi = warp_sum(hi);
      __syncthreads();
      if (tid < 128 && (tid & 31) == 0) ends[0][tid / 32] = lo, ends[1][tid / 32] = hi;
      __syncthreads();
      if (tid < 2 && (P.D > 0 || tid == 1))
        acc[tid == 0 ? 0 : 2 * P.D] = ends[tid][0] + ends[tid][1] + ends[tid][2] + ends[tid][3];
      __syncthreads();
      float* dst = P.dw_part + (static_cast<size_t>(h) * P.parts + b * gridDim.x + blockIdx.x) * W;
      for (int x = tid; x < W; x += kNT) dst[x] = acc[x];
      __syncthreads();
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = j0 + 4 * ty + r;
    if (j >= P.nk) continue;
    E *kr = row_ptr<E>(P.d_k, b, hk, j), *vr = row_ptr<E>(P.d_v, b, hk, j);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (4 * tx + c < P.d) {
        kr[4 * tx + c] = from_f32<E>(dk[r][c] * P.scale);
        vr[4 * tx + c] = from_f32<E>(dv[r][c]);
      }
  }
}

template <typename... A>
cudaError_t launch(void (*kern)(A...), dim3 grid, size_t smem, cudaStream_t st, A... args) {
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  kern<<<grid, kNT, smem, st>>>(args...);
  return cudaGetLastError();
}

size_t table_bytes(const AttnParams& P) { return P.w ? (2 * P.D + 1) * sizeof(float) : 0; }

template <typename E>
cudaError_t fwd(const AttnParams& P, cudaStream_t st) {
  return launch(simt_fwd_kernel<E>, dim3((P.nq + kT - 1) / kT, P.H, P.B),
                4 * kTile * sizeof(float) + table_bytes(P), st, P);
}
template <typename E>
cudaError_t bwd(const AttnParams& P, cudaStream_t st) {
  const size_t acc = P.dw_part ? (2 * P.D + 1) * sizeof(float) : 0;
  if (P.nq > 0) {
    const cudaError_t e = launch(simt_dq_kernel<E>, dim3((P.nq + kT - 1) / kT, P.H, P.B),
                                 6 * kTile * sizeof(float) + table_bytes(P), st, P);
    if (e != cudaSuccess) return e;
  }
  if (P.nk == 0) return cudaSuccess;
  return launch(simt_dkv_kernel<E>, dim3((P.nk + kT - 1) / kT, P.Hkv, P.B),
                8 * kTile * sizeof(float) + table_bytes(P) + acc, st, P);
}

}  // namespace

cudaError_t launch_attn_simt_fwd(const AttnParams& P, int dtype, cudaStream_t st) {
  return dtype == DFS_F32 ? fwd<float>(P, st) : dtype == DFS_BF16 ? fwd<__nv_bfloat16>(P, st) : fwd<__half>(P, st);
}
cudaError_t launch_attn_simt_bwd(const AttnParams& P, int dtype, cudaStream_t st) {
  return dtype == DFS_F32 ? bwd<float>(P, st) : dtype == DFS_BF16 ? bwd<__nv_bfloat16>(P, st) : bwd<__half>(P, st);
}

// ---------------------------------------------------------------- one token over a cache
namespace {

constexpr int kDecThreads = 128;
constexpr int kDecKeys = 128;   // keys of a tile: one per thread
constexpr int kDecHeads = 8;    // query heads of one CTA

// grid (head chunks of a key head, key heads, batch), one CTA walks every visible tile
template <typename E>
__global__ void __launch_bounds__(kDecThreads) decode_kernel(AttnParams P) {
  extern __shared__ float tabs[];  // kDecHeads tables
  __shared__ float qs[kDecHeads][kT], ps[kDecHeads][kDecKeys], red[kDecThreads][kDecHeads];
  __shared__ float ms[kDecHeads], ls[kDecHeads], shr[kDecHeads];
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, g0 = blockIdx.x * kDecHeads;
  const int ng = min(kDecHeads, P.G - g0), W = 2 * P.D + 1;
  const int len = min(max(P.lengths[b], 0), P.nk), p = len - 1;
  for (int x = tid; x < kDecHeads * kT; x += kDecThreads) {
    const int g = x / kT, c = x % kT;
    qs[g][c] = g < ng && c < P.d ? to_f32<E>(row_ptr<E>(P.q, b, hk * P.G + g0 + g, 0)[c]) : 0.0f;
  }
  if (P.w)
    for (int g = 0; g < ng; ++g)
      load_bias_table(tabs + g * W, P.w, P.lut, P.D, P.nb, P.wdtype, hk * P.G + g0 + g, kLog2e, tid, kDecThreads);
  if (tid < kDecHeads) ms[tid] = -INFINITY, ls[tid] = 0.0f;
  __syncthreads();
  const int lo = max(0, len - P.window), ns = min(P.sinks, lo);  // keys [0, ns) and [lo, len)
  const int total = ns + (len - lo);
  const int c = tid % kT, half = tid / kT;  // value column and half of the tile's keys
  float o[kDecHeads];
#pragma unroll
  for (int g = 0; g < kDecHeads; ++g) o[g] = 0.0f;
  for (int x0 = 0; x0 < total; x0 += kDecKeys) {
    const int x = x0 + tid, j = x < ns ? x : lo + (x - ns);
    float s[kDecHeads];
#pragma unroll
    for (int g = 0; g < kDecHeads; ++g) s[g] = 0.0f;
    if (x < total) {
      const E* kr = row_ptr<E>(P.k, b, hk, j);
      for (int e = 0; e < P.d; ++e) {
        const float kv = to_f32<E>(kr[e]);
#pragma unroll
        for (int g = 0; g < kDecHeads; ++g) s[g] = fmaf(kv, qs[g][e], s[g]);
      }
    }
#pragma unroll
    for (int g = 0; g < kDecHeads; ++g) {
      const float bias = P.w && g < ng ? tabs[g * W + min(p - j, P.D) + P.D] : 0.0f;
      ps[g][tid] = x < total ? fmaf(s[g], P.scale2, bias) : -INFINITY;
    }
    __syncthreads();
    for (int g = tid / 32; g < ng; g += kDecThreads / 32) {
      float v[kDecKeys / 32], top = -INFINITY;
#pragma unroll
      for (int r = 0; r < kDecKeys / 32; ++r) top = fmaxf(top, v[r] = ps[g][(tid & 31) + 32 * r]);
      top = warp_max(top);
      const float mn = fmaxf(ms[g], top), ref = mn == -INFINITY ? 0.0f : mn;
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < kDecKeys / 32; ++r) {
        v[r] = exp2f(v[r] - ref);
        sum += v[r];
        ps[g][(tid & 31) + 32 * r] = v[r];
      }
      sum = warp_sum(sum);
      __syncwarp();
      if ((tid & 31) == 0) {
        const float k = exp2f(ms[g] - ref);
        shr[g] = k;
        ls[g] = ls[g] * k + sum;
        ms[g] = mn;
      }
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < kDecHeads; ++g) o[g] *= g < ng ? shr[g] : 0.0f;
    if (c < P.d)
      for (int r = half * (kDecKeys / 2); r < (half + 1) * (kDecKeys / 2) && x0 + r < total; ++r) {
        const int xx = x0 + r, jj = xx < ns ? xx : lo + (xx - ns);
        const float v = to_f32<E>(row_ptr<E>(P.v, b, hk, jj)[c]);
#pragma unroll
        for (int g = 0; g < kDecHeads; ++g) o[g] = fmaf(ps[g][r], v, o[g]);
      }
    __syncthreads();
  }
#pragma unroll
  for (int g = 0; g < kDecHeads; ++g) red[tid][g] = o[g];
  __syncthreads();
  if (half == 0 && c < P.d)
    for (int g = 0; g < ng; ++g)
      row_ptr<E>(P.o, b, hk * P.G + g0 + g, 0)[c] =
          from_f32<E>(ls[g] > 0.0f ? (red[tid][g] + red[tid + kT][g]) / ls[g] : 0.0f);
}

template <typename E>
cudaError_t decode(const AttnParams& P, cudaStream_t st) {
  const size_t smem = kDecHeads * table_bytes(P);
  const cudaError_t e =
      cudaFuncSetAttribute(decode_kernel<E>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  decode_kernel<E><<<dim3((P.G + kDecHeads - 1) / kDecHeads, P.Hkv, P.B), kDecThreads, smem, st>>>(P);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_decode(const AttnParams& P, int dtype, cudaStream_t st) {
  return dtype == DFS_F32 ? decode<float>(P, st) : dtype == DFS_BF16 ? decode<__nv_bfloat16>(P, st)
                                                                    : decode<__half>(P, st);
}

}  // namespace dfs
