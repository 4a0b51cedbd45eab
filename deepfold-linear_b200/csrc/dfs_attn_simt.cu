// dfs_attn_simt.cu -- local attention on the fp32 pipes: every type, any strides.
//
// The exact-product path: fp32 operands run here because a tensor-core product
// of fp32 operands keeps 11 bits of each.  16-bit operands whose addresses or
// strides are not multiples of 16 bytes run here too.
//
// One CTA owns 64 queries (forward, dQ) or 64 keys (dK, dV) of one head and
// walks the tiles of 64 that its rows see; 128 threads hold 8 x 4 pairs each.
// Every tile lies in shared memory as its rows do in global memory, and products
// read the operand whose rows they contract along in pieces of four (so no tile is
// needed twice, transposed): 32 FMAs for three 16-byte reads, two of them the same
// for 16 lanes, so the FMA pipes are the bound and shared memory is not.  The
// forward keeps the running maximum and sum of each row; the backward recomputes p
// from the saved log-sum, so its passes need no reductions across threads.
//
// Measured (fp32, causal, a bias): forward of 16 heads of 4096 at d = 64, 1.37 ms,
// 25 TFLOP/s of 74; with both gradients 7.1 ms.  (Transposed copies in shared
// memory and 4 x 4 pairs a thread: 2.1 and 11.3 ms.)  A third of the instructions
// are not products, and 12 warps an SM leave half of the issue slots empty.
#include "dfs_attn.cuh"

namespace dfs {
namespace {

constexpr int kT = 64;        // tile edge, and the padded head dim
constexpr int kLd = kT + 4;   // row pitch: 16-byte aligned, 8 rows' pieces on different banks
constexpr int kNT = 128;
constexpr int kR = 8;         // rows ty + 8 r of a thread; its columns are tx + 16 c (pairs) or 4 tx + c (head dim)
constexpr int kTile = kT * kLd;

// s[r][c] = sum over k < K (a multiple of 4) of A[ty + 8 r][k] * B[tx + 16 c][k]
DFS_DEV void product_nt(const float* A, const float* B, int K, int ty, int tx, float (&s)[kR][4]) {
  float2 t[kR][4];  // sums of the even and of the odd k
#pragma unroll
  for (int r = 0; r < kR; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) t[r][c] = make_float2(0.0f, 0.0f);
#pragma unroll 2
  for (int k = 0; k < K; k += 4) {
    float4 b[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) b[c] = *reinterpret_cast<const float4*>(B + (tx + 16 * c) * kLd + k);
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const float4 a = *reinterpret_cast<const float4*>(A + (ty + 8 * r) * kLd + k);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        t[r][c] = __ffma2_rn(make_float2(a.x, a.y), make_float2(b[c].x, b[c].y), t[r][c]);
        t[r][c] = __ffma2_rn(make_float2(a.z, a.w), make_float2(b[c].z, b[c].w), t[r][c]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kR; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) s[r][c] = t[r][c].x + t[r][c].y;
}

// acc[r][c] += sum over the 64 rows k of B of A[ty + 8 r][k] * B[k][4 tx + c]
DFS_DEV void product_nn(const float* A, const float* B, int ty, int tx, float (&acc)[kR][4]) {
#pragma unroll 2
  for (int k = 0; k < kT; k += 4) {
    float a[kR][4];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const float4 x = *reinterpret_cast<const float4*>(A + (ty + 8 * r) * kLd + k);
      a[r][0] = x.x, a[r][1] = x.y, a[r][2] = x.z, a[r][3] = x.w;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float4 b = *reinterpret_cast<const float4*>(B + (k + u) * kLd + 4 * tx);
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        acc[r][0] = fmaf(a[r][u], b.x, acc[r][0]);
        acc[r][1] = fmaf(a[r][u], b.y, acc[r][1]);
        acc[r][2] = fmaf(a[r][u], b.z, acc[r][2]);
        acc[r][3] = fmaf(a[r][u], b.w, acc[r][3]);
      }
    }
  }
}

DFS_DEV void zero(float (&a)[kR][4]) {
#pragma unroll
  for (int r = 0; r < kR; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) a[r][c] = 0.0f;
}

// Rows [n0, n0 + 64) of (b, h) into T[row][c], zeros beyond n, beyond d and where
// the mask hides the row.  kVec: fp32 rows on 16-byte boundaries, d a multiple of 4.
template <typename E, bool kVec>
DFS_DEV void load_tile(const Strided& s, int b, int h, int n0, int n, int d, const uint8_t* mask, float* T, int tid) {
  if constexpr (kVec) {
    float4 v[kT * kT / 4 / kNT];
#pragma unroll
    for (int u = 0; u < kT * kT / 4 / kNT; ++u) {
      const int x = tid + u * kNT, r = x / 16, c = x % 16 * 4, row = n0 + r;
      v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (row < n && c < d && (mask == nullptr || mask[row] != 0))
        v[u] = *reinterpret_cast<const float4*>(row_ptr<float>(s, b, h, row) + c);
    }
#pragma unroll
    for (int u = 0; u < kT * kT / 4 / kNT; ++u) {
      const int x = tid + u * kNT;
      *reinterpret_cast<float4*>(T + x / 16 * kLd + x % 16 * 4) = v[u];
    }
  } else {
#pragma unroll 8
    for (int x = tid; x < kT * kT; x += kNT) {
      const int r = x / kT, c = x % kT, row = n0 + r;
      float v = 0.0f;
      if (row < n && c < d && (mask == nullptr || mask[row] != 0)) v = to_f32<E>(row_ptr<E>(s, b, h, row)[c]);
      T[r * kLd + c] = v;
    }
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

// Whether every pair of 64 queries from position p0 and 64 keys from j0 is visible and has the far bias of its side
// (1: at or beyond the table's end, -1: the other; 0: look at each).  rows: the tiles are whole and unmasked.
DFS_DEV int plain_side(const AttnParams& P, int p0, int j0, bool rows) {
  const int lo = p0 - j0 - (kT - 1), hi = p0 - j0 + (kT - 1);  // the distances
  if (!rows || (P.causal && lo < 0) || lo <= -P.window || hi >= P.window) return 0;
  return P.w == nullptr || lo >= P.D ? 1 : hi <= -P.D ? -1 : 0;
}

// Key tiles of 64 seen by positions p0..p1: the sink tiles [0, ns), then the window's [t0, t1), which go on to the last
// sink where the sinks reach into them or (without causality) past them.
struct KeyTiles {
  int ns, t0, t1;
  DFS_DEV KeyTiles(const AttnParams& P, int p0, int p1) {
    int lo, hi;
    near_keys(P, p0, p1, lo, hi);
    t0 = lo / kT;
    t1 = hi > lo ? (hi + kT - 1) / kT : t0;
    ns = (sink_keys(P, p1) + kT - 1) / kT;
    if (hi > lo && ns > t0) t1 = max(t1, ns), ns = t0;
  }
  DFS_DEV int count() const { return ns + (t1 - t0); }
  DFS_DEV int operator[](int x) const { return x < ns ? x : t0 + (x - ns); }
};

template <typename E, bool kVec>
__global__ void __launch_bounds__(kNT, 3) simt_fwd_kernel(AttnParams P) {
  extern __shared__ __align__(16) float sm[];
  float *Q = sm, *K = Q + kTile, *V = K + kTile, *Pr = V + kTile, *tab = nullptr;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / P.G, tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int i0 = (gridDim.x - 1 - blockIdx.x) * kT, dk = (P.d + 3) / 4 * 4;  // causal: longest first
  if (P.w) {
    tab = Pr + kTile;
    load_bias_table(tab, P, h, tid, kNT);
  }
  const uint8_t* mask = P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr;
  load_tile<E, kVec>(P.q, b, h, i0, P.nq, P.d, nullptr, Q, tid);
  const KeyTiles tiles(P, i0 + P.qs, min(i0 + kT, P.nq) - 1 + P.qs);
  float o[kR][4], m[kR], l[kR];
  zero(o);
#pragma unroll
  for (int r = 0; r < kR; ++r) m[r] = -INFINITY, l[r] = 0.0f;
  for (int x = 0; x < tiles.count(); ++x) {
    const int j0 = tiles[x] * kT;
    __syncthreads();
    load_tile<E, kVec>(P.k, b, hk, j0, P.nk, P.d, mask, K, tid);
    load_tile<E, kVec>(P.v, b, hk, j0, P.nk, P.d, mask, V, tid);
    __syncthreads();
    float s[kR][4];
    product_nt(Q, K, dk, ty, tx, s);
    const int side = plain_side(P, i0 + P.qs, j0, mask == nullptr && i0 + kT <= P.nq && j0 + kT <= P.nk);
    const float far = P.w ? tab[side > 0 ? 2 * P.D : 0] : 0.0f;
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const int i = i0 + ty + 8 * r;
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = side != 0 ? fmaf(s[r][c], P.scale2, far) : logit2(P, tab, mask, s[r][c], i, j0 + tx + 16 * c);
        top = fmaxf(top, s[r][c]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float mn = fmaxf(m[r], top), ref = mn == -INFINITY ? 0.0f : mn;
      const float shrink = exp2f(m[r] - ref);
      float sum = 0.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float p = exp2f(s[r][c] - ref);
        sum += p;
        Pr[(ty + 8 * r) * kLd + tx + 16 * c] = p;
        o[r][c] *= shrink;
      }
      l[r] = l[r] * shrink + sum;  // this thread's columns
      m[r] = mn;
    }
    __syncthreads();
    product_nn(Pr, V, ty, tx, o);
  }
#pragma unroll
  for (int r = 0; r < kR; ++r)
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
#pragma unroll
  for (int r = 0; r < kR; ++r) {
    const int i = i0 + ty + 8 * r;
    if (i >= P.nq) continue;
    const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];  // a sum that is NaN stays one, here and in lse
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
      P.lse[(static_cast<size_t>(b) * P.H + h) * P.nq + i] = l[r] == 0.0f ? INFINITY : m[r] + log2f(l[r]);
  }
}

// dQ of 64 queries, and D_i for the key pass.  Here D_i = sum_c dO_ic O_ic comes
// from O (with what its rounding took, where the forward kept that); the key pass
// gets D_i + sum_j dS_ij, which is sum_j p_ij dP_ij in fp32 (sum_j p_ij = 1).  The
// sums of dS by bucket need that: they cancel within a row, and from a bfloat16 O
// alone they were 4e-3 off.
template <typename E, bool kVec>
__global__ void __launch_bounds__(kNT, 2) simt_dq_kernel(AttnParams P) {
  extern __shared__ __align__(16) float sm[];
  float *Q = sm, *dO = Q + kTile, *K = dO + kTile, *V = K + kTile, *dS = V + kTile;
  float* tab = dS + kTile;                 // 2 D + 1
  __shared__ float Drow[kT];
  const int h = blockIdx.y, b = blockIdx.z, hk = h / P.G, tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int i0 = (gridDim.x - 1 - blockIdx.x) * kT, dk = (P.d + 3) / 4 * 4;  // causal: longest first
  if (P.w) load_bias_table(tab, P, h, tid, kNT);
  const uint8_t* mask = P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr;
  load_tile<E, kVec>(P.q, b, h, i0, P.nq, P.d, nullptr, Q, tid);
  load_tile<E, kVec>(P.d_o, b, h, i0, P.nq, P.d, nullptr, dO, tid);
  __syncthreads();
  if (tid < kT) {
    float s = 0.0f;
    const int i = i0 + tid;
    if (i < P.nq) {
      const E* orow = row_ptr<E>(P.o, b, h, i);
      const E* rest = nullptr;
      if (P.o_lo) rest = reinterpret_cast<const E*>(P.o_lo) + (orow - reinterpret_cast<const E*>(P.o.p));
      for (int c = 0; c < P.d; ++c)
        s = fmaf(dO[tid * kLd + c], to_f32<E>(orow[c]) + (rest ? to_f32<E>(rest[c]) : 0.0f), s);
    }
    Drow[tid] = s;
  }
  __syncthreads();
  float lse[kR], Di[kR], rest[kR], dq[kR][4];
  zero(dq);
#pragma unroll
  for (int r = 0; r < kR; ++r) {
    const int i = i0 + ty + 8 * r;
    lse[r] = i < P.nq ? P.lse[(static_cast<size_t>(b) * P.H + h) * P.nq + i] : INFINITY;
    Di[r] = Drow[ty + 8 * r];
    rest[r] = 0.0f;
  }
  const KeyTiles tiles(P, i0 + P.qs, min(i0 + kT, P.nq) - 1 + P.qs);
  for (int x = 0; x < tiles.count(); ++x) {
    const int j0 = tiles[x] * kT;
    __syncthreads();
    load_tile<E, kVec>(P.k, b, hk, j0, P.nk, P.d, mask, K, tid);
    load_tile<E, kVec>(P.v, b, hk, j0, P.nk, P.d, mask, V, tid);
    __syncthreads();
    float p[kR][4], dp[kR][4];
    product_nt(Q, K, dk, ty, tx, p);
    const int side = plain_side(P, i0 + P.qs, j0, mask == nullptr && i0 + kT <= P.nq && j0 + kT <= P.nk);
    const float far = P.w ? tab[side > 0 ? 2 * P.D : 0] : 0.0f;
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int i = i0 + ty + 8 * r, j = j0 + tx + 16 * c;
        const float x = side != 0 ? fmaf(p[r][c], P.scale2, far) : logit2(P, P.w ? tab : nullptr, mask, p[r][c], i, j);
        p[r][c] = exp2f(x - lse[r]);
      }
    product_nt(dO, V, dk, ty, tx, dp);
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float ds = p[r][c] * (dp[r][c] - Di[r]);
        rest[r] += ds;
        dS[(ty + 8 * r) * kLd + tx + 16 * c] = ds;
      }
    __syncthreads();
    product_nn(dS, K, ty, tx, dq);
  }
#pragma unroll
  for (int r = 0; r < kR; ++r) {
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) rest[r] += __shfl_xor_sync(0xffffffffu, rest[r], w);
    const int i = i0 + ty + 8 * r;
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
template <typename E, bool kVec>
__global__ void __launch_bounds__(kNT, 2) simt_dkv_kernel(AttnParams P) {
  extern __shared__ __align__(16) float sm[];
  float *K = sm, *V = K + kTile, *Q = V + kTile, *dO = Q + kTile;
  float *Pt = dO + kTile, *dSt = Pt + kTile, *tab = dSt + kTile;  // P and dS transposed: [key][query]
  const int W = 2 * P.D + 1;
  float* acc = tab + (P.w ? W : 0);  // 2 D + 1
  __shared__ float ends[2][4];
  const bool dw = P.dw_part != nullptr;
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int j0 = blockIdx.x * kT, j1 = min(j0 + kT, P.nk), kd = (P.d + 3) / 4 * 4;
  const uint8_t* mask = P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr;
  load_tile<E, kVec>(P.k, b, hk, j0, P.nk, P.d, mask, K, tid);
  load_tile<E, kVec>(P.v, b, hk, j0, P.nk, P.d, mask, V, tid);
  // queries that see some key of the tile: [i_lo, i_hi)
  int i_lo = P.causal ? j0 - P.qs : j0 - P.window + 1 - P.qs, i_hi = j1 - 1 + P.window - P.qs;
  if (j0 < P.sinks) {
    i_hi = P.nq;
    if (!P.causal) i_lo = 0;
  }
  i_lo = max(i_lo, 0);
  i_hi = min(i_hi, P.nq);
  float dk[kR][4], dv[kR][4];
  zero(dk);
  zero(dv);
  for (int g = 0; g < P.G; ++g) {
    const int h = hk * P.G + g;
    if (P.w) {
      __syncthreads();
      load_bias_table(tab, P, h, tid, kNT);
    }
    if (dw)
      for (int x = tid; x < W; x += kNT) acc[x] = 0.0f;
    float lo = 0.0f, hi = 0.0f;  // this thread's sums of the distances beyond the table's ends
    const float* lse = P.lse + (static_cast<size_t>(b) * P.H + h) * P.nq;
    const float* Dv = P.dsum + (static_cast<size_t>(b) * P.H + h) * P.nq;
    for (int i0 = i_lo / kT * kT; i0 < i_hi; i0 += kT) {
      __syncthreads();
      load_tile<E, kVec>(P.q, b, h, i0, P.nq, P.d, nullptr, Q, tid);
      load_tile<E, kVec>(P.d_o, b, h, i0, P.nq, P.d, nullptr, dO, tid);
      __syncthreads();
      float p[kR][4], dp[kR][4];
      product_nt(K, Q, kd, ty, tx, p);
      const int side = plain_side(P, i0 + P.qs, j0, mask == nullptr && i0 + kT <= P.nq && j0 + kT <= P.nk);
      const float far = P.w ? tab[side > 0 ? 2 * P.D : 0] : 0.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int i = i0 + tx + 16 * c;
        const float ls = i < P.nq ? lse[i] : INFINITY;
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const int j = j0 + ty + 8 * r;
          const float x =
              side != 0 ? fmaf(p[r][c], P.scale2, far) : logit2(P, P.w ? tab : nullptr, mask, p[r][c], i, j);
          p[r][c] = exp2f(x - ls);
          Pt[(ty + 8 * r) * kLd + tx + 16 * c] = p[r][c];
        }
      }
      product_nt(V, dO, kd, ty, tx, dp);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int i = i0 + tx + 16 * c;
        const float Di = i < P.nq ? Dv[i] : 0.0f;
#pragma unroll
        for (int r = 0; r < kR; ++r) dSt[(ty + 8 * r) * kLd + tx + 16 * c] = p[r][c] * (dp[r][c] - Di);
      }
      __syncthreads();
      product_nn(Pt, dO, ty, tx, dv);
      product_nn(dSt, Q, ty, tx, dk);
      if (dw && tid < 2 * kT - 1) {  // thread tid owns the tile's diagonal e = query - key
        const int e = tid - (kT - 1);
        float t = 0.0f;
        for (int i = max(0, e); i < min(kT, kT + e); ++i) t += dSt[(i - e) * kLd + i];
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
      if ((tid & 31) == 0) ends[0][tid / 32] = lo, ends[1][tid / 32] = hi;
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
  for (int r = 0; r < kR; ++r) {
    const int j = j0 + ty + 8 * r;
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

// K over a grid with `tiles` tiles and `tables` bias tables (or sums by distance) in shared memory; most: the tables
// that it can have
template <auto K>
cudaError_t launch(dim3 grid, int tiles, int tables, int most, cudaStream_t st, const AttnParams& P) {
  auto bytes = [=](int n, int D) { return (tiles * kTile + n * (2 * D + 1)) * sizeof(float); };
  const cudaError_t e = prepare_kernel<K>(bytes(most, DFS_MAX_BUCKET_DISTANCE));
  if (e != cudaSuccess) return e;
  K<<<grid, kNT, bytes(tables, P.D), st>>>(P);
  return cudaGetLastError();
}

template <typename E, bool kVec>
cudaError_t fwd(const AttnParams& P, cudaStream_t st) {
  return launch<simt_fwd_kernel<E, kVec>>(dim3((P.nq + kT - 1) / kT, P.H, P.B), 4, P.w != nullptr, 1, st, P);
}
template <typename E, bool kVec>
cudaError_t bwd(const AttnParams& P, cudaStream_t st) {
  const int table = P.w != nullptr, sums = P.dw_part != nullptr;
  if (P.nq > 0 && P.H > 0) {
    const cudaError_t e =
        launch<simt_dq_kernel<E, kVec>>(dim3((P.nq + kT - 1) / kT, P.H, P.B), 5, table, 1, st, P);
    if (e != cudaSuccess) return e;
  }
  if (P.nk == 0) return cudaSuccess;
  return launch<simt_dkv_kernel<E, kVec>>(dim3((P.nk + kT - 1) / kT, P.Hkv, P.B), 6, table + sums, 2, st, P);
}

}  // namespace

cudaError_t launch_attn_simt_fwd(const AttnParams& P, int dtype, bool vec, cudaStream_t st) {
  if (dtype == DFS_F32) return vec ? fwd<float, true>(P, st) : fwd<float, false>(P, st);
  return dtype == DFS_BF16 ? fwd<__nv_bfloat16, false>(P, st) : fwd<__half, false>(P, st);
}
cudaError_t launch_attn_simt_bwd(const AttnParams& P, int dtype, bool vec, cudaStream_t st) {
  if (dtype == DFS_F32) return vec ? bwd<float, true>(P, st) : bwd<float, false>(P, st);
  return dtype == DFS_BF16 ? bwd<__nv_bfloat16, false>(P, st) : bwd<__half, false>(P, st);
}

}  // namespace dfs
