// dfs_attn_decode.cu -- local attention for one query per sequence over a cache
// (bf16, fp16 whose rows can be copied in 16-byte pieces).
//
// Reading the visible cache rows is all the time there is: 256 bytes of K and V
// a key at d = 64 for 4 d operations a query head.  A cluster of up to 8 CTAs
// shares one key head of one sequence and splits its visible keys (the sinks,
// then the window, as one list) into equal runs; each CTA copies tiles of 64 keys
// through a ring of shared-memory stages and its 4 warps take 16 keys each:
// S = Q K^T and O += P V for the group's heads as mma.sync m16n8k16 (16 heads by
// 8 keys; the tensor-core rate does not matter here, the small shape does).  Every
// warp keeps its own maximum and sum; warps join through shared memory, CTAs
// through distributed shared memory, in a fixed order and without a second launch.
#include <type_traits>

#include "dfs_attn.cuh"

namespace dfs {
namespace {

constexpr int kThreads = 128;
constexpr int kKeys = 64;          // keys of a tile
constexpr int kStages = 3;
constexpr int kHeads = 16;         // query heads of a CTA: the rows of an m16n8k16 product
constexpr int kPitch = 72;         // elements of a staged row: 144 bytes keep ldmatrix free of conflicts
constexpr int kTileElems = kKeys * kPitch;
constexpr int kMaxSplit = 8;

struct DecodeShared {
  float m[4][kHeads], l[4][kHeads];       // the warps' maxima and sums
  float cm[kHeads], cl[kHeads];           // the CTA's, read by the cluster
  float o[kHeads][68];                    // the CTA's sums of P V, read by the cluster
};

DFS_DEV void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {  // bytes 16, or 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
DFS_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
DFS_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

DFS_DEV void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
DFS_DEV void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <bool BF16>
DFS_DEV void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF16>
DFS_DEV uint32_t pack(float lo, float hi) {
  uint32_t r;
  if (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// grid (split, key heads x head chunks, batch), clusters of `split` CTAs
template <typename E>
__global__ void __launch_bounds__(kThreads) decode_mma_kernel(AttnParams P, int split, int chunks) {
  constexpr bool BF16 = std::is_same<E, __nv_bfloat16>::value;
  extern __shared__ __align__(16) unsigned char raw[];
  E* stage = reinterpret_cast<E*>(raw);  // [kStages][2][kKeys][kPitch]: K, V
  DecodeShared& S = *reinterpret_cast<DecodeShared*>(raw + kStages * 2 * kTileElems * sizeof(E));
  float* tab = reinterpret_cast<float*>(&S + 1);  // [heads][D + 1] bias of delta = 0 .. D
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, rank = blockIdx.x;
  const int hk = blockIdx.y / chunks, g0 = blockIdx.y % chunks * kHeads, b = blockIdx.z;
  const int ng = min(kHeads, P.G - g0), h0 = hk * P.G + g0;
  const int len = min(max(P.lengths[b], 0), P.nk), p = len - 1;
  const int lo = max(0, len - P.window), ns = min(P.sinks, lo), total = ns + (len - lo);
  const int tiles = (total + kKeys - 1) / kKeys, per = (tiles + split - 1) / split;
  const int t0 = min(rank * per, tiles), t1 = min(t0 + per, tiles);
  const int ksteps = (P.d + 15) / 16, pieces = 2 * ksteps;

  const E* kb = row_ptr<E>(P.k, b, hk, 0);
  const E* vb = row_ptr<E>(P.v, b, hk, 0);
  auto load = [&](int t) {  // one commit group, empty beyond the run
    if (t < t1) {
      E* ks = stage + (t - t0) % kStages * 2 * kTileElems;
      const int c = tid % 8;
#pragma unroll
      for (int r = tid / 8; r < kKeys; r += kThreads / 8) {
        const int x = t * kKeys + r, j = x < ns ? x : lo + (x - ns);
        if (c < pieces) {
          const uint32_t bytes = x < total && 8 * c < P.d ? 16u : 0u;  // rows and columns beyond: zeros
          const int64_t jj = bytes ? j : 0;
          const int cc = bytes ? 8 * c : 0;
          cp_async16(smem_u32(ks + r * kPitch + 8 * c), kb + jj * P.k.sn + cc, bytes);
          cp_async16(smem_u32(ks + kTileElems + r * kPitch + 8 * c), vb + jj * P.v.sn + cc, bytes);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load(t0 + s);

  // Q as the A operand: rows lane / 4 and + 8, columns 2 (lane % 4).. of each k step
  const int g = lane / 4, q2 = 2 * (lane % 4);
  uint32_t qa[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = g + 8 * (e & 1), col = 16 * k + q2 + 8 * (e >> 1);
      qa[k][e] = 0;
      if (row < ng && col < P.d) qa[k][e] = *reinterpret_cast<const uint32_t*>(row_ptr<E>(P.q, b, h0 + row, 0) + col);
    }
  // the far bias of this thread's two heads; the table where this run comes near the query
  float far[2] = {0.0f, 0.0f};
  const int last = t1 > t0 ? min(t1 * kKeys, total) - 1 : -1;  // the run's newest key
  const bool near_run = P.w && last >= 0 && p - (last < ns ? last : lo + (last - ns)) < P.D;
  if (P.w) {
    const int bk = min(max(P.lut[2 * P.D], 0), P.nb - 1);
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (g + 8 * r < ng) far[r] = load_as_f32<void>(P.w, static_cast<size_t>(h0 + g + 8 * r) * P.nb + bk, P.wdtype) * kLog2e;
  }
  if (near_run)
    for (int x = tid; x < ng * (P.D + 1); x += kThreads) {
      const int bk = min(max(P.lut[P.D + x % (P.D + 1)], 0), P.nb - 1);
      tab[x] = load_as_f32<void>(P.w, static_cast<size_t>(h0 + x / (P.D + 1)) * P.nb + bk, P.wdtype) * kLog2e;
    }

  float o[8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;

  for (int t = t0; t < t1; ++t) {
    cp_async_wait<kStages - 2>();
    __syncthreads();  // tile t is in; everybody is done with tile t - 1
    load(t + kStages - 1);
    const E* ks = stage + (t - t0) % kStages * 2 * kTileElems + 16 * warp * kPitch;
    const E* vs = ks + kTileElems;
    float s[2][4] = {};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < ksteps) {
        uint32_t kf[4];
        ldsm4(smem_u32(ks + ((lane / 16) * 8 + lane % 8) * kPitch + 16 * k + (lane / 8 % 2) * 8), kf);
        mma16<BF16>(s[0], qa[k], kf[0], kf[1]);
        mma16<BF16>(s[1], qa[k], kf[2], kf[3]);
      }
    const int x0 = t * kKeys + 16 * warp + q2;
    const int xl = min(t * kKeys + 16 * warp + 15, total - 1);
    const bool near = near_run && p - (xl < ns ? xl : lo + (xl - ns)) < P.D;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int x = x0 + 8 * n + (e & 1), r = e >> 1;
        float bias = far[r];
        if (near && x < total && g + 8 * r < ng) {
          const int j = x < ns ? x : lo + (x - ns);
          bias = tab[(g + 8 * r) * (P.D + 1) + min(p - j, P.D)];
        }
        s[n][e] = x < total ? fmaf(s[n][e], P.scale2, bias) : -INFINITY;
        top[r] = fmaxf(top[r], s[n][e]);
      }
    uint32_t pa[4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float mn = fmaxf(m[r], top[r]), ref = mn == -INFINITY ? 0.0f : mn;
      const float shrink = ex2(m[r] - ref);
      m[r] = mn;
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float a = ex2(s[n][2 * r] - ref), c = ex2(s[n][2 * r + 1] - ref);
        sum += a + c;
        pa[2 * n + r] = pack<BF16>(a, c);
      }
      l[r] = l[r] * shrink + sum;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        o[n][2 * r] *= shrink;
        o[n][2 * r + 1] *= shrink;
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (n < ksteps) {
        uint32_t vf[4];
        ldsm4t(smem_u32(vs + (lane % 16) * kPitch + 16 * n + (lane / 16) * 8), vf);
        mma16<BF16>(o[2 * n], pa, vf[0], vf[1]);
        mma16<BF16>(o[2 * n + 1], pa, vf[2], vf[3]);
      }
  }
  cp_async_wait<0>();
  // join the warps: maxima and sums, then each warp in turn adds its part
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (lane % 4 == 0) {
      S.m[warp][g + 8 * r] = m[r];
      S.l[warp][g + 8 * r] = l[r];
    }
  }
  __syncthreads();
  float f[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = g + 8 * r;
    const float top = fmaxf(fmaxf(S.m[0][row], S.m[1][row]), fmaxf(S.m[2][row], S.m[3][row]));
    const float ref = top == -INFINITY ? 0.0f : top;
    f[r] = ex2(m[r] - ref);
    if (warp == 0 && lane % 4 == 0) {
      S.cm[row] = top;
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) sum += S.l[w][row] * ex2(S.m[w][row] - ref);
      S.cl[row] = sum;
    }
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (warp == w)
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float* at = &S.o[g + 8 * (e >> 1)][8 * n + q2 + (e & 1)];
          const float v = o[n][e] * f[e >> 1];
          *at = w == 0 ? v : *at + v;
        }
    __syncthreads();
  }
  // join the CTAs: this one finishes every split-th head
  if (split > 1) cluster_sync();
  for (int x = tid; x < ng * P.d; x += kThreads) {
    const int head = x / P.d, c = x % P.d;
    if (head % split != rank) continue;
    float top = -INFINITY, sum = 0.0f, acc = 0.0f;
    if (split == 1) {
      sum = S.cl[head];
      acc = S.o[head][c];
    } else {
      const uint32_t am = smem_u32(&S.cm[head]), al = smem_u32(&S.cl[head]), ao = smem_u32(&S.o[head][c]);
      for (int r = 0; r < split; ++r) top = fmaxf(top, dsmem_ld(dsmem_addr(am, r)));
      const float ref = top == -INFINITY ? 0.0f : top;
      for (int r = 0; r < split; ++r) {
        const float k = ex2(dsmem_ld(dsmem_addr(am, r)) - ref);
        sum += dsmem_ld(dsmem_addr(al, r)) * k;
        acc += dsmem_ld(dsmem_addr(ao, r)) * k;
      }
    }
    row_ptr<E>(P.o, b, h0 + head, 0)[c] = from_f32<E>(sum > 0.0f ? acc / sum : 0.0f);
  }
  if (split > 1) cluster_sync();  // nobody leaves while its memory is read
}

template <typename E>
cudaError_t launch(const AttnParams& P, cudaStream_t st) {
  const int chunks = (P.G + kHeads - 1) / kHeads, heads = P.G < kHeads ? P.G : kHeads;
  // CTAs: about four an SM (as many as its shared memory holds), so that short batches are split and large
  // ones are not, with a tile of keys for each at least
  const long problems = static_cast<long>(P.B) * P.Hkv * chunks;
  const long seen = P.window < P.nk ? static_cast<long>(P.window) + P.sinks : P.nk;
  const long tiles = ((seen < P.nk ? seen : P.nk) + kKeys - 1) / kKeys;
  int split = 1;
  while (split < kMaxSplit && split * problems < 4 * 148 && 2 * split <= tiles) split *= 2;
  const size_t smem = kStages * 2 * kTileElems * sizeof(E) + sizeof(DecodeShared) +
                      (P.w ? heads * (P.D + 1) * sizeof(float) : 0);
  auto kern = decode_mma_kernel<E>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(split, P.Hkv * chunks, P.B);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, P, split, chunks);
}

}  // namespace

cudaError_t launch_decode_mma(const AttnParams& P, int dtype, cudaStream_t st) {
  return dtype == DFS_BF16 ? launch<__nv_bfloat16>(P, st) : launch<__half>(P, st);
}

}  // namespace dfs
