// dfs_attn_tc.cu -- local attention forward on the tensor cores (bf16, fp16).
//
// One CTA owns 128 queries of one head and walks the tiles of 128 keys that they
// see.  Warps 0-3 hold a query row per thread: they read S = Q K^T from TMEM,
// keep the running maximum and sum, and write P (16 bit) back to TMEM, from where
// it is the A operand of O += P V.  Warp 4 issues the MMAs (the next tile's S
// while this one's exponentials run), warp 5 stages K and V by TMA and finds the
// tiles; a tile whose keys are all masked is never announced.
#include "dfs_attn_tc.cuh"

namespace dfs {
namespace {

constexpr int kFwdThreads = 192;
constexpr int kKStages = 3, kVStages = 2, kInfo = 4;
// the running maximum may lag by this much (log2) before O is rescaled: P stays
// below 2^8, far inside fp16, and the sums are fp32
constexpr float kLag = 8.0f;

struct FwdShared {
  uint64_t q_full, k_full[kKStages], k_empty[kKStages], v_full[kVStages], v_empty[kVStages];
  uint64_t s_full, s_free, p_ready, pv_done;
  TileInfo info[kInfo];
  uint32_t tmem;
};

// TMEM columns: S 0-127, P 128-191, O 192-255
constexpr uint32_t kColS = 0, kColP = 128, kColO = 192;

template <bool BF16>
__global__ void __launch_bounds__(kFwdThreads, 2) tc_fwd_kernel(const __grid_constant__ TcParams T) {
  extern __shared__ unsigned char raw[];
  const AttnParams& P = T.a;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gen = raw + (base - smem_u32(raw));
  const uint32_t sQ = base, sK = base + kTcTileBytes, sV = sK + kKStages * kTcTileBytes;
  FwdShared& S = *reinterpret_cast<FwdShared*>(gen + (1 + kKStages + kVStages) * kTcTileBytes);
  float* tab = reinterpret_cast<float*>(&S + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / P.G;
  const int i0 = (gridDim.x - 1 - blockIdx.x) * kTcRows;  // causal: the longest rows first
  const int p0 = i0 + P.qs;
  bool err = false;
  if (threadIdx.x == 0) {
    mbar_init(&S.q_full, 1);
    for (int s = 0; s < kKStages; ++s) mbar_init(&S.k_full[s], 1), mbar_init(&S.k_empty[s], 1);
    for (int s = 0; s < kVStages; ++s) mbar_init(&S.v_full[s], 1), mbar_init(&S.v_empty[s], 1);
    mbar_init(&S.s_full, 1);
    mbar_init(&S.s_free, 128);
    mbar_init(&S.p_ready, 128);
    mbar_init(&S.pv_done, 1);
    fence_mbar_init();
  }
  if (warp == 4) tmem_alloc(&S.tmem, 256);
  if (P.w) load_bias_ext(tab, P, h, threadIdx.x, kFwdThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = S.tmem;

  if (warp == 5) {  // ---- producer
    const uint8_t* mask = P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr;
    const TcKeyTiles tiles(P, p0, min(i0 + kTcRows, P.nq) - 1 + P.qs);
    if (lane == 0) {
      mbar_arrive_expect_tx(smem_u32(&S.q_full), kTcTileBytes);
      tma_load_4d(sQ, &T.q, 0, i0, h, b, smem_u32(&S.q_full));
    }
    int t = 0;
    for (int x = 0; x <= tiles.count() && !err; ++x) {
      const int j0 = x < tiles.count() ? tiles[x] * kTcRows : -1;
      uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
      if (j0 >= 0 && mask != nullptr) {
        key_bits(mask, j0, P.nk, lane, bits);
        if ((bits[0] | bits[1] | bits[2] | bits[3]) == 0) continue;
      }
      const int ks = t % kKStages, vs = t % kVStages;
      if (!mbar_wait(&S.k_empty[ks], ((t / kKStages) & 1) ^ 1)) { err = true; break; }
      if (lane == 0) {
        TileInfo& f = S.info[t % kInfo];
        f.at = j0;
#pragma unroll
        for (int w = 0; w < 4; ++w) f.bits[w] = bits[w];
        if (j0 < 0) {
          mbar_arrive(&S.k_full[ks]);
        } else {
          mbar_arrive_expect_tx(smem_u32(&S.k_full[ks]), kTcTileBytes);
          tma_load_4d(sK + ks * kTcTileBytes, &T.k, 0, j0, hk, b, smem_u32(&S.k_full[ks]));
        }
      }
      if (j0 < 0) break;
      if (!mbar_wait(&S.v_empty[vs], ((t / kVStages) & 1) ^ 1)) { err = true; break; }
      if (lane == 0) {
        mbar_arrive_expect_tx(smem_u32(&S.v_full[vs]), kTcTileBytes);
        tma_load_4d(sV + vs * kTcTileBytes, &T.v, 0, j0, hk, b, smem_u32(&S.v_full[vs]));
      }
      ++t;
    }
  } else if (warp == 4) {  // ---- MMA
    const uint32_t id_s = tc_idesc(128, 128, BF16, false);
    const int dp = (P.d + 15) / 16 * 16;
    const uint32_t id_o = tc_idesc(128, dp, BF16, true);
    err = !mbar_wait(&S.q_full, 0);
    // announce tile t: its S, or the end
    auto start = [&](int t, bool& end) {
      const int ks = t % kKStages;
      if (!mbar_wait(&S.k_full[ks], (t / kKStages) & 1)) return false;
      end = S.info[t % kInfo].at < 0;
      if (t > 0 && !mbar_wait(&S.s_free, (t - 1) & 1)) return false;
      tc_fence_after();
      if (lane == 0) {
        if (end) {
          mbar_arrive(&S.s_full);
        } else {
          tc_mma_kk(tm + kColS, sQ, sK + ks * kTcTileBytes, id_s, dp / 16);
          mma_commit(&S.k_empty[ks]);
          mma_commit(&S.s_full);
        }
      }
      __syncwarp();
      return true;
    };
    bool end = false;
    if (!err) err = !start(0, end);
    for (int t = 0; !end && !err; ++t) {
      uint32_t bits[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) bits[w] = S.info[t % kInfo].bits[w];
      bool next_end = false;
      if (!start(t + 1, next_end)) { err = true; break; }
      const int vs = t % kVStages;
      if (!mbar_wait(&S.v_full[vs], (t / kVStages) & 1)) { err = true; break; }
      if (P.mask != nullptr && (bits[0] & bits[1] & bits[2] & bits[3]) != ~0u) {
        // a hidden key's V may hold anything, and 0 x NaN is NaN: zero its row
        unsigned char* vt = gen + (1 + kKStages + vs) * kTcTileBytes;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          for (int r = lane / 8; r < 32; r += 4)
            if (!((bits[w] >> r) & 1u))
              *reinterpret_cast<uint4*>(vt + (32 * w + r) * 128 + (lane % 8) * 16) = make_uint4(0, 0, 0, 0);
        fence_async_smem();
        __syncwarp();
      }
      if (!mbar_wait(&S.p_ready, t & 1)) { err = true; break; }
      tc_fence_after();
      if (lane == 0) {
        tc_mma_ts(tm + kColO, tm + kColP, sV + vs * kTcTileBytes, id_o, t > 0);
        mma_commit(&S.v_empty[vs]);
        mma_commit(&S.pv_done);
      }
      __syncwarp();
      end = next_end;
    }
  } else {  // ---- softmax: a query row per thread
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const int row = warp * 32 + lane, i = i0 + row, p = p0 + row;
    const int E = bias_ext(P.D);
    float m = -INFINITY, l = 0.0f;
    int t = 0;
    for (;; ++t) {
      if (!mbar_wait(&S.s_full, t & 1)) { err = true; break; }
      const int j0 = S.info[t % kInfo].at;
      if (j0 < 0) break;
      uint32_t bits[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) bits[w] = S.info[t % kInfo].bits[w];
      tc_fence_after();
      uint32_t sr[4][32];
#pragma unroll
      for (int w = 0; w < 4; ++w) tmem_ld32_async(tm + lanes + kColS + 32 * w, sr[w]);
#pragma unroll
      for (int w = 0; w < 4; ++w) tmem_wait_ld(sr[w]);
      tc_fence_before();
      mbar_arrive(&S.s_free);
      // logits in log2 units are mul * s + add
      float mul = P.scale2, add = 0.0f;
      if (P.w) {
        const int dlo = p0 - j0 - 127, dhi = p0 - j0 + 127;
        if (dlo >= P.D) {
          add = tab[E + P.D];
        } else if (dhi <= -P.D) {
          add = tab[E - P.D];
        } else {
          const float* at = tab + (E + p - j0);
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int c = 0; c < 32; ++c)
              sr[w][c] = __float_as_uint(fmaf(__uint_as_float(sr[w][c]), P.scale2, at[-(32 * w + c)]));
          mul = 1.0f;
        }
      }
      if (!all_visible(P, p0, j0) || (bits[0] & bits[1] & bits[2] & bits[3]) != ~0u) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t vis = bits[w] & row_bits(P, p, j0, w);
#pragma unroll
          for (int c = 0; c < 32; ++c) sr[w][c] = (vis >> c) & 1u ? sr[w][c] : 0xff800000u;
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float v[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(sr[w][c]);
        top = fmaxf(top, max32(v));
      }
      top = fmaf(top, mul, add);
      if (t > 0 && !mbar_wait(&S.pv_done, (t - 1) & 1)) { err = true; break; }
      const bool raise = top > m + kLag || (m == -INFINITY && top > -INFINITY);
      if (__any_sync(0xffffffffu, raise)) {
        const float mn = raise ? top : m;
        const float f = raise ? ex2(m - mn) : 1.0f;  // m = -inf: 0, and O is 0 there
        m = mn;
        l *= f;
        if (t > 0) {
          tc_fence_after();
          for (int c = 0; c < P.d; c += 32) {
            uint32_t o[32];
            tmem_ld32_async(tm + lanes + kColO + c, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st32(tm + lanes + kColO + c, o);
          }
        }
      }
      const float off = add - (m == -INFINITY ? 0.0f : m);
      float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const int w = 2 * half + c / 16, e = 2 * (c % 16);
          float2 x = make_float2(__uint_as_float(sr[w][e]), __uint_as_float(sr[w][e + 1]));
          x = fma2(x, make_float2(mul, mul), make_float2(off, off));
          x = make_float2(ex2(x.x), ex2(x.y));
          sum = __fadd2_rn(sum, x);
          pk[c] = pack16<BF16>(x.x, x.y);
        }
        tmem_st32(tm + lanes + kColP + 32 * half, pk);
      }
      l += sum.x + sum.y;
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&S.p_ready);
    }
    if (!err && t > 0) err = !mbar_wait(&S.pv_done, (t - 1) & 1);
    tc_fence_after();
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    using E16 = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    for (int c0 = 0; c0 < P.d; c0 += 32) {
      uint32_t o[32];
      if (t > 0) {  // warp-collective
        tmem_ld32_async(tm + lanes + kColO + c0, o);
        tmem_wait_ld(o);
      }
      if (i < P.nq) {
        E16* dst = row_ptr<E16>(P.o, b, h, i) + c0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c0 + 8 * e < P.d) {
            uint32_t r[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              r[u] = l > 0.0f ? pack16<BF16>(__uint_as_float(o[8 * e + 2 * u]) * inv,
                                             __uint_as_float(o[8 * e + 2 * u + 1]) * inv)
                              : 0u;
            *reinterpret_cast<uint4*>(dst + 8 * e) = make_uint4(r[0], r[1], r[2], r[3]);
          }
      }
    }
    if (P.lse && i < P.nq)
      P.lse[(static_cast<size_t>(b) * P.H + h) * P.nq + i] = l > 0.0f ? m + lg2(l) : INFINITY;
  }
  if (err) report_timeout(P.status);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 4) tmem_dealloc(tm, 256);
}

}  // namespace

bool tc_tmap(CUtensorMap* tm, const Strided& s, bool bf16, int d, int n, int heads, int B) {
  return make_tmap_4d(tm, s.p, bf16 ? DFS_BF16 : DFS_F16, d, n, heads, B, s.sn, s.sh, s.sb, 64, kTcRows);
}

cudaError_t launch_attn_tc_fwd(const AttnParams& P, int dtype, cudaStream_t st) {
  const bool bf16 = dtype == DFS_BF16;
  TcParams T;
  T.a = P;
  if (!tc_tmap(&T.q, P.q, bf16, P.d, P.nq, P.H, P.B) || !tc_tmap(&T.k, P.k, bf16, P.d, P.nk, P.Hkv, P.B) ||
      !tc_tmap(&T.v, P.v, bf16, P.d, P.nk, P.Hkv, P.B))
    return cudaErrorInvalidValue;
  T.d_o = T.q;
  const size_t smem = 1024 + (1 + kKStages + kVStages) * kTcTileBytes + sizeof(FwdShared) + bias_ext_bytes(P);
  auto kern = bf16 ? tc_fwd_kernel<true> : tc_fwd_kernel<false>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  kern<<<dim3((P.nq + kTcRows - 1) / kTcRows, P.H, P.B), kFwdThreads, smem, st>>>(T);
  return cudaGetLastError();
}

}  // namespace dfs
