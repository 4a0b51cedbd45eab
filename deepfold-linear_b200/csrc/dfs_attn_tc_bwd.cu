// dfs_attn_tc_bwd.cu -- local attention backward on the tensor cores (bf16, fp16).
//
// Two passes, neither with atomics, so gradients repeat bit for bit:
//   dQ pass   one CTA per 128 queries of a head, over the key tiles they see:
//             S = Q K^T, dP = dO V^T, p = 2^(S - lse), dS = p (dP - D), dQ += dS K;
//             D comes from the rounded O, and D + sum_j dS_ij = sum_j p_ij dP_ij (in
//             fp32) goes to the key pass, whose bias sums cancel within a row;
//   dK/dV pass  one CTA per 128 keys of a key head, over the query tiles (of every
//             head of the group) that see them, on transposed tiles: S^T = K Q^T,
//             dP^T = V dO^T, dV += P^T dO, dK += dS^T Q; and the sums of dS by distance.
// The alternative is one pass with dQ added up in memory: 5 products a tile pair
// instead of 7 and one exponential instead of two, but 32 KB of fp32 atomics (in
// varying order) a tile pair.
//
// Both: warps 0-7 work element by element (a TMEM row and half of a tile's columns
// each), warp 8 issues the MMAs (the next tile's S and dP while this one's
// elements are worked on), warp 9 stages tiles by TMA and announces them.
#include "dfs_attn_tc.cuh"

namespace dfs {
namespace {

constexpr int kBwdThreads = 320;
constexpr int kWork = 256;     // threads of the element warps
constexpr int kStages = 3, kInfo = 4;

// TMEM columns (512 allocated)
constexpr uint32_t kColS = 0, kColDP = 128, kColP = 256, kColDS = 320, kColA = 384, kColB = 448;

struct BwdShared {
  uint64_t own_full, full[kStages], empty[kStages];
  uint64_t s_full, s_free, ds_ready, acc_done;
  TileInfo info[kInfo];
  alignas(16) float stat[kStages][2][kTcRows];  // dK/dV pass: lse and D of the stage's queries
  float half[2][kTcRows];           // dQ pass: two half rows' sums
  float ends[2][kWork / 32];
  float diag[2][kWork / 32][96];    // dK/dV pass: a warp's strip's diagonals, two tiles in turn
  uint32_t tmem;
};

DFS_DEV void work_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <bool BF16>
struct E16 {
  using T = __half;
};
template <>
struct E16<true> {
  using T = __nv_bfloat16;
};

// 32 of a row's gradient values, scaled, to global memory (columns c0.. of d)
template <bool BF16>
DFS_DEV void store_row32(const Strided& s, int b, int h, int row, int c0, int d, const uint32_t (&v)[32], float mul,
                         bool zero) {
  auto* dst = row_ptr<typename E16<BF16>::T>(s, b, h, row) + c0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c0 + 8 * e < d) {
      uint32_t r[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        r[u] = zero ? 0u
                    : pack16<BF16>(__uint_as_float(v[8 * e + 2 * u]) * mul, __uint_as_float(v[8 * e + 2 * u + 1]) * mul);
      *reinterpret_cast<uint4*>(dst + 8 * e) = make_uint4(r[0], r[1], r[2], r[3]);
    }
}

template <bool BF16>
__global__ void __launch_bounds__(kBwdThreads, 1) tc_dq_kernel(const __grid_constant__ TcParams T) {
  extern __shared__ unsigned char raw[];
  const AttnParams& P = T.a;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gen = raw + (base - smem_u32(raw));
  const uint32_t sQ = base, sO = sQ + kTcTileBytes, sK = sO + kTcTileBytes, sV = sK + kStages * kTcTileBytes;
  BwdShared& S = *reinterpret_cast<BwdShared*>(gen + (2 + 2 * kStages) * kTcTileBytes);
  float* tab = reinterpret_cast<float*>(&S + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / P.G;
  const int i0 = (gridDim.x - 1 - blockIdx.x) * kTcRows, p0 = i0 + P.qs;
  bool err = false;
  if (threadIdx.x == 0) {
    mbar_init(&S.own_full, 1);
    for (int s = 0; s < kStages; ++s) mbar_init(&S.full[s], 1), mbar_init(&S.empty[s], 1);
    mbar_init(&S.s_full, 1);
    mbar_init(&S.s_free, kWork);
    mbar_init(&S.ds_ready, kWork);
    mbar_init(&S.acc_done, 1);
    fence_mbar_init();
  }
  if (warp == 8) tmem_alloc(&S.tmem, 512);
  if (P.w) load_bias_ext(tab, P, h, threadIdx.x, kBwdThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = S.tmem;

  if (warp == 9) {  // ---- producer
    const uint8_t* mask = P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr;
    const TcKeyTiles tiles(P, p0, min(i0 + kTcRows, P.nq) - 1 + P.qs);
    if (lane == 0) {
      mbar_arrive_expect_tx(smem_u32(&S.own_full), 2 * kTcTileBytes);
      tma_load_4d(sQ, &T.q, 0, i0, h, b, smem_u32(&S.own_full));
      tma_load_4d(sO, &T.d_o, 0, i0, h, b, smem_u32(&S.own_full));
    }
    int t = 0;
    for (int x = 0; x <= tiles.count(); ++x) {
      const int j0 = x < tiles.count() ? tiles[x] * kTcRows : -1;
      uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
      if (j0 >= 0 && mask != nullptr) {
        key_bits(mask, j0, P.nk, lane, bits);
        if ((bits[0] | bits[1] | bits[2] | bits[3]) == 0) continue;
      }
      const int s = t % kStages;
      if (!mbar_wait(&S.empty[s], ((t / kStages) & 1) ^ 1)) { err = true; break; }
      if (lane == 0) {
        TileInfo& f = S.info[t % kInfo];
        f.at = j0;
#pragma unroll
        for (int w = 0; w < 4; ++w) f.bits[w] = bits[w];
        if (j0 < 0) {
          mbar_arrive(&S.full[s]);
        } else {
          mbar_arrive_expect_tx(smem_u32(&S.full[s]), 2 * kTcTileBytes);
          tma_load_4d(sK + s * kTcTileBytes, &T.k, 0, j0, hk, b, smem_u32(&S.full[s]));
          tma_load_4d(sV + s * kTcTileBytes, &T.v, 0, j0, hk, b, smem_u32(&S.full[s]));
        }
      }
      ++t;
    }
  } else if (warp == 8) {  // ---- MMA
    const int dp = (P.d + 15) / 16 * 16;
    const uint32_t id_s = tc_idesc(128, 128, BF16, false), id_a = tc_idesc(128, dp, BF16, true);
    err = !mbar_wait(&S.own_full, 0);
    auto start = [&](int t, bool& end) {
      const int s = t % kStages;
      if (!mbar_wait(&S.full[s], (t / kStages) & 1)) return false;
      const TileInfo& f = S.info[t % kInfo];
      end = f.at < 0;
      if (!end && P.mask != nullptr) {
        // a hidden key's K may hold anything, and 0 x NaN is NaN in dS K: zero its row
        unsigned char* kt = gen + (2 + s) * kTcTileBytes;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t bw = f.bits[w];
          if (bw != ~0u)
            for (int r = lane / 8; r < 32; r += 4)
              if (!((bw >> r) & 1u))
                *reinterpret_cast<uint4*>(kt + (32 * w + r) * 128 + (lane % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
        __syncwarp();
      }
      if (t > 0 && !mbar_wait(&S.s_free, (t - 1) & 1)) return false;
      tc_fence_after();
      if (lane == 0) {
        if (end) {
          mbar_arrive(&S.s_full);
        } else {
          tc_mma_kk(tm + kColS, sQ, sK + s * kTcTileBytes, id_s, dp / 16);
          tc_mma_kk(tm + kColDP, sO, sV + s * kTcTileBytes, id_s, dp / 16);
          mma_commit(&S.s_full);
        }
      }
      __syncwarp();
      return true;
    };
    bool end = false;
    if (!err) err = !start(0, end);
    for (int t = 0; !end && !err; ++t) {
      bool next_end = false;
      if (!start(t + 1, next_end)) { err = true; break; }
      if (!mbar_wait(&S.ds_ready, t & 1)) { err = true; break; }
      tc_fence_after();
      if (lane == 0) {
        tc_mma_ts(tm + kColA, tm + kColDS, sK + (t % kStages) * kTcTileBytes, id_a, t > 0);
        mma_commit(&S.empty[t % kStages]);
        mma_commit(&S.acc_done);
      }
      __syncwarp();
      end = next_end;
    }
  } else {  // ---- elements: warp w has TMEM lanes 32 (w % 4).. and columns 64 (w / 4)..
    const int row = (warp % 4) * 32 + lane, ch = warp / 4, i = i0 + row, p = p0 + row;
    const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const int E = bias_ext(P.D);
    using T16 = typename E16<BF16>::T;
    const size_t stat = (static_cast<size_t>(b) * P.H + h) * P.nq + i;
    float D = 0.0f;
    if (i < P.nq) {
      const T16* orow = row_ptr<T16>(P.o, b, h, i) + 32 * ch;
      const T16* drow = row_ptr<T16>(P.d_o, b, h, i) + 32 * ch;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (32 * ch + 8 * e < P.d) {
          const uint4 x = *reinterpret_cast<const uint4*>(orow + 8 * e), y = *reinterpret_cast<const uint4*>(drow + 8 * e);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float2 f = unpack16<BF16>(xs[u]), g = unpack16<BF16>(ys[u]);
            D = fmaf(f.x, g.x, fmaf(f.y, g.y, D));
          }
        }
    }
    S.half[ch][row] = D;
    work_barrier();
    D = S.half[0][row] + S.half[1][row];
    const float lse = i < P.nq ? P.lse[stat] : INFINITY;
    float2 rest = make_float2(0.0f, 0.0f);
    int t = 0;
    for (;; ++t) {
      if (!mbar_wait(&S.s_full, t & 1)) { err = true; break; }
      const int j0 = S.info[t % kInfo].at;
      if (j0 < 0) break;
      uint32_t bits[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) bits[w] = S.info[t % kInfo].bits[w];
      tc_fence_after();
      uint32_t sr[2][32], dr[2][32];
#pragma unroll
      for (int w = 0; w < 2; ++w) tmem_ld32_async(tm + lanes + kColS + 64 * ch + 32 * w, sr[w]);
#pragma unroll
      for (int w = 0; w < 2; ++w) tmem_ld32_async(tm + lanes + kColDP + 64 * ch + 32 * w, dr[w]);
#pragma unroll
      for (int w = 0; w < 2; ++w) tmem_wait_ld(sr[w]);
#pragma unroll
      for (int w = 0; w < 2; ++w) tmem_wait_ld(dr[w]);
      tc_fence_before();
      mbar_arrive(&S.s_free);
      float mul = P.scale2, off = -lse;
      if (P.w) {
        const int dlo = p0 - j0 - 127, dhi = p0 - j0 + 127;
        if (dlo >= P.D) {
          off = tab[E + P.D] - lse;
        } else if (dhi <= -P.D) {
          off = tab[E - P.D] - lse;
        } else {
          const float* at = tab + (E + p - j0 - 64 * ch);
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int c = 0; c < 32; ++c)
              sr[w][c] = __float_as_uint(fmaf(__uint_as_float(sr[w][c]), P.scale2, at[-(32 * w + c)]));
          mul = 1.0f;
        }
      }
      if (!all_visible(P, p0, j0) || (bits[0] & bits[1] & bits[2] & bits[3]) != ~0u) {
        // a hidden key's logit is -inf, and its dP (0 or, from hidden memory, anything) is 0
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t vis = (ch ? bits[2 + w] : bits[w]) & row_bits(P, p, j0, 2 * ch + w);
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const bool on = (vis >> c) & 1u;
            sr[w][c] = on ? sr[w][c] : 0xff800000u;
            dr[w][c] = on ? dr[w][c] : 0u;
          }
        }
      }
      if (t > 0 && !mbar_wait(&S.acc_done, (t - 1) & 1)) { err = true; break; }
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        const int w = c / 16, e = 2 * (c % 16);
        float2 x = make_float2(__uint_as_float(sr[w][e]), __uint_as_float(sr[w][e + 1]));
        x = fma2(x, make_float2(mul, mul), make_float2(off, off));
        x = make_float2(ex2(x.x), ex2(x.y));
        const float2 dp = make_float2(__uint_as_float(dr[w][e]), __uint_as_float(dr[w][e + 1]));
        const float2 ds = __fmul2_rn(x, __fadd2_rn(dp, make_float2(-D, -D)));
        rest = __fadd2_rn(rest, ds);
        pk[c] = pack16<BF16>(ds.x, ds.y);
      }
      tmem_st32(tm + lanes + kColDS + 32 * ch, pk);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&S.ds_ready);
    }
    if (!err && t > 0) err = !mbar_wait(&S.acc_done, (t - 1) & 1);
    tc_fence_after();
    uint32_t v[32];
    const int c0 = 32 * ch;
    if (t > 0 && c0 < P.d) {
      tmem_ld32_async(tm + lanes + kColA + c0, v);
      tmem_wait_ld(v);
    }
    if (i < P.nq && c0 < P.d) store_row32<BF16>(P.d_q, b, h, i, c0, P.d, v, P.scale, t == 0);
    work_barrier();
    S.half[ch][row] = rest.x + rest.y;
    work_barrier();
    if (ch == 0 && i < P.nq) P.dsum[stat] = D + (S.half[0][row] + S.half[1][row]);
  }
  if (err) report_timeout(P.status);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tm, 512);
}

template <bool BF16>
__global__ void __launch_bounds__(kBwdThreads, 1) tc_dkv_kernel(const __grid_constant__ TcParams T) {
  extern __shared__ unsigned char raw[];
  const AttnParams& P = T.a;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gen = raw + (base - smem_u32(raw));
  const uint32_t sK = base, sV = sK + kTcTileBytes, sQ = sV + kTcTileBytes, sO = sQ + kStages * kTcTileBytes;
  BwdShared& S = *reinterpret_cast<BwdShared*>(gen + (2 + 2 * kStages) * kTcTileBytes);
  float* tab = reinterpret_cast<float*>(&S + 1);
  const int W = 2 * P.D + 1;
  float* acc = tab + (P.w ? 2 * bias_ext(P.D) + 1 : 0);  // W sums by distance
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int hk = blockIdx.y, b = blockIdx.z, j0 = blockIdx.x * kTcRows;
  bool err = false;
  if (threadIdx.x == 0) {
    mbar_init(&S.own_full, 1);
    for (int s = 0; s < kStages; ++s) mbar_init(&S.full[s], 1), mbar_init(&S.empty[s], 1);
    mbar_init(&S.s_full, 1);
    mbar_init(&S.s_free, kWork);
    mbar_init(&S.ds_ready, kWork);
    mbar_init(&S.acc_done, 1);
    fence_mbar_init();
  }
  if (warp == 8) tmem_alloc(&S.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = S.tmem;

  // queries that see some key of the tile: [i_lo, i_hi)
  int i_lo = P.causal ? j0 - P.qs : j0 - P.window + 1 - P.qs;
  int i_hi = min(j0 + kTcRows, P.nk) - 1 + P.window - P.qs;
  if (j0 < P.sinks) {
    i_hi = P.nq;
    if (!P.causal) i_lo = 0;
  }
  i_lo = max(i_lo, 0) / kTcRows;
  i_hi = (min(i_hi, P.nq) + kTcRows - 1) / kTcRows;  // in tiles

  if (warp == 9) {  // ---- producer
    uint32_t bits[4];
    key_bits(P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr, j0, P.nk, lane, bits);
    const int per = (bits[0] | bits[1] | bits[2] | bits[3]) == 0 ? 0 : max(0, i_hi - i_lo);
    if (lane == 0) {
      mbar_arrive_expect_tx(smem_u32(&S.own_full), 2 * kTcTileBytes);
      tma_load_4d(sK, &T.k, 0, j0, hk, b, smem_u32(&S.own_full));
      tma_load_4d(sV, &T.v, 0, j0, hk, b, smem_u32(&S.own_full));
    }
    const int total = per * P.G;
    for (int t = 0; t <= total; ++t) {
      const int s = t % kStages;
      const int g = t < total ? t / per : 0, h = hk * P.G + g, i0 = t < total ? (i_lo + t % per) * kTcRows : -1;
      float st[2][4];
      if (i0 >= 0) {
        const size_t at = (static_cast<size_t>(b) * P.H + h) * P.nq;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = i0 + 4 * lane + e;
          st[0][e] = i < P.nq ? P.lse[at + i] : INFINITY;
          st[1][e] = i < P.nq ? P.dsum[at + i] : 0.0f;
        }
      }
      if (!mbar_wait(&S.empty[s], ((t / kStages) & 1) ^ 1)) { err = true; break; }
      if (i0 >= 0) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          *reinterpret_cast<float4*>(&S.stat[s][k][4 * lane]) = make_float4(st[k][0], st[k][1], st[k][2], st[k][3]);
      }
      __syncwarp();
      if (lane == 0) {
        TileInfo& f = S.info[t % kInfo];
        f.at = i0;
        f.head = g;
#pragma unroll
        for (int w = 0; w < 4; ++w) f.bits[w] = bits[w];
        if (i0 < 0) {
          mbar_arrive(&S.full[s]);
        } else {
          mbar_arrive_expect_tx(smem_u32(&S.full[s]), 2 * kTcTileBytes);
          tma_load_4d(sQ + s * kTcTileBytes, &T.q, 0, i0, h, b, smem_u32(&S.full[s]));
          tma_load_4d(sO + s * kTcTileBytes, &T.d_o, 0, i0, h, b, smem_u32(&S.full[s]));
        }
      }
    }
  } else if (warp == 8) {  // ---- MMA
    const int dp = (P.d + 15) / 16 * 16;
    const uint32_t id_s = tc_idesc(128, 128, BF16, false), id_a = tc_idesc(128, dp, BF16, true);
    err = !mbar_wait(&S.own_full, 0);
    auto start = [&](int t, bool& end) {
      const int s = t % kStages;
      if (!mbar_wait(&S.full[s], (t / kStages) & 1)) return false;
      end = S.info[t % kInfo].at < 0;
      if (t > 0 && !mbar_wait(&S.s_free, (t - 1) & 1)) return false;
      tc_fence_after();
      if (lane == 0) {
        if (end) {
          mbar_arrive(&S.s_full);
        } else {
          tc_mma_kk(tm + kColS, sK, sQ + s * kTcTileBytes, id_s, dp / 16);
          tc_mma_kk(tm + kColDP, sV, sO + s * kTcTileBytes, id_s, dp / 16);
          mma_commit(&S.s_full);
        }
      }
      __syncwarp();
      return true;
    };
    bool end = false;
    if (!err) err = !start(0, end);
    for (int t = 0; !end && !err; ++t) {
      bool next_end = false;
      if (!start(t + 1, next_end)) { err = true; break; }
      if (!mbar_wait(&S.ds_ready, t & 1)) { err = true; break; }
      tc_fence_after();
      if (lane == 0) {
        const int s = t % kStages;
        tc_mma_ts(tm + kColA, tm + kColP, sO + s * kTcTileBytes, id_a, t > 0);
        tc_mma_ts(tm + kColB, tm + kColDS, sQ + s * kTcTileBytes, id_a, t > 0);
        mma_commit(&S.empty[s]);
        mma_commit(&S.acc_done);
      }
      __syncwarp();
      end = next_end;
    }
  } else {  // ---- elements: a key row and half of the tile's queries per thread
    const int row = (warp % 4) * 32 + lane, ch = warp / 4, j = j0 + row, tid = threadIdx.x;
    const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const int E = bias_ext(P.D);
    const bool dw = P.dw_part != nullptr;
    float lo = 0.0f, hi = 0.0f;  // sums of dS beyond the table's ends
    int head = -1, strip = 0;
    // this head's sums by distance, to memory (the element threads together)
    auto flush = [&]() {
      if (P.D == 0) hi += lo, lo = 0.0f;
      const float a = warp_sum(lo), c = warp_sum(hi);
      if (lane == 0) S.ends[0][warp] = a, S.ends[1][warp] = c;
      work_barrier();
      if (tid < 2 && (P.D > 0 || tid == 1)) {
        float s = 0.0f;
        for (int w = 0; w < kWork / 32; ++w) s += S.ends[tid][w];
        acc[tid == 0 ? 0 : 2 * P.D] += s;
      }
      work_barrier();
      float* dst = P.dw_part + (static_cast<size_t>(hk * P.G + head) * P.parts + b * gridDim.x + blockIdx.x) * W;
      for (int x = tid; x < W; x += kWork) dst[x] = acc[x];
      lo = hi = 0.0f;
    };
    // the heads from `from` on have no tile here: their sums are zero
    auto zero_heads = [&](int from) {
      for (int g = from; g < P.G; ++g) {
        float* dst = P.dw_part + (static_cast<size_t>(hk * P.G + g) * P.parts + b * gridDim.x + blockIdx.x) * W;
        for (int x = tid; x < W; x += kWork) dst[x] = 0.0f;
      }
    };
    int t = 0;
    for (;; ++t) {
      if (!mbar_wait(&S.s_full, t & 1)) { err = true; break; }
      const int i0 = S.info[t % kInfo].at, g = S.info[t % kInfo].head;
      if (i0 < 0) break;
      if (g != head) {
        if (dw && head >= 0) flush();
        work_barrier();  // nobody reads the old tables any more
        head = g;
        if (P.w) load_bias_ext(tab, P, hk * P.G + g, tid, kWork);
        if (dw)
          for (int x = tid; x < W; x += kWork) acc[x] = 0.0f;
        work_barrier();
      }
      const uint32_t kbits = S.info[t % kInfo].bits[warp % 4];
      const bool whole = (S.info[t % kInfo].bits[0] & S.info[t % kInfo].bits[1] & S.info[t % kInfo].bits[2] &
                          S.info[t % kInfo].bits[3]) == ~0u;
      const float* lse = S.stat[t % kStages][0] + 64 * ch;
      const float* Dv = S.stat[t % kStages][1] + 64 * ch;
      tc_fence_after();
      uint32_t sr[2][32], dr[2][32];
#pragma unroll
      for (int w = 0; w < 2; ++w) tmem_ld32_async(tm + lanes + kColS + 64 * ch + 32 * w, sr[w]);
#pragma unroll
      for (int w = 0; w < 2; ++w) tmem_ld32_async(tm + lanes + kColDP + 64 * ch + 32 * w, dr[w]);
#pragma unroll
      for (int w = 0; w < 2; ++w) tmem_wait_ld(sr[w]);
#pragma unroll
      for (int w = 0; w < 2; ++w) tmem_wait_ld(dr[w]);
      tc_fence_before();
      mbar_arrive(&S.s_free);
      const int p0 = i0 + P.qs;
      float mul = P.scale2, add = 0.0f;
      int side = 0;  // where the tile's distances lie: in the table, or beyond an end
      const int dlo = p0 - j0 - 127, dhi = p0 - j0 + 127;
      if (P.w) {
        if (dlo >= P.D) {
          add = tab[E + P.D];
          side = 1;
        } else if (dhi <= -P.D) {
          add = tab[E - P.D];
          side = -1;
        } else {
          const float* at = tab + (E + p0 + 64 * ch - j);
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int c = 0; c < 32; ++c)
              sr[w][c] = __float_as_uint(fmaf(__uint_as_float(sr[w][c]), P.scale2, at[32 * w + c]));
          mul = 1.0f;
        }
      }
      if (!all_visible(P, p0, j0) || !whole) {
        // queries [a, b) of the tile see this key through the window, all from `from` on as a sink
        const bool on = (kbits >> lane) & 1u;
        const int a = P.causal ? j - p0 : j - P.window + 1 - p0, z = j + P.window - p0;
        const int from = P.causal ? j - p0 : 0;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t vis = range_word(a, z, 2 * ch + w);
          if (j < P.sinks) vis |= range_word(from, kTcRows, 2 * ch + w);
          if (!on) vis = 0;
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const bool k = (vis >> c) & 1u;
            sr[w][c] = k ? sr[w][c] : 0xff800000u;
            dr[w][c] = k ? dr[w][c] : 0u;
          }
        }
      }
      if (t > 0 && !mbar_wait(&S.acc_done, (t - 1) & 1)) { err = true; break; }
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 32; c += 2) {  // four queries
        const int w = c / 16, e = 2 * (c % 16);
        const float4 ls = *reinterpret_cast<const float4*>(lse + 2 * c);
        const float4 dd = *reinterpret_cast<const float4*>(Dv + 2 * c);
        const float2 l2[2] = {make_float2(ls.x, ls.y), make_float2(ls.z, ls.w)};
        const float2 d2[2] = {make_float2(dd.x, dd.y), make_float2(dd.z, dd.w)};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float2 x = make_float2(__uint_as_float(sr[w][e + 2 * u]), __uint_as_float(sr[w][e + 2 * u + 1]));
          x = fma2(x, make_float2(mul, mul), fma2(l2[u], make_float2(-1.0f, -1.0f), make_float2(add, add)));
          x = make_float2(ex2(x.x), ex2(x.y));
          pk[c + u] = pack16<BF16>(x.x, x.y);
          const float2 dp = make_float2(__uint_as_float(dr[w][e + 2 * u]), __uint_as_float(dr[w][e + 2 * u + 1]));
          const float2 ds = __fmul2_rn(x, fma2(d2[u], make_float2(-1.0f, -1.0f), dp));
          dr[w][e + 2 * u] = __float_as_uint(ds.x);
          dr[w][e + 2 * u + 1] = __float_as_uint(ds.y);
        }
      }
      tmem_st32(tm + lanes + kColP + 32 * ch, pk);
#pragma unroll
      for (int c = 0; c < 32; ++c)
        pk[c] = pack16<BF16>(__uint_as_float(dr[c / 16][2 * (c % 16)]), __uint_as_float(dr[c / 16][2 * (c % 16) + 1]));
      tmem_st32(tm + lanes + kColDS + 32 * ch, pk);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&S.ds_ready);
      if (dw) {
        if (side != 0) {
          float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int c = 0; c < 32; ++c)
            s2 = __fadd2_rn(s2, make_float2(__uint_as_float(dr[c / 16][2 * (c % 16)]),
                                            __uint_as_float(dr[c / 16][2 * (c % 16) + 1])));
          if (side > 0) hi += s2.x + s2.y;
          else lo += s2.x + s2.y;
        } else {
          // Diagonals of this warp's strip (32 keys x 64 queries): the running sum of a diagonal moves one
          // lane up as the query advances, and is complete once lane 31 has added its element.
          float* out = S.diag[strip][warp];
          float run = 0.0f;
#pragma unroll
          for (int c = 0; c < 64; ++c) {
            run += __uint_as_float(dr[c / 32][c % 32]);
            if (c < 63) {
              if (lane == 31) out[c] = run;
              run = __shfl_up_sync(0xffffffffu, run, 1);
              if (lane == 0) run = 0.0f;
            }
          }
          out[94 - lane] = run;  // slot x + 31 for diagonal x = query - key of the strip
          work_barrier();
          if (tid < 2 * kTcRows - 1) {
            const int e = tid - (kTcRows - 1);  // query - key within the tile
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kWork / 32; ++w) {
              const int x = e - 64 * (w / 4) + 32 * (w % 4) + 31;
              if (x >= 0 && x < 95) s += S.diag[strip][w][x];
            }
            const int delta = p0 - j0 + e;
            if (delta <= -P.D) lo += s;
            else if (delta >= P.D) hi += s;
            else acc[delta + P.D] += s;
          }
          strip ^= 1;
        }
      }
    }
    if (dw) {
      if (head >= 0) flush();
      zero_heads(head + 1);
    }
    if (!err && t > 0) err = !mbar_wait(&S.acc_done, (t - 1) & 1);
    tc_fence_after();
    const int c0 = 32 * ch;
    if (c0 < P.d) {
      uint32_t v[32];
      if (t > 0) {
        tmem_ld32_async(tm + lanes + kColA + c0, v);
        tmem_wait_ld(v);
      }
      if (j < P.nk) store_row32<BF16>(P.d_v, b, hk, j, c0, P.d, v, 1.0f, t == 0);
      if (t > 0) {
        tmem_ld32_async(tm + lanes + kColB + c0, v);
        tmem_wait_ld(v);
      }
      if (j < P.nk) store_row32<BF16>(P.d_k, b, hk, j, c0, P.d, v, P.scale, t == 0);
    }
  }
  if (err) report_timeout(P.status);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tm, 512);
}

}  // namespace

cudaError_t launch_attn_tc_bwd(const AttnParams& P, int dtype, cudaStream_t st) {
  const bool bf16 = dtype == DFS_BF16;
  TcParams T;
  T.a = P;
  if (!tc_tmap(&T.q, P.q, bf16, P.d, P.nq, P.H, P.B) || !tc_tmap(&T.k, P.k, bf16, P.d, P.nk, P.Hkv, P.B) ||
      !tc_tmap(&T.v, P.v, bf16, P.d, P.nk, P.Hkv, P.B) || !tc_tmap(&T.d_o, P.d_o, bf16, P.d, P.nq, P.H, P.B))
    return cudaErrorInvalidValue;
  const size_t smem = 1024 + (2 + 2 * kStages) * kTcTileBytes + sizeof(BwdShared) + bias_ext_bytes(P) +
                      (P.w ? (2 * P.D + 1) * sizeof(float) : 0);
  auto dq = bf16 ? tc_dq_kernel<true> : tc_dq_kernel<false>;
  auto dkv = bf16 ? tc_dkv_kernel<true> : tc_dkv_kernel<false>;
  cudaError_t e = cudaFuncSetAttribute(dq, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(dkv, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  dq<<<dim3((P.nq + kTcRows - 1) / kTcRows, P.H, P.B), kBwdThreads, smem, st>>>(T);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  dkv<<<dim3((P.nk + kTcRows - 1) / kTcRows, P.Hkv, P.B), kBwdThreads, smem, st>>>(T);
  return cudaGetLastError();
}

}  // namespace dfs
