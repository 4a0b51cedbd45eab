// dfs_attn_tc.cu -- local attention forward on the tensor cores (bf16, fp16).
//
// One CTA owns 128 queries of one head and walks the tiles of 128 keys that they
// see.  Warps 0-7 work on S = Q K^T element by element, a TMEM row and half of the
// tile's columns per thread: running maximum (joined between a row's two threads)
// and sum, and P (16 bit) back to TMEM, from where it is the A operand of
// O += P V.  Warp 8 issues the MMAs (the next tile's S while this one's
// exponentials run), warp 9 stages K and V by TMA and finds the tiles; a tile
// whose keys are all masked is never announced, and a warp does nothing for a
// block of 32 x 32 pairs that are all hidden.
//
// At d <= 64 the exponentials bound it: 16384 a tile at 16 a clock are 1024
// clocks, the two products 512.  So part of them run on the FMA pipes, and two
// CTAs share an SM (256 of its 512 TMEM columns each), with 16 element warps
// between them to cover TMEM and barrier latencies.
#include <type_traits>

#include "dfs_attn_tc.cuh"

namespace dfs {
namespace {

// 384 threads x 80 registers at launch = 256 x 104 (elements) + 128 x 32 (MMA, TMA and two idle warps)
constexpr int kFwdThreads = 384;
constexpr int kElementRegs = 104, kOtherRegs = 32;
static_assert(256 * kElementRegs + 128 * kOtherRegs <= kFwdThreads * 80, "register shares");
constexpr int kWork = 256;  // threads of the element warps
constexpr int kKStages = 3, kVStages = 2, kInfo = 4;
// the running maximum may lag by this much (log2) before O is rescaled: P stays
// below 2^8, far inside fp16, and the sums are fp32
constexpr float kLag = 8.0f;
// below any sum with a visible key in it (which holds a term of at least 2^-8)
constexpr float kNone = 1e-30f;
constexpr int kPolyEvery = 3;

struct FwdShared {
  uint64_t q_full, k_full[kKStages], k_empty[kKStages], v_full[kVStages], v_empty[kVStages];
  uint64_t s_full, s_free, p_ready, pv_done;
  TileInfo info[kInfo];
  float top[2][2][kTcRows];  // a row's two maxima, two tiles in turn
  float sum[2][kTcRows];
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
  const int warp = warp_index(), lane = threadIdx.x % 32;
  const int h = blockIdx.x % P.H, b = blockIdx.x / P.H % P.B, hk = h / P.G;
  const int i0 = ((P.nq - 1) / kTcRows - static_cast<int>(blockIdx.x / P.H / P.B)) * kTcRows;  // causal: longest first
  const int p0 = i0 + P.qs;
  bool err = false;
  if (warp >= 8) {
    regs_down<kOtherRegs>();  // one instruction for the whole warpgroup
    if (warp == 9) {  // ---- producer
      if (lane == 0) {
        prefetch_tmap(&T.q);
        prefetch_tmap(&T.k);
        prefetch_tmap(&T.v);
        mbar_init(&S.q_full, 1);
        for (int s = 0; s < kKStages; ++s) mbar_init(&S.k_full[s], 1), mbar_init(&S.k_empty[s], 1);
        for (int s = 0; s < kVStages; ++s) mbar_init(&S.v_full[s], 1), mbar_init(&S.v_empty[s], 1);
        mbar_init(&S.s_full, 1);
        mbar_init(&S.s_free, kWork);
        mbar_init(&S.p_ready, kWork);
        mbar_init(&S.pv_done, 1);
        fence_mbar_init();
      }
      __syncwarp();
      setup_arrive<kFwdThreads>();
      const uint8_t* mask = P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr;
      const TcKeyTiles<kTcRows> tiles(P, p0, min(i0 + kTcRows, P.nq) - 1 + P.qs);
      if (lane == 0) {
        mbar_arrive_expect_tx(smem_u32(&S.q_full), kTcTileBytes);
        tma_load_4d(sQ, &T.q, 0, i0, h, b, smem_u32(&S.q_full));
      }
      int t = 0;
      for (int x = 0; x <= tiles.count(); ++x) {
        const int j0 = x < tiles.count() ? tiles[x] * kTcRows : -1;
        uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
        if (j0 >= 0 && mask != nullptr) {
          key_bits(mask, j0, P.nk, lane, bits);
          if ((bits[0] | bits[1] | bits[2] | bits[3]) == 0) continue;
        }
        const int ks = t % kKStages, vs = t % kVStages;
        if (!tc_wait(&S.k_empty[ks], ((t / kKStages) & 1) ^ 1)) { err = true; break; }
        if (lane == 0 && j0 >= 0) {
          mbar_expect_tx(smem_u32(&S.k_full[ks]), kTcTileBytes);
          tma_load_4d(sK + ks * kTcTileBytes, &T.k, 0, j0, hk, b, smem_u32(&S.k_full[ks]));
        }
        describe_tile(P, S.info[t % kInfo], j0, h, p0, j0, kTcRows, kTcRows, bits, lane);
        if (lane == 0) mbar_arrive(&S.k_full[ks]);
        if (j0 < 0) break;
        if (!tc_wait(&S.v_empty[vs], ((t / kVStages) & 1) ^ 1)) { err = true; break; }
        if (lane == 0) {
          mbar_arrive_expect_tx(smem_u32(&S.v_full[vs]), kTcTileBytes);
          tma_load_4d(sV + vs * kTcTileBytes, &T.v, 0, j0, hk, b, smem_u32(&S.v_full[vs]));
        }
        ++t;
      }
    } else if (warp == 8) {  // ---- MMA
      tmem_alloc(&S.tmem, 256);
      tc_fence_before();
      setup_wait<kFwdThreads>();
      tc_fence_after();
      const uint32_t tm = S.tmem;
      const uint32_t id_s = tc_idesc(128, 128, BF16, false);
      const int dp = (P.d + 15) / 16 * 16;
      const uint32_t id_o = tc_idesc(128, dp, BF16, true);
      err = !tc_wait(&S.q_full, 0);
      // announce tile t: its S, or the end
      auto start = [&](int t, bool& end) {
        const int ks = t % kKStages;
        if (!tc_wait(&S.k_full[ks], (t / kKStages) & 1)) return false;
        end = S.info[t % kInfo].at < 0;
        if (t > 0 && !tc_wait(&S.s_free, (t - 1) & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          if (end) {
            mbar_arrive(&S.s_full);
          } else {
            tc_mma_kk(tm + kColS, tc_desc(sQ), tc_desc(sK + ks * kTcTileBytes), id_s, dp / 16);
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
        if (!tc_wait(&S.v_full[vs], (t / kVStages) & 1)) { err = true; break; }
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
        if (!tc_wait(&S.p_ready, t & 1)) { err = true; break; }
        tc_fence_after();
        if (elect_one()) {
          tc_mma_ts<8>(tm + kColO, tm + kColP, tc_desc(sV + vs * kTcTileBytes), id_o, t > 0);
          mma_commit(&S.v_empty[vs]);
          mma_commit(&S.pv_done);
        }
        __syncwarp();
        end = next_end;
      }
    } else if (warp != 8) {  // ---- the warpgroup's idle warps
      setup_wait<kFwdThreads>();
    }
  } else {  // ---- elements: warp w has rows 32 (w % 4).. and columns 64 (w / 4)..
    setup_wait<kFwdThreads>();
    tc_fence_after();
    regs_up<kElementRegs>();
    const uint32_t tm = S.tmem;
    if (P.w) {
      load_bias_ext(tab, P, h, threadIdx.x, kWork);
      asm volatile("bar.sync 5, 256;" ::: "memory");
    }
    const int wq = warp % 4, ch = warp / 4;
    const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
    const int row = wq * 32 + lane, i = i0 + row, p = p0 + row;
    const int E = bias_ext(P.D), c0 = 32 * ch;  // c0: this thread's columns of O
    float m = -INFINITY;
    float2 l = make_float2(0.0f, 0.0f);
    const float far_hi = P.w ? tab[E + P.D] : 0.0f, far_lo = P.w ? tab[E - P.D] : 0.0f;
    // One tile, S on its way to sr.  Plain tiles (all but a row's first and last few) need no look at masks
    // or distances; the others are taken apart into blocks of 32 x 32.
    auto step = [&](auto is_plain, int t, uint32_t (&sr)[2][32], int j0, const uint32_t (&bits)[2],
                    const int (&cls)[2], float far) -> bool {
      constexpr bool kPlain = decltype(is_plain)::value;
      bool live[2] = {true, true}, whole[2] = {true, true};
      uint32_t vis[2] = {~0u, ~0u};
      float mul[2] = {P.scale2, P.scale2}, add[2] = {far, far};  // logits (log2 units) are mul s + add
      int side[2] = {1, 1};
      if (!kPlain) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          live[u] = (cls[u] & 3) != kHidden;
          whole[u] = (cls[u] & 3) == kWhole;
          if (live[u] && !whole[u]) vis[u] = bits[u] & key_word(P, p, j0 + 32 * u);
          side[u] = (cls[u] >> 2) - 1;
          mul[u] = side[u] == 0 ? 1.0f : P.scale2;
          add[u] = side[u] == 1 ? far_hi : side[u] == -1 ? far_lo : 0.0f;
        }
      }
      tmem_wait_ld(sr[0]);
      tmem_wait_ld(sr[1]);
      tc_fence_before();
      mbar_arrive(&S.s_free);
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (!kPlain) {
          if (!live[u]) continue;
          if (side[u] == 0) {
            const float* tb = tab + (E + p - j0 - 32 * u);
#pragma unroll
            for (int c = 0; c < 32; ++c) sr[u][c] = __float_as_uint(fmaf(__uint_as_float(sr[u][c]), P.scale2, tb[-c]));
          }
          if (!whole[u]) {
#pragma unroll
            for (int c = 0; c < 32; ++c) sr[u][c] = (vis[u] >> c) & 1u ? sr[u][c] : 0xff800000u;
          }
        }
        top = fmaxf(top, fmaf(max32u(sr[u]), mul[u], add[u]));
      }
      S.top[t & 1][ch][row] = top;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + wq) : "memory");
      top = fmaxf(top, S.top[t & 1][ch ^ 1][row]);
      if (t > 0 && !tc_wait(&S.pv_done, (t - 1) & 1)) return false;
      const bool raise = top > m + kLag || (m == -INFINITY && top > -INFINITY);
      if (__any_sync(0xffffffffu, raise)) {
        const float mn = raise ? top : m;
        const float g = raise ? ex2(m - mn) : 1.0f;  // m = -inf: 0, and O is 0 there
        m = mn;
        l = mul2(l, both(g));
        if (t > 0 && c0 < P.d) {
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 32; c += 8) {  // 8 at a time: S fills the registers
            uint32_t o[8];
            tmem_ld8(tm + lanes + kColO + c0 + c, o);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * g);
            tmem_st8(tm + lanes + kColO + c0 + c, o);
          }
        }
      }
      const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t pk[16];
        if (kPlain || live[u]) {
          const float2 mu = both(mul[u]), off = both(add[u] - ref);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float2 s = make_float2(__uint_as_float(sr[u][2 * c]), __uint_as_float(sr[u][2 * c + 1]));
            const float2 x = exp2_pair<kPolyEvery>(fma2(s, mu, off), c);
            l = add2_ftz(l, x);
            pk[c] = pack16<BF16>(x.x, x.y);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 16; ++c) pk[c] = 0;
        }
        tmem_st16(tm + lanes + kColP + 32 * ch + 16 * u, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&S.p_ready);
      return true;
    };
    int t = 0;
    for (;; ++t) {
      if (!tc_wait(&S.s_full, t & 1)) { err = true; break; }
      const TileInfo& f = S.info[t % kInfo];
      const int at = f.at;
      if (at < 0) break;
      const bool plain = f.plain;
      const int tile_side = f.side;
      const int j0 = at + 64 * ch;
      const uint32_t bits[2] = {f.bits[2 * ch], f.bits[2 * ch + 1]};
      const int cls[2] = {f.cls[4 * wq + 2 * ch], f.cls[4 * wq + 2 * ch + 1]};
      tc_fence_after();
      uint32_t sr[2][32];
      tmem_ld32_async(tm + lanes + kColS + 64 * ch, sr[0]);
      tmem_ld32_async(tm + lanes + kColS + 64 * ch + 32, sr[1]);
      if (plain)
        err = !step(std::true_type(), t, sr, j0, bits, cls, tile_side > 0 ? far_hi : tile_side < 0 ? far_lo : 0.0f);
      else
        err = !step(std::false_type(), t, sr, j0, bits, cls, 0.0f);
      if (err) break;
    }
    if (!err && t > 0) err = !tc_wait(&S.pv_done, (t - 1) & 1);
    tc_fence_after();
    S.sum[ch][row] = l.x + l.y;
    asm volatile("bar.sync %0, 64;" ::"r"(1 + wq) : "memory");
    const float total = S.sum[0][row] + S.sum[1][row];
    const bool none = !(total > kNone) && total == total;
    const float inv = 1.0f / total;
    using E16 = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    if (c0 < P.d) {
      uint32_t o[32];
      if (t > 0) {  // warp-collective
        tmem_ld32_async(tm + lanes + kColO + c0, o);
        tmem_wait_ld(o);
      }
      if (i < P.nq) {
        E16* dst = row_ptr<E16>(P.o, b, h, i) + c0;
        E16* rest = P.o_lo ? reinterpret_cast<E16*>(P.o_lo) + (dst - reinterpret_cast<E16*>(P.o.p)) : nullptr;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c0 + 8 * e < P.d) {
            uint32_t r[4], lo[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const float x = none ? 0.0f : __uint_as_float(o[8 * e + 2 * u]) * inv;
              const float y = none ? 0.0f : __uint_as_float(o[8 * e + 2 * u + 1]) * inv;
              r[u] = pack16<BF16>(x, y);
              const float2 back = unpack16<BF16>(r[u]);
              lo[u] = pack16<BF16>(x - back.x, y - back.y);
            }
            *reinterpret_cast<uint4*>(dst + 8 * e) = make_uint4(r[0], r[1], r[2], r[3]);
            if (rest) *reinterpret_cast<uint4*>(rest + 8 * e) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
      }
    }
    if (P.lse && ch == 0 && i < P.nq)
      P.lse[(static_cast<size_t>(b) * P.H + h) * P.nq + i] = none ? INFINITY : m + lg2(total);
  }
  if (err) report_timeout(P.status);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(S.tmem, 256);
}

}  // namespace

bool tc_tmap(CUtensorMap* tm, const Strided& s, bool bf16, int d, int n, int heads, int B, int rows) {
  return make_tmap_4d(tm, s.p, bf16 ? DFS_BF16 : DFS_F16, d, n, heads, B, s.sn, s.sh, s.sb, 64, rows);
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
  const int share = 256 * kElementRegs + 128 * kOtherRegs;
  const unsigned grid = tc_grid(P.nq, P.H, P.B);
  const cudaError_t e = bf16 ? prepare_kernel<tc_fwd_kernel<true>>(smem, kFwdThreads, share)
                             : prepare_kernel<tc_fwd_kernel<false>>(smem, kFwdThreads, share);
  if (e != cudaSuccess) return e;
  if (bf16)
    tc_fwd_kernel<true><<<grid, kFwdThreads, smem, st>>>(T);
  else
    tc_fwd_kernel<false><<<grid, kFwdThreads, smem, st>>>(T);
  return cudaGetLastError();
}

}  // namespace dfs
