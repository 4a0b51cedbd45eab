// dfs_attn_tc.cu -- local attention forward on the tensor cores (bf16, fp16).
//
// One CTA owns 128 queries of one head and walks the tiles of 64 keys that they
// see.  Warps 0-3 hold a query row per thread: S = Q K^T from TMEM, the running
// maximum and sum, and P (16 bit) back to TMEM over the S it came from, where it is
// the A operand of O += P V.  Warp 4 issues the MMAs, each tile's S behind the
// product that reads the tile before's P, warp 5 stages K and V by TMA and finds
// the tiles; a tile whose keys are all masked is never announced, and a warp does
// nothing for a block of 32 x 32 pairs that are all hidden.
//
// At d <= 64 the exponentials bound it (8192 a tile at 16 a clock: 512 clocks, the
// two products 320), if the chain S -> P -> O of one tile after the other does not
// (1600 clocks for a CTA alone): so the tiles are narrow (64 + 64 TMEM columns), and
// four CTAs share an SM.  Measured (bfloat16, d = 64): 8192 tokens of 16 / 4 heads,
// window 4096, 155 us, 660 TFLOP/s, an exponential pipe 60 % busy; 8 x 1024 of 16
// heads, window 256 in both directions, 32 us.  While all SMs have four CTAs a tile
// takes 560 clocks of each: 76 us of the 155 for the first wave, and 44 for the longest
// row of the second, alone.  Where the other 35 go has not been measured.  Slower at the same sizes: 128-key tiles with 256 or 512 threads, two S
// buffers and two CTAs an SM (155 to 170 us), part of the exponentials as a
// polynomial on the FMA pipes, and every row shared by two CTAs (157 us).
#include <algorithm>
#include <type_traits>

#include "dfs_attn_tc.cuh"

namespace dfs {
namespace {

// 256 threads x 64 registers at launch = 128 x 96 (elements) + 128 x 32 (MMA, TMA and two idle warps)
constexpr int kFwdThreads = 256;
constexpr int kElementRegs = 96, kOtherRegs = 32;
static_assert(128 * kElementRegs + 128 * kOtherRegs <= kFwdThreads * 64, "register shares");
constexpr int kMmaWarp = 4, kTmaWarp = 5;
constexpr int kStages = 2, kInfo = 4;
constexpr int kHalfBytes = kTcTileBytes / 2;  // a tile of 64 keys
// the running maximum may lag by this much (log2) before O is rescaled: P stays
// below 2^8, far inside fp16, and the sums are fp32
constexpr float kLag = 8.0f;
// below any sum with a visible key in it (which holds a term of at least 2^-8)
constexpr float kNone = 1e-30f;

struct FwdShared {
  uint64_t q_full, full[kStages], empty[kStages];
  uint64_t s_full, p_ready, o_done, products;
  TileInfo info[kInfo];
  uint32_t tmem;
  int uses;  // of the ring of stages
};

// TMEM columns (128 allocated): S, and P over its first half; O
constexpr uint32_t kColS = 0, kColO = 64;

// Parts of a tile whose keys a cluster shares, over the staged tiles once all products are done
constexpr int kPartPitch = 68;
struct FwdPart {
  float o[kTcRows * kPartPitch];  // not normalised
  float m[kTcRows], l[kTcRows];
};
static_assert(sizeof(FwdPart) <= kTcTileBytes + 2 * kStages * kHalfBytes, "parts over the staged tiles");

// This CTA's share of the joined rows, 16 lanes a row (whole rows of the other CTAs' memory at once).  The remote
// reads of 8 / N rows are on their way together; one after the other they took as long as several tiles.
template <bool BF16, int N>
DFS_DEV void join_rows(const AttnParams& P, const FwdPart& part, int b, int h, int i0, int rank) {
  using E16 = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  constexpr int kRows = 8 / N;  // rows of a thread at a time; 8 rows of the CTA's 128 / N at once
  const int c = threadIdx.x % 16 * 4;
#pragma unroll 1
  for (int r0 = rank * (kTcRows / N) + threadIdx.x / 16; r0 < (rank + 1) * (kTcRows / N); r0 += 8 * kRows) {
    float m[kRows][N], l[kRows][N];
    float4 v[kRows][N];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int r = r0 + 8 * u;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        m[u][k] = dsmem_ld(dsmem_addr(smem_u32(&part.m[r]), k));
        l[u][k] = dsmem_ld(dsmem_addr(smem_u32(&part.l[r]), k));
        v[u][k] = dsmem_ld4(dsmem_addr(smem_u32(&part.o[r * kPartPitch + c]), k));
      }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int at = i0 + r0 + 8 * u;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int k = 0; k < N; ++k) top = fmaxf(top, m[u][k]);
      const float ref = top == -INFINITY ? 0.0f : top;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float f = ex2(m[u][k] - ref);
        sum = fmaf(l[u][k], f, sum);
        acc = make_float4(fmaf(v[u][k].x, f, acc.x), fmaf(v[u][k].y, f, acc.y), fmaf(v[u][k].z, f, acc.z),
                          fmaf(v[u][k].w, f, acc.w));
      }
      if (at >= P.nq || c >= P.d) continue;
      const bool none = !(sum > kNone) && sum == sum;
      const float inv = none ? 0.0f : 1.0f / sum;
      acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      const uint2 out = make_uint2(pack16<BF16>(acc.x, acc.y), pack16<BF16>(acc.z, acc.w));
      E16* dst = row_ptr<E16>(P.o, b, h, at) + c;
      *reinterpret_cast<uint2*>(dst) = out;
      if (P.o_lo) {
        const float2 lo = unpack16<BF16>(out.x), hi = unpack16<BF16>(out.y);
        *reinterpret_cast<uint2*>(reinterpret_cast<E16*>(P.o_lo) + (dst - reinterpret_cast<E16*>(P.o.p))) =
            make_uint2(pack16<BF16>(acc.x - lo.x, acc.y - lo.y), pack16<BF16>(acc.z - hi.x, acc.w - hi.y));
      }
      if (P.lse && c == 0)
        P.lse[(static_cast<size_t>(b) * P.H + h) * P.nq + at] = none ? INFINITY : top + lg2(sum);
    }
  }
}

// kSplit: a cluster of T.split CTAs shares each tile of queries, a run of the key tiles for each, joined in order
// through distributed shared memory.
template <bool BF16, bool kSplit>
__global__ void __launch_bounds__(kFwdThreads, 4) tc_fwd_kernel(const __grid_constant__ TcParams T) {
  extern __shared__ unsigned char raw[];
  const AttnParams& P = T.a;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gen = raw + (base - smem_u32(raw));
  const uint32_t sQ = base, sK = base + kTcTileBytes, sV = sK + kStages * kHalfBytes;
  FwdShared& S = *reinterpret_cast<FwdShared*>(gen + kTcTileBytes + 2 * kStages * kHalfBytes);
  float* tab = reinterpret_cast<float*>(&S + 1);
  const int warp = warp_index(), lane = threadIdx.x % 32;
  const int split = kSplit ? T.split : 1, rank = blockIdx.x % split;
  const unsigned unit = blockIdx.x / split;
  const int h = unit % P.H, b = unit / P.H % P.B, hk = h / P.G;
  const int i0 = ((P.nq - 1) / kTcRows - static_cast<int>(unit / P.H / P.B)) * kTcRows;  // causal: longest first
  const int p0 = i0 + P.qs;
  bool err = false;
  if (warp >= kMmaWarp) {
    regs_down<kOtherRegs>();  // one instruction for the whole warpgroup
    if (warp == kTmaWarp) {  // ---- producer
      if (lane == 0) {
        prefetch_tmap(&T.q);
        prefetch_tmap(&T.k);
        prefetch_tmap(&T.v);
        mbar_init(&S.q_full, 1);
        for (int s = 0; s < kStages; ++s) mbar_init(&S.full[s], 1), mbar_init(&S.empty[s], 1);
        mbar_init(&S.s_full, 1);
        mbar_init(&S.p_ready, 4);
        mbar_init(&S.o_done, 1);
        mbar_init(&S.products, 1);
        fence_mbar_init();
      }
      __syncwarp();
      setup_arrive<kFwdThreads>();
      wait_previous();
      const uint8_t* mask = P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr;
      const TcKeyTiles<kTcHalf> tiles(P, p0, min(i0 + kTcRows, P.nq) - 1 + P.qs);
      if (lane == 0) {
        mbar_arrive_expect_tx(smem_u32(&S.q_full), kTcTileBytes);
        tma_load_4d(sQ, &T.q, 0, i0, h, b, smem_u32(&S.q_full));
      }
      const PlainTiles<4, 2> plain(P);
      const int count = tiles.count(), x1 = count * (rank + 1) / split;
      uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
      int t = 0;
      for (int x = count * rank / split; x <= x1; ++x) {
        const int j0 = x < x1 ? tiles[x] * kTcHalf : -1;
        if (j0 >= 0 && mask != nullptr) {
          key_bits(mask, j0, P.nk, lane, bits);
          if ((bits[0] | bits[1]) == 0) continue;
        }
        const int s = t % kStages;
        if (!tc_wait(&S.empty[s], ((t / kStages) & 1) ^ 1)) { err = true; break; }
        if (lane == 0 && j0 >= 0) {
          const uint32_t bar = smem_u32(&S.full[s]);
          mbar_expect_tx(bar, 2 * kHalfBytes);
          tma_load_4d(sK + s * kHalfBytes, &T.k, 0, j0, hk, b, bar);
          tma_load_4d(sV + s * kHalfBytes, &T.v, 0, j0, hk, b, bar);
        }
        describe_tile(P, plain, S.info[t % kInfo], j0, h, p0, j0, (bits[0] & bits[1]) == ~0u, bits, lane);
        if (lane == 0) mbar_arrive(&S.full[s]);
        ++t;
      }
      if (lane == 0) S.uses = t;
    } else if (warp == kMmaWarp) {  // ---- MMA
      tmem_alloc(&S.tmem, 128);
      allow_next();
      tc_fence_before();
      setup_wait<kFwdThreads>();
      tc_fence_after();
      const uint32_t tm = S.tmem;
      const int dp = (P.d + 15) / 16 * 16;
      const uint32_t id_s = tc_idesc(128, 64, BF16, false), id_o = tc_idesc(128, dp, BF16, true);
      auto wait_tile = [&](int t, bool& end) {
        if (!tc_wait(&S.full[t % kStages], (t / kStages) & 1)) return false;
        end = S.info[t % kInfo].at < 0;
        return true;
      };
      auto start = [&](int t, bool end) {  // one lane: tile t's S, or the end
        if (end) {
          mbar_arrive(&S.s_full);
        } else {
          tc_mma_kk(tm + kColS, tc_desc(sQ), tc_desc(sK + t % kStages * kHalfBytes), id_s, dp / 16);
          mma_commit(&S.s_full);
        }
      };
      err = !tc_wait(&S.q_full, 0);
      bool end = false;
      if (!err) err = !wait_tile(0, end);
      if (!err && elect_one()) start(0, end);
      __syncwarp();
      for (int t = 0; !end && !err; ++t) {
        const int s = t % kStages;
        const TileInfo& f = S.info[t % kInfo];
        if (P.mask != nullptr && !f.plain) {
          const uint32_t bits[2] = {f.bits[0], f.bits[1]};
          // a hidden key's V may hold anything, and 0 x NaN is NaN: zero its row
          unsigned char* vt = gen + kTcTileBytes + (kStages + s) * kHalfBytes;
#pragma unroll
          for (int w = 0; w < 2; ++w)
            for (int r = lane / 8; r < 32; r += 4)
              if (!((bits[w] >> r) & 1u))
                *reinterpret_cast<uint4*>(vt + (32 * w + r) * 128 + (lane % 8) * 16) = make_uint4(0, 0, 0, 0);
          fence_async_smem();
          __syncwarp();
        }
        if (!wait_tile(t + 1, end) || !tc_wait(&S.p_ready, t & 1)) { err = true; break; }
        tc_fence_after();
        if (elect_one()) {
          tc_mma_ts<4>(tm + kColO, tm + kColS, tc_desc(sV + s * kHalfBytes), id_o, t > 0);
          if (end) mma_commit(&S.o_done);
          // The next S overwrites the P that this product reads: MMAs of one thread execute in the order of
          // their issue, and the commit that announces S covers the product too.
          start(t + 1, end);
          mma_commit(&S.empty[s]);  // covers more than the stage's products, which are done before the rest
        }
        __syncwarp();
      }
    } else {  // ---- the warpgroup's idle warps
      setup_wait<kFwdThreads>();
    }
    if (kSplit) {
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  } else {  // ---- elements: a query row per thread
    setup_wait<kFwdThreads>();
    tc_fence_after();
    regs_up<kElementRegs>();
    const uint32_t tm = S.tmem;
    wait_previous();
    if (P.w) {
      load_bias_ext(tab, P, h, threadIdx.x, 128);
      asm volatile("bar.sync 5, 128;" ::: "memory");
    }
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const int row = warp * 32 + lane, i = i0 + row, p = p0 + row;
    const int E = bias_ext(P.D);
    float m = -INFINITY;
    float2 l = both(0.0f);
    const float far_hi = P.w ? tab[E + P.D] : 0.0f, far_lo = P.w ? tab[E - P.D] : 0.0f;
    // One tile, S on its way to sr.  Plain tiles (all but a row's first and last few) need no look at masks
    // or distances; the others come as blocks of 32 x 32.
    auto step = [&](auto is_plain, int t, uint32_t (&sr)[2][32], const TileInfo& f, float far) {
      constexpr bool kPlain = decltype(is_plain)::value;
      float mul[2] = {P.scale2, P.scale2}, add[2] = {far, far};  // logits (log2 units) are mul s + add
      int cls[2] = {kWhole, kWhole};
      uint32_t vis[2] = {~0u, ~0u};
      const int j0 = f.at;
      if (!kPlain) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          cls[u] = f.cls[2 * warp + u];
          const int side = (cls[u] >> 2) - 1;
          if ((cls[u] & 3) == kPartial) vis[u] = f.bits[u] & key_word(P, p, j0 + 32 * u);
          mul[u] = side == 0 ? 1.0f : P.scale2;
          add[u] = side == 1 ? far_hi : side == -1 ? far_lo : 0.0f;
        }
      }
      tmem_wait_ld(sr[0]);
      tmem_wait_ld(sr[1]);
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (!kPlain) {
          if ((cls[u] & 3) == kHidden) continue;
          if ((cls[u] >> 2) == 1) {
            const float* tb = tab + (E + p - j0 - 32 * u);
#pragma unroll
            for (int c = 0; c < 32; ++c) sr[u][c] = __float_as_uint(fmaf(__uint_as_float(sr[u][c]), P.scale2, tb[-c]));
          }
          if ((cls[u] & 3) == kPartial) {
#pragma unroll
            for (int c = 0; c < 32; ++c) sr[u][c] = (vis[u] >> c) & 1u ? sr[u][c] : 0xff800000u;
          }
        }
        top = fmaxf(top, fmaf(max32u(sr[u]), mul[u], add[u]));
      }
      const bool raise = top > m + kLag || (m == -INFINITY && top > -INFINITY);
      if (__any_sync(0xffffffffu, raise)) {
        const float mn = raise ? top : m;
        const float g = raise ? ex2(m - mn) : 1.0f;  // m = -inf: 0, and O is 0 there
        m = mn;
        l = mul2(l, both(g));
        if (t > 0) {
#pragma unroll 1
          for (int c = 0; c < P.d; c += 8) {  // 8 at a time: S fills the registers
            uint32_t o[8];
            tmem_ld8(tm + lanes + kColO + c, o);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * g);
            tmem_st8(tm + lanes + kColO + c, o);
          }
        }
      }
      const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t pk[16];
        if (kPlain || (cls[u] & 3) != kHidden) {
          const float2 mu = both(mul[u]), off = both(add[u] - ref);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float2 x = make_float2(__uint_as_float(sr[u][2 * c]), __uint_as_float(sr[u][2 * c + 1]));
            x = fma2(x, mu, off);
            x = make_float2(ex2(x.x), ex2(x.y));
            l = add2(l, x);
            pk[c] = pack16<BF16>(x.x, x.y);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 16; ++c) pk[c] = 0;
        }
        tmem_st16(tm + lanes + kColS + 16 * u, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(&S.p_ready, lane);
    };
    int t = 0;
    for (;; ++t) {
      if (!tc_wait(&S.s_full, t & 1)) { err = true; break; }
      const TileInfo& f = S.info[t % kInfo];
      if (f.at < 0) break;
      const int plain = f.plain, side = f.side;
      tc_fence_after();
      uint32_t sr[2][32];
      tmem_ld32_async(tm + lanes + kColS, sr[0]);
      tmem_ld32_async(tm + lanes + kColS + 32, sr[1]);
      if (plain)
        step(std::true_type(), t, sr, f, side > 0 ? far_hi : far_lo);
      else
        step(std::false_type(), t, sr, f, 0.0f);
    }
    if (!err && t > 0) err = !tc_wait(&S.o_done, 0);
    tc_fence_after();
    const float total = l.x + l.y;
    const bool none = !(total > kNone) && total == total;
    const float inv = 1.0f / total;
    using E16 = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    if (kSplit) {
      FwdPart& part = *reinterpret_cast<FwdPart*>(gen);
#pragma unroll
      for (int c0 = 0; c0 < 64; c0 += 32) {
        if (c0 >= P.d) break;
        uint32_t o[32] = {};
        if (t > 0) {
          tmem_ld32_async(tm + lanes + kColO + c0, o);
          tmem_wait_ld(o);
        }
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *reinterpret_cast<uint4*>(&part.o[row * kPartPitch + c0 + e]) =
              make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      }
      part.m[row] = m;
      part.l[row] = total;
      __syncwarp();
      cluster_sync();
      if (split == 2) join_rows<BF16, 2>(P, part, b, h, i0, rank);
      else if (split == 4) join_rows<BF16, 4>(P, part, b, h, i0, rank);
      else join_rows<BF16, 8>(P, part, b, h, i0, rank);
      __syncwarp();
      cluster_sync();  // nobody leaves while its memory is read
    }
#pragma unroll
    for (int c0 = 0; c0 < 64 && !kSplit; c0 += 32) {
      if (c0 >= P.d) break;
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
    if (!kSplit && P.lse && i < P.nq)
      P.lse[(static_cast<size_t>(b) * P.H + h) * P.nq + i] = none ? INFINITY : m + lg2(total);
  }
  end_block<kStages>(err, P.status, warp == kTmaWarp, warp == kMmaWarp, &S.q_full, S.full, S.uses, &S.products);
  if (warp == kMmaWarp) tmem_dealloc(S.tmem, 128);
}

}  // namespace

bool tc_tmap(CUtensorMap* tm, const Strided& s, bool bf16, int d, int n, int heads, int B, int rows) {
  return make_tmap_4d(tm, s.p, bf16 ? DFS_BF16 : DFS_F16, d, n, heads, B, s.sn, s.sh, s.sb, 64, rows);
}

cudaError_t launch_attn_tc_fwd(const AttnParams& P, int dtype, cudaStream_t st) {
  const bool bf16 = dtype == DFS_BF16;
  TcParams T;
  T.a = P;
  const size_t fixed = 1024 + kTcTileBytes + 2 * kStages * kHalfBytes + sizeof(FwdShared);
  const size_t smem = fixed + bias_ext_bytes(P), most = fixed + ext_table_bytes(DFS_MAX_BUCKET_DISTANCE);
  const int share = 128 * kElementRegs + 128 * kOtherRegs;
  // Few queries over many keys: a cluster of CTAs shares them, until every SM has four and while each has four
  // tiles; with sixteen each, until every SM has had eight (a wave that is not full ends with its longest CTA).
  // Measured (bfloat16, d = 64, causal): 5 queries of 16 heads over 8192 keys 110 -> 28 us, 8 heads of 1024 18.6 ->
  // 12.7; 16 heads of 4096 97 -> 62, but 32 heads of 2048 with a window of 512, ten tiles a CTA, 29 -> 36.
  const unsigned grid = tc_grid(P.nq, P.H, P.B);
  const int64_t seen = std::min<int64_t>(P.nk, int64_t{P.window} * (P.causal ? 1 : 2) + kTcRows + P.sinks) / kTcHalf;
  T.split = 1;
  while (T.split < 8 && 8 * T.split <= seen && 2u * T.split * grid <= (32 * T.split <= seen ? 8u : 4u) * 148)
    T.split *= 2;
  auto run = [&](auto kern, cudaError_t e) {
    if (e != cudaSuccess) return e;
    if (!tc_tmap(&T.q, P.q, bf16, P.d, P.nq, P.H, P.B) ||
        !tc_tmap(&T.k, P.k, bf16, P.d, P.nk, P.Hkv, P.B, kTcHalf) ||
        !tc_tmap(&T.v, P.v, bf16, P.d, P.nk, P.Hkv, P.B, kTcHalf))
      return cudaErrorInvalidValue;
    T.d_o = T.q;
    return launch_clusters(kern, grid * T.split, T.split, kFwdThreads, smem, st, T);
  };
  if (T.split > 1)
    return bf16 ? run(tc_fwd_kernel<true, true>, prepare_kernel<tc_fwd_kernel<true, true>>(most, kFwdThreads, share))
                : run(tc_fwd_kernel<false, true>, prepare_kernel<tc_fwd_kernel<false, true>>(most, kFwdThreads, share));
  return bf16 ? run(tc_fwd_kernel<true, false>, prepare_kernel<tc_fwd_kernel<true, false>>(most, kFwdThreads, share))
              : run(tc_fwd_kernel<false, false>, prepare_kernel<tc_fwd_kernel<false, false>>(most, kFwdThreads, share));
}

}  // namespace dfs
