// dfs_attn_tc_bwd.cu -- local attention backward on the tensor cores (bf16, fp16).
//
// Two passes, neither with atomics, so gradients repeat bit for bit:
//   dQ pass   one CTA per 128 queries of a head, over the key tiles they see:
//             S = Q K^T, dP = dO V^T, p = 2^(S - lse), dS = p (dP - D), dQ += dS K;
//             D = sum_c dO O comes from O and what its rounding took, and D + sum_j dS_ij,
//             which is sum_j p_ij dP_ij in fp32, goes to the key pass, whose bias sums
//             cancel within a row;
//   dK/dV pass  one CTA per 128 keys of a key head, over the query tiles (of every
//             head of the group) that see them, on transposed tiles: S^T = K Q^T,
//             dP^T = V dO^T, dV += P^T dO, dK += dS^T Q; and the sums of dS by distance.
// The alternative is one pass with dQ added up in memory: 5 products a tile pair
// instead of 7 and one exponential instead of two, but 32 KB of fp32 atomics (in
// varying order) a tile pair.
//
// Both stream tiles of 64 rows past their own 128 and run two CTAs an SM (256 TMEM
// columns each), so that one's products, TMEM traffic, start and end overlap the
// other's arithmetic; with 128-row tiles and one CTA an SM of twice the element
// warps the same work took about twice as long.  Warps 0-7 work element by element
// (a TMEM row and half of a tile's columns per thread: blocks of 32 x 32 per warp,
// skipped where all is hidden), warp 8 issues the MMAs, warp 9 stages tiles by TMA
// and announces them.
//
// Measured (bfloat16, d = 64, 8192 tokens of 16 heads, window 1024, a bias): dQ pass
// 95 us, dK/dV pass 133 us, together 350 TFLOP/s of the 10 d a visible pair needs.
// No pipe is more than half busy.  A key tile's step is a chain of about 2500 clocks:
// 650 for the four products (their operands' way out of shared memory, not the
// tensor cores), 450 through TMEM, 900 of arithmetic, the rest waits' wake-ups; two
// CTAs, which is what TMEM holds, overlap theirs.  Slower: one CTA an SM with two
// groups of element warps and three buffers (20 us), and P and dS handed over one
// after the other, so that half of the products run behind the other half's
// arithmetic (13 us: twice the waits and reads).  Where few key heads would leave
// SMs idle, the key pass spreads a tile's steps over CTAs and joins them in 32 bits
// (16 / 2 heads of 2048 tokens: 351 -> 108 us).
#include <type_traits>

#include "dfs_attn_tc.cuh"

namespace dfs {
namespace {

// 384 threads x 80 registers at launch = 256 x 104 (elements) + 128 x 32 (MMA, TMA and two idle warps)
constexpr int kBwdThreads = 384;
constexpr int kElementRegs = 104, kOtherRegs = 32;
static_assert(256 * kElementRegs + 128 * kOtherRegs <= kBwdThreads * 80, "register shares");
constexpr int kWork = 256;     // threads of the element warps
constexpr int kMmaWarp = 8, kTmaWarp = 9;
constexpr int kStages = 3, kInfo = 4;
constexpr int kHalfBytes = kTcTileBytes / 2;  // a streamed tile

// TMEM columns (256 allocated): S and dP (64 each), then the dQ pass's dQ and dS, or dV and dK.  The dK/dV pass
// writes P and dS over the S and dP that it has read, a warp within its own 32 columns.
constexpr uint32_t kColS = 0, kColDP = 64, kColA = 128, kColB = 192;
constexpr uint32_t kColDS = 192;              // dQ pass

struct BwdShared {
  uint64_t own_full, full[kStages], empty[kStages];
  uint64_t s_full, s_free, ds_ready, acc_done, products;
  TileInfo info[kInfo];
  alignas(16) float stat[kStages][2][kTcHalf];  // dK/dV pass: -lse and -D of the stage's queries
  float part[2][kTcRows];           // dQ pass: a row's two partial sums
  float ends[2][kWork / 32];
  float diag[kWork / 32][32];       // dK/dV pass: diagonals of a warp's block that ended at lane 31
  uint32_t tmem;
  int uses;  // of the ring of stages
};

DFS_DEV void work_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Barriers of a key-pass element warp up to a head's first tile, as the `entered`-th of its unit: two a head for the
// tables, and with sums by distance two for the flush of each head before it.
__host__ __device__ constexpr int barriers_before(int entered, bool dw) {
  return entered == 0 ? 0 : 2 * entered + (dw ? 2 * (entered - 1) : 0);
}
// Those that are left, the last head's flush among them, for a unit of `heads`
__host__ __device__ constexpr int barriers_left(int heads, int entered, bool dw) {
  return barriers_before(heads, dw) + (dw && heads > 0 ? 2 : 0) - barriers_before(entered, dw);
}
static_assert(barriers_left(0, 0, true) == 0 && barriers_left(3, 0, true) == 12 && barriers_left(3, 3, true) == 2 &&
                  barriers_left(3, 1, false) == 4 && barriers_left(3, 3, false) == 0,
              "as the key pass's loop has them");

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
        r[u] = zero ? 0u : pack16<BF16>(__uint_as_float(v[8 * e + 2 * u]) * mul,
                                        __uint_as_float(v[8 * e + 2 * u + 1]) * mul);
      *reinterpret_cast<uint4*>(dst + 8 * e) = make_uint4(r[0], r[1], r[2], r[3]);
    }
}

template <bool BF16>
__global__ void __launch_bounds__(kBwdThreads, 2) tc_dq_kernel(const __grid_constant__ TcParams T) {
  extern __shared__ unsigned char raw[];
  const AttnParams& P = T.a;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gen = raw + (base - smem_u32(raw));
  const uint32_t sQ = base, sO = sQ + kTcTileBytes, sK = sO + kTcTileBytes, sV = sK + kStages * kHalfBytes;
  BwdShared& S = *reinterpret_cast<BwdShared*>(gen + 2 * kTcTileBytes + 2 * kStages * kHalfBytes);
  float* tab = reinterpret_cast<float*>(&S + 1);
  const int warp = warp_index(), lane = threadIdx.x % 32;
  const int h = blockIdx.x % P.H, b = blockIdx.x / P.H % P.B, hk = h / P.G;
  const int i0 = ((P.nq - 1) / kTcRows - static_cast<int>(blockIdx.x / P.H / P.B)) * kTcRows;  // causal: longest first
  const int p0 = i0 + P.qs;
  bool err = false;

  if (warp >= kMmaWarp) {
    regs_down<kOtherRegs>();  // one instruction for the whole warpgroup
    if (warp == kTmaWarp) {  // ---- producer
      if (lane == 0) {
        prefetch_tmap(&T.q);
        prefetch_tmap(&T.k);
        prefetch_tmap(&T.v);
        prefetch_tmap(&T.d_o);
        mbar_init(&S.own_full, 1);
        for (int s = 0; s < kStages; ++s) mbar_init(&S.full[s], 1), mbar_init(&S.empty[s], 1);
        mbar_init(&S.s_full, 1);
        mbar_init(&S.s_free, kWork / 32);
        mbar_init(&S.ds_ready, kWork / 32);
        mbar_init(&S.acc_done, 1);
        mbar_init(&S.products, 1);
        fence_mbar_init();
      }
      __syncwarp();
      setup_arrive<kBwdThreads>();
      wait_previous();
      const uint8_t* mask = P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr;
      const TcKeyTiles<kTcHalf> tiles(P, p0, min(i0 + kTcRows, P.nq) - 1 + P.qs);
      if (lane == 0) {
        mbar_arrive_expect_tx(smem_u32(&S.own_full), 2 * kTcTileBytes);
        tma_load_4d(sQ, &T.q, 0, i0, h, b, smem_u32(&S.own_full));
        tma_load_4d(sO, &T.d_o, 0, i0, h, b, smem_u32(&S.own_full));
      }
      const PlainTiles<4, 2> plain(P);
      const int count = tiles.count();
      uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
      int t = 0;
      for (int x = 0; x <= count; ++x) {
        const int j0 = x < count ? tiles[x] * kTcHalf : -1;
        if (j0 >= 0 && mask != nullptr) {
          key_bits(mask, j0, P.nk, lane, bits);
          if ((bits[0] | bits[1]) == 0) continue;
        }
        const int s = t % kStages;
        if (!tc_wait(&S.empty[s], ((t / kStages) & 1) ^ 1)) { err = true; break; }
        if (lane == 0 && j0 >= 0) {
          mbar_expect_tx(smem_u32(&S.full[s]), 2 * kHalfBytes);
          tma_load_4d(sK + s * kHalfBytes, &T.k, 0, j0, hk, b, smem_u32(&S.full[s]));
          tma_load_4d(sV + s * kHalfBytes, &T.v, 0, j0, hk, b, smem_u32(&S.full[s]));
        }
        describe_tile(P, plain, S.info[t % kInfo], j0, h, p0, j0, (bits[0] & bits[1]) == ~0u, bits, lane);
        if (lane == 0) mbar_arrive(&S.full[s]);
        ++t;
      }
      if (lane == 0) S.uses = t;
    } else if (warp == kMmaWarp) {  // ---- MMA
      tmem_alloc(&S.tmem, 256);
      allow_next();
      tc_fence_before();
      setup_wait<kBwdThreads>();
      tc_fence_after();
      const uint32_t tm = S.tmem;
      const int dp = (P.d + 15) / 16 * 16;
      const uint32_t id_s = tc_idesc(128, 64, BF16, false), id_a = tc_idesc(128, dp, BF16, true);
      err = !tc_wait(&S.own_full, 0);
      auto start = [&](int t, bool& end) {
        const int s = t % kStages;
        if (!tc_wait(&S.full[s], (t / kStages) & 1)) return false;
        const TileInfo& f = S.info[t % kInfo];
        end = f.at < 0;
        if (!end && P.mask != nullptr && !f.plain) {
          // a hidden key's K may hold anything, and 0 x NaN is NaN in dS K: zero its row
          unsigned char* kt = gen + 2 * kTcTileBytes + s * kHalfBytes;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t bw = f.bits[w];
            if (bw != ~0u)
              for (int r = lane / 8; r < 32; r += 4)
                if (!((bw >> r) & 1u))
                  *reinterpret_cast<uint4*>(kt + (32 * w + r) * 128 + (lane % 8) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
          __syncwarp();
        }
        if (t > 0 && !tc_wait(&S.s_free, (t - 1) & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          if (end) {
            mbar_arrive(&S.s_full);
          } else {
            tc_mma_kk(tm + kColS, tc_desc(sQ), tc_desc(sK + s * kHalfBytes), id_s, dp / 16);
            tc_mma_kk(tm + kColDP, tc_desc(sO), tc_desc(sV + s * kHalfBytes), id_s, dp / 16);
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
        if (!tc_wait(&S.ds_ready, t & 1)) { err = true; break; }
        tc_fence_after();
        if (elect_one()) {
          tc_mma_ts<4>(tm + kColA, tm + kColDS, tc_desc(sK + (t % kStages) * kHalfBytes), id_a, t > 0);
          mma_commit(&S.empty[t % kStages]);
          mma_commit(&S.acc_done);
        }
        __syncwarp();
        end = next_end;
      }
    } else {  // ---- the warpgroup's idle warps
      setup_wait<kBwdThreads>();
    }
  } else {  // ---- elements: warp w has TMEM lanes 32 (w % 4).. and columns 32 (w / 4)..
    setup_wait<kBwdThreads>();
    tc_fence_after();
    regs_up<kElementRegs>();
    const uint32_t tm = S.tmem;
    wait_previous();
    if (P.w) load_bias_ext(tab, P, h, threadIdx.x, kWork);  // read after the barrier below
    const int wq = warp % 4, cg = warp / 4, row = wq * 32 + lane, i = i0 + row, p = p0 + row;
    const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
    const int E = bias_ext(P.D), c0 = 32 * cg;  // c0: this thread's columns of d
    using T16 = typename E16<BF16>::T;
    const size_t stat = (static_cast<size_t>(b) * P.H + h) * P.nq + i;
    float D = 0.0f;
    if (i < P.nq) {
      const T16* orow = row_ptr<T16>(P.o, b, h, i) + c0;
      const T16* rest = P.o_lo ? reinterpret_cast<const T16*>(P.o_lo) + (orow - reinterpret_cast<const T16*>(P.o.p))
                               : nullptr;
      const T16* drow = row_ptr<T16>(P.d_o, b, h, i) + c0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c0 + 8 * e < P.d) {
          const uint4 x = *reinterpret_cast<const uint4*>(orow + 8 * e);
          const uint4 y = *reinterpret_cast<const uint4*>(drow + 8 * e);
          const uint4 z = rest ? *reinterpret_cast<const uint4*>(rest + 8 * e) : make_uint4(0, 0, 0, 0);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w}, zs[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float2 f = unpack16<BF16>(xs[u]), g = unpack16<BF16>(ys[u]), r = unpack16<BF16>(zs[u]);
            D = fmaf(f.x + r.x, g.x, fmaf(f.y + r.y, g.y, D));
          }
        }
    }
    S.part[cg][row] = D;
    work_barrier();
    D = S.part[0][row] + S.part[1][row];
    const float lse = i < P.nq ? P.lse[stat] : INFINITY;
    float2 rest = both(0.0f);
    const float far_hi = P.w ? tab[E + P.D] : 0.0f, far_lo = P.w ? tab[E - P.D] : 0.0f;
    // One tile, S and dP on their way to sr and dr (plain tiles: see TileInfo).
    auto step = [&](auto is_plain, int t, uint32_t (&sr)[32], uint32_t (&dr)[32], int j0, uint32_t bits,
                    int cls, float far) -> bool {
      constexpr bool kPlain = decltype(is_plain)::value;
      bool whole = true, live = true;
      uint32_t vis = ~0u;
      int side = 1;
      float mul = P.scale2;
      if (!kPlain) {
        live = (cls & 3) != kHidden;
        whole = (cls & 3) == kWhole;
        if (live && !whole) vis = bits & key_word(P, p, j0);
        side = (cls >> 2) - 1;
        far = side == 1 ? far_hi : side == -1 ? far_lo : 0.0f;
        if (side == 0) mul = 1.0f;
      }
      tmem_wait_ld(sr);
      tmem_wait_ld(dr);
      tc_fence_before();
      warp_arrive(&S.s_free, lane);
      uint32_t pk[16];
      if (kPlain || live) {
        if (!kPlain && side == 0) {
          const float* tb = tab + (E + p - j0);
#pragma unroll
          for (int c = 0; c < 32; ++c) sr[c] = __float_as_uint(fmaf(__uint_as_float(sr[c]), P.scale2, tb[-c]));
        }
        if (!kPlain && !whole) {
          // a hidden key's logit is -inf, and its dP (from hidden memory: anything) 0
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const bool on = (vis >> c) & 1u;
            sr[c] = on ? sr[c] : 0xff800000u;
            dr[c] = on ? dr[c] : 0u;
          }
        }
        const float2 mul_2 = both(mul), off = both(far - lse);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float2 s = make_float2(__uint_as_float(sr[2 * c]), __uint_as_float(sr[2 * c + 1]));
          const float2 dp = make_float2(__uint_as_float(dr[2 * c]), __uint_as_float(dr[2 * c + 1]));
          const float2 x = fma2(s, mul_2, off);
          const float2 ds = mul2(make_float2(ex2(x.x), ex2(x.y)), add2(dp, both(-D)));
          rest = add2(rest, ds);
          pk[c] = pack16<BF16>(ds.x, ds.y);
        }
      } else {
#pragma unroll
        for (int c = 0; c < 16; ++c) pk[c] = 0;
      }
      if (t > 0 && !tc_wait(&S.acc_done, (t - 1) & 1)) return false;
      tmem_st16(tm + lanes + kColDS + 16 * cg, pk);
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(&S.ds_ready, lane);
      return true;
    };
    int t = 0;
    for (;; ++t) {
      if (!tc_wait(&S.s_full, t & 1)) { err = true; break; }
      const TileInfo& f = S.info[t % kInfo];
      const int at = f.at, j0 = at + 32 * cg;
      if (at < 0) break;
      const int plain = f.plain, tile_side = f.side;
      const uint32_t bits = f.bits[cg];
      const int cls = f.cls[2 * wq + cg];
      tc_fence_after();
      uint32_t sr[32], dr[32];
      tmem_ld32_async(tm + lanes + kColS + 32 * cg, sr);
      tmem_ld32_async(tm + lanes + kColDP + 32 * cg, dr);
      if (plain)
        err = !step(std::true_type(), t, sr, dr, j0, bits, cls, tile_side > 0 ? far_hi : tile_side < 0 ? far_lo : 0.0f);
      else
        err = !step(std::false_type(), t, sr, dr, j0, bits, cls, 0.0f);
      if (err) break;
    }
    if (!err && t > 0) err = !tc_wait(&S.acc_done, (t - 1) & 1);
    tc_fence_after();
    if (c0 < P.d) {
      uint32_t v[32];
      if (t > 0) {
        tmem_ld32_async(tm + lanes + kColA + c0, v);
        tmem_wait_ld(v);
      }
      if (i < P.nq) store_row32<BF16>(P.d_q, b, h, i, c0, P.d, v, P.scale, t == 0);
    }
    work_barrier();
    S.part[cg][row] = rest.x + rest.y;
    work_barrier();
    if (cg == 0 && i < P.nq)
      P.dsum[stat] = D + (S.part[0][row] + S.part[1][row]);
  }
  end_block<kStages>(err, P.status, warp == kTmaWarp, warp == kMmaWarp, &S.own_full, S.full, S.uses, &S.products);
  if (warp == kMmaWarp) tmem_dealloc(S.tmem, 256);
}

template <bool BF16>
__global__ void __launch_bounds__(kBwdThreads, 2) tc_dkv_kernel(const __grid_constant__ TcParams T) {
  extern __shared__ unsigned char raw[];
  const AttnParams& P = T.a;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gen = raw + (base - smem_u32(raw));
  const uint32_t sK = base, sV = sK + kTcTileBytes, sQ = sV + kTcTileBytes, sO = sQ + kStages * kHalfBytes;
  BwdShared& S = *reinterpret_cast<BwdShared*>(gen + 2 * kTcTileBytes + 2 * kStages * kHalfBytes);
  float* tab = reinterpret_cast<float*>(&S + 1);
  const int W = 2 * P.D + 1;
  float* acc = tab + (P.w ? 2 * bias_ext(P.D) + 1 : 0);  // a table of W sums by distance for each element warp
  const int warp = warp_index(), lane = threadIdx.x % 32;
  const int hk = blockIdx.x % P.Hkv, b = blockIdx.x / P.Hkv % P.B, unit = blockIdx.x / P.Hkv / P.B;
  // Units: first the far segments of the sinks' tiles (the queries beyond their window, which see the sinks
  // only; without them those tiles' CTAs would walk every query tile), then the key tiles.
  const int far_units = P.sink_tiles * P.far_segs;
  const bool far_unit = unit < far_units;
  const int near = unit - far_units, tile = far_unit ? unit / P.far_segs : near / P.near_segs, j0 = tile * kTcRows;
  const int sink_rows = P.far_segs > 0 ? min(max(P.sinks - j0, 0), kTcRows) : 0;  // rows that are joined afterwards
  bool err = false;

  // queries that see some key of the tile, in tiles of queries: [i_lo, i_hi); this unit's steps [first, last)
  // of (head, query tile)
  int i_lo = P.causal ? j0 - P.qs : j0 - P.window + 1 - P.qs;
  int i_hi = min(j0 + kTcRows, P.nk) - 1 + P.window - P.qs;
  if (j0 < P.sinks) {
    if (P.far_segs == 0) i_hi = P.nq;
    if (!P.causal) i_lo = 0;
  }
  i_lo = max(i_lo, 0) / kTcHalf;
  i_hi = (max(min(i_hi, P.nq), 0) + kTcHalf - 1) / kTcHalf;
  if (far_unit) {
    i_lo = max(i_lo, i_hi);
    i_hi = (P.nq + kTcHalf - 1) / kTcHalf;
  }
  const int per = max(0, i_hi - i_lo);
  const int len = far_unit ? P.far_len : (per * P.G + P.near_segs - 1) / P.near_segs;
  const int first = min((far_unit ? unit % P.far_segs : near % P.near_segs) * len, per * P.G);
  const int last = min(first + len, per * P.G);

  if (warp >= kMmaWarp) {
    regs_down<kOtherRegs>();  // one instruction for the whole warpgroup
    if (warp == kTmaWarp) {  // ---- producer
      if (lane == 0) {
        prefetch_tmap(&T.q);
        prefetch_tmap(&T.k);
        prefetch_tmap(&T.v);
        prefetch_tmap(&T.d_o);
        mbar_init(&S.own_full, 1);
        for (int s = 0; s < kStages; ++s) mbar_init(&S.full[s], 1), mbar_init(&S.empty[s], 1);
        mbar_init(&S.s_full, 1);
        mbar_init(&S.ds_ready, kWork / 32);
        mbar_init(&S.acc_done, 1);
        mbar_init(&S.products, 1);
        fence_mbar_init();
      }
      __syncwarp();
      setup_arrive<kBwdThreads>();
      wait_previous();
      uint32_t bits[4];
      key_bits(P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr, j0, P.nk, lane, bits);
      const int total = (bits[0] | bits[1] | bits[2] | bits[3]) == 0 ? 0 : last - first;
      if (lane == 0) {
        mbar_arrive_expect_tx(smem_u32(&S.own_full), 2 * kTcTileBytes);
        tma_load_4d(sK, &T.k, 0, j0, hk, b, smem_u32(&S.own_full));
        tma_load_4d(sV, &T.v, 0, j0, hk, b, smem_u32(&S.own_full));
      }
      const PlainTiles<2, 4> plain(P);
      const bool whole = (bits[0] & bits[1] & bits[2] & bits[3]) == ~0u;
      int g = total > 0 ? first / per : 0, it = total > 0 ? first - g * per : 0;  // head and query tile of the step
      float st[2][2];
      auto load_stats = [&](int g, int it) {  // -lse and -D of two queries a lane, a step ahead
        const size_t at = (static_cast<size_t>(b) * P.H + hk * P.G + g) * P.nq;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = (i_lo + it) * kTcHalf + 2 * lane + e;
          st[0][e] = i < P.nq ? -P.lse[at + i] : -INFINITY;
          st[1][e] = i < P.nq ? -P.dsum[at + i] : 0.0f;
        }
      };
      if (total > 0) load_stats(g, it);
      int t = 0;
      for (; t <= total; ++t) {
        const int s = t % kStages, i0 = t < total ? (i_lo + it) * kTcHalf : -1, now = g;
        if (!tc_wait(&S.empty[s], ((t / kStages) & 1) ^ 1)) { err = true; break; }
        if (i0 >= 0) {
          if (lane == 0) {
            const uint32_t bar = smem_u32(&S.full[s]);
            mbar_expect_tx(bar, 2 * kHalfBytes);
            tma_load_4d(sQ + s * kHalfBytes, &T.q, 0, i0, hk * P.G + g, b, bar);
            tma_load_4d(sO + s * kHalfBytes, &T.d_o, 0, i0, hk * P.G + g, b, bar);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k)
            *reinterpret_cast<float2*>(&S.stat[s][k][2 * lane]) = make_float2(st[k][0], st[k][1]);
          if (++it == per) it = 0, ++g;
          if (t + 1 < total) load_stats(g, it);
        }
        describe_tile(P, plain, S.info[t % kInfo], i0, now, i0 + P.qs, j0, whole, bits, lane);
        if (lane == 0) mbar_arrive(&S.full[s]);
      }
      if (lane == 0) S.uses = t;
    } else if (warp == kMmaWarp) {  // ---- MMA
      tmem_alloc(&S.tmem, 256);
      allow_next();
      tc_fence_before();
      setup_wait<kBwdThreads>();
      tc_fence_after();
      const uint32_t tm = S.tmem;
      const int dp = (P.d + 15) / 16 * 16;
      const uint32_t id_s = tc_idesc(128, 64, BF16, false), id_a = tc_idesc(128, dp, BF16, true);
      err = !tc_wait(&S.own_full, 0);
      auto wait_tile = [&](int t, bool& end) {
        if (!tc_wait(&S.full[t % kStages], (t / kStages) & 1)) return false;
        end = S.info[t % kInfo].at < 0;
        return true;
      };
      auto start = [&](int t) {  // one lane: tile t's S and dP
        const int s = t % kStages;
        tc_mma_kk(tm + kColS, tc_desc(sK), tc_desc(sQ + s * kHalfBytes), id_s, dp / 16);
        tc_mma_kk(tm + kColDP, tc_desc(sV), tc_desc(sO + s * kHalfBytes), id_s, dp / 16);
        mma_commit(&S.s_full);
      };
      bool end = false;
      if (!err) err = !wait_tile(0, end);
      if (!err && !end && elect_one()) start(0);
      __syncwarp();
      for (int t = 0; !end && !err; ++t) {
        if (!wait_tile(t + 1, end) || !tc_wait(&S.ds_ready, t & 1)) { err = true; break; }
        tc_fence_after();
        if (elect_one()) {
          const int s = t % kStages;
          tc_mma_ts<4, true>(tm + kColA, tm + kColS, tc_desc(sO + s * kHalfBytes), id_a, t > 0);
          tc_mma_ts<4, true>(tm + kColB, tm + kColDP, tc_desc(sQ + s * kHalfBytes), id_a, t > 0);
          mma_commit(&S.empty[s]);
          mma_commit(&S.acc_done);
          // The next S and dP overwrite the P and dS that these products read: MMAs of one thread execute in
          // the order of their issue, and the commit below covers all of them.
          if (!end) start(t + 1);
        }
        __syncwarp();
      }
    } else {  // ---- the warpgroup's idle warps
      setup_wait<kBwdThreads>();
    }
  } else {  // ---- elements: a key row and half of the tile's queries per thread
    setup_wait<kBwdThreads>();
    tc_fence_after();
    regs_up<kElementRegs>();
    const uint32_t tm = S.tmem;
    wait_previous();
    const int wq = warp % 4, cg = warp / 4, row = wq * 32 + lane, j = j0 + row, tid = threadIdx.x;
    const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
    const int E = bias_ext(P.D);
    const bool dw = P.dw_part != nullptr;
    float lo = 0.0f, hi = 0.0f;  // sums of dS beyond the table's ends
    int head = -1;
    float far_hi = 0.0f, far_lo = 0.0f;
    auto dw_row = [&](int g) {
      return P.dw_part + (static_cast<size_t>(hk * P.G + g) * P.parts + b * (P.parts / P.B) + unit) * W;
    };
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
      float* dst = dw_row(head);
      for (int x = tid; x < W; x += kWork) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kWork / 32; ++w) s += acc[w * W + x];
        dst[x] = s;
      }
      lo = hi = 0.0f;
    };
    // heads that have no tile here: their sums are zero
    auto zero_heads = [&](int from, int to) {
      for (int g = from; g < to; ++g) {
        float* dst = dw_row(g);
        for (int x = tid; x < W; x += kWork) dst[x] = 0.0f;
      }
    };
    // One block, S^T and dP^T on their way to sr and dr: P and dS to TMEM, over S and dP, and the block's sum of dS
    // to `sum`; a block that is not plain also leaves dS in dr.
    auto step = [&](auto is_plain, int t, uint32_t (&sr)[32], uint32_t (&dr)[32], int pw, uint32_t vis, int cls,
                    float far, float2& sum) {
      constexpr bool kPlain = decltype(is_plain)::value;
      const float* lse = S.stat[t % kStages][0] + 32 * cg;
      const float* Dv = S.stat[t % kStages][1] + 32 * cg;
      float mul = P.scale2;
      if (!kPlain) {
        const int side = (cls >> 2) - 1;
        far = side == 1 ? far_hi : side == -1 ? far_lo : 0.0f;
        if (side == 0) mul = 1.0f;
      }
      tmem_wait_ld(sr);
      tmem_wait_ld(dr);
      if (!kPlain) {
        if ((cls >> 2) == 1) {
          const float* tb = tab + (E + pw - j);
#pragma unroll
          for (int c = 0; c < 32; ++c) sr[c] = __float_as_uint(fmaf(__uint_as_float(sr[c]), P.scale2, tb[c]));
        }
        if ((cls & 3) == kPartial) {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const bool on = (vis >> c) & 1u;
            sr[c] = on ? sr[c] : 0xff800000u;
            dr[c] = on ? dr[c] : 0u;
          }
        }
      }
      const float2 mul_2 = both(mul), far_2 = both(far);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {  // 16 queries at a time: registers
        uint32_t pp[8], ps[8];
#pragma unroll
        for (int c = 0; c < 8; c += 2) {
          const float4 ls = *reinterpret_cast<const float4*>(lse + 16 * hf + 2 * c);
          const float4 dd = *reinterpret_cast<const float4*>(Dv + 16 * hf + 2 * c);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float2 l2 = u ? make_float2(ls.z, ls.w) : make_float2(ls.x, ls.y);
            const float2 d2 = u ? make_float2(dd.z, dd.w) : make_float2(dd.x, dd.y);
            const int e = 16 * hf + 2 * (c + u);
            const float2 s = make_float2(__uint_as_float(sr[e]), __uint_as_float(sr[e + 1]));
            const float2 dp = make_float2(__uint_as_float(dr[e]), __uint_as_float(dr[e + 1]));
            float2 x = fma2(s, mul_2, add2(l2, far_2));
            x = make_float2(ex2(x.x), ex2(x.y));
            const float2 ds = mul2(x, add2(dp, d2));
            sum = add2(sum, ds);
            pp[c + u] = pack16<BF16>(x.x, x.y);
            ps[c + u] = pack16<BF16>(ds.x, ds.y);
            if (!kPlain) {
              dr[e] = __float_as_uint(ds.x);
              dr[e + 1] = __float_as_uint(ds.y);
            }
          }
        }
        tmem_st8(tm + lanes + kColS + 32 * cg + 8 * hf, pp);
        tmem_st8(tm + lanes + kColDP + 32 * cg + 8 * hf, ps);
      }
    };
    int t = 0;
    for (;; ++t) {
      // what the producer says of the tile, while its S and dP are computed
      if (!tc_wait(&S.full[t % kStages], (t / kStages) & 1)) { err = true; break; }
      const TileInfo& f = S.info[t % kInfo];
      const int i0 = f.at, g = f.head;
      if (i0 < 0) break;
      if (g != head) {
        if (dw) {
          if (head >= 0) flush();
          zero_heads(head + 1, g);
        }
        work_barrier();  // nobody reads the old tables any more
        head = g;
        if (P.w) load_bias_ext(tab, P, hk * P.G + g, tid, kWork);
        if (dw)
          for (int x = tid; x < kWork / 32 * W; x += kWork) acc[x] = 0.0f;
        work_barrier();
        if (P.w) far_hi = tab[E + P.D], far_lo = tab[E - P.D];
      }
      const int plain = f.plain, tile_side = f.side, cls = f.cls[4 * cg + wq];
      const uint32_t kbits = f.bits[wq];
      const int p0 = i0 + P.qs, pw = p0 + 32 * cg;
      const bool live = plain || (cls & 3) != kHidden;
      const uint32_t vis = (kbits >> lane) & 1u ? query_word(P, j, pw) : 0u;
      float2 sum = both(0.0f);
      uint32_t sr[32], dr[32];
      if (!tc_wait(&S.s_full, t & 1)) { err = true; break; }
      if (live) {
        tc_fence_after();
        tmem_ld32_async(tm + lanes + kColS + 32 * cg, sr);
        tmem_ld32_async(tm + lanes + kColDP + 32 * cg, dr);
        if (plain)
          step(std::true_type(), t, sr, dr, pw, vis, cls, tile_side > 0 ? far_hi : far_lo, sum);
        else
          step(std::false_type(), t, sr, dr, pw, vis, cls, 0.0f, sum);
      } else {
        const uint32_t none[16] = {};
        tc_fence_after();
        tmem_st16(tm + lanes + kColS + 32 * cg, none);
        tmem_st16(tm + lanes + kColDP + 32 * cg, none);
      }
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(&S.ds_ready, lane);
      if (!dw) continue;
      if (tile_side != 0) {
        if (tile_side > 0) hi += sum.x + sum.y;
        else lo += sum.x + sum.y;
        continue;
      }
      if (!live) continue;
      // Diagonals of this warp's block of 32 keys x 32 queries: the running sum of a diagonal moves one lane up
      // as the query advances, and is complete once lane 31 has added its element.  Two chains, of the first and of
      // the last 16 queries, halve the way of dependent shuffles; the first one's sums then go on where the
      // second one's diagonals are.  The sums go to a table of this warp's own, while it would wait for the next
      // tile's S: with one table and a join of the warps a tile, such tiles took half as long again.
      float* out = S.diag[warp];
      float up = 0.0f, run = 0.0f;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        up += __uint_as_float(dr[c]);
        run += __uint_as_float(dr[c + 16]);
        if (c < 15) {
          if (lane == 31) out[c] = up, out[c + 16] = run;  // slot x + 31 for diagonal x = query - key of the block
          up = __shfl_up_sync(0xffffffffu, up, 1);
          run = __shfl_up_sync(0xffffffffu, run, 1);
          if (lane == 0) up = run = 0.0f;
        }
      }
      __syncwarp();
      const float done = lane < 15 ? out[lane] : lane < 16 ? 0.0f : lane == 31 ? up : out[46 - lane] + up;
      up = __shfl_up_sync(0xffffffffu, up, 16);
      if (lane >= 16) run += up;
      float* mine = acc + warp * W;
      auto add = [&](int slot, float v) {
        const int delta = pw - (j0 + 32 * wq) + slot - 31;
        if (delta <= -P.D) lo += v;
        else if (delta >= P.D) hi += v;
        else mine[delta + P.D] += v;
      };
      if (lane != 15) add(lane < 15 ? lane : 46 - lane, done);
      add(62 - lane, run);
    }
    if (err) {
      // A wait of this warp gave up, where the others' may not have: it takes part in the barriers that are left, the
      // same number for every warp, so that nobody waits for it for good.
      uint32_t bits[4];
      key_bits(P.mask ? P.mask + static_cast<size_t>(b) * P.nk : nullptr, j0, P.nk, lane, bits);
      const int g0 = per > 0 ? first / per : 0;
      const int heads = (bits[0] | bits[1] | bits[2] | bits[3]) != 0 && last > first ? (last - 1) / per - g0 + 1 : 0;
      for (int n = barriers_left(heads, head < 0 ? 0 : head - g0 + 1, dw); n > 0; --n) work_barrier();
    } else if (dw) {
      if (head >= 0) flush();
      zero_heads(head + 1, P.G);
    }
    if (!err && t > 0) err = !tc_wait(&S.acc_done, (t - 1) & 1);
    tc_fence_after();
    const int c0 = 32 * cg;
    if (c0 < P.d) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {  // dV, dK
        uint32_t v[32];
        if (t > 0) {
          tmem_ld32_async(tm + lanes + (which ? kColB : kColA) + c0, v);
          tmem_wait_ld(v);
        }
        if (j >= P.nk) continue;
        if (!far_unit && P.near_segs > 1) {
          // joined in 32 bits: [key head][key tile][segment][row][dV, dK][64]
          const size_t per_head = static_cast<size_t>((P.nk + kTcRows - 1) / kTcRows) * P.near_segs;
          float* dst = P.near_part + ((static_cast<size_t>(b) * P.Hkv + hk) * per_head + near) * (kTcRows * 128) +
                       row * 128 + 64 * which + c0;
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (c0 + e < P.d)
              *reinterpret_cast<float4*>(dst + e) =
                  t > 0 ? make_float4(__uint_as_float(v[e]), __uint_as_float(v[e + 1]), __uint_as_float(v[e + 2]),
                                      __uint_as_float(v[e + 3]))
                        : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        } else if (row < sink_rows) {
          // joined in 32 bits: [key head][sink tile][key tile, segments][sink row][dV, dK][64]
          const size_t seg = far_unit ? unit % P.far_segs + 1 : 0;
          float* dst = P.sink_part +
                       (((static_cast<size_t>(b) * P.Hkv + hk) * P.sink_tiles + tile) * (P.far_segs + 1) + seg) *
                           (min(P.sinks, kTcRows) * 128) + row * 128 + 64 * which + c0;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c0 + e < P.d) dst[e] = t > 0 ? __uint_as_float(v[e]) : 0.0f;
        } else if (!far_unit) {
          store_row32<BF16>(which ? P.d_k : P.d_v, b, hk, j, c0, P.d, v, which ? P.scale : 1.0f, t == 0);
        }
      }
    }
  }
  end_block<kStages>(err, P.status, warp == kTmaWarp, warp == kMmaWarp, &S.own_full, S.full, S.uses, &S.products);
  if (warp == kMmaWarp) tmem_dealloc(S.tmem, 256);
}

// Joins the parts of a row's dV and dK in order: those of its tile's segments, and a sink's far segments (where
// tiles have one segment, sinks' own tiles are part 0 of the latter).  grid (32 rows each, key heads, batch), four
// values of a row a thread at a time.
constexpr int kJoinRows = 32;
template <bool BF16>
__global__ void __launch_bounds__(256) join_kernel(AttnParams P) {
  wait_previous();
  allow_next();
  const int tile = blockIdx.x / (kTcRows / kJoinRows), r0 = blockIdx.x % (kTcRows / kJoinRows) * kJoinRows;
  const int hk = blockIdx.y, b = blockIdx.z, j0 = tile * kTcRows, tiles = (P.nk + kTcRows - 1) / kTcRows;
  const size_t head = static_cast<size_t>(b) * P.Hkv + hk;
  const bool near = P.near_segs > 1;
  const int sinks = tile < P.sink_tiles ? min(min(P.sinks, P.nk) - j0, kTcRows) : 0;
  const int rows = near ? min(P.nk - j0, kTcRows) : sinks, pitch = min(P.sinks, kTcRows) * 128;
  const float* np = P.near_part + (head * tiles + tile) * P.near_segs * (kTcRows * 128);
  const float* sp = P.sink_part + (head * P.sink_tiles + tile) * (P.far_segs + 1) * pitch;
  for (int x = threadIdx.x; x < kJoinRows * 32; x += 256) {
    const int row = r0 + x / 32, which = x % 32 / 16, c = x % 16 * 4;
    if (row >= rows || c >= P.d) continue;
    const int at = row * 128 + 64 * which + c;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](const float* part) {
      const float4 v = *reinterpret_cast<const float4*>(part + at);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    };
    if (near) {
#pragma unroll 4
      for (int k = 0; k < P.near_segs; ++k) add(np + static_cast<size_t>(k) * (kTcRows * 128));
    }
    if (row < sinks) {
#pragma unroll 8
      for (int k = near; k <= P.far_segs; ++k) add(sp + static_cast<size_t>(k) * pitch);
    }
    using T16 = typename E16<BF16>::T;
    const float mul = which ? P.scale : 1.0f;
    T16* out = row_ptr<T16>(which ? P.d_k : P.d_v, b, hk, j0 + row) + c;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack16<BF16>(s.x * mul, s.y * mul), pack16<BF16>(s.z * mul, s.w * mul));
  }
}

}  // namespace

template <bool BF16>
static cudaError_t launch_bwd(const AttnParams& P, cudaStream_t st) {
  TcParams T;
  T.a = P;
  auto maps = [&](int q_rows, int k_rows) {
    return tc_tmap(&T.q, P.q, BF16, P.d, P.nq, P.H, P.B, q_rows) &&
           tc_tmap(&T.d_o, P.d_o, BF16, P.d, P.nq, P.H, P.B, q_rows) &&
           tc_tmap(&T.k, P.k, BF16, P.d, P.nk, P.Hkv, P.B, k_rows) &&
           tc_tmap(&T.v, P.v, BF16, P.d, P.nk, P.Hkv, P.B, k_rows);
  };
  const size_t fixed = 1024 + 2 * kTcTileBytes + 2 * kStages * kHalfBytes + sizeof(BwdShared);
  const size_t smem = fixed + bias_ext_bytes(P);
  // Tables of distances up to 371 leave room for two CTAs an SM (8192 tokens, both directions: 363 us there, 441 at 372)
  auto sums = [](int D) { return kWork / 32 * (2 * D + 1) * sizeof(float); };
  const size_t smem_keys = smem + (P.dw_part ? sums(P.D) : 0);
  const size_t most = fixed + ext_table_bytes(DFS_MAX_BUCKET_DISTANCE);
  const int share = 256 * kElementRegs + 128 * kOtherRegs;
  cudaError_t e = prepare_kernel<tc_dq_kernel<BF16>>(most, kBwdThreads, share);
  if (e == cudaSuccess)
    e = prepare_kernel<tc_dkv_kernel<BF16>>(most + sums(DFS_MAX_BUCKET_DISTANCE), kBwdThreads, share);
  if (e != cudaSuccess) return e;
  if (!maps(kTcRows, kTcHalf)) return cudaErrorInvalidValue;
  e = launch_dependent(tc_dq_kernel<BF16>, tc_grid(P.nq, P.H, P.B), kBwdThreads, smem, st, T);
  if (e != cudaSuccess) return e;
  if (!maps(kTcHalf, kTcRows)) return cudaErrorInvalidValue;
  const unsigned tiles = (P.nk + kTcRows - 1) / kTcRows, units = tiles * P.near_segs + P.sink_tiles * P.far_segs;
  e = launch_dependent(tc_dkv_kernel<BF16>, units * P.Hkv * P.B, kBwdThreads, smem_keys, st, T);
  const unsigned joined = P.near_segs > 1 ? tiles : P.sink_tiles;
  if (e != cudaSuccess || joined == 0) return e;
  return launch_dependent(join_kernel<BF16>, dim3(joined * (kTcRows / kJoinRows), P.Hkv, P.B), 256, 0, st, P);
}

cudaError_t launch_attn_tc_bwd(const AttnParams& P, int dtype, cudaStream_t st) {
  return dtype == DFS_BF16 ? launch_bwd<true>(P, st) : launch_bwd<false>(P, st);
}

}  // namespace dfs
