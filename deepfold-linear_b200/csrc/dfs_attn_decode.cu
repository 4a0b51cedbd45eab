// dfs_attn_decode.cu -- local attention for one query per sequence over a cache
// (bf16, fp16 whose rows can be copied in 16-byte pieces).
//
// Reading the visible cache rows is all the time there is: 256 bytes of K and V
// a key at d = 64 for 4 d operations a query head.  A cluster of up to 16 CTAs
// shares one key head of one sequence and splits the tiles of 128 keys that hold
// visible ones (the sinks' and the window's) into equal runs.  In a CTA one warp
// keeps TMA copies in flight through a ring of stages and four warps take 32 keys
// of a tile each: S = Q K^T and O += P V for the group's heads as mma.sync
// m16n8k16 (16 heads by 8 keys; the tensor-core rate does not matter here, the
// small shape does).  Every warp keeps its own maximum and sum; warps join through
// shared memory, CTAs through distributed shared memory, in a fixed order and
// without a second launch.
//
// Measured: 12 sequences of 32 / 8 heads over up to 32768 keys (float16, d = 64)
// 111 us, 5.8 TB/s; 64 ragged sequences of 16 / 4 heads, window 4096, 47 us, 4.3
// TB/s (a run of eight tiles hardly fills the ring before it drains); one sequence,
// window 1024, 8 us, of which the launch is most.  (Copies by the threads
// themselves, 16 bytes each, cost 440 instructions a warp per 64 keys and held the
// reads to 4.2 TB/s.  A ring of six tiles where a CTA has its SM alone was slower:
// clusters of sixteen then find no room.)
#include <algorithm>
#include <type_traits>

#include "dfs_attn_tc.cuh"

namespace dfs {
namespace {

constexpr int kThreads = 160;      // four warps of products, one of copies
constexpr int kStages = 2;         // of K and V tiles: 64 KB, three CTAs an SM
constexpr int kHeads = 16;         // query heads of a CTA: the rows of an m16n8k16 product

// What a CTA found, read by its cluster: maxima, sums and sums of P V
template <int N>
struct Found {
  float m[N], l[N];
  float o[N][68];
};

struct DecodeShared {
  uint64_t full[kStages], empty[kStages];
  float m[4][kHeads], l[4][kHeads];       // the warps' maxima and sums
  Found<kHeads> found;
};

struct DecodeParams {
  CUtensorMap k, v;
  AttnParams a;
  int split, chunks;
};

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
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte of 16-byte piece c of row r of a tile (128-byte rows, 128-byte swizzle)
DFS_DEV uint32_t piece_at(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// Joins the cluster's CTAs in order, and writes the outputs: this one finishes every split-th head.
template <typename E, int N, int kBlock>
DFS_DEV void join_cluster(const AttnParams& P, const Found<N>& F, int b, int h0, int ng, int rank, int split) {
  if (split > 1) cluster_sync();
  for (int x = threadIdx.x; x < ng * P.d; x += kBlock) {
    const int head = x / P.d, c = x % P.d;
    if (head % split != rank) continue;
    float top = -INFINITY, sum = 0.0f, acc = 0.0f;
    if (split == 1) {
      sum = F.l[head];
      acc = F.o[head][c];
    } else {
      const uint32_t am = smem_u32(&F.m[head]), al = smem_u32(&F.l[head]), ao = smem_u32(&F.o[head][c]);
      for (int r = 0; r < split; ++r) top = fmaxf(top, dsmem_ld(dsmem_addr(am, r)));
      const float ref = top == -INFINITY ? 0.0f : top;
      for (int r = 0; r < split; ++r) {
        const float k = exp2f(dsmem_ld(dsmem_addr(am, r)) - ref);
        sum += dsmem_ld(dsmem_addr(al, r)) * k;
        acc += dsmem_ld(dsmem_addr(ao, r)) * k;
      }
    }
    // nothing visible: 0 exactly; a sum that is NaN (a NaN, or a logit of +inf) stays one
    row_ptr<E>(P.o, b, h0 + head, 0)[c] = from_f32<E>(sum == 0.0f ? 0.0f : acc / sum);
  }
  if (split > 1) cluster_sync();  // nobody leaves while its memory is read
}

// grid (split, key heads x head chunks, batch), clusters of `split` CTAs
template <typename E>
__global__ void __launch_bounds__(kThreads) decode_mma_kernel(const __grid_constant__ DecodeParams T) {
  constexpr bool BF16 = std::is_same<E, __nv_bfloat16>::value;
  extern __shared__ unsigned char raw[];
  const AttnParams& P = T.a;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  unsigned char* gen = raw + (base - smem_u32(raw));
  DecodeShared& S = *reinterpret_cast<DecodeShared*>(gen + kStages * 2 * kTcTileBytes);
  float* tab = reinterpret_cast<float*>(&S + 1);  // [heads][D + 1] bias of delta = 0 .. D
  const int tid = threadIdx.x, warp = warp_index(), lane = tid % 32, rank = blockIdx.x, split = T.split;
  const int hk = blockIdx.y / T.chunks, g0 = blockIdx.y % T.chunks * kHeads, b = blockIdx.z;
  const int ng = min(kHeads, P.G - g0), h0 = hk * P.G + g0;
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&S.full[s], 1), mbar_init(&S.empty[s], 4);
    fence_mbar_init();
    prefetch_tmap(&T.k);
    prefetch_tmap(&T.v);
  }
  allow_next();
  wait_previous();
  const int len = seq_length(P, b), p = len - 1;
  const int lo = max(0, len - P.window), ns = min(P.sinks, lo);  // keys [0, ns) and [lo, len) are visible
  const int w0 = lo / kTcRows, sink_tiles = min((ns + kTcRows - 1) / kTcRows, w0);
  const int tiles = len > 0 ? sink_tiles + (len + kTcRows - 1) / kTcRows - w0 : 0;
  const int per = (tiles + split - 1) / split, t0 = min(rank * per, tiles), t1 = min(t0 + per, tiles);
  auto tile_key = [&](int t) { return (t < sink_tiles ? t : w0 + (t - sink_tiles)) * kTcRows; };
  const int ksteps = (P.d + 15) / 16;
  bool err = false;
  __syncthreads();
  const int t_near = t1 - 1;  // the run's newest tile
  const bool near_run = P.w && t1 > t0 && p - min(tile_key(t_near) + kTcRows - 1, p) < P.D;
  if (warp == 4) {
    int t = t0;
    for (; t < t1; ++t) {
      const int s = (t - t0) % kStages;
      if (!tc_wait(&S.empty[s], (((t - t0) / kStages) & 1) ^ 1)) { err = true; break; }
      if (lane == 0) {
        const uint32_t bar = smem_u32(&S.full[s]), dst = base + s * 2 * kTcTileBytes;
        mbar_arrive_expect_tx(bar, 2 * kTcTileBytes);
        tma_load_4d(dst, &T.k, 0, tile_key(t), hk, b, bar);
        tma_load_4d(dst + kTcTileBytes, &T.v, 0, tile_key(t), hk, b, bar);
      }
      __syncwarp();
    }
    // (always: a common question whether anybody gave up cost the other warps 1.5 us of 46, this 0.3)
    land_copies<kStages>(S.full, t - t0);
  }
  // the table where this run comes near the query (the copies are on their way)
  if (near_run && warp < 4)
    for (int x = tid; x <= P.D; x += 128) {
      const int bk = P.lut[P.D + x];
#pragma unroll 4
      for (int r = 0; r < ng; ++r) tab[r * (P.D + 1) + x] = bias_weight(P, h0 + r, bk);
    }

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
  if (P.w) {
    const int bk = P.lut[2 * P.D];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (g + 8 * r < ng) far[r] = bias_weight(P, h0 + g + 8 * r, bk);
  }
  if (near_run && warp < 4) asm volatile("bar.sync 1, 128;" ::: "memory");

  float o[8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;

  for (int t = t0; warp < 4 && t < t1; ++t) {
    const int st = (t - t0) % kStages;
    if (!tc_wait(&S.full[st], ((t - t0) / kStages) & 1)) { err = true; break; }
    const int j0 = tile_key(t) + 32 * warp;  // this warp's 32 keys
    const uint32_t ks = base + st * 2 * kTcTileBytes + 32 * warp * 128, vs = ks + kTcTileBytes;
    const bool edge = j0 + 32 > len || (j0 < lo && j0 + 32 > ns);  // some key of the 32 is hidden
    if (edge) {
      // a hidden row may hold anything, and 0 x NaN is NaN: zero its V
      unsigned char* vt = gen + (st * 2 + 1) * kTcTileBytes + 32 * warp * 128;
      for (int r = lane / 8; r < 32; r += 4)
        if (j0 + r >= len || (j0 + r < lo && j0 + r >= ns))
          *reinterpret_cast<uint4*>(vt + r * 128 + lane % 8 * 16) = make_uint4(0, 0, 0, 0);
      fence_async_smem();  // before the stage's next copy
      __syncwarp();
    }
    float s[4][4] = {};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < ksteps) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          uint32_t kf[4];
          ldsm4(ks + piece_at(16 * n + (lane / 16) * 8 + lane % 8, 2 * k + lane / 8 % 2), kf);
          mma16<BF16>(s[2 * n], qa[k], kf[0], kf[1]);
          mma16<BF16>(s[2 * n + 1], qa[k], kf[2], kf[3]);
        }
      }
    const bool near = near_run && p - min(j0 + 31, p) < P.D;
    float top[2] = {-INFINITY, -INFINITY};
    if (near) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + 8 * n + q2 + (e & 1), row = min(g + 8 * (e >> 1), ng - 1);
          s[n][e] = fmaf(s[n][e], P.scale2, tab[row * (P.D + 1) + min(max(p - j, 0), P.D)]);
        }
    } else {
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = fmaf(s[n][e], P.scale2, far[e >> 1]);
    }
    if (edge) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + 8 * n + q2 + (e & 1);
          if (j >= len || (j < lo && j >= ns)) s[n][e] = -INFINITY;
        }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
    uint32_t pa[2][4];
    float shrink[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float mn = fmaxf(m[r], top[r]), ref = mn == -INFINITY ? 0.0f : mn;
      shrink[r] = ex2(m[r] - ref);
      m[r] = mn;
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float a = ex2(s[n][2 * r] - ref), c = ex2(s[n][2 * r + 1] - ref);
        sum += a + c;
        pa[n / 2][2 * (n % 2) + r] = pack16<BF16>(a, c);
      }
      l[r] = l[r] * shrink[r] + sum;
    }
    if (__any_sync(0xffffffffu, shrink[0] != 1.0f || shrink[1] != 1.0f)) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= shrink[e >> 1];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (n < ksteps) {
          uint32_t vf[4];
          ldsm4t(vs + piece_at(16 * k + lane % 16, 2 * n + lane / 16), vf);
          mma16<BF16>(o[2 * n], pa[k], vf[0], vf[1]);
          mma16<BF16>(o[2 * n + 1], pa[k], vf[2], vf[3]);
        }
    __syncwarp();
    if (lane == 0) mbar_arrive(&S.empty[st]);
  }
  // join the warps: maxima and sums, then each warp in turn adds its part
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (warp < 4 && lane % 4 == 0) {
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
      S.found.m[row] = top;
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) sum += S.l[w][row] * ex2(S.m[w][row] - ref);
      S.found.l[row] = sum;
    }
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (warp == w)
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float* at = &S.found.o[g + 8 * (e >> 1)][8 * n + q2 + (e & 1)];
          const float v = o[n][e] * f[e >> 1];
          *at = w == 0 ? v : *at + v;
        }
    __syncthreads();
  }
  if (err) report_timeout(P.status);
  join_cluster<E, kHeads, kThreads>(P, S.found, b, h0, ng, rank, split);
}

// The same for every type and any strides, on the fp32 pipes: fp32 operands, and 16-bit ones that TMA cannot
// stage.  Sixteen lanes take a key at a time, four columns each, for four query heads; of four keys' products the
// sixteen sums end one to a lane (reduced and scattered together, a shuffle a sum), so a lane has one exponential.
// kVec: fp32 rows on 16-byte boundaries.  Measured (fp32): 64 sequences of 16 / 4 heads, 4096 keys of 512 bytes each:
// 112 us, 4.8 TB/s; 8 of 32 / 8 heads over 16384 keys: 96 us, 5.6 TB/s.
constexpr int kAnyThreads = 128, kAnyHeads = 4, kAnyKeys = 4;
constexpr int kAnyTeams = kAnyThreads / 16, kAnyStep = kAnyTeams * kAnyKeys;  // keys of the CTA at once

template <typename E, bool kVec>
__global__ void __launch_bounds__(kAnyThreads, 4) decode_any_kernel(AttnParams P, int split, int chunks) {
  extern __shared__ float tab[];  // [heads][D + 1] bias of delta = 0 .. D
  __shared__ Found<kAnyHeads> F;
  __shared__ float tm[kAnyTeams][kAnyHeads], tl[kAnyTeams][kAnyHeads];
  const int tid = threadIdx.x, lane = tid % 32, team = tid / 16, at = tid % 16, rank = blockIdx.x;
  const int hk = blockIdx.y / chunks, g0 = blockIdx.y % chunks * kAnyHeads, b = blockIdx.z;
  const int ng = min(kAnyHeads, P.G - g0), h0 = hk * P.G + g0;
  const int head = at % kAnyHeads, key = at / kAnyHeads;  // of the sum that ends in this lane
  allow_next();
  wait_previous();
  const int len = seq_length(P, b), p = len - 1;
  const int lo = max(0, len - P.window), ns = min(P.sinks, lo), total = ns + len - lo;  // keys [0, ns), [lo, len)
  const int per = ((total + split - 1) / split + kAnyStep - 1) / kAnyStep * kAnyStep;
  const int x0 = static_cast<int>(min(static_cast<int64_t>(rank) * per, static_cast<int64_t>(total)));
  const int x1 = static_cast<int>(min(static_cast<int64_t>(x0) + per, static_cast<int64_t>(total)));
  auto key_at = [&](int x) { return x < ns ? x : lo + (x - ns); };
  auto col = [&](int e) { return kVec ? 4 * at + e : at + 16 * e; };
  float far = 0.0f;
  bool near_run = false;
  if (P.w) {
    near_run = x1 > x0 && p - key_at(x1 - 1) < P.D;
    auto weight = [&](int r, int x) { return bias_weight(P, h0 + r, P.lut[P.D + x]); };
    if (near_run)
      for (int x = tid; x < ng * (P.D + 1); x += kAnyThreads) tab[x] = weight(x / (P.D + 1), x % (P.D + 1));
    far = weight(min(head, ng - 1), P.D);
  }
  float q[kAnyHeads][4], o[kAnyHeads][4];
#pragma unroll
  for (int h = 0; h < kAnyHeads; ++h)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[h][e] = 0.0f;
      q[h][e] = h < ng && col(e) < P.d ? to_f32<E>(row_ptr<E>(P.q, b, h0 + h, 0)[col(e)]) : 0.0f;
    }
  __syncthreads();
  float m = -INFINITY, l = 0.0f;
  auto row4 = [&](const Strided& s, int j, bool on, float (&v)[4]) {  // zeros for a key that is not visible
    const E* row = row_ptr<E>(s, b, hk, j);
    if (kVec) {
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (on && 4 * at < P.d) x = __ldcs(reinterpret_cast<const float4*>(row) + at);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = on && col(e) < P.d ? to_f32<E>(row[col(e)]) : 0.0f;
    }
  };
  for (int xb = x0; xb < x1; xb += kAnyStep) {
    const int xt = xb + team * kAnyKeys;
    float k[kAnyKeys][4], v[kAnyKeys][4];
#pragma unroll
    for (int r = 0; r < kAnyKeys; ++r) row4(P.k, key_at(min(xt + r, x1 - 1)), xt + r < x1, k[r]);
#pragma unroll
    for (int r = 0; r < kAnyKeys; ++r) row4(P.v, key_at(min(xt + r, x1 - 1)), xt + r < x1, v[r]);
    float s[16];
#pragma unroll
    for (int r = 0; r < kAnyKeys; ++r)
#pragma unroll
      for (int h = 0; h < kAnyHeads; ++h) {
        float t = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) t = fmaf(q[h][e], k[r][e], t);
        s[r * kAnyHeads + h] = t;
      }
#pragma unroll
    for (int w = 8; w > 0; w >>= 1)
#pragma unroll
      for (int i = 0; i < w; ++i) {
        const bool up = at & w;
        const float keep = up ? s[i + w] : s[i], send = up ? s[i] : s[i + w];
        s[i] = keep + __shfl_xor_sync(0xffffffffu, send, w);
      }
    const int x = xt + key;
    float val = -INFINITY;
    if (x < x1)
      val = fmaf(s[0], P.scale2,
                 near_run ? tab[min(head, ng - 1) * (P.D + 1) + min(p - key_at(x), P.D)] : far);
    float top = fmaxf(val, __shfl_xor_sync(0xffffffffu, val, 4));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.0f : mn;
    if (__any_sync(0xffffffffu, mn != m)) {
      const float shrink = exp2f(m - ref);
      l *= shrink;
#pragma unroll
      for (int h = 0; h < kAnyHeads; ++h) {
        const float f = __shfl_sync(0xffffffffu, shrink, h, 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[h][e] *= f;
      }
      m = mn;
    }
    const float pr = exp2f(val - ref);
    l += pr;
#pragma unroll
    for (int r = 0; r < kAnyKeys; ++r)
#pragma unroll
      for (int h = 0; h < kAnyHeads; ++h) {
        const float f = __shfl_sync(0xffffffffu, pr, r * kAnyHeads + h, 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[h][e] = fmaf(f, v[r][e], o[h][e]);
      }
  }
  // join the teams: two of a warp by a shuffle, the warps in turn
  l += __shfl_xor_sync(0xffffffffu, l, 4);
  l += __shfl_xor_sync(0xffffffffu, l, 8);
  if (key == 0) tm[team][head] = m, tl[team][head] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int t = 0; t < kAnyTeams; ++t) top = fmaxf(top, tm[t][head]);
  const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int t = 0; t < kAnyTeams; ++t) sum += tl[t][head] * exp2f(tm[t][head] - ref);
  if (tid < kAnyHeads) F.m[head] = top, F.l[head] = sum;
  const float scale = exp2f(m - ref);
#pragma unroll
  for (int h = 0; h < kAnyHeads; ++h) {
    const float f = __shfl_sync(0xffffffffu, scale, h, 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[h][e] *= f;
      o[h][e] += __shfl_xor_sync(0xffffffffu, o[h][e], 16);
    }
  }
#pragma unroll
  for (int w = 0; w < kAnyThreads / 32; ++w) {
    if (tid / 32 == w && lane < 16)
#pragma unroll
      for (int h = 0; h < kAnyHeads; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) F.o[h][col(e)] = w == 0 ? o[h][e] : F.o[h][col(e)] + o[h][e];
    __syncthreads();
  }
  join_cluster<E, kAnyHeads, kAnyThreads>(P, F, b, h0, ng, rank, split);
}

// How many CTAs share a (sequence, key head): until there are twice the CTAs that fit at once (`resident` an SM),
// so that ragged lengths even out, while each has 128 keys; short batches are split and large ones are not.  Sixteen
// only while no SM gets more than two, for they have to find room together (bfloat16, d = 64, 32768 keys: 8 key heads
// 38 -> 26 us with sixteen, 32 key heads 51 -> 58).
int split_of(const AttnParams& P, int chunks, int resident) {
  const long problems = static_cast<long>(P.B) * P.Hkv * chunks;
  const long tiles = (std::min<long>(static_cast<long>(P.window) + P.sinks, P.nk) + kTcRows - 1) / kTcRows;
  int split = 1;
  while (split < 8 && split * problems < 2 * resident * 148 && 2 * split <= tiles) split *= 2;
  return split == 8 && 16 * problems <= 2 * 148 && 16 <= tiles ? 16 : split;
}

template <typename E>
cudaError_t launch(const AttnParams& P, cudaStream_t st) {
  DecodeParams T;
  T.a = P;
  const bool bf16 = std::is_same<E, __nv_bfloat16>::value;
  if (!tc_tmap(&T.k, P.k, bf16, P.d, P.nk, P.Hkv, P.B) || !tc_tmap(&T.v, P.v, bf16, P.d, P.nk, P.Hkv, P.B))
    return cudaErrorInvalidValue;
  T.chunks = (P.G + kHeads - 1) / kHeads;
  T.split = split_of(P, T.chunks, 3);
  const size_t fixed = 1024 + kStages * 2 * kTcTileBytes + sizeof(DecodeShared);
  const size_t smem = fixed + (P.w ? std::min(P.G, kHeads) * (P.D + 1) * sizeof(float) : 0);
  const cudaError_t e =
      prepare_kernel<decode_mma_kernel<E>>(fixed + kHeads * (DFS_MAX_BUCKET_DISTANCE + 1) * sizeof(float));
  if (e != cudaSuccess) return e;
  return launch_clusters(decode_mma_kernel<E>, dim3(T.split, P.Hkv * T.chunks, P.B), T.split, kThreads, smem, st, T);
}

template <typename E, bool kVec>
cudaError_t launch_any(const AttnParams& P, cudaStream_t st) {
  const int chunks = (P.G + kAnyHeads - 1) / kAnyHeads, split = split_of(P, chunks, 4);
  const size_t smem = P.w ? kAnyHeads * (P.D + 1) * sizeof(float) : 0;
  return launch_clusters(decode_any_kernel<E, kVec>, dim3(split, P.Hkv * chunks, P.B), split, kAnyThreads, smem, st, P,
                         split, chunks);
}

}  // namespace

cudaError_t launch_decode_mma(const AttnParams& P, int dtype, cudaStream_t st) {
  return dtype == DFS_BF16 ? launch<__nv_bfloat16>(P, st) : launch<__half>(P, st);
}

cudaError_t launch_decode_any(const AttnParams& P, int dtype, bool vec, cudaStream_t st) {
  if (dtype == DFS_F32) return vec ? launch_any<float, true>(P, st) : launch_any<float, false>(P, st);
  return dtype == DFS_BF16 ? launch_any<__nv_bfloat16, false>(P, st) : launch_any<__half, false>(P, st);
}

}  // namespace dfs
