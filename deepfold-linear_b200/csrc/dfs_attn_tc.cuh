// dfs_attn_tc.cuh -- shared by the tensor-core local-attention kernels: operand
// staging, TMEM operands, tile information, bias tables.
#pragma once

#include "dfs_attn.cuh"
#include "dfs_tma.cuh"

namespace dfs {

constexpr int kTcRows = 128;              // rows of a CTA's own tile
constexpr int kTcTileBytes = 128 * 128;   // 128 rows of 64 16-bit elements, 128-byte swizzle
constexpr int kTcHalf = 64;               // rows of the tiles it walks

struct TcParams {
  CUtensorMap q, k, v, d_o;
  AttnParams a;
  int split = 1;  // CTAs that share a tile of queries
};

// instruction descriptor, kind::f16; b_mn: B is stored with its N index contiguous
__host__ __device__ constexpr uint32_t tc_idesc(int M, int N, bool bf16, bool b_mn) {
  return idesc_f16(M, N, bf16) | (static_cast<uint32_t>(b_mn) << 16);
}

// D(tmem) (+)= A(tmem) * B(smem): A's 16-bit elements lie two to a 32-bit column
DFS_DEV void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accum));
}

// The setup barrier of a block: the TMA warp, which initialises the mbarriers, only
// arrives and starts its copies at once; everybody else waits for the mbarriers,
// the TMEM address and each other.
template <int N>
DFS_DEV void setup_arrive() { asm volatile("bar.arrive 8, %0;" ::"n"(N) : "memory"); }
template <int N>
DFS_DEV void setup_wait() { asm volatile("bar.sync 8, %0;" ::"n"(N) : "memory"); }
DFS_DEV void prefetch_tmap(const CUtensorMap* tm) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tm)) : "memory");
}

// maximum of 32 values held as bits
DFS_DEV float max32u(const uint32_t (&v)[32]) {
  float a[3];
#pragma unroll
  for (int i = 0; i < 3; ++i)
    a[i] = fmax3(__uint_as_float(v[3 * i]), __uint_as_float(v[3 * i + 1]), __uint_as_float(v[3 * i + 2]));
#pragma unroll
  for (int i = 9; i + 1 < 32; i += 2)
    a[(i / 2) % 3] = fmax3(a[(i / 2) % 3], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
  return fmaxf(fmax3(a[0], a[1], a[2]), __uint_as_float(v[31]));
}

// One lane of a converged warp.  The compiler keeps what that lane computes in
// uniform registers, where the MMA takes its descriptors from; a branch on the
// lane number moved each there one by one, and issuing 8 MMAs took 600 clocks.
DFS_DEV bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
DFS_DEV float4 dsmem_ld4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
DFS_DEV int warp_index() { return __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x / 32), 0); }

// Descriptors of a tile at `s`: rows as the M or N index (a step of 16 along d is
// +2 in the address field), or as the contraction index (16 rows: +128).
DFS_DEV uint64_t tc_desc(uint32_t s) { return sw128_desc(s, 1024, 1024); }

// Product over d of two tiles whose rows are the M and N indices
DFS_DEV void tc_mma_kk(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, int ksteps) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < ksteps) mma_f16(d_tmem, a + 2 * k, b + 2 * k, idesc, k > 0);
}
// 128 x dp product over the 16 kSteps rows of B: A in TMEM, its 8 columns a step side
// by side, or (kSpread) two steps at the start of every 32 columns
template <int kSteps, bool kSpread = false>
DFS_DEV void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc, bool accum) {
#pragma unroll
  for (int k = 0; k < kSteps; ++k)
    mma_f16_ts(d_tmem, a_tmem + (kSpread ? 32 * (k / 2) + 8 * (k % 2) : 8 * k), b + 128 * k, idesc, accum || k > 0);
}

DFS_DEV void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr)
      : "memory");
}
DFS_DEV void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
DFS_DEV void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
DFS_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

DFS_DEV void tma_load_4d(uint32_t dst, const CUtensorMap* tm, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

template <bool BF16>
DFS_DEV uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool BF16>
DFS_DEV float2 unpack16(uint32_t x) {
  if (BF16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  const __half2 h = *reinterpret_cast<const __half2*>(&x);
  return __half22float2(h);
}

// Packed fp32 pairs.
DFS_DEV float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
DFS_DEV float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
DFS_DEV float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
DFS_DEV float2 both(float x) { return make_float2(x, x); }

// Wait for the phase with the given parity; false after some seconds (2^20 tries,
// each of which sleeps for 1.5 to 4 us by itself: measured).  No clock is read
// and the loop is short, for warps wait much of the time.
DFS_DEV bool tc_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  for (int tries = 1 << 20; tries > 0; --tries) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}

// A warp's arrival, after everything its lanes did before.
DFS_DEV void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// A wait that gave up: tell the host (status may be mapped host memory: a plain store)
DFS_DEV void report_timeout(int32_t* status) {
  if (status != nullptr) *reinterpret_cast<volatile int32_t*>(status) = DFS_ERR_DEVICE_TIMEOUT;
}

// A block that some wait of its warps made give up must not end before what it has started, for its shared memory and
// TMEM go to the next one: copies into the last stages of a ring of kStages (uses 0 .. n - 1 of it) ...
template <int kStages>
DFS_DEV void land_copies(uint64_t* full, int n) {
  for (int u = max(0, n - kStages); u < n; ++u) tc_wait(&full[u % kStages], (u / kStages) & 1);
}
// ... and the products that this warp's elected lane has issued.  (Where none gave up, somebody waited for all of them.)
DFS_DEV void end_products(uint64_t* bar) {
  if (elect_one()) mma_commit(bar);
  __syncwarp();
  tc_wait(bar, 0);
}
// The end of a block: err: a wait of this thread gave up; `uses` of the ring, written by the TMA warp.
template <int kStages>
DFS_DEV void end_block(bool err, int32_t* status, bool tma, bool mma, uint64_t* own, uint64_t* full, const int& uses,
                       uint64_t* products) {
  tc_fence_before();
  if (__syncthreads_or(err)) {
    if (err) report_timeout(status);
    if (tma) tc_wait(own, 0), land_copies<kStages>(full, uses);
    if (mma) end_products(products);
    __syncthreads();
  }
  tc_fence_after();
}

// Registers of this warpgroup (four warps) from here on.  The shares of a block
// must not add up to more than it was launched with.
template <int N>
DFS_DEV void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
DFS_DEV void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Bits c of [0, 128) with a <= c < b, as four words
DFS_DEV uint32_t range_word(int a, int b, int w) {
  const int lo = min(max(a - 32 * w, 0), 32), hi = min(max(b - 32 * w, 0), 32);
  const uint32_t below_hi = hi == 32 ? 0xffffffffu : (1u << hi) - 1u;
  const uint32_t below_lo = lo == 32 ? 0xffffffffu : (1u << lo) - 1u;
  return below_hi & ~below_lo;
}

// The bias table widened by its end values, so that a tile whose distances
// reach into the table needs no clamp: tab[delta + ext], ext = D + 255.
DFS_DEV int bias_ext(int D) { return D + 255; }
DFS_DEV void load_bias_ext(float* tab, const AttnParams& P, int h, int tid, int nthreads) {
  const int E = bias_ext(P.D), W = 2 * E + 1;
  for (int x0 = tid; x0 < W; x0 += 4 * nthreads) {  // four entries' look-ups in flight: each is two dependent loads
    int b[4];
    float v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = min(max(x0 + u * nthreads - E, -P.D), P.D) + P.D;
      b[u] = P.lut[at];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = bias_weight(P, h, b[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (x0 + u * nthreads < W) tab[x0 + u * nthreads] = v[u];
  }
}
constexpr size_t ext_table_bytes(int D) { return (2 * (D + 255) + 1) * sizeof(float); }
inline size_t bias_ext_bytes(const AttnParams& P) { return P.w ? ext_table_bytes(P.D) : 0; }

// One tile as the producer announces it: first key (or query) row, -1 for the
// end; whether it is plain (all pairs visible, one bias for all) and where its
// distances lie (1 beyond the bias table's far end, -1 beyond the other, 0 in
// it); for a tile that is not plain, the key mask's bits and the class of each of
// its blocks of 32 x 32, so that the element warps need no look at positions for
// most of them.
enum { kHidden = 0, kWhole = 1, kPartial = 2 };
struct TileInfo {
  int at, plain, side, head;
  uint32_t bits[4];
  uint8_t cls[16];  // kind | (side + 1) << 2
};

// Mask bits of keys [j0, j0 + 128) (a full warp; all lanes get the four words)
DFS_DEV void key_bits(const uint8_t* mask, int j0, int nk, int lane, uint32_t (&bits)[4]) {
  uint32_t nib = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int j = j0 + 4 * lane + e;
    if (j < nk && (mask == nullptr || mask[j] != 0)) nib |= 1u << e;
  }
  const uint32_t part = nib << (4 * (lane & 7));
#pragma unroll
  for (int w = 0; w < 4; ++w) bits[w] = __reduce_or_sync(0xffffffffu, (lane >> 3) == w ? part : 0u);
}

// Key tiles of kRows seen by positions p0..p1: the sink tiles [0, ns), then the window's [t0, t1), which go on to the
// last sink where the sinks reach into them or (without causality) past them.
template <int kRows>
struct TcKeyTiles {
  int ns, t0, t1;
  DFS_DEV TcKeyTiles(const AttnParams& P, int p0, int p1) {
    int lo, hi;
    near_keys(P, p0, p1, lo, hi);
    t0 = lo / kRows;
    t1 = hi > lo ? (hi + kRows - 1) / kRows : t0;
    ns = (sink_keys(P, p1) + kRows - 1) / kRows;
    if (hi > lo && ns > t0) t1 = max(t1, ns), ns = t0;
  }
  DFS_DEV int count() const { return ns + (t1 - t0); }
  DFS_DEV int operator[](int x) const { return x < ns ? x : t0 + (x - ns); }
};

// Visible keys j0..j0+31 for position p, the mask apart.
DFS_DEV uint32_t key_word(const AttnParams& P, int p, int j0) {
  const int top = min(P.causal ? p + 1 : P.nk, P.nk);
  return range_word(p - P.window + 1 - j0, min(top, p + P.window) - j0, 0) | range_word(0, min(P.sinks, top) - j0, 0);
}
// Visible queries at positions p0..p0+31 for key j, the mask apart.
DFS_DEV uint32_t query_word(const AttnParams& P, int j, int p0) {
  uint32_t v = range_word(P.causal ? j - p0 : j - P.window + 1 - p0, j + P.window - p0, 0);
  if (j < P.sinks) v |= range_word(P.causal ? j - p0 : 0, 32, 0);
  return v;
}
// Class of the block of 32 queries from position p0 and 32 keys from j0, whose mask bits are `bits`; o = p0 - j0.
DFS_DEV int block_class(const AttnParams& P, int o, int j0, uint32_t bits) {
  const int far = o < 0 ? -o : o;
  const bool hidden = bits == 0 || j0 >= P.nk || (P.causal && o < -31) || (far >= P.window + 31 && j0 >= P.sinks);
  const bool whole = bits == ~0u && j0 + 31 < P.nk && (!P.causal || o >= 31) &&
                     (far < P.window - 31 || j0 + 31 < P.sinks);
  const int side = P.w == nullptr || o - 31 >= P.D ? 1 : o + 31 <= -P.D ? -1 : 0;
  return (hidden ? kHidden : whole ? kWhole : kPartial) | (side + 1) << 2;
}
// The tiles of 32 NP queries x 32 NJ keys that are plain, the key mask apart, by o = (first query's position) -
// (first key): all distances beyond the bias table, all inside the window.  Two comparisons a tile keep the
// producer's chain of instructions shorter than a tile's work; it runs alone, without the instruction cache to
// itself, and classing every tile's blocks (600 clocks) held everybody up.
template <int NP, int NJ>
struct PlainTiles {
  int a1, b1, a2, b2;
  DFS_DEV explicit PlainTiles(const AttnParams& P) {
    const int w = P.window - 1, low = P.w ? P.D : P.causal ? 0 : -w;
    a1 = low + 32 * NJ - 1;        // beyond the far end (or anywhere, without a bias)
    b1 = w - (32 * NP - 1);
    a2 = -w + 32 * NJ - 1;         // beyond the other end
    b2 = P.w && !P.causal ? -P.D - (32 * NP - 1) : a2 - 1;
  }
  DFS_DEV int side(int o) const { return o >= a1 && o <= b1 ? 1 : o >= a2 && o <= b2 ? -1 : 0; }  // 0: not plain
};

// What the producer (a full warp) says of the tile of 32 NP queries from position p0 and 32 NJ keys from j0 with
// the given mask bits (all ones if `whole`); -1 for `at`: the end.  A lane per block, joined by votes.
template <int NP, int NJ>
DFS_DEV void describe_tile(const AttnParams& P, const PlainTiles<NP, NJ>& plain, TileInfo& f, int at, int head, int p0,
                           int j0, bool whole_mask, const uint32_t (&bits)[4], int lane) {
  static_assert(NP * NJ <= 16, "blocks of a tile");
  int side = plain.side(p0 - j0);
  const bool easy = at < 0 || (side != 0 && whole_mask && j0 + 32 * NJ <= P.nk);
  if (!easy) {
    const int jb = lane % NJ, pb = lane / NJ % NP;
    uint32_t own = bits[0];
#pragma unroll
    for (int w = 1; w < NJ; ++w) own = jb == w ? bits[w] : own;
    const int jl = j0 + 32 * jb, cls = block_class(P, p0 + 32 * pb - jl, jl, own);
    if (lane < NP * NJ) f.cls[lane] = static_cast<uint8_t>(cls);  // (the other lanes repeat blocks)
    if (lane < NJ) f.bits[lane] = own;
    side = __all_sync(0xffffffffu, (cls >> 2) == 2) ? 1 : __all_sync(0xffffffffu, (cls >> 2) == 0) ? -1 : 0;
  }
  if (lane == 0) {
    f.at = at;
    f.head = head;
    f.side = side;
    f.plain = easy;
  }
  __syncwarp();
}

// A strided (B, heads, n, d) operand of 16-bit elements as {d, n, heads, B}, boxes of 64 x rows.
bool tc_tmap(CUtensorMap* tm, const Strided& s, bool bf16, int d, int n, int heads, int B, int rows = kTcRows);

// One CTA per tile of each (head, batch element), heads fastest and tiles slowest:
// the CTAs with the most tiles to walk start first, over all heads.  (Tiles
// fastest left a head's longest CTA among the last: 35 % of SM time idle at
// N = 4096, causal.)
inline unsigned tc_grid(int n, int heads, int B) {
  return static_cast<unsigned>((n + kTcRows - 1) / kTcRows) * heads * B;
}

// A dependent launch (launch_dependent) whose blocks come in clusters of `size` along x.
template <typename... Params, typename... Args>
cudaError_t launch_clusters(void (*kern)(Params...), dim3 grid, int size, int threads, size_t smem, cudaStream_t st,
                            const Args&... args) {
  if (size > 8) {  // beyond what every device has: opted in
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = size;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = size > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

cudaError_t launch_attn_tc_fwd(const AttnParams& P, int dtype, cudaStream_t st);
cudaError_t launch_attn_tc_bwd(const AttnParams& P, int dtype, cudaStream_t st);

}  // namespace dfs
