// dfs_attn.cu -- C entry points of the local attention (include/dfsink.h):
// argument checks, workspace layout and the choice of kernels.
#include <algorithm>
#include <cmath>

#include "dfs_attn_tc.cuh"

using namespace dfs;

namespace {

constexpr int kMaxHeadDim = 64;
constexpr int kMaxRows = 1 << 28;   // positions and distances stay inside 32 bits
constexpr int kWindowAll = 1 << 30;

bool type_ok(int t) { return t == DFS_BF16 || t == DFS_F16 || t == DFS_F32; }

// DFS_OK, or why the problem cannot run
int problem_status(const dfs_attn_problem* p, const dfs_relbias* b) {
  if (!p || p->B < 0 || p->H < 0 || p->H_kv < 0 || p->n_q < 0 || p->n_k < 0 || p->d < 1 || !type_ok(p->dtype) ||
      p->window < 0 || p->sinks < 0 || !std::isfinite(p->scale))
    return DFS_ERR_INVALID_ARGUMENT;
  if (p->H > 0 && (p->H_kv == 0 || p->H % p->H_kv != 0)) return DFS_ERR_INVALID_ARGUMENT;
  if (b && b->weight &&
      (!b->lut || b->num_buckets < 1 || b->max_distance < 0 || b->max_distance > DFS_MAX_BUCKET_DISTANCE ||
       !type_ok(b->dtype)))
    return DFS_ERR_INVALID_ARGUMENT;
  if (p->d > kMaxHeadDim || p->n_q > kMaxRows || p->n_k > kMaxRows || p->q_start > kMaxRows ||
      p->q_start < -kMaxRows || p->B > 65535 || p->H > 65535)
    return DFS_ERR_UNSUPPORTED;
  return DFS_OK;
}

Strided strided(const dfs_strided& s) { return {static_cast<char*>(s.ptr), s.stride_b, s.stride_h, s.stride_n}; }

AttnParams params(const dfs_attn_problem* p, const dfs_attn_args* a) {
  AttnParams P = {};
  P.q = strided(a->q);
  P.k = strided(a->k);
  P.v = strided(a->v);
  P.o = strided(a->o);
  P.d_o = strided(a->d_o);
  P.d_q = strided(a->d_q);
  P.d_k = strided(a->d_k);
  P.d_v = strided(a->d_v);
  P.lse = a->lse;
  P.o_lo = p->dtype != DFS_F32 ? static_cast<char*>(a->o_lo) : nullptr;
  P.mask = a->mask;
  P.w = a->bias.weight;
  P.lut = a->bias.lut;
  P.nb = a->bias.num_buckets;
  P.D = a->bias.weight ? a->bias.max_distance : 0;
  P.wdtype = a->bias.dtype;
  P.status = a->status;
  P.B = p->B;
  P.H = p->H;
  P.Hkv = p->H_kv;
  P.G = p->H_kv > 0 ? p->H / p->H_kv : 1;
  P.nq = p->n_q;
  P.nk = p->n_k;
  P.d = p->d;
  P.causal = p->causal != 0;
  P.window = p->window == 0 ? kWindowAll : p->window < kWindowAll ? p->window : kWindowAll;
  P.sinks = p->sinks;
  P.qs = p->q_start;
  P.scale = p->scale;
  P.scale2 = p->scale * kLog2e;
  return P;
}

size_t round256(size_t x) { return (x + 255) / 256 * 256; }
size_t dsum_bytes(const dfs_attn_problem* p) {
  return round256(sizeof(float) * static_cast<size_t>(p->B) * p->H * p->n_q);
}
// The backward's key pass: units of work of a batch element and key head, each a CTA that walks steps of (head of
// the group, query tile).  Every query sees the sinks, so the CTAs of their key tiles would walk all query tiles,
// with the others done long before; where the queries beyond the window are many, they are cut into segments of
// their own of about an ordinary tile's length.  And where few key heads leave SMs idle, every tile's steps are cut
// into segments of at least four, up to two CTAs an SM (16 / 2 heads, 2048 tokens: see the key pass).
struct KeyUnits {
  int tiles, sink_tiles, far_segs, far_len, near_segs;
  int count() const { return tiles * near_segs + sink_tiles * far_segs; }
};
KeyUnits key_units(const dfs_attn_problem* p, int tile, int q_tile) {
  KeyUnits u{(p->n_k + tile - 1) / tile, 0, 0, 0, 1};
  if (q_tile == 0 || p->H_kv == 0 || u.tiles == 0) return u;
  const int64_t G = p->H / p->H_kv, q_tiles = (p->n_q + q_tile - 1) / q_tile;
  const int64_t seen = p->window == 0 ? q_tiles : (int64_t{tile} + p->window) / q_tile + 1;
  const int64_t steps = std::min<int64_t>(seen, q_tiles) * G;  // of an ordinary tile
  const int64_t ctas = int64_t{u.tiles} * p->H_kv * std::max(p->B, 1);
  u.near_segs = static_cast<int>(std::clamp<int64_t>(std::min<int64_t>(2 * 148 / ctas, steps / 4), 1, 32));
  if (p->window == 0 || p->sinks == 0) return u;
  const int64_t last = std::min(tile, p->n_k) - 1;  // key of the first tile
  const int64_t near_end = std::clamp<int64_t>(last + p->window - p->q_start, 0, p->n_q);
  const int64_t far = (q_tiles - (near_end + q_tile - 1) / q_tile) * G;  // of the first tile, the most
  const int64_t sink_tiles = (std::min(p->sinks, p->n_k) + tile - 1) / tile;
  // (with many sinks longer ones, so that their parts are no more than the key tiles)
  const int64_t len = std::max<int64_t>({steps / u.near_segs, 8, (far * sink_tiles + u.tiles - 1) / u.tiles});
  if (far < 2 * len) return u;
  u.sink_tiles = static_cast<int>(sink_tiles);
  u.far_segs = static_cast<int>((far + len - 1) / len);
  u.far_len = static_cast<int>(len);
  return u;
}
size_t near_part_bytes(const dfs_attn_problem* p, const KeyUnits& u) {
  return u.near_segs == 1 ? 0 : sizeof(float) * kTcRows * 128 * p->B * p->H_kv * u.tiles * u.near_segs;
}
size_t sink_part_bytes(const dfs_attn_problem* p, const KeyUnits& u) {
  return sizeof(float) * 128 * static_cast<size_t>(std::min<int>(p->sinks, kTcRows)) * p->B * p->H_kv * u.sink_tiles *
         (u.far_segs > 0 ? u.far_segs + 1 : 0);
}
constexpr int kSimtTile = 64;

// Whether an operand can be staged by TMA (and stored in 16-byte pieces): its address and the strides of
// its extents above 1 are multiples of 16 bytes.
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool staged(const dfs_strided& s, int n, int heads, int B, int piece = 8) {  // piece: elements of 16 bytes
  auto ok = [=](int64_t stride, int extent) { return extent <= 1 || (stride > 0 && stride % piece == 0); };
  return aligned16(s.ptr) && ok(s.stride_n, n) && ok(s.stride_h, heads) && ok(s.stride_b, B);
}
// The tensor-core kernels: 16-bit operands that TMA can stage.  fp32 operands keep all their bits on the
// SIMT kernels; a scale that is not positive would turn the running maximum of raw products around.
bool tensor_cores(const dfs_attn_problem* p, const dfs_attn_args* a) {
  const int64_t tiles = (std::max(p->n_q, p->n_k) + kTcRows - 1) / kTcRows + (p->n_q + kTcHalf - 1) / kTcHalf;
  return tiles * p->B * p->H < (int64_t{1} << 31) && p->dtype != DFS_F32 && p->d % 8 == 0 && p->scale > 0.0f &&
         p->H > 0 && p->n_q > 0 && p->n_k > 0 && tmap_available() && aligned16(a->o_lo) &&
         staged(a->q, p->n_q, p->H, p->B) && staged(a->o, p->n_q, p->H, p->B) &&
         staged(a->k, p->n_k, p->H_kv, p->B) && staged(a->v, p->n_k, p->H_kv, p->B);
}
// fp32 operands whose rows the other kernels read in 16-byte pieces
bool vector_rows(const dfs_attn_problem* p, const dfs_attn_args* a) {
  return p->dtype == DFS_F32 && p->d % 4 == 0 && staged(a->k, p->n_k, p->H_kv, p->B, 4) &&
         staged(a->v, p->n_k, p->H_kv, p->B, 4);
}
int rc(cudaError_t e) { return e == cudaSuccess ? DFS_OK : DFS_ERR_CUDA; }

}  // namespace

extern "C" int dfs_window_attn_fwd(const dfs_attn_problem* p, const dfs_attn_args* a, void* stream) {
  if (!a) return DFS_ERR_INVALID_ARGUMENT;
  const int s = problem_status(p, &a->bias);
  if (s != DFS_OK) return s;
  if (p->B == 0 || p->H == 0 || p->n_q == 0) return DFS_OK;
  if (!a->q.ptr || !a->o.ptr || (p->n_k > 0 && (!a->k.ptr || !a->v.ptr))) return DFS_ERR_INVALID_ARGUMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const AttnParams P = params(p, a);
  if (tensor_cores(p, a)) return rc(launch_attn_tc_fwd(P, p->dtype, st));
  return rc(launch_attn_simt_fwd(P, p->dtype, vector_rows(p, a) && staged(a->q, p->n_q, p->H, p->B, 4), st));
}

extern "C" size_t dfs_window_attn_bwd_work(const dfs_attn_problem* p, const dfs_relbias* b) {
  if (problem_status(p, b) != DFS_OK) return 0;
  const KeyUnits u = key_units(p, kTcRows, kTcHalf);
  size_t n = dsum_bytes(p) + round256(sink_part_bytes(p, u)) + near_part_bytes(p, u);
  if (b && b->weight) {
    const int units = std::max(u.count(), key_units(p, kSimtTile, 0).count());  // whichever kernels run
    n += sizeof(float) * static_cast<size_t>(p->H) * p->B * units * (2 * b->max_distance + 1);
  }
  return n;
}

extern "C" int dfs_window_attn_bwd(const dfs_attn_problem* p, const dfs_attn_args* a, void* work, size_t work_bytes,
                                   void* stream) {
  if (!a) return DFS_ERR_INVALID_ARGUMENT;
  const int s = problem_status(p, &a->bias);
  if (s != DFS_OK) return s;
  if (p->H == 0 && (p->B == 0 || p->H_kv == 0 || p->n_k == 0)) return DFS_OK;  // (else d_k and d_v are zeros)
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool dw = a->d_weight != nullptr && a->bias.weight != nullptr;
  if (a->d_weight && !a->bias.weight) return DFS_ERR_INVALID_ARGUMENT;
  if (p->B == 0)  // d_weight alone has elements: sums of nothing
    return !dw ? DFS_OK
               : rc(launch_bucket_sums(nullptr, p->H, 0, a->bias.max_distance, a->bias.lut, a->bias.num_buckets,
                                       a->bias.dtype, a->d_weight, st));
  if ((p->n_q > 0 && p->H > 0 && (!a->q.ptr || !a->o.ptr || !a->d_o.ptr || !a->d_q.ptr || !a->lse || !work)) ||
      (p->n_k > 0 && (!a->k.ptr || !a->v.ptr || !a->d_k.ptr || !a->d_v.ptr)))
    return DFS_ERR_INVALID_ARGUMENT;
  if (work_bytes < dfs_window_attn_bwd_work(p, dw ? &a->bias : nullptr)) return DFS_ERR_WORKSPACE;
  AttnParams P = params(p, a);
  P.dsum = static_cast<float*>(work);
  const bool tc = tensor_cores(p, a) && staged(a->d_o, p->n_q, p->H, p->B) && staged(a->d_q, p->n_q, p->H, p->B) &&
                  staged(a->d_k, p->n_k, p->H_kv, p->B) && staged(a->d_v, p->n_k, p->H_kv, p->B);
  const KeyUnits u = tc ? key_units(p, kTcRows, kTcHalf) : key_units(p, kSimtTile, 0);
  P.parts = p->B * u.count();
  P.sink_tiles = u.sink_tiles;
  P.far_segs = u.far_segs;
  P.far_len = u.far_len;
  P.near_segs = u.near_segs;
  char* at = static_cast<char*>(work) + dsum_bytes(p);
  P.sink_part = reinterpret_cast<float*>(at);
  at += round256(sink_part_bytes(p, u));
  P.near_part = reinterpret_cast<float*>(at);
  if (dw) P.dw_part = reinterpret_cast<float*>(at + near_part_bytes(p, u));
  if (p->n_q > 0 || p->n_k > 0) {
    const bool vec = vector_rows(p, a) && staged(a->q, p->n_q, p->H, p->B, 4) && staged(a->d_o, p->n_q, p->H, p->B, 4);
    const int r = rc(tc ? launch_attn_tc_bwd(P, p->dtype, st) : launch_attn_simt_bwd(P, p->dtype, vec, st));
    if (r != DFS_OK) return r;
  }
  if (!dw || p->H == 0) return DFS_OK;
  return rc(launch_bucket_sums(P.dw_part, p->H, P.parts, P.D, P.lut, P.nb, P.wdtype, a->d_weight, st));
}

static int decode(const dfs_attn_problem* p, const dfs_attn_args* a, const void* lengths, bool wide, void* stream) {
  if (!a) return DFS_ERR_INVALID_ARGUMENT;
  const int s = problem_status(p, &a->bias);
  if (s != DFS_OK) return s;
  if (p->n_q != 1) return DFS_ERR_INVALID_ARGUMENT;
  if (p->B == 0 || p->H == 0) return DFS_OK;
  if (!a->q.ptr || !a->o.ptr || !lengths || (p->n_k > 0 && (!a->k.ptr || !a->v.ptr))) return DFS_ERR_INVALID_ARGUMENT;
  AttnParams P = params(p, a);
  P.causal = 1;
  P.mask = nullptr;
  P.lengths = lengths;
  P.wide_lengths = wide;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // cache tiles staged by TMA, 4-byte reads of q
  const bool rows = p->dtype != DFS_F32 && p->d % 8 == 0 && p->n_k > 0 && tmap_available() &&
                    staged(a->q, 1, p->H, p->B) && staged(a->k, p->n_k, p->H_kv, p->B) &&
                    staged(a->v, p->n_k, p->H_kv, p->B);
  if (rows) return rc(launch_decode_mma(P, p->dtype, st));
  return rc(launch_decode_any(P, p->dtype, vector_rows(p, a), st));
}

extern "C" int dfs_window_attn_decode(const dfs_attn_problem* p, const dfs_attn_args* a, const int32_t* lengths,
                                      void* stream) {
  return decode(p, a, lengths, false, stream);
}
extern "C" int dfs_window_attn_decode_i64(const dfs_attn_problem* p, const dfs_attn_args* a, const int64_t* lengths,
                                          void* stream) {
  return decode(p, a, lengths, true, stream);
}
