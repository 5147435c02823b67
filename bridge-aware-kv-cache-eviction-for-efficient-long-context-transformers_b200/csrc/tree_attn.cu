// Attention of drafted tokens over a paged KV cache (tree attention): a tree of draft nodes, a
// chain of new tokens, or one decoded token per sequence.
//
// Sequence i has len tokens in its pages, of which the last m = num_nodes[i] are its nodes;
// c = len - m are context. Node t sees every key j < c, and of the nodes (key c + u) its
// ancestors and itself (parents), the u with tree_mask[t, u], or u <= t (neither given):
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max),  lse = max + log sum p_j,
// 0 and -inf where nothing is seen and for t >= m. Unseen places are selected away, never
// multiplied by 0, so NaN or infinities there do not reach the output.
//
// The G = Hq / Hkv query heads of a KV head and the T nodes form G*T rows that share every
// key, row = t * G + g: a key is read once for all of them.

#include "cab_host.h"
#include "cab_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

namespace cab {
namespace tree {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  return static_cast<float>(x);
}
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  return static_cast<T>(x);
}

struct Params {
  const void *q, *k, *v;
  void* out;
  float* lse;
  int64_t qs[3], os[3], ks[3], vs[3];  // q / out {n, h, t}, pages {p, h, s}
  const int32_t *table, *lens, *rows, *nodes, *parents;
  const uint8_t* mask;
  int64_t table_stride, parents_stride, mask_stride;
  int64_t pages, page_size, width, num_rows;
  int32_t n, Hq, Hkv, G, T, D;
  float scale_log2;
  int32_t splits;
  float *part_o, *part_ml;
};

struct Seq {
  int32_t row, len, m, ctx;  // a sequence that does not fit its row has len = m = 0
};

__device__ __forceinline__ Seq load_seq(const Params& p, int i) {
  Seq s{0, 0, 0, 0};
  const int row = p.rows ? p.rows[i] : i;
  if (row < 0 || row >= p.num_rows) return s;
  const int len = p.lens[row];
  const int m = p.nodes ? p.nodes[i] : p.T;
  if (m < 0 || m > p.T || len < m || len > p.width * p.page_size) return s;
  s.row = row;
  s.len = len;
  s.m = m;
  s.ctx = len - m;
  return s;
}

// Whether node t sees node u (both < m). A parent that does not come before its child ends
// the walk: such a node is taken for a root.
__device__ __forceinline__ bool sees(const Params& p, int i, int t, int u) {
  if (p.parents) {
    const int32_t* up = p.parents + i * p.parents_stride;
    int x = t;
    while (x > u) {
      const int y = up[x];
      if (y >= x) return false;
      x = y;
    }
    return x == u;
  }
  if (p.mask) return p.mask[i * p.mask_stride + static_cast<int64_t>(t) * p.T + u] != 0;
  return u <= t;
}

// Keys that the rows up to node t_last can see: with a mask any node may see any other.
__device__ __forceinline__ int key_limit(const Params& p, const Seq& s, int t_last) {
  return s.ctx + (p.mask ? s.m : min(s.m, t_last + 1));
}

// ------------------------------------------------------------------ CUDA-core path
// fp32 arithmetic for any type, page size and head_dim <= 256: float32 caches, and shapes the
// tensor-core path does not take. One CTA per (sequence, KV head, 16 rows, key split); a warp
// owns 4 rows, a lane one key of the 32-key tile for the scores and a set of columns for the
// output, so the row maximum and sum stay in the warp.
constexpr int kRowsTile = 16, kKeysTile = 32, kSimtThreads = 128;

template <typename T, int DC>
__global__ void __launch_bounds__(kSimtThreads) simt_kernel(const Params p) {
  extern __shared__ float sm[];
  const int Dp = (p.D + 3) & ~3, ld = Dp + 4;
  float* sQ = sm;                    // [16][Dp]
  float* sK = sQ + kRowsTile * Dp;   // [32][ld]
  float* sV = sK + kKeysTile * ld;   // [32][Dp]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = p.G * p.T, tiles_r = (R + kRowsTile - 1) / kRowsTile;
  const int unit = blockIdx.x, split = blockIdx.y;
  const int rt = unit % tiles_r, hk = (unit / tiles_r) % p.Hkv, i = unit / (tiles_r * p.Hkv);
  const int row0 = rt * kRowsTile;
  const Seq s = load_seq(p, i);
  const int keys = s.m > 0 ? key_limit(p, s, min(p.T - 1, (row0 + kRowsTile - 1) / p.G)) : 0;
  const int tiles = (keys + kKeysTile - 1) / kKeysTile;
  const int per = (tiles + p.splits - 1) / p.splits;
  const int t_lo = min(tiles, split * per), t_hi = min(tiles, t_lo + per);

  for (int e = threadIdx.x; e < kRowsTile * Dp; e += kSimtThreads) {
    const int r = e / Dp, d = e - r * Dp, row = row0 + r;
    float x = 0.f;
    if (row < R && d < p.D)
      x = to_f32(static_cast<const T*>(p.q)[i * p.qs[0] + (hk * p.G + row % p.G) * p.qs[1] + (row / p.G) * p.qs[2] + d]);
    sQ[e] = x;
  }
  float acc[4][DC], m[4], l[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < DC; ++c) acc[r][c] = 0.f;
  }
  const int32_t* table = p.table + s.row * p.table_stride;
  for (int tile = t_lo; tile < t_hi; ++tile) {
    const int key0 = tile * kKeysTile;
    __syncthreads();
    for (int e = threadIdx.x; e < kKeysTile * Dp; e += kSimtThreads) {
      const int j = e / Dp, d = e - j * Dp, key = key0 + j;
      float a = 0.f, b = 0.f;
      if (key < keys && d < p.D) {
        const int64_t pg = table[key / p.page_size], slot = key % p.page_size;
        if (pg >= 0 && pg < p.pages) {
          a = to_f32(static_cast<const T*>(p.k)[pg * p.ks[0] + hk * p.ks[1] + slot * p.ks[2] + d]);
          b = to_f32(static_cast<const T*>(p.v)[pg * p.vs[0] + hk * p.vs[1] + slot * p.vs[2] + d]);
        }
      }
      sK[j * ld + d] = a;
      sV[j * Dp + d] = b;
    }
    __syncthreads();
    float sc[4] = {0.f, 0.f, 0.f, 0.f};
    const float4* kr = reinterpret_cast<const float4*>(sK + lane * ld);
    for (int d = 0; d < Dp / 4; ++d) {
      const float4 kk = kr[d];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float4 qq = reinterpret_cast<const float4*>(sQ + (warp * 4 + r) * Dp)[d];
        sc[r] = fmaf(qq.x, kk.x, fmaf(qq.y, kk.y, fmaf(qq.z, kk.z, fmaf(qq.w, kk.w, sc[r]))));
      }
    }
    const int key = key0 + lane;
    bool there = key < keys;
    if (there) {
      const int64_t pg = table[key / p.page_size];
      there = pg >= 0 && pg < p.pages;
    }
    uint32_t seen[4];
    float pr[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = (row0 + warp * 4 + r) / p.G;
      const bool ok = there && t < s.m && (key < s.ctx || sees(p, i, t, key - s.ctx));
      seen[r] = __ballot_sync(0xffffffffu, ok);
      float x = ok ? sc[r] * p.scale_log2 : -INFINITY, mx = x;
#pragma unroll
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float mn = fmaxf(m[r], mx);
      const float alpha = m[r] == -INFINITY ? 0.f : ex2(m[r] - mn);
      pr[r] = x == -INFINITY ? 0.f : ex2(x - mn);  // unseen, or a score of -inf
      float sum = pr[r];
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[r] = l[r] * alpha + sum;
      m[r] = mn;
#pragma unroll
      for (int c = 0; c < DC; ++c) acc[r][c] *= alpha;
    }
    for (int j = 0; j < kKeysTile; ++j) {
      float vv[DC];
#pragma unroll
      for (int c = 0; c < DC; ++c) vv[c] = lane + 32 * c < Dp ? sV[j * Dp + lane + 32 * c] : 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float w = __shfl_sync(0xffffffffu, pr[r], j);
        if (seen[r] >> j & 1u) {
#pragma unroll
          for (int c = 0; c < DC; ++c) acc[r][c] = fmaf(w, vv[c], acc[r][c]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = row0 + warp * 4 + r;
    if (row >= R) continue;
    if (p.splits == 1) {
      const int h = hk * p.G + row % p.G, t = row / p.G;
      T* o = static_cast<T*>(p.out) + i * p.os[0] + h * p.os[1] + t * p.os[2];
      const float inv = l[r] != 0.f ? 1.f / l[r] : 0.f;  // a row without keys gives 0; NaN stays NaN
#pragma unroll
      for (int c = 0; c < DC; ++c)
        if (lane + 32 * c < p.D) o[lane + 32 * c] = from_f32<T>(acc[r][c] * inv);
      if (p.lse && lane == 0) p.lse[(static_cast<int64_t>(i) * p.Hq + h) * p.T + t] = (m[r] + log2f(l[r])) * kLn2;
    } else {
      const int64_t slot = (static_cast<int64_t>(unit) * p.splits + split) * kRowsTile + warp * 4 + r;
#pragma unroll
      for (int c = 0; c < DC; ++c)
        if (lane + 32 * c < p.D) p.part_o[slot * p.D + lane + 32 * c] = acc[r][c];
      if (lane == 0) {
        p.part_ml[slot * 2] = m[r];
        p.part_ml[slot * 2 + 1] = l[r];
      }
    }
  }
}

// Joins the splits of a row: one warp per row, always in the order of the keys.
template <typename T, int DC>
__global__ void __launch_bounds__(kSimtThreads) simt_join_kernel(const Params p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = p.G * p.T, tiles_r = (R + kRowsTile - 1) / kRowsTile;
  const int64_t total = static_cast<int64_t>(p.n) * p.Hkv * tiles_r * kRowsTile;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  if (x >= total) return;
  const int64_t unit = x / kRowsTile;
  const int r = static_cast<int>(x - unit * kRowsTile);
  const int rt = static_cast<int>(unit % tiles_r), hk = static_cast<int>(unit / tiles_r % p.Hkv);
  const int64_t i = unit / tiles_r / p.Hkv;
  const int row = rt * kRowsTile + r;
  if (row >= R) return;
  float m = -INFINITY;
  for (int k = lane; k < p.splits; k += 32) m = fmaxf(m, p.part_ml[((unit * p.splits + k) * kRowsTile + r) * 2]);
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float acc[DC], l = 0.f;
#pragma unroll
  for (int c = 0; c < DC; ++c) acc[c] = 0.f;
  for (int k = 0; k < p.splits; ++k) {
    const int64_t slot = (unit * p.splits + k) * kRowsTile + r;
    const float mk = p.part_ml[slot * 2], lk = p.part_ml[slot * 2 + 1];
    if (mk == -INFINITY && lk == 0.f) continue;
    const float w = ex2(mk - m);
    l = fmaf(w, lk, l);
#pragma unroll
    for (int c = 0; c < DC; ++c)
      if (lane + 32 * c < p.D) acc[c] = fmaf(w, p.part_o[slot * p.D + lane + 32 * c], acc[c]);
  }
  const int h = hk * p.G + row % p.G, t = row / p.G;
  T* o = static_cast<T*>(p.out) + i * p.os[0] + h * p.os[1] + t * p.os[2];
  const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int c = 0; c < DC; ++c)
    if (lane + 32 * c < p.D) o[lane + 32 * c] = from_f32<T>(acc[c] * inv);
  if (p.lse && lane == 0) p.lse[(i * p.Hq + h) * p.T + t] = (m + log2f(l)) * kLn2;
}

// ------------------------------------------------------------------ host side
inline int simt_splits(int64_t units, int64_t tokens) {
  const int64_t want = (static_cast<int64_t>(current_sm_count()) * 6 + units - 1) / units;
  return static_cast<int>(std::max<int64_t>(1, std::min({want, (tokens + kKeysTile - 1) / kKeysTile, (int64_t)64})));
}

struct Layout {
  bool tc;
  int splits;
  int64_t units;
  size_t part_o, part_ml, total;
};

inline Layout layout(int64_t n, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int64_t page_size, int64_t width, int dtype) {
  Layout L{};
  (void)dtype;
  const int64_t R = Hq / Hkv * T;
  L.units = n * Hkv * ((R + kRowsTile - 1) / kRowsTile);
  L.splits = simt_splits(L.units, width * page_size);
  if (L.splits > 1) {
    const size_t slots = static_cast<size_t>(L.units) * L.splits * kRowsTile;
    L.part_o = 0;
    L.part_ml = (slots * D * 4 + 15) & ~size_t(15);
    L.total = L.part_ml + slots * 8;
  }
  return L;
}

template <typename T, int DC>
int launch_simt(const Params& p, int64_t units, cudaStream_t st) {
  const int Dp = (p.D + 3) & ~3;
  const size_t smem = static_cast<size_t>(kRowsTile * Dp + kKeysTile * (Dp + 4) + kKeysTile * Dp) * 4;
  if (smem > 48 * 1024) cudaFuncSetAttribute(simt_kernel<T, DC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  simt_kernel<T, DC><<<dim3(static_cast<unsigned>(units), static_cast<unsigned>(p.splits)), kSimtThreads, smem, st>>>(p);
  if (int rc = check_launch("tree_attn simt_kernel")) return rc;
  if (p.splits == 1) return CAB_OK;
  simt_join_kernel<T, DC><<<static_cast<unsigned>((units * kRowsTile + 3) / 4), kSimtThreads, 0, st>>>(p);
  return check_launch("tree_attn simt_join_kernel");
}

template <typename T>
int launch_simt_d(const Params& p, int64_t units, cudaStream_t st) {
  if (p.D <= 64) return launch_simt<T, 2>(p, units, st);
  if (p.D <= 128) return launch_simt<T, 4>(p, units, st);
  return launch_simt<T, 8>(p, units, st);
}

inline int check_sizes(const cab_page_cache* c, int64_t n, int64_t Hq, int64_t T) {
  if (int rc = pages::check_cache(c, "tree_attn", true, false)) return rc;
  if (n <= 0 || Hq <= 0 || T <= 0) return fail(CAB_ERR_INVALID_ARG, "tree_attn: non-positive size");
  if (Hq % c->heads != 0) return fail(CAB_ERR_INVALID_ARG, "tree_attn: Hq %% Hkv != 0");
  if (c->dim > 256) return fail(CAB_ERR_UNSUPPORTED, "tree_attn: head_dim %lld (at most 256)", (long long)c->dim);
  if (n > pages::kMaxRows || Hq > 65536 || T > 65536 || n * Hq * T >= (int64_t)1 << 31)
    return fail(CAB_ERR_UNSUPPORTED, "tree_attn: more than 2^31 rows, or a size above 65536");
  return CAB_OK;
}

}  // namespace tree
}  // namespace cab

extern "C" int cab_tree_attn_workspace_size(const cab_page_cache* cache, int64_t n, int64_t Hq, int64_t T, size_t* bytes) {
  using namespace cab;
  if (!bytes) return fail(CAB_ERR_INVALID_ARG, "tree_attn_workspace_size: NULL output");
  if (int rc = tree::check_sizes(cache, n, Hq, T)) return rc;
  *bytes = tree::layout(n, Hq, cache->heads, T, cache->dim, cache->page_size, cache->width, cache->dtype).total;
  return CAB_OK;
}

extern "C" int cab_tree_attn_fwd(const cab_page_cache* cache, int64_t layer, const void* q, void* out, float* lse,
                                 int64_t n, int64_t Hq, int64_t T, const int64_t* q_strides, const int64_t* o_strides,
                                 const int32_t* rows, const int32_t* num_nodes, const int32_t* parents,
                                 int64_t parents_stride, const uint8_t* tree_mask, int64_t mask_stride,
                                 float softmax_scale, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace cab;
  using namespace cab::tree;
  if (int rc = check_sizes(cache, n, Hq, T)) return rc;
  if (!q || !out || !q_strides || !o_strides) return fail(CAB_ERR_INVALID_ARG, "tree_attn: NULL pointer");
  if (layer < 0 || layer >= cache->layers) return fail(CAB_ERR_INVALID_ARG, "tree_attn: layer %lld of %lld", (long long)layer, (long long)cache->layers);
  if (!rows && n > cache->rows) return fail(CAB_ERR_INVALID_ARG, "tree_attn: more sequences than rows");
  if (parents && tree_mask) return fail(CAB_ERR_INVALID_ARG, "tree_attn: parents or a mask, not both");
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale)) return fail(CAB_ERR_INVALID_ARG, "tree_attn: softmax_scale must be > 0 and finite");
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] < 0 || o_strides[i] < 0) return fail(CAB_ERR_INVALID_ARG, "tree_attn: negative stride");
  const Layout L = layout(n, Hq, cache->heads, T, cache->dim, cache->page_size, cache->width, cache->dtype);
  if (L.total > 0 && (!workspace || workspace_bytes < L.total))
    return fail(CAB_ERR_WORKSPACE, "tree_attn: workspace of %zu bytes needed, %zu given", L.total, workspace_bytes);
  if (L.total > 0 && !aligned16(workspace)) return fail(CAB_ERR_INVALID_ARG, "tree_attn: workspace must be 16-byte aligned");
  if (L.units >= (int64_t)1 << 31) return fail(CAB_ERR_UNSUPPORTED, "tree_attn: too many row tiles");
  const int64_t es = static_cast<int64_t>(dtype_size(cache->dtype));
  Params p{};
  p.q = q;
  p.k = static_cast<const uint8_t*>(cache->k_pages) + layer * cache->k_strides[0] * es;
  p.v = static_cast<const uint8_t*>(cache->v_pages) + layer * cache->v_strides[0] * es;
  p.out = out;
  p.lse = lse;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = q_strides[i];
    p.os[i] = o_strides[i];
    p.ks[i] = cache->k_strides[i + 1];
    p.vs[i] = cache->v_strides[i + 1];
  }
  p.table = cache->block_table;
  p.lens = cache->seq_lens;
  p.rows = rows;
  p.nodes = num_nodes;
  p.parents = parents;
  p.mask = tree_mask;
  p.table_stride = cache->table_stride;
  p.parents_stride = parents_stride;
  p.mask_stride = mask_stride;
  p.pages = cache->pages;
  p.page_size = cache->page_size;
  p.width = cache->width;
  p.num_rows = cache->rows;
  p.n = static_cast<int32_t>(n);
  p.Hq = static_cast<int32_t>(Hq);
  p.Hkv = static_cast<int32_t>(cache->heads);
  p.G = p.Hq / p.Hkv;
  p.T = static_cast<int32_t>(T);
  p.D = static_cast<int32_t>(cache->dim);
  p.scale_log2 = softmax_scale * kLog2e;
  p.splits = L.splits;
  if (L.total > 0) {
    p.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + L.part_o);
    p.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + L.part_ml);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case CAB_DTYPE_F32: return launch_simt_d<float>(p, L.units, st);
    case CAB_DTYPE_F16: return launch_simt_d<__half>(p, L.units, st);
    default: return launch_simt_d<__nv_bfloat16>(p, L.units, st);
  }
}
