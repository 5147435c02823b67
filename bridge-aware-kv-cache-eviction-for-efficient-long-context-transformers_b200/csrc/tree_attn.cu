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
#include <type_traits>

namespace cab {
namespace tree {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int64_t kMaxTokens = 0x7fffffff - 512;  // of a row: positions up to two 128-key tiles past it fit 32 bits
constexpr int kMaxTree = 1024;  // nodes of a tree given by parents: a query walks up its ancestors

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
  int32_t least;      // tensor-core path: tiles a CTA takes at least
  int32_t part_rows;  // rows of a partial slot
  int32_t out_vec;    // out rows start on 16 bytes
  int32_t whole_units;  // no unit is cut: none can be longer than a few tiles
  int32_t in_vec;       // CUDA-core path: K / V rows can be read 4 elements at a time
  float *part_o, *part_ml;
  int64_t* before;  // [n + 1] more than kScan sequences: the weight before each, for the join
};

struct Seq {
  int32_t row, len, m, ctx;  // a sequence that does not fit its row has len = m = 0
};

__device__ __forceinline__ Seq load_seq(const Params& p, int i) {
  Seq s{0, 0, 0, 0};
  if (i >= p.n) return s;
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
// tensor-core path does not take. Up to 8 rows of a KV head take few_rows_kernel (below); more rows, or
// rows that are not 8 columns on 16 bytes, this kernel: one CTA per (sequence, KV head, 4 * RW rows, key
// split). A warp owns RW rows and a lane one key of the 32-key tile for the scores, so a row's maximum and
// sum are warp reductions; for the output a lane owns the columns lane + 32 c. Four threads fetch a key: its
// page is looked up once, then its K and V rows come in 4-element vectors. Bound by shared-memory reads: per
// 4 dims 4 wavefronts of keys and one of each row's query for 4 * RW multiply-adds, so more than 16 rows
// take RW = 8, others RW = 4 to spread them over the warps. 2 trees of 128 nodes, 16 / 4 heads of 128 over
// 2000 tokens, float32: 238 us, 18 TFLOP/s; 4 of 40 nodes, 8 / 2 heads, up to 1000 tokens: 47 us.
constexpr int kKeysTile = 32, kSimtThreads = 128;

template <typename T>
struct Vec4;
template <>
struct Vec4<float> {
  using type = float4;
  static __device__ __forceinline__ float4 widen(float4 v) { return v; }
};
template <>
struct Vec4<__half> {
  using type = uint2;
  static __device__ __forceinline__ float4 widen(uint2 v) {
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&v.x)), b = __half22float2(*reinterpret_cast<__half2*>(&v.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
};
template <>
struct Vec4<__nv_bfloat16> {
  using type = uint2;
  static __device__ __forceinline__ float4 widen(uint2 v) {
    const float2 a = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v.x)),
                 b = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
};

template <typename T, int DC, int RW>
__global__ void __launch_bounds__(kSimtThreads) simt_kernel(const __grid_constant__ Params p) {
  extern __shared__ float sm[];
  constexpr int kRowsTile = 4 * RW;
  using V4 = typename Vec4<T>::type;
  const int Dp = (p.D + 3) & ~3, ld = Dp + 4;
  float* sQ = sm;                    // [rows][Dp]
  float* sK = sQ + kRowsTile * Dp;   // [32][ld]
  float* sV = sK + kKeysTile * ld;   // [32][Dp]
  float* sP = sV + kKeysTile * Dp;   // [rows][32]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int R = p.G * p.T, tiles_r = (R + kRowsTile - 1) / kRowsTile;
  const int unit = blockIdx.x, split = blockIdx.y;
  const int rt = unit % tiles_r, hk = (unit / tiles_r) % p.Hkv, i = unit / (tiles_r * p.Hkv);
  const int row0 = rt * kRowsTile;
  const Seq s = load_seq(p, i);
  const int keys = s.m > 0 && row0 / p.G < s.m ? key_limit(p, s, min(p.T - 1, (row0 + kRowsTile - 1) / p.G)) : 0;
  const int tiles = (keys + kKeysTile - 1) / kKeysTile;
  const int per = (tiles + p.splits - 1) / p.splits;
  const int t_lo = min(tiles, split * per), t_hi = min(tiles, t_lo + per);
  const uint32_t S = static_cast<uint32_t>(p.page_size);
  const int32_t* table = p.table + s.row * p.table_stride;
  // the key this thread fetches a quarter of
  const int fk = threadIdx.x >> 2, part = threadIdx.x & 3;
  auto page_at = [&](int tile) -> int {  // of that key; -1: none
    const int key = tile * kKeysTile + fk;
    if (tile >= t_hi || key >= keys) return -1;
    const int pg = table[static_cast<uint32_t>(key) / S];
    return pg < 0 || pg >= p.pages ? -1 : pg;
  };
  int page = page_at(t_lo);

  {
    float q[RW][DC];  // this warp's rows, all in flight
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      const int row = row0 + warp * RW + r, t = row / p.G;
      const T* src = static_cast<const T*>(p.q) + i * p.qs[0] + (hk * p.G + row - t * p.G) * p.qs[1] + t * p.qs[2];
#pragma unroll
      for (int c = 0; c < DC; ++c) q[r][c] = row < R && lane + 32 * c < p.D ? to_f32(src[lane + 32 * c]) : 0.f;
    }
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
      for (int c = 0; c < DC; ++c)
        if (lane + 32 * c < Dp) sQ[(warp * RW + r) * Dp + lane + 32 * c] = q[r][c];
  }
  float acc[RW][DC], m[RW], l[RW];
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < DC; ++c) acc[r][c] = 0.f;
  }
  for (int tile = t_lo; tile < t_hi; ++tile) {
    const int key0 = tile * kKeysTile;
    const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);  // four lanes a key
    const int next_page = page_at(tile + 1);
    __syncthreads();
    if (lane < 8) reinterpret_cast<uint32_t*>(sP)[warp * 8 + lane] = there >> (4 * lane) & 1u;  // before P is written
    {
      const int64_t slot = static_cast<uint32_t>(key0 + fk) % S;
      const T* k = static_cast<const T*>(p.k) + page * p.ks[0] + hk * p.ks[1] + slot * p.ks[2];
      const T* v = static_cast<const T*>(p.v) + page * p.vs[0] + hk * p.vs[1] + slot * p.vs[2];
      float* dk = sK + fk * ld;
      float* dv = sV + fk * Dp;
      if (p.in_vec) {
        constexpr int kChunks = DC * 2;  // 32 DC columns, 4 threads of 4
        V4 a[kChunks], b[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int d = 16 * c + 4 * part;
          if (page >= 0 && d < p.D) {
            a[c] = *reinterpret_cast<const V4*>(k + d);
            b[c] = *reinterpret_cast<const V4*>(v + d);
          } else {
            a[c] = b[c] = V4{};
          }
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int d = 16 * c + 4 * part;
          if (d < Dp) {
            *reinterpret_cast<float4*>(dk + d) = Vec4<T>::widen(a[c]);
            *reinterpret_cast<float4*>(dv + d) = Vec4<T>::widen(b[c]);
          }
        }
      } else {
        for (int d = part; d < Dp; d += 4) {
          const bool ok = page >= 0 && d < p.D;
          dk[d] = ok ? to_f32(k[d]) : 0.f;
          dv[d] = ok ? to_f32(v[d]) : 0.f;
        }
      }
    }
    page = next_page;
    __syncthreads();
    const bool key_there = reinterpret_cast<const uint32_t*>(sP)[lane] != 0u;
    float sc[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) sc[r] = 0.f;
    const float4* kr = reinterpret_cast<const float4*>(sK + lane * ld);
    const float4* qr = reinterpret_cast<const float4*>(sQ + warp * RW * Dp);
#pragma unroll 4
    for (int d = 0; d < Dp / 4; ++d) {
      const float4 kk = kr[d];
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        const float4 qq = qr[r * (Dp / 4) + d];
        sc[r] = fmaf(qq.x, kk.x, fmaf(qq.y, kk.y, fmaf(qq.z, kk.z, fmaf(qq.w, kk.w, sc[r]))));
      }
    }
    const int key = key0 + lane;
    uint32_t seen[RW], all = 0xffffffffu;
    __syncthreads();  // every warp has read the keys' flags
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      const int t = (row0 + warp * RW + r) / p.G;
      const bool ok = key_there && t < s.m && (key < s.ctx || (key < keys && sees(p, i, t, key - s.ctx)));
      seen[r] = __ballot_sync(0xffffffffu, ok);
      all &= seen[r];
      const float x = ok ? sc[r] * p.scale_log2 : -INFINITY;
      float mx = x;
#pragma unroll
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float mn = fmaxf(m[r], mx);
      const float alpha = m[r] == -INFINITY ? 0.f : ex2(m[r] - mn);
      const float w = x == -INFINITY ? 0.f : ex2(x - mn);  // unseen, or a score of -inf
      l[r] = l[r] * alpha + w;                             // this lane's keys; the lanes are added at the end
      m[r] = mn;
      sP[(warp * RW + r) * 32 + lane] = w;
      if (alpha != 1.f) {
#pragma unroll
        for (int c = 0; c < DC; ++c) acc[r][c] *= alpha;
      }
    }
    __syncwarp();
    const float4* pr = reinterpret_cast<const float4*>(sP + warp * RW * 32);
    if (all == 0xffffffffu) {
#pragma unroll 2
      for (int j = 0; j < kKeysTile; j += 4) {
        float vv[4][DC];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int c = 0; c < DC; ++c) vv[u][c] = lane + 32 * c < Dp ? sV[(j + u) * Dp + lane + 32 * c] : 0.f;
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          const float4 w = pr[r * 8 + j / 4];
#pragma unroll
          for (int c = 0; c < DC; ++c)
            acc[r][c] = fmaf(w.x, vv[0][c], fmaf(w.y, vv[1][c], fmaf(w.z, vv[2][c], fmaf(w.w, vv[3][c], acc[r][c]))));
        }
      }
    } else {  // unseen keys are left out, not multiplied by 0
      for (int j = 0; j < kKeysTile; ++j) {
        float vv[DC];
#pragma unroll
        for (int c = 0; c < DC; ++c) vv[c] = lane + 32 * c < Dp ? sV[j * Dp + lane + 32 * c] : 0.f;
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          if (seen[r] >> j & 1u) {
            const float w = sP[(warp * RW + r) * 32 + j];
#pragma unroll
            for (int c = 0; c < DC; ++c) acc[r][c] = fmaf(w, vv[c], acc[r][c]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    const int row = row0 + warp * RW + r;
#pragma unroll
    for (int o = 16; o; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
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
      const int64_t slot = (static_cast<int64_t>(unit) * kRowsTile + warp * RW + r) * p.splits + split;
#pragma unroll
      for (int c = 0; c < DC; ++c)
        if (lane + 32 * c < p.D) p.part_o[slot * p.D + lane + 32 * c] = acc[r][c];
      if (lane == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(m[r], l[r]);
    }
  }
}

// Up to 8 rows: no tile in shared memory, the products are vector by vector. LK = D / 8 lanes (8, 16 or
// 32) hold 8 columns of the queries and sums each and take a key together: its K and V rows come straight
// from global memory, the score is a sum over the lanes, and each group of lanes keeps a maximum, sums and
// output of its own, joined at the end. A warp takes 32 keys at a time, whose pages its lanes look up
// together. Bound by the loads in flight: two keys' rows a lane. 16 rows of 1 to 2k tokens, 8 heads of
// 128, float32, one token: 59 us (149 us by tiles of 16 rows, of which one is used); 3 rows of 0.9 to 1.5k
// tokens, 8 heads of 64, 5 nodes: 18 us with the join (23 us by tiles), the latency of the loads.
constexpr int kFewRows = 8;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const float4 a = Vec4<T>::widen(make_uint2(v.x, v.y)), b = Vec4<T>::widen(make_uint2(v.z, v.w));
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
}

template <typename T, int LK, int RM>
__global__ void __launch_bounds__(kSimtThreads) few_rows_kernel(const __grid_constant__ Params p) {
  constexpr int kGroups = 32 / LK, kCols = 8 * LK;
  __shared__ float s_acc[4][RM][kCols], s_m[4][RM], s_l[4][RM];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = lane / LK, col = (lane % LK) * 8;
  const int R = p.G * p.T, unit = blockIdx.x, split = blockIdx.y, hk = unit % p.Hkv, i = unit / p.Hkv;
  const Seq s = load_seq(p, i);
  const int keys = s.len;
  const int chunks = (keys + 31) / 32, per = (chunks + p.splits - 1) / p.splits;
  const int c_lo = min(chunks, split * per), c_hi = min(chunks, c_lo + per);
  const uint32_t S = static_cast<uint32_t>(p.page_size);
  const int32_t* table = p.table + s.row * p.table_stride;
  const bool there = col < p.D;
  const T* kbase = static_cast<const T*>(p.k) + hk * p.ks[1] + col;
  const T* vbase = static_cast<const T*>(p.v) + hk * p.vs[1] + col;
  float q[RM][8], acc[RM][8], m[RM], l[RM];
  uint32_t live = 0u;
#pragma unroll
  for (int r = 0; r < RM; ++r) {
    const int t = r / p.G;
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) q[r][e] = acc[r][e] = 0.f;
    if (r < R && t < s.m) {
      live |= 1u << r;
      const T* src = static_cast<const T*>(p.q) + i * p.qs[0] + (hk * p.G + r - t * p.G) * p.qs[1] + t * p.qs[2] + col;
#pragma unroll
      for (int e = 0; e < 8; ++e) q[r][e] = there ? to_f32(src[e]) * p.scale_log2 : 0.f;
    }
  }
  for (int c = c_lo + warp; c < c_hi; c += 4) {
    const int mine = c * 32 + lane;
    int page = -1;
    uint32_t slot = 0u;
    if (mine < keys) {
      const uint32_t j = static_cast<uint32_t>(mine) / S;
      slot = static_cast<uint32_t>(mine) - j * S;
      page = table[j];
      if (page >= p.pages) page = -1;
    }
#pragma unroll 1
    for (int sub = 0; sub < LK; sub += 2) {
      float kk[2][8], vv[2][8];
      uint32_t vis[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int x = (sub + u) * kGroups + grp, key = c * 32 + x;
        const int64_t pg = __shfl_sync(0xffffffffu, page, x), sl = __shfl_sync(0xffffffffu, slot, x);
        vis[u] = pg < 0 ? 0u : live;
        if (pg >= 0 && key >= s.ctx) {
#pragma unroll 1
          for (int r = 0; r < R; ++r)
            if (live >> r & 1u && !sees(p, i, r / p.G, key - s.ctx)) vis[u] &= ~(1u << r);
        }
        if (vis[u] != 0u && there) {
          load8(kbase + pg * p.ks[0] + sl * p.ks[2], kk[u]);
          load8(vbase + pg * p.vs[0] + sl * p.vs[2], vv[u]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) kk[u][e] = vv[u][e] = 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float x[RM];
#pragma unroll
        for (int r = 0; r < RM; ++r) {
          x[r] = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[r] = fmaf(q[r][e], kk[u][e], x[r]);
        }
#pragma unroll
        for (int o = LK / 2; o; o >>= 1)
#pragma unroll
          for (int r = 0; r < RM; ++r) x[r] += __shfl_xor_sync(0xffffffffu, x[r], o);
#pragma unroll
        for (int r = 0; r < RM; ++r) {
          if (!(vis[u] >> r & 1u) || x[r] == -INFINITY) continue;  // unseen, or a weight of 0
          if (x[r] > m[r]) {
            const float alpha = ex2(m[r] - x[r]);  // from -inf: 0
            l[r] *= alpha;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[r][e] *= alpha;
            m[r] = x[r];
          }
          const float w = ex2(x[r] - m[r]);
          l[r] += w;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[r][e] = fmaf(w, vv[u][e], acc[r][e]);
        }
      }
    }
  }
  // the groups of a warp, then the warps
#pragma unroll
  for (int r = 0; r < RM; ++r) {
#pragma unroll
    for (int o = LK; o < 32; o <<= 1) {
      const float mo = __shfl_xor_sync(0xffffffffu, m[r], o), lo = __shfl_xor_sync(0xffffffffu, l[r], o);
      const float mn = fmaxf(m[r], mo), ref = mn == -INFINITY ? 0.f : mn, a = ex2(m[r] - ref), b = ex2(mo - ref);
      l[r] = l[r] * a + lo * b;
      m[r] = mn;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[r][e] = acc[r][e] * a + __shfl_xor_sync(0xffffffffu, acc[r][e], o) * b;
    }
    if (lane < LK) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s_acc[warp][r][col + e] = acc[r][e];
      if (lane == 0) {
        s_m[warp][r] = m[r];
        s_l[warp][r] = l[r];
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < R * kCols; e += kSimtThreads) {
    const int r = e / kCols, d = e - r * kCols;
    const float mm = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    const float ref = mm == -INFINITY ? 0.f : mm;
    float o = 0.f, ll = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float a = ex2(s_m[w][r] - ref);
      o = fmaf(a, s_acc[w][r][d], o);
      ll = fmaf(a, s_l[w][r], ll);
    }
    if (p.splits == 1) {
      const int t = r / p.G, h = hk * p.G + r - t * p.G;
      if (d < p.D)
        static_cast<T*>(p.out)[i * p.os[0] + h * p.os[1] + t * p.os[2] + d] = from_f32<T>(ll != 0.f ? o / ll : 0.f);
      if (p.lse && d == 0) p.lse[(static_cast<int64_t>(i) * p.Hq + h) * p.T + t] = (mm + log2f(ll)) * kLn2;
    } else {
      const int64_t slot = (static_cast<int64_t>(unit) * RM + r) * p.splits + split;
      if (d < p.D) p.part_o[slot * p.D + d] = o;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(mm, ll);
    }
  }
}

// Joins the splits of a row: one warp per row, always in the order of the keys. The splits'
// weights are computed by a lane each, so the sums' loads do not wait for one another.
template <typename T, int DC>
__global__ void __launch_bounds__(kSimtThreads) simt_join_kernel(const __grid_constant__ Params p, int rows_tile) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = p.G * p.T, tiles_r = (R + rows_tile - 1) / rows_tile;
  const int64_t total = static_cast<int64_t>(p.n) * p.Hkv * tiles_r * rows_tile;
  const int64_t x = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  const int64_t unit = x / rows_tile;
  const int rt = static_cast<int>(unit % tiles_r), hk = static_cast<int>(unit / tiles_r % p.Hkv);
  const int64_t i = unit / tiles_r / p.Hkv;
  const int row = rt * rows_tile + static_cast<int>(x - unit * rows_tile);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (x >= total || row >= R) return;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + x * p.splits;
  const float* po = p.part_o + x * p.splits * p.D;
  float m = -INFINITY, l = 0.f, acc[DC];
#pragma unroll
  for (int c = 0; c < DC; ++c) acc[c] = 0.f;
  for (int k0 = 0; k0 < p.splits; k0 += 32) {
    const float2 own = k0 + lane < p.splits ? ml[k0 + lane] : make_float2(-INFINITY, 0.f);
    float mx = own.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = ex2(m - ref), w = own.x == -INFINITY && own.y == 0.f ? 0.f : ex2(own.x - ref);
    float lw = w * own.y;
#pragma unroll
    for (int o = 16; o; o >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, o);
    l = fmaf(l, alpha, lw);
    m = mn;
#pragma unroll
    for (int c = 0; c < DC; ++c) acc[c] *= alpha;
    const int n = min(32, p.splits - k0);
#pragma unroll 8
    for (int k = 0; k < n; ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
#pragma unroll
      for (int c = 0; c < DC; ++c)
        if (lane + 32 * c < p.D) acc[c] = fmaf(wk, po[static_cast<int64_t>(k0 + k) * p.D + lane + 32 * c], acc[c]);
    }
  }
  const int h = hk * p.G + row % p.G, t = row / p.G;
  T* o = static_cast<T*>(p.out) + i * p.os[0] + h * p.os[1] + t * p.os[2];
  const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int c = 0; c < DC; ++c)
    if (lane + 32 * c < p.D) o[lane + 32 * c] = from_f32<T>(acc[c] * inv);
  if (p.lse && lane == 0) p.lse[(i * p.Hq + h) * p.T + t] = (m + log2f(l)) * kLn2;
}

// ------------------------------------------------------------------ tensor-core path
// bf16 / f16, head_dim 64 or 128. The G * T rows of a (sequence, KV head) are cut into groups
// of whole nodes, at most 128 rows, the M of tcgen05.mma. Up to kMaxShare groups are worked on side by side by as many CTAs, so
// that a K / V tile comes from HBM once and for the others from L2. A unit is (sequence, KV head, such a
// set of groups); the units' 128-key tiles form one flat list that is cut into equal ranges, one
// per set of CTAs (persistent, one CTA per SM), so ragged lengths balance and one long sequence
// fills the GPU; a unit cut between ranges leaves partial sums that join_kernel adds in key order.
//
// Tile g of a CTA: S = Q K^T (128 x 128, K-major operands from shared memory) into one of three
// TMEM buffers; p = 2^(s - m) by one thread per row, written over S as 16-bit, the products' operand
// type: the tensor pipe takes no float32, and a second product for the bits cut off would double its work and the
// weights' TMEM traffic. A weight is off by half a step at most (bf16 2^-8, fp16 2^-11, relative), the
// output by less, since the errors of many keys are independent: against 64 bits 0.0023 relative for bf16, 0.0017
// without this rounding. The weights' sum is taken before it, in float32. O += P V (P from TMEM, V MN-major as it lies in
// the pages). S(g + 3) reuses the buffer once PV(g) has completed. Two sets of four warps take turns,
// one tile each: a set takes its tile's maxima, gets the rows' reference m from the other set's tile
// before, passes m on and then computes the weights, so that on each SM quarter one warp's exponentials
// (the special function unit's 1024 clocks a tile, as many as the products take) run under the other's
// loads and maxima. (Both sets on one tile, half the keys each, wait for one another: 2050 clocks a tile.)
// m, and with it O, changes only when a maximum exceeds it by more than 2^8.
//
// Warps 0 and 3 look up the pages and load K and V by TMA (one box per page and 64 columns, a lane
// each; a page number outside the pool reads zeros), so loads are issued from two warps (one warp
// gives 5.3 TB/s with 16-token pages, two 5.9, copy peak 6.55). Tiles that reach into the nodes or past the
// length are masked per row, a bit a key, and V rows past the length and values of nodes that
// are not finite are zeroed in shared memory, so that 0 * NaN cannot enter a product; a seen value
// that is not finite is added back to the rows that see it (fix_up).
//
// Measured (B200): 32 rows of 0.8 to 8k tokens, 32 / 8 heads of 128, one token, 16-token pages: 606 MB
// from HBM (each key and value once) in 111 us, 5.5 TB/s = 0.83 of the copy rate; the rest is the first tiles'
// latency (table, page and tile one after the other, 7 us), and the join. 4 trees of 64 nodes over 65,536
// tokens (275 GFLOP, 256 rows a KV head): 265 us = 1.04 PFLOP/s alone, 0.33 ms in a loop, where the 1 kW cap
// lowers the clock to 1.3 - 1.6 GHz; 1.08 GB from HBM, so the CTAs side by side share each tile through L2.
// Before that: one tile a time on two streams with an O each 407 us; 64 keys a thread 361 us.
//
// A parity wait must not meet a barrier two phases away from its own. Each loader and issuer waits for every phase
// of its barriers in turn. A softmax set skips the other set's tiles; what ties it to them is the hand-over of m,
// and between segments the meeting over O (rows that are nodes) or over the cleaned V (every live group's last
// tile holds its own nodes, so only a range's last segment has no such meeting). A group without a node would
// have neither, so it takes no tiles at all: its rows' zeros are written straight away.

constexpr int kTcThreads = 384;  // warps 0 / 3: K / V loads, 1: S, 2: PV, 4-11: softmax and epilogue
constexpr float kRescaleThreshold = 8.0f;
constexpr int kBufs = 3;
constexpr uint32_t kTmemO = 384;
constexpr int kMaxShare = 4;
constexpr int kLostRing = 16;  // tiles between the K loads and the softmax, at most kStages + 3
constexpr int kUnitCost = 4;
constexpr int kScan = 128;  // sequences up to which the join adds up the weights itself, before it waits
// Table rows of at most this many tiles are not cut: no join (one token over 299: 19 -> 15 us). The host knows the
// table's width alone, not the lengths, so short rows of a wide table take the general path.
constexpr int kWholeTiles = 4;

template <int D>
struct Cfg {
  static constexpr int kTile = 128 * D * 2;  // bytes of a K, V or Q tile
  static constexpr int kAtoms = D / 64;
  static constexpr int kStages = D == 128 ? 3 : 6;  // of K, and of V
  // with as many stages as S / P buffers S(g) completed frees K stage g % 3, PV(g) V stage g % 3
  static constexpr bool kOneSignal = kStages == kBufs;
  static constexpr int kXchg = 2 * 2 * 128 * 4;  // references m [tile parity][row], sums [set][row]
  static constexpr int kBars = (4 * kStages + 3 * kBufs + 6) * 8 + 32 + kLostRing;
  static constexpr int kBytes = (1 + 2 * kStages) * kTile + kXchg + kBars;
  static constexpr int kSmem = kBytes + 1024 < 232448 ? kBytes + 1024 : 232448;  // the kernel checks that it fits
  static_assert(kBytes <= 232448, "shared memory");
};

// How the nodes are shared out: groups of `nodes` whole nodes (their G rows each, at most 128 rows), `wide`
// groups side by side, `sets` of them per KV head.
struct Share {
  int nodes, groups, wide, sets;
};
__host__ __device__ __forceinline__ Share share_of(int G, int T) {
  Share s;
  s.nodes = 128 / G;
  s.groups = (T + s.nodes - 1) / s.nodes;
  s.sets = (s.groups + kMaxShare - 1) / kMaxShare;
  s.wide = (s.groups + s.sets - 1) / s.sets;
  return s;
}

struct Walk {  // a range of the flat list, unit by unit
  int b, hk, set, tiles, at;  // place `at` of the unit's weight; it has `tiles` tiles
  int left;                   // tiles (units, where units stay whole) of the range not yet walked
  Seq s;
};

// Keys that groups [g0, g1] of sequence s can see, 0 where none of their rows is a node.
__device__ __forceinline__ int group_keys(const Params& p, const Share& sh, const Seq& s, int g0, int g1) {
  return g0 * sh.nodes < s.m ? key_limit(p, s, min(p.T, (g1 + 1) * sh.nodes) - 1) : 0;
}
__device__ __forceinline__ int tiles_of(int keys) { return max(1, (keys + 127) / 128); }  // at least one, for the zeros
__device__ __forceinline__ int unit_tiles(const Params& p, const Share& sh, const Seq& s, int set) {
  return tiles_of(group_keys(p, sh, s, set * sh.wide, min(sh.groups, (set + 1) * sh.wide) - 1));
}
// What a unit counts in the flat list, and the units of one KV head of a sequence. Starting and
// ending a unit costs about as much as kUnitCost tiles, which stand before its tiles in the list.
__device__ __forceinline__ int unit_weight(const Params& p, const Share& sh, const Seq& s, int set) {
  return p.whole_units ? 1 : kUnitCost + unit_tiles(p, sh, s, set);
}
__device__ __forceinline__ int head_weight(const Params& p, const Share& sh, const Seq& s) {
  if (p.whole_units) return sh.sets;
  int sum = 0;
  for (int g = 0; g < sh.sets; ++g) sum += unit_weight(p, sh, s, g);
  return sum;
}

__device__ __forceinline__ void walk_next(const Params& p, const Share& sh, Walk& w) {  // to the next unit's first tile
  w.left -= p.whole_units ? 1 : min(w.left, kUnitCost + w.tiles - w.at);
  w.at = 0;
  if (w.left == 0) return;
  if (++w.set == sh.sets) {
    w.set = 0;
    if (++w.hk == p.Hkv) {
      w.hk = 0;
      w.s = load_seq(p, ++w.b);
    }
  }
  w.tiles = unit_tiles(p, sh, w.s, w.set);
}
// The walk's segment: group grp's tiles [first, first + count) (the unit's longest group has them all). A group
// without a node has no tiles to compute, and `zeros` where its one place in the list is in the range.
struct Segment {
  int first, count;
  bool zeros;
};
__device__ __forceinline__ Segment segment_of(const Params& p, const Share& sh, const Walk& w, int grp) {
  if (grp >= sh.groups) return Segment{0, 0, false};
  const int keys = group_keys(p, sh, w.s, grp, grp), own = min(w.tiles, tiles_of(keys));
  const int first = p.whole_units ? 0 : max(0, w.at - kUnitCost);
  const int end = p.whole_units ? own : min(own, w.at + w.left - kUnitCost), count = max(0, end - first);
  return keys > 0 ? Segment{first, count, false} : Segment{0, 0, count > 0};
}

// Where range c starts. (A 64-bit division takes several hundred clocks, a 32-bit one about a hundred.)
__device__ __forceinline__ int64_t range_start(int64_t total, int64_t ranges, int64_t c) {
  const uint64_t x = static_cast<uint64_t>(total) * static_cast<uint64_t>(c);
  return x >> 32 == 0 ? static_cast<uint32_t>(x) / static_cast<uint32_t>(ranges) : x / static_cast<uint64_t>(ranges);
}
__device__ __forceinline__ int range_count(int64_t total, int most, int least) {
  if (total >= static_cast<int64_t>(most) * least) return most;
  return (static_cast<int>(total) + least - 1) / least;
}

// Warp-wide: the weight of all units.
__device__ __forceinline__ int64_t total_weight(const Params& p, const Share& sh) {
  const int lane = threadIdx.x & 31;
  int64_t sum = 0;
  for (int b = lane; b < p.n; b += 32) sum += static_cast<int64_t>(head_weight(p, sh, load_seq(p, b))) * p.Hkv;
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
struct Begin {
  int b, offset, left;
};
__device__ __forceinline__ Begin find_range(const Params& p, const Share& sh, int range, int most) {
  const int lane = threadIdx.x & 31;
  int64_t own = 0;  // up to 32 sequences: one reading for the total and the place
  if (p.n <= 32 && lane < p.n) own = static_cast<int64_t>(head_weight(p, sh, load_seq(p, lane))) * p.Hkv;
  int64_t total = own;
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (p.n > 32) total = total_weight(p, sh);
  const int ranges = range_count(total, most, p.least);
  if (range >= ranges) return Begin{0, 0, 0};
  const int64_t f0 = range_start(total, ranges, range), f1 = range_start(total, ranges, range + 1);
  int64_t base = 0;
  for (int b0 = 0; b0 < p.n; b0 += 32) {
    const int b = b0 + lane;
    if (p.n > 32) own = b < p.n ? static_cast<int64_t>(head_weight(p, sh, load_seq(p, b))) * p.Hkv : 0;  // L1
    int64_t inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, base + inc > f0);
    if (hit) {
      const int l = __ffs(hit) - 1;
      return Begin{b0 + l, static_cast<int>(f0 - base - __shfl_sync(0xffffffffu, inc - own, l)), static_cast<int>(f1 - f0)};
    }
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
  return Begin{0, 0, 0};
}

__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

struct Bits {
  uint64_t lo, hi;
};

// Which of the keys key0 .. key0 + 127 node t of sequence b sees.
__device__ __forceinline__ Bits seen_bits(const Params& p, const Seq& s, int b, int t, int key0, bool bad_pages) {
  const int c = s.ctx - key0;
  Bits w{low_bits(c), low_bits(c - 64)};
  if (p.parents) {
    const int32_t* up = p.parents + b * p.parents_stride;
    for (int x = t; x >= 0;) {
      const int y = up[x], at = c + x;
      if (at < 0) break;
      if (at < 64) w.lo |= 1ull << at;
      else if (at < 128) w.hi |= 1ull << (at - 64);
      if (y >= x) break;
      x = y;
    }
  } else if (p.mask) {
    const uint8_t* row = p.mask + b * p.mask_stride + static_cast<int64_t>(t) * p.T - c;
    const int end = min(128, c + s.m);
#pragma unroll 1
    for (int at0 = max(c, 0); at0 < end; at0 += 16) {
      uint32_t v[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) v[u] = at0 + u < end ? row[at0 + u] : 0u;
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const uint64_t bit = v[u] != 0u ? 1ull << ((at0 + u) & 63) : 0ull;
        if (at0 + u < 64) w.lo |= bit;
        else w.hi |= bit;
      }
    }
  } else {
    w.lo = low_bits(c + t + 1);
    w.hi = low_bits(c + t + 1 - 64);
  }
  if (bad_pages) {
    for (int j = 0; j < 128 && key0 + j < s.len; ++j) {
      const int pg = p.table[s.row * p.table_stride + (key0 + j) / p.page_size];
      if (pg < 0 || pg >= p.pages) {
        if (j < 64) w.lo &= ~(1ull << j);
        else w.hi &= ~(1ull << (j - 64));
      }
    }
  }
  return w;
}

// Adds to 32 columns of a row's sum the values that are not finite of the nodes it sees among
// keys [lo, hi): they were taken out of the product.
template <typename T>
__device__ __forceinline__ void fix_up(const Params& p, const Seq& s, int b, int hk, int t, int lo, int hi, int col, float* o) {
  for (int key = max(lo, s.ctx); key < min(hi, s.len); ++key) {
    if (!sees(p, b, t, key - s.ctx)) continue;
    const int64_t pg = p.table[s.row * p.table_stride + key / p.page_size], slot = key % p.page_size;
    if (pg < 0 || pg >= p.pages) continue;
    const T* v = static_cast<const T*>(p.v) + pg * p.vs[0] + hk * p.vs[1] + slot * p.vs[2] + col;
    for (int d = 0; d < 32; ++d) {
      const float x = to_f32(v[d]);
      if (!isfinite(x)) o[d] += x;
    }
  }
}

// Row r of a V tile: past the length it becomes 0; of a node, elements that are not finite do. Returns
// whether there were any.
template <int D, bool kBF16>
__device__ __forceinline__ bool clean_v_row(uint8_t* tile, int r, int key, const Seq& s) {
  constexpr uint32_t kExp = kBF16 ? 0x7F807F80u : 0x7C007C00u, kOne = kBF16 ? 0x00800080u : 0x04000400u;
  auto chunk = [&](int x) { return reinterpret_cast<uint4*>(tile + (x >> 3) * 16384 + sw128_offset(r, x & 7)); };
  if (key >= s.len) {
#pragma unroll
    for (int c = 0; c < D / 8; ++c) *chunk(c) = make_uint4(0, 0, 0, 0);
    return false;
  }
  uint32_t hit = 0u;  // an exponent of ones carries into the bit above it
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    const uint4 v = *chunk(c);
    hit |= ((v.x & kExp) + kOne) | ((v.y & kExp) + kOne) | ((v.z & kExp) + kOne) | ((v.w & kExp) + kOne);
  }
  if ((hit & 0x80008000u) == 0u) return false;
  for (int c = 0; c < D / 8; ++c) {
    uint4 v = *chunk(c);
    uint32_t* e = reinterpret_cast<uint32_t*>(&v);
    for (int k = 0; k < 4; ++k) {
      const uint32_t h = ((e[k] & kExp) + kOne) & 0x80008000u;
      if (h & 0x8000u) e[k] &= 0xFFFF0000u;
      if (h & 0x80000000u) e[k] &= 0x0000FFFFu;
    }
    *chunk(c) = v;
  }
  return true;
}

template <bool kBF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (kBF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

__device__ __forceinline__ void softmax_sync() {  // the 256 threads of the softmax warps
  asm volatile("barrier.cta.sync 5, 256;" ::: "memory");
}
// The two warps of a row quarter: a meeting of both, and a handing on from the warp of one tile to that
// of the next (barriers by the parity of the tile).
__device__ __forceinline__ void pair_sync(int quad) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(1 + quad) : "memory"); }
__device__ __forceinline__ void hand_on(int quad, int parity) {
  asm volatile("barrier.cta.arrive %0, 64;" ::"r"(6 + 2 * quad + parity) : "memory");
}
__device__ __forceinline__ void take_over(int quad, int parity) {
  asm volatile("barrier.cta.sync %0, 64;" ::"r"(6 + 2 * quad + parity) : "memory");
}

__device__ __forceinline__ float2 ffma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The 64 weights of a row's half tile from its scores: writes P and returns their sum. An unseen key's
// score is -inf, its weight 0.
template <bool kBF16>
__device__ __forceinline__ float weights(const uint32_t (&s)[64], float scale, float sub, uint32_t t_p) {
  const float2 sc = make_float2(scale, scale), nm = make_float2(-sub, -sub);
  float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t y[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int c = 32 * h + 2 * k;
      const float2 x = ffma2(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sc, nm);
      const float p0 = ex2(x.x), p1 = ex2(x.y);
      acc[k & 1] = fadd2(acc[k & 1], make_float2(p0, p1));
      y[k] = pack2<kBF16>(p0, p1);
    }
    tmem_st16(t_p + 16 * h, y);
  }
  return (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
}

template <int D, bool kBF16>
__global__ void __launch_bounds__(kTcThreads, 1)
    tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
              const __grid_constant__ CUtensorMap qmap, const __grid_constant__ Params p) {
  using C = Cfg<D>;
  using InT = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = base;
  uint8_t* sK = sQ + C::kTile;
  uint8_t* sV = sK + kStages * C::kTile;
  float* xchg = reinterpret_cast<float*>(sV + kStages * C::kTile);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(xchg + C::kXchg / 4);
  uint64_t* v_full = k_full + kStages;
  uint64_t* k_empty = v_full + kStages;    // unused with kOneSignal
  uint64_t* v_empty = k_empty + kStages;   // unused with kOneSignal
  uint64_t* s_full = v_empty + kStages;    // [3] S(g) is there
  uint64_t* p_full = s_full + kBufs;       // [3] P(g) is there (4 warps)
  uint64_t* buf_free = p_full + kBufs;     // [3] PV(g) has completed
  uint64_t* q_full = buf_free + kBufs;     // [2] Q of the segment is there
  uint64_t* q_free = q_full + 2;           // [2] the segment's products with Q have completed
  uint64_t* drain = q_free + 2;            // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  int* odd = abort_flag + 1;       // [2] the last odd / even tail segment (from 1) with values of nodes that are not finite
  int* begin = odd + 2;            // the range: first sequence, weight before it in there, own weight
  uint8_t* lost = reinterpret_cast<uint8_t*>(begin + 3);  // [kLostRing] tile has a page outside the pool
  {
    uint32_t dyn;
    asm volatile("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dyn));
    if (base + C::kBytes > smem_raw + dyn) {
      if (threadIdx.x == 0) atomicOr(&g_device_status, CAB_DEVICE_LAYOUT);
      return;  // shared memory does not start where expected: nothing was touched
    }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Share sh = share_of(p.G, p.T);
  const int range = blockIdx.x / sh.wide, side = blockIdx.x % sh.wide;

  if (warp == 0) {
    // The barriers lie in one row: K / V stages, s_full (2: the product, and the issuer itself, which passes
    // on what the K loader wrote), p_full (4 warps), buf_free, q_full, q_free, drain; a lane each.
    constexpr int kAll = 4 * kStages + 3 * kBufs + 6;
    for (int i = lane; i < kAll; i += 32) {
      const int j = i - 4 * kStages;
      mbar_init(&k_full[i], j < 0 ? 1 : j < kBufs ? 2 : j < 2 * kBufs ? 4 : 1);
    }
    if (lane == 0) {
      *abort_flag = 0;
      odd[0] = odd[1] = 0;
    }
    fence_barrier_init();
  }
  if (threadIdx.x == 32) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
    prefetch_tensormap(&qmap);
  }
  if (warp == 2) tmem_alloc(tmem_slot, 512);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the inputs of this call may be the kernel before's results
  // Only now, with the kernel before complete, may the join start: it reads the lengths before its own wait.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == 0) {
    __syncwarp();
    const Begin x = find_range(p, sh, range, gridDim.x / sh.wide);
    if (lane == 0) {
      begin[0] = x.b;
      begin[1] = x.offset;
      begin[2] = x.left;
    }
    __syncwarp();
  }
  tc_fence_before_sync();
  if (warp == 0) asm volatile("barrier.cta.arrive 14, %0;" ::"n"(kTcThreads) : "memory");  // K needs nobody else
  else asm volatile("barrier.cta.sync 14, %0;" ::"n"(kTcThreads) : "memory");
  tc_fence_after_sync();
  const uint32_t tmem = warp == 0 ? 0u : *tmem_slot;

  // Up to 64 rows leave room for two Q buffers in the tile; the products read 128 rows from there all the
  // same, and what lies behind a buffer's rows only reaches rows of S that nobody uses.
  const uint32_t q_bufs = min(sh.nodes, p.T) * p.G <= 64 ? 2 : 1;
  constexpr uint32_t kHalfQ = 64 * 128;

  Walk w;
  w.b = begin[0];
  w.left = begin[2];
  w.hk = w.set = w.at = 0;
  w.tiles = 1;
  if (w.left > 0) {
    w.s = load_seq(p, w.b);
    const int per_head = head_weight(p, sh, w.s);
    int rem = begin[1];
    w.hk = rem / per_head;
    rem -= w.hk * per_head;
    while (rem >= unit_weight(p, sh, w.s, w.set)) rem -= unit_weight(p, sh, w.s, w.set++);
    w.tiles = unit_tiles(p, sh, w.s, w.set);
    w.at = rem;
  }

  if (warp == 0 || warp == 3) {
    // ---------------------------------------------------------------- loads: warp 0 K, warp 3 V
    const bool is_k = warp == 0;
    const CUtensorMap* map = is_k ? &kmap : &vmap;
    uint8_t* ring = is_k ? sK : sV;
    uint64_t* full = is_k ? k_full : v_full;
    uint64_t* empty = C::kOneSignal ? (is_k ? s_full : buf_free) : (is_k ? k_empty : v_empty);
    const int S = static_cast<int>(p.page_size);
    const int per_tile = S < 128 ? 128 / S : 1;
    const int pi = lane / C::kAtoms, a = lane % C::kAtoms;
    const bool mine = pi < per_tile;
    const uint32_t off = a * 16384 + pi * (S < 128 ? S * 128 : 0);
    uint32_t g = 0, nq = 0;
    bool ok = true;
    for (; w.left > 0 && ok; walk_next(p, sh, w)) {
      const Segment sg = segment_of(p, sh, w, w.set * sh.wide + side);
      const int T = sg.count;
      if (T == 0) continue;
      const int held = (w.s.len + S - 1) / S;
      const int32_t* row = p.table + w.s.row * p.table_stride;
      // the page of this lane's box in tile i of the segment (the number past the pool: zeros)
      auto page_of = [&](int i) -> int {
        const int j = (sg.first + i) * 128 / S + (S < 128 ? pi : 0);
        if (!mine || i >= T || j >= held) return static_cast<int>(p.pages);
        const int q = row[j];
        return q < 0 || q >= p.pages ? -1 : q;  // -1: a page outside the pool
      };
      int e0 = page_of(0), e1 = page_of(1);  // read two tiles ahead
      // Q into its buffer once the buffer's last reader has completed: with two buffers the segment before
      // the previous one, so Q is there ahead of its segment.
      auto load_q = [&]() -> bool {
        const uint32_t qb = nq & (q_bufs - 1), use = nq >> (q_bufs - 1);
        ++nq;
        const bool got = __all_sync(0xffffffffu, mbar_wait(&q_free[qb], (use & 1) ^ 1, abort_flag));
        if (got && lane == 0) {
          const int nodes = min(sh.nodes, p.T);
          mbar_arrive_expect_tx(&q_full[qb], nodes * p.G * D * 2);
#pragma unroll
          for (int k = 0; k < C::kAtoms; ++k)
            tma_load_5d(sQ + qb * kHalfQ + k * 16384, &qmap, &q_full[qb], 64 * k, 0, (w.set * sh.wide + side) * sh.nodes, w.hk, w.b);
        }
        __syncwarp();
        return got;
      };
      if (is_k) ok = load_q();
      if (!ok) break;
      for (int i = 0; i < T; ++i, ++g) {
        const int e2 = page_of(i + 2);
        const uint32_t st = g % kStages;
        // tile g - kStages, the stage's last reader, has completed
        ok = mbar_wait(&empty[st], ((g / kStages) & 1) ^ 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const bool bad = __any_sync(0xffffffffu, e0 < 0);
        if (lane == 0) {
          if (is_k) *reinterpret_cast<volatile uint8_t*>(&lost[g % kLostRing]) = bad;
          mbar_arrive_expect_tx(&full[st], C::kTile);
        }
        __syncwarp();
        if (mine)
          tma_load_4d(ring + st * C::kTile + off, map, &full[st], 64 * a, S < 128 ? 0 : (sg.first + i) * 128 % S, w.hk,
                      e0 < 0 ? static_cast<int>(p.pages) : e0);
        __syncwarp();
        e0 = e1;
        e1 = e2;
      }
    }
    if (!ok) {  // copies still in flight land before the CTA ends
      for (uint32_t k = 1; k <= kStages && k <= g; ++k) (void)mbar_wait(&full[(g - k) % kStages], ((g - k) / kStages) & 1, nullptr);
      for (uint32_t k = 1; k <= q_bufs && k <= nq; ++k) (void)mbar_wait(&q_full[(nq - k) % q_bufs], (nq - k) / q_bufs & 1, nullptr);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- S = Q K^T
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_f16(128, 128, kBF16 ? 1 : 0, 0, 0);
      const uint64_t dQ = make_smem_desc(smem_u32(sQ), 16, 1024, 2);
      const uint64_t dK = make_smem_desc(smem_u32(sK), 16, 1024, 2);
      uint32_t g = 0, seg = 0;
      bool ok = true;
      for (; w.left > 0 && ok; walk_next(p, sh, w)) {
        const int T = segment_of(p, sh, w, w.set * sh.wide + side).count;
        if (T == 0) continue;
        const uint32_t qb = seg & (q_bufs - 1);
        if (!mbar_wait(&q_full[qb], seg >> (q_bufs - 1) & 1, abort_flag)) break;
        ++seg;
        const uint64_t dq = dQ + static_cast<uint64_t>(qb * (kHalfQ >> 4));
        for (int i = 0; i < T; ++i, ++g) {
          const uint32_t st = g % kStages, buf = g % kBufs;
          if (!mbar_wait(&k_full[st], (g / kStages) & 1, abort_flag) ||
              !mbar_wait(&buf_free[buf], ((g / kBufs) & 1) ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint64_t dk = dK + static_cast<uint64_t>((st * C::kTile) >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t o = (kk >> 2) * (16384 >> 4) + (kk & 3) * (32 >> 4);
            mma_f16_ss(tmem + buf * 128, dq + o, dk + o, idesc, kk > 0 ? 1u : 0u);
          }
          if constexpr (!C::kOneSignal) mma_commit(&k_empty[st]);
          mma_commit(&s_full[buf]);
          mbar_arrive(&s_full[buf]);
        }
        mma_commit(&q_free[qb]);
      }
      mma_commit(&drain[0]);
      (void)mbar_wait(&drain[0], 0, nullptr);
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---------------------------------------------------------------- O += P V
    if (p.n > kScan && blockIdx.x == 0 && !p.whole_units) {  // while the first tiles are on their way
      int64_t base = 0;
      for (int b0 = 0; b0 < p.n; b0 += 32) {
        const int b = b0 + lane;
        int64_t inc = b < p.n ? static_cast<int64_t>(head_weight(p, sh, load_seq(p, b))) * p.Hkv : 0;
        const int64_t own = inc;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += u;
        }
        if (b < p.n) p.before[b] = base + inc - own;
        base += __shfl_sync(0xffffffffu, inc, 31);
      }
      if (lane == 0) p.before[p.n] = base;
      __syncwarp();
    }
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_f16(128, D, kBF16 ? 1 : 0, 0, 1);
      const uint64_t dV = make_smem_desc(smem_u32(sV), 16384, 1024, 2);
      uint32_t g = 0;
      bool ok = true;
      for (; w.left > 0 && ok; walk_next(p, sh, w)) {
        const int T = segment_of(p, sh, w, w.set * sh.wide + side).count;
        for (int i = 0; i < T; ++i, ++g) {
          const uint32_t st = g % kStages, buf = g % kBufs;
          // V normally lands early; P(g) is the event waited on last. The previous segment's O has been
          // read before the first P is released.
          if (!mbar_wait(&v_full[st], (g / kStages) & 1, abort_flag) ||
              !mbar_wait(&p_full[buf], (g / kBufs) & 1, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint64_t dv = dV + static_cast<uint64_t>((st * C::kTile) >> 4);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            mma_f16_ts(tmem + kTmemO, tmem + buf * 128 + kk * 8,
                       dv + static_cast<uint64_t>(kk * (2048 >> 4)), idesc, (i > 0 || kk > 0) ? 1u : 0u);
          if constexpr (!C::kOneSignal) mma_commit(&v_empty[st]);
          mma_commit(&buf_free[buf]);
        }
      }
      mma_commit(&drain[1]);
      (void)mbar_wait(&drain[1], 0, nullptr);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax and epilogue
    // Warp w owns TMEM lanes 32 * (w & 3) .. + 31 (rows); set kb = (w - 4) / 4 takes every other tile.
    // A wait that gave up does not end the loops: the barriers stay matched, and every later wait
    // returns at once.
    const int quad = warp & 3, kb = (warp - 4) >> 2, r = quad * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_o = tmem + lanes + kTmemO;
    float *ref = xchg, *sums = xchg + 256;
    uint32_t g0 = 0;  // tiles of earlier segments
    // Segments that reach into their nodes. A warp that sets odd[] for tail segment x + 2 has met the others in
    // x + 1, so all of them have read it for x: two words, by the segment's parity.
    int tails = 0;
    for (; w.left > 0; walk_next(p, sh, w)) {
      const int grp = w.set * sh.wide + side;
      const Segment sg = segment_of(p, sh, w, grp);
      const int T = sg.count;
      const int t = grp * sh.nodes + r / p.G, rows = min(sh.nodes, p.T - grp * sh.nodes) * p.G;
      if (sg.zeros && r < rows) {  // no row of the group is a node; the row's two threads take half the columns each
        const int h = w.hk * p.G + r % p.G;
        InT* orow = static_cast<InT*>(p.out) + w.b * p.os[0] + h * p.os[1] + t * p.os[2] + kb * (D / 2);
        if (p.out_vec) {
#pragma unroll
          for (int c = 0; c < D / 2; c += 8) *reinterpret_cast<uint4*>(orow + c) = make_uint4(0u, 0u, 0u, 0u);
        } else {
          for (int c = 0; c < D / 2; ++c) orow[c] = from_f32<InT>(0.f);
        }
        if (p.lse && kb == 0) p.lse[(static_cast<int64_t>(w.b) * p.Hq + h) * p.T + t] = -INFINITY;
      }
      if (T == 0) continue;
      const Seq q = w.s;
      const bool live = r < rows && t < q.m;
      const bool any_live = __any_sync(0xffffffffu, live);
      const int key_lo = sg.first * 128, keys = group_keys(p, sh, q, grp, grp);
      const bool has_tail = key_lo + T * 128 > q.ctx;
      tails += has_tail;
      float m_run = -INFINITY, l = 0.f;  // this set's sum, relative to its last m
      for (int i = kb; i < T; i += 2) {
        const uint32_t g = g0 + i, buf = g % kBufs;
        const uint32_t t_s = tmem + lanes + buf * 128;  // S in, P out
        const int key0 = key_lo + i * 128;
        // S(g - 3) has completed: this set, or the other before they last met, waited for it or for a later tile
        (void)mbar_wait(&s_full[buf], (g / kBufs) & 1, abort_flag);
        tc_fence_after_sync();
        const bool bad = *reinterpret_cast<volatile uint8_t*>(&lost[g % kLostRing]) != 0;
        const bool masked = bad || key0 + 128 > q.ctx;  // some keys are nodes, past the length or on a lost page
        Bits see{~0ull, ~0ull};
        if (masked) {
          see = Bits{0ull, 0ull};
          // S(g) came after PV(g - 3), so V(g)'s barrier is at most this phase behind; P(g) is not
          // released before V(g) is clean, and PV(g) frees V(g)
          const uint32_t st = g % kStages;
          (void)mbar_wait(&v_full[st], (g / kStages) & 1, abort_flag);
          if (key0 + r >= q.ctx) {
            if (clean_v_row<D, kBF16>(sV + st * C::kTile, r, key0 + r, q)) *reinterpret_cast<volatile int*>(&odd[tails & 1]) = tails;
            fence_proxy_async_smem();
          }
          if (live) see = seen_bits(p, q, w.b, t, key0, bad);
        }
        __syncwarp();  // waits and masks end lane by lane; the TMEM loads want the whole warp
        if (any_live) {
          uint32_t s[64];
          auto load_half = [&](int h) {
            tmem_ld32(t_s + 64 * h, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
            tmem_ld32(t_s + 64 * h + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
            tmem_wait_ld();
            const uint64_t word = h ? see.hi : see.lo;
            if (__any_sync(0xffffffffu, word != ~0ull)) {  // else all of the warp's rows see the whole half
              const uint32_t lo = static_cast<uint32_t>(word), hi = static_cast<uint32_t>(word >> 32);
#pragma unroll
              for (int c = 0; c < 64; ++c)
                if (!((c < 32 ? lo : hi) >> (c & 31) & 1u)) s[c] = 0xff800000u;  // -inf
            }
          };
          float m8[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) m8[u] = -INFINITY;
#pragma unroll
          for (int h = 1; h >= 0; --h) {  // the first half last: its scores are in registers for the weights
            load_half(h);
#pragma unroll
            for (int c = 0; c < 64; c += 2)
              m8[(c >> 1) & 7] = fmax3(m8[(c >> 1) & 7], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
          }
          const float m_tile = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])), fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7]))) *
                               p.scale_log2;
          float m_prev = -INFINITY;
          if (i > 0) {
            take_over(quad, (i - 1) & 1);
            m_prev = ref[((i - 1) & 1) * 128 + r];
          }
          const float m_new = m_prev == -INFINITY || m_tile > m_prev + kRescaleThreshold ? m_tile : m_prev;
          if (i + 1 < T) {
            ref[(i & 1) * 128 + r] = m_new;
            hand_on(quad, i & 1);
          }
          if (m_run != m_new) l *= ex2(m_run - m_new);  // from -inf: l is 0
          m_run = m_new;
          const float sub = m_new == -INFINITY ? 0.f : m_new;  // nothing above -inf so far: weights 0
          __syncwarp();
          l += weights<kBF16>(s, p.scale_log2, sub, t_s);
          load_half(1);
          l += weights<kBF16>(s, p.scale_log2, sub, t_s + 32);
          const bool grown = live && m_prev != -INFINITY && m_new != m_prev;  // rows past the last hold anything
          if (__any_sync(0xffffffffu, grown)) {
            // PV(g - 1) has completed: its barrier's phase before, PV(g - 4), was needed by S(g - 1)
            (void)mbar_wait(&buf_free[(g - 1) % kBufs], ((g - 1) / kBufs) & 1, abort_flag);
            __syncwarp();
            tc_fence_after_sync();
            const float alpha = grown ? ex2(m_prev - m_new) : 1.f;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t x[32];
              tmem_ld32(t_o + c, x);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * alpha);
              tmem_st32(t_o + c, x);
            }
          }
          tmem_wait_st();
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf]);
      }
      g0 += T;

      // epilogue: the row's two threads take half the columns each
      if (any_live) {
        const int last = (T - 1) & 1;
        if (kb == last) ref[last * 128 + r] = m_run;
        pair_sync(quad);
        const float m_end = ref[last * 128 + r];
        if (m_run != m_end) l *= ex2(m_run - m_end);
        m_run = m_end;
        sums[kb * 128 + r] = l;
        pair_sync(quad);
        l += sums[(kb ^ 1) * 128 + r];
        // the last tile's S was seen by one of the pair, so its PV's barrier is at most this phase behind
        (void)mbar_wait(&buf_free[(g0 - 1) % kBufs], ((g0 - 1) / kBufs) & 1, abort_flag);
        tc_fence_after_sync();
      }
      if (has_tail) softmax_sync();  // all warps have cleaned their part of V
      if (quad * 32 < rows) {
        const bool mend = has_tail && *reinterpret_cast<volatile int*>(&odd[tails & 1]) == tails;
        const bool whole = T == tiles_of(keys);
        const float inv = live && l != 0.f ? 1.f / l : 0.f;
        const int h = w.hk * p.G + r % p.G;
        InT* orow = static_cast<InT*>(p.out) + w.b * p.os[0] + h * p.os[1] + t * p.os[2] + kb * (D / 2);
        const int slot = 2 * static_cast<int>(blockIdx.x) + (w.left == begin[2] ? 0 : 1);
        const int64_t prow = static_cast<int64_t>(slot) * p.part_rows + r;
#pragma unroll
        for (int c = 0; c < D / 2; c += 32) {
          uint32_t x[32];
          __syncwarp();  // from the meetings, or from the columns before
          if (any_live) {
            tmem_ld32(t_o + kb * (D / 2) + c, x);
            tmem_wait_ld();
          }
          if (r >= rows) continue;
          if (mend && live) {
            float more[32];  // rare: kept out of the sum's registers
#pragma unroll
            for (int k = 0; k < 32; ++k) more[k] = 0.f;
            fix_up<InT>(p, q, w.b, w.hk, t, key_lo, key_lo + T * 128, kb * (D / 2) + c, more);
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) + more[k]);
          }
          if (!live) {
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = 0u;
          }
          if (whole) {
            if (p.out_vec) {
#pragma unroll
              for (int k = 0; k < 32; k += 8) {
                uint32_t y[4];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                  y[u] = pack2<kBF16>(__uint_as_float(x[k + 2 * u]) * inv, __uint_as_float(x[k + 2 * u + 1]) * inv);
                *reinterpret_cast<uint4*>(orow + c + k) = make_uint4(y[0], y[1], y[2], y[3]);
              }
            } else {
#pragma unroll
              for (int k = 0; k < 32; ++k) orow[c + k] = from_f32<InT>(__uint_as_float(x[k]) * inv);
            }
          } else {
            uint4* po = reinterpret_cast<uint4*>(p.part_o + prow * D + kb * (D / 2) + c);
#pragma unroll
            for (int k = 0; k < 8; ++k) po[k] = make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
          }
        }
        if (r < rows && kb == 0) {
          if (whole) {
            const float m_ref = m_run == -INFINITY ? 0.f : m_run;
            if (p.lse) p.lse[(static_cast<int64_t>(w.b) * p.Hq + h) * p.T + t] = live ? (m_ref + log2f(l)) * kLn2 : -INFINITY;
          } else {
            p.part_ml[prow * 2] = live ? m_run : -INFINITY;
            p.part_ml[prow * 2 + 1] = live ? l : 0.f;
          }
        }
      }
      tc_fence_before_sync();
      if (any_live) pair_sync(quad);  // both have read O: the next segment's products may overwrite it
    }
  }
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

// Adds a cut unit's partial sums: one warp per row, in key order. Up to kScan sequences the search for the unit
// reads lens, rows and nodes ahead of the wait for tc_kernel, which is sound because tc_kernel lets this kernel
// start only after its own wait: whatever wrote them has completed by then.
template <int D, bool kBF16>
__global__ void __launch_bounds__(512) join_kernel(const __grid_constant__ Params p, int ctas_max) {
  using InT = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  __shared__ int s_c0, s_c1, s_first;
  const Share sh = share_of(p.G, p.T);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = blockIdx.x % sh.groups, hk = blockIdx.x / sh.groups % p.Hkv, b = blockIdx.x / sh.groups / p.Hkv;
  const int set = grp / sh.wide, side = grp % sh.wide;
  if (p.n > kScan) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 0) {
    int64_t total = 0, before = 0;
    if (p.n > kScan) {
      total = p.before[p.n];
      before = p.before[b];
    } else {
      for (int i = lane; i < p.n; i += 32) {
        const int64_t x = static_cast<int64_t>(head_weight(p, sh, load_seq(p, i))) * p.Hkv;
        total += x;
        if (i < b) before += x;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
      }
    }
    const Seq s = load_seq(p, b);
    before += static_cast<int64_t>(hk) * head_weight(p, sh, s);
    for (int g = 0; g < set; ++g) before += unit_weight(p, sh, s, g);
    const int64_t start = before + kUnitCost, end = start + tiles_of(group_keys(p, sh, s, grp, grp));  // of its tiles
    const int64_t ranges = range_count(total, ctas_max / sh.wide, p.least);
    // the range of place f is the largest c with total * c / ranges <= f
    int64_t c0 = (start * ranges + ranges - 1) / total, c1 = ((end - 1) * ranges + ranges - 1) / total;
    while (range_start(total, ranges, c0) > start) --c0;
    while (c0 + 1 < ranges && range_start(total, ranges, c0 + 1) <= start) ++c0;
    while (range_start(total, ranges, c1) > end - 1) --c1;
    while (c1 + 1 < ranges && range_start(total, ranges, c1 + 1) <= end - 1) ++c1;
    if (lane == 0) {
      s_c0 = static_cast<int>(c0);
      s_c1 = static_cast<int>(c1);
      s_first = range_start(total, ranges, c0) >= before;  // the unit begins range c0
    }
  }
  __syncthreads();
  const int c0 = s_c0, c1 = s_c1;
  // Every block waits, also one without work: a kernel launched behind this one takes its end for the end of both.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (c0 == c1) return;
  const int rr = blockIdx.y * (blockDim.x >> 5) + warp, t = grp * sh.nodes + rr / p.G;
  if (rr >= sh.nodes * p.G || t >= p.T) return;
  auto part = [&](int c) -> int64_t {  // the row's place in range c's partial slot
    return (2 * (static_cast<int64_t>(c) * sh.wide + side) + (c == c0 && !s_first ? 1 : 0)) * p.part_rows + rr;
  };
  float m = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) m = fmaxf(m, p.part_ml[part(c) * 2]);
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float m_ref = m == -INFINITY ? 0.f : m;
  constexpr int kV = D / 32;
  float acc[kV], l = 0.f;
#pragma unroll
  for (int k = 0; k < kV; ++k) acc[k] = 0.f;
#pragma unroll 4
  for (int c = c0; c <= c1; ++c) {
    const int64_t x = part(c);
    const float wgt = ex2(p.part_ml[x * 2] - m_ref);
    l = fmaf(wgt, p.part_ml[x * 2 + 1], l);
#pragma unroll
    for (int k = 0; k < kV; ++k) acc[k] = fmaf(wgt, p.part_o[x * D + lane * kV + k], acc[k]);
  }
  const int h = hk * p.G + rr % p.G;
  InT* o = static_cast<InT*>(p.out) + b * p.os[0] + h * p.os[1] + t * p.os[2] + lane * kV;
  const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int k = 0; k < kV; ++k) o[k] = from_f32<InT>(m == -INFINITY && l == 0.f ? 0.f : acc[k] * inv);
  if (p.lse && lane == 0) p.lse[(static_cast<int64_t>(b) * p.Hq + h) * p.T + t] = (m_ref + log2f(l)) * kLn2;
}

// ------------------------------------------------------------------ host side
// Whether K and V rows can be read 8 columns at a time.
inline bool rows_in_8(const cab_page_cache* c) {
  const int64_t es = static_cast<int64_t>(dtype_size(static_cast<int>(c->dtype)));
  if (c->dim % 8 != 0 || !aligned16(c->k_pages) || !aligned16(c->v_pages)) return false;
  for (int i = 0; i < 4; ++i)
    if (c->k_strides[i] * es % 16 != 0 || c->v_strides[i] * es % 16 != 0) return false;
  return true;
}
// Rows of a CTA on the CUDA-core path.
inline int simt_rows(const cab_page_cache* c, int64_t R) { return R <= kFewRows && rows_in_8(c) ? kFewRows : R <= 16 ? 16 : 32; }
// Key splits: as many CTAs as fit the GPU at once (registers: 3 an SM with 32 rows, else 4; one more split
// would be a second wave, 287 us instead of 238 for 2 x 128 nodes of 16 / 4 heads over 2000 tokens), none
// without a tile of the longest row the table allows.
inline int simt_splits(int64_t units, int64_t tokens, int rows) {
  const int64_t want = static_cast<int64_t>(current_sm_count()) * (rows == 32 ? 3 : 4) / units;
  const int least = rows == kFewRows ? 128 : kKeysTile;  // few rows: 32 keys for each warp
  return static_cast<int>(std::max<int64_t>(1, std::min({want, (tokens + least - 1) / least, (int64_t)64})));
}

struct Layout {
  bool tc, whole;
  int splits, part_rows, ctas, rows;
  int64_t units;
  size_t part_o, part_ml, before, total;
};

inline bool use_tensor_cores(const cab_page_cache* c, int64_t G) {
  if (c->dtype != CAB_DTYPE_BF16 && c->dtype != CAB_DTYPE_F16) return false;
  if ((c->dim != 64 && c->dim != 128) || G > 128) return false;
  const int64_t S = c->page_size;
  if (!(S == 8 || S == 16 || S == 32 || S == 64 || S % 128 == 0)) return false;
  if (!aligned16(c->k_pages) || !aligned16(c->v_pages)) return false;
  for (int i = 0; i < 4; ++i)
    for (int64_t x : {c->k_strides[i], c->v_strides[i]})
      if (x % 8 != 0 || x >= (int64_t)1 << 39) return false;
  return true;
}

inline Layout layout(const cab_page_cache* c, int64_t n, int64_t Hq, int64_t T) {
  Layout L{};
  const int64_t G = Hq / c->heads, R = G * T, D = c->dim;
  L.tc = use_tensor_cores(c, G);
  if (L.tc) {
    const Share sh = share_of(static_cast<int>(G), static_cast<int>(T));
    L.units = n * c->heads * sh.groups;
    L.part_rows = static_cast<int>(G * std::min<int64_t>(T, sh.nodes));
    L.whole = c->width * c->page_size <= kWholeTiles * 128;
    L.ctas = current_sm_count();
    if (L.whole) return L;
    const size_t slots = static_cast<size_t>(L.ctas) * 2 * L.part_rows;
    L.part_ml = slots * D * 4;
    L.before = (L.part_ml + slots * 8 + 15) & ~size_t(15);
    L.total = L.before + (n > kScan ? static_cast<size_t>(n + 1) * 8 : 0);
    return L;
  }
  L.rows = simt_rows(c, R);
  const int64_t rows = L.rows;
  L.units = n * c->heads * ((R + rows - 1) / rows);
  L.splits = simt_splits(L.units, c->width * c->page_size, L.rows);
  if (L.splits > 1) {
    const size_t slots = static_cast<size_t>(L.units) * L.splits * rows;
    L.part_ml = (slots * D * 4 + 15) & ~size_t(15);
    L.total = L.part_ml + slots * 8;
  }
  return L;
}

inline int page_map(CUtensorMap* map, const void* base, const cab_page_cache* c, const int64_t* st) {
  const uint64_t dims[4] = {static_cast<uint64_t>(c->dim), static_cast<uint64_t>(c->page_size),
                            static_cast<uint64_t>(c->heads), static_cast<uint64_t>(c->pages)};
  const uint64_t strides[3] = {static_cast<uint64_t>(st[3]) * 2, static_cast<uint64_t>(st[2]) * 2, static_cast<uint64_t>(st[1]) * 2};
  const uint32_t box[4] = {64, static_cast<uint32_t>(std::min<int64_t>(c->page_size, 128)), 1, 1};
  return make_tensor_map(map, tma_type(static_cast<int>(c->dtype)), 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The query as [n, Hkv, T, G, D]: a box is the G rows of a group's nodes (64 columns of them).
inline int query_map(CUtensorMap* map, const void* q, const Params& p, int64_t dtype) {
  const uint64_t dims[5] = {static_cast<uint64_t>(p.D), static_cast<uint64_t>(p.G), static_cast<uint64_t>(p.T),
                            static_cast<uint64_t>(p.Hkv), static_cast<uint64_t>(p.n)};
  const uint64_t strides[4] = {static_cast<uint64_t>(p.qs[1]) * 2, static_cast<uint64_t>(p.qs[2]) * 2,
                               static_cast<uint64_t>(p.qs[1]) * 2 * p.G, static_cast<uint64_t>(p.qs[0]) * 2};
  const uint32_t box[5] = {64, static_cast<uint32_t>(p.G), static_cast<uint32_t>(std::min(p.T, 128 / p.G)), 1, 1};
  return make_tensor_map(map, tma_type(static_cast<int>(dtype)), 5, q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int D, bool kBF16>
int launch_tc(const CUtensorMap& km, const CUtensorMap& vm, const CUtensorMap& qm, const Params& p, const Layout& L,
              cudaStream_t st) {
  using C = Cfg<D>;
  if (int rc = pages::allow_smem<tc_kernel<D, kBF16>>(C::kSmem, "tree_attn tc_kernel")) return rc;
  pages::launch_after(tc_kernel<D, kBF16>, dim3(L.ctas), kTcThreads, st, C::kSmem, 1, km, vm, qm, p);
  if (int rc = check_launch("tree_attn tc_kernel")) return rc;
  if (L.whole) return CAB_OK;
  // A block's rows share the search for their unit: 16 where a unit has many (36.5 -> 34.7 us on a 300-token
  // chunk), 8 where that leaves too few blocks (22.9 us against 23.6 on trees of 50 rows).
  const int rows = L.part_rows > 64 ? 16 : 8;
  pages::launch_after(join_kernel<D, kBF16>, dim3(static_cast<unsigned>(L.units), static_cast<unsigned>((L.part_rows + rows - 1) / rows)),
                      32 * rows, st, 0, 1, p, L.ctas);
  return check_launch("tree_attn join_kernel");
}

template <typename T, int DC, int RW>
int launch_simt(const Params& p, int64_t units, cudaStream_t st) {
  auto smem_of = [](int Dp) { return static_cast<size_t>(4 * RW * (Dp + 32) + kKeysTile * (Dp + 4) + kKeysTile * Dp) * 4; };
  const size_t smem = smem_of((p.D + 3) & ~3);
  if (int rc = pages::allow_smem<simt_kernel<T, DC, RW>>(smem_of(32 * DC), "tree_attn simt_kernel")) return rc;
  pages::launch_after(simt_kernel<T, DC, RW>, dim3(static_cast<unsigned>(units), static_cast<unsigned>(p.splits)), kSimtThreads, st, smem, 1, p);
  if (int rc = check_launch("tree_attn simt_kernel")) return rc;
  if (p.splits == 1) return CAB_OK;
  pages::launch_after(simt_join_kernel<T, DC>, dim3(static_cast<unsigned>(units * RW)), kSimtThreads, st, 0, 1, p, 4 * RW);
  return check_launch("tree_attn simt_join_kernel");
}

template <typename T, int DC, int LK>
int launch_simt_rows(const Params& p, const Layout& L, cudaStream_t st) {
  if (L.rows == 16) return launch_simt<T, DC, 4>(p, L.units, st);
  if (L.rows == 32) return launch_simt<T, DC, 8>(p, L.units, st);
  const dim3 grid(static_cast<unsigned>(L.units), static_cast<unsigned>(p.splits));
  const int R = p.G * p.T;  // fewer rows, fewer registers and more loads in flight
  if (R <= 2) pages::launch_after(few_rows_kernel<T, LK, 2>, grid, kSimtThreads, st, 0, 1, p);
  else pages::launch_after(few_rows_kernel<T, LK, kFewRows>, grid, kSimtThreads, st, 0, 1, p);
  if (int rc = check_launch("tree_attn few_rows_kernel")) return rc;
  if (p.splits == 1) return CAB_OK;
  const int rows = R <= 2 ? 2 : kFewRows;
  pages::launch_after(simt_join_kernel<T, DC>, dim3(static_cast<unsigned>((L.units * rows + 3) / 4)), kSimtThreads, st, 0, 1, p, rows);
  return check_launch("tree_attn simt_join_kernel");
}

template <typename T>
int launch_simt_d(const Params& p, const Layout& L, cudaStream_t st) {
  if (p.D <= 64) return launch_simt_rows<T, 2, 8>(p, L, st);
  if (p.D <= 128) return launch_simt_rows<T, 4, 16>(p, L, st);
  return launch_simt_rows<T, 8, 32>(p, L, st);
}

inline int check_sizes(const cab_page_cache* c, int64_t n, int64_t Hq, int64_t T) {
  if (int rc = pages::check_cache(c, "tree_attn", true, false)) return rc;
  if (n <= 0 || Hq <= 0 || T <= 0) return fail(CAB_ERR_INVALID_ARG, "tree_attn: non-positive size");
  if (Hq % c->heads != 0) return fail(CAB_ERR_INVALID_ARG, "tree_attn: Hq %% Hkv != 0");
  if (c->width * c->page_size > kMaxTokens)
    return fail(CAB_ERR_UNSUPPORTED, "tree_attn: table rows for more than %lld tokens", (long long)kMaxTokens);
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
  *bytes = tree::layout(cache, n, Hq, T).total;
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
  if (parents && T > kMaxTree) return fail(CAB_ERR_UNSUPPORTED, "tree_attn: %lld nodes given by parents (at most %d)", (long long)T, kMaxTree);
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale)) return fail(CAB_ERR_INVALID_ARG, "tree_attn: softmax_scale must be > 0 and finite");
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] < 0 || o_strides[i] < 0) return fail(CAB_ERR_INVALID_ARG, "tree_attn: negative stride");
  for (int i = 0; i < 3; ++i)
    if (o_strides[i] == 0 && (i == 0 ? n : i == 1 ? Hq : T) > 1)
      return fail(CAB_ERR_INVALID_ARG, "tree_attn: rows of the output in one place (stride 0)");
  const Layout L = layout(cache, n, Hq, T);
  if (L.total > 0 && (!workspace || workspace_bytes < L.total))
    return fail(CAB_ERR_WORKSPACE, "tree_attn: workspace of %zu bytes needed, %zu given", L.total, workspace_bytes);
  if (L.total > 0 && !aligned16(workspace)) return fail(CAB_ERR_INVALID_ARG, "tree_attn: workspace must be 16-byte aligned");
  if (L.tc) {  // what the ranges count in 32 bits
    const Share sh = share_of(static_cast<int>(Hq / cache->heads), static_cast<int>(T));
    if (cache->heads * sh.sets * (cache->width * cache->page_size / 128 + 1 + kUnitCost) >= (int64_t)1 << 31)
      return fail(CAB_ERR_UNSUPPORTED, "tree_attn: more than 2^31 tiles a sequence");
  }
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
    p.before = reinterpret_cast<int64_t*>(static_cast<uint8_t*>(workspace) + L.before);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (L.tc) {
    if (!aligned16(q)) return fail(CAB_ERR_INVALID_ARG, "tree_attn: q must be 16-byte aligned");
    p.least = L.whole ? 1 : 2;
    p.whole_units = L.whole;
    p.part_rows = L.part_rows;
    p.out_vec = aligned16(out);
    for (int i = 0; i < 3; ++i) {
      if (q_strides[i] <= 0 || q_strides[i] % 8 != 0)
        return fail(CAB_ERR_INVALID_ARG, "tree_attn: q strides must be positive multiples of 16 bytes");
      p.out_vec = p.out_vec && o_strides[i] % 8 == 0;
    }
    CUtensorMap km{}, vm{}, qm{};
    if (int rc = query_map(&qm, q, p, cache->dtype)) return rc;
    if (int rc = page_map(&km, p.k, cache, cache->k_strides)) return rc;
    if (int rc = page_map(&vm, p.v, cache, cache->v_strides)) return rc;
    if (cache->dtype == CAB_DTYPE_BF16)
      return cache->dim == 128 ? launch_tc<128, true>(km, vm, qm, p, L, st) : launch_tc<64, true>(km, vm, qm, p, L, st);
    return cache->dim == 128 ? launch_tc<128, false>(km, vm, qm, p, L, st) : launch_tc<64, false>(km, vm, qm, p, L, st);
  }
  // four elements at a time where every row of K and V starts on their size
  p.in_vec = cache->dim % 4 == 0;
  for (const void* x : {p.k, p.v}) p.in_vec = p.in_vec && reinterpret_cast<uintptr_t>(x) % (4 * es) == 0;
  for (int i = 0; i < 3; ++i) p.in_vec = p.in_vec && p.ks[i] % 4 == 0 && p.vs[i] % 4 == 0;
  switch (cache->dtype) {
    case CAB_DTYPE_F32: return launch_simt_d<float>(p, L, st);
    case CAB_DTYPE_F16: return launch_simt_d<__half>(p, L, st);
    default: return launch_simt_d<__nv_bfloat16>(p, L, st);
  }
}
