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
  int32_t least;      // tensor-core path: tiles a CTA takes at least
  int32_t part_rows;  // rows of a partial slot
  int32_t out_vec;    // out rows start on 16 bytes
  float *part_o, *part_ml;
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

// ------------------------------------------------------------------ tensor-core path
// bf16 / f16, head_dim 64 or 128. A unit is (sequence, KV head, row group); a row group is up
// to 128 rows (kDual false) or 256 (kDual true) of the G * T rows that share the head's keys. The
// units' 128-key tiles form one flat list that is cut into equal ranges, one per CTA
// (persistent, one CTA per SM), so ragged lengths balance and a single long sequence fills the
// GPU; a unit cut between CTAs leaves partial sums that join_kernel adds in key order.
//
// Two streams of work share the tensor pipe, so one's softmax runs under the other's products:
// with kDual the two 128-row halves of the group against the same K/V tile; else the even and
// the odd key tiles of one 128-row group, each with its own O, maximum and sum, merged at the
// end of the range. Stream s, its tile i:
//   S = Q K^T (tcgen05.mma, 128 x 128, K-major from shared memory) -> 128 TMEM columns,
//   p = 2^(s - m) by four warps, one thread per row, written as 16-bit over the S columns
//   (the products' operand type; its sum is taken before the rounding, in float32),
//   O += P V (P from TMEM, V MN-major from its natural layout).
// One thread issues all products in the order PV(i), S(i + 1) per stream, so completion of S(i + 1)
// implies that of PV(i): O may be rescaled then (only when the maximum has grown by more than
// 2^8), and S(i + 1) may overwrite P(i).
//
// Warp 0 looks up the pages and loads K and V tiles by TMA (one box per page and 64 columns)
// through one ring of stages; a page number outside the pool reads zeros. Tiles that reach into the nodes
// or past the length are masked per row by a 128-bit word, and the unused or unseen rows of V that are not
// finite are zeroed in shared memory, so that 0 * NaN cannot enter a product; a seen value that is not
// finite is added back to the rows that see it (fix_up).

constexpr int kTcThreads = 384;  // warp 0: TMA, warp 1: products, warps 4-7 / 8-11: streams 0 / 1
constexpr float kRescaleThreshold = 8.0f;
constexpr uint32_t kTmemO = 256;

template <int D, bool kDual>
struct Cfg {
  static constexpr int kTile = 128 * D * 2;  // bytes of a K, V or Q tile
  static constexpr int kAtoms = D / 64;
  static constexpr int kQTiles = kDual ? 2 : 1;
  static constexpr int kRows = 128 * kQTiles;
  static constexpr int kStages = (7 - kQTiles) * (D == 64 ? 2 : 1);
  static constexpr int kBars = (2 * kStages + 8) * 8 + 64;
  static constexpr int kSmem = kQTiles * kTile + kStages * kTile + kBars + 1024;
  static_assert(kSmem <= 232448, "shared memory");
};

struct Walk {  // a range of the flat tile list, unit by unit
  int b, hk, grp, tiles, at;  // tile `at` of `tiles`
  int left;                   // tiles of the range not yet walked
  Seq s;
};

template <int kRows>
__device__ __forceinline__ int unit_keys(const Params& p, const Seq& s, int grp) {
  const int t0 = grp * kRows / p.G;
  return t0 < s.m ? key_limit(p, s, min(p.T - 1, (grp * kRows + kRows - 1) / p.G)) : 0;
}
template <int kRows>
__device__ __forceinline__ int unit_tiles(const Params& p, const Seq& s, int grp) {
  return max(1, (unit_keys<kRows>(p, s, grp) + 127) / 128);
}
template <int kRows>
__device__ __forceinline__ int seq_tiles(const Params& p, const Seq& s) {  // of one KV head
  const int groups = (p.G * p.T + kRows - 1) / kRows;
  int sum = 0;
  for (int g = 0; g < groups; ++g) sum += unit_tiles<kRows>(p, s, g);
  return sum;
}

template <int kRows>
__device__ __forceinline__ void walk_next(const Params& p, Walk& w) {  // to the next unit's first tile
  const int groups = (p.G * p.T + kRows - 1) / kRows;
  w.left -= min(w.left, w.tiles - w.at);
  w.at = 0;
  if (++w.grp == groups) {
    w.grp = 0;
    if (++w.hk == p.Hkv) {
      w.hk = 0;
      ++w.b;
      if (w.left > 0) w.s = load_seq(p, w.b);
    }
  }
  if (w.left > 0) w.tiles = unit_tiles<kRows>(p, w.s, w.grp);
}

__host__ __device__ __forceinline__ int64_t range_start(int64_t total, int64_t ctas, int64_t c) { return total * c / ctas; }
__device__ __forceinline__ int range_ctas(int64_t total, int ctas, int least) {
  return static_cast<int>(min(static_cast<int64_t>(ctas), (total + least - 1) / least));
}

// Warp-wide: the total number of tiles, and the sequence that holds flat tile `f` with the tiles before it.
template <int kRows>
__device__ __forceinline__ int64_t total_tiles(const Params& p) {
  const int lane = threadIdx.x & 31;
  int64_t sum = 0;
  for (int b = lane; b < p.n; b += 32) sum += static_cast<int64_t>(seq_tiles<kRows>(p, load_seq(p, b))) * p.Hkv;
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
template <int kRows>
__device__ __forceinline__ void find_seq(const Params& p, int64_t f, int* b_out, int64_t* before) {
  const int lane = threadIdx.x & 31;
  int64_t base = 0;
  for (int b0 = 0; b0 < p.n; b0 += 32) {
    const int b = b0 + lane;
    const int64_t own = b < p.n ? static_cast<int64_t>(seq_tiles<kRows>(p, load_seq(p, b))) * p.Hkv : 0;
    int64_t inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, base + inc > f);
    if (hit) {
      const int l = __ffs(hit) - 1;
      *b_out = b0 + l;
      *before = base + __shfl_sync(0xffffffffu, inc - own, l);
      return;
    }
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
  *b_out = p.n - 1;
  *before = base;
}

struct Bits {
  uint64_t lo, hi;
};
__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// Which of the keys key0 .. key0 + 127 node t of sequence b sees.
__device__ __noinline__ Bits seen_bits(const Params& p, const Seq& s, int b, int t, int key0, bool bad_pages) {
  const int c = s.ctx - key0;
  Bits w{low_bits(c), low_bits(c - 64)};
  if (p.parents) {
    const int32_t* up = p.parents + b * p.parents_stride;
    for (int x = t; x >= 0;) {
      const int at = c + x;
      if (at < 0) break;
      if (at < 64) w.lo |= 1ull << at;
      else if (at < 128) w.hi |= 1ull << (at - 64);
      const int y = up[x];
      if (y >= x) break;
      x = y;
    }
  } else if (p.mask) {
    const uint8_t* row = p.mask + b * p.mask_stride + static_cast<int64_t>(t) * p.T;
    for (int at = max(c, 0); at < min(128, c + s.m); ++at)
      if (row[at - c]) {
        if (at < 64) w.lo |= 1ull << at;
        else w.hi |= 1ull << (at - 64);
      }
  } else {
    w.lo = low_bits(c + t + 1);
    w.hi = low_bits(c + t + 1 - 64);
  }
  if (bad_pages) {
    for (int j = 0; j < 128; ++j) {
      const int key = key0 + j;
      if (key >= s.len) break;
      const int pg = p.table[s.row * p.table_stride + key / p.page_size];
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
__device__ __noinline__ void fix_up(const Params& p, const Seq& s, int b, int hk, int t, int lo, int hi, int col, float* o) {
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

// Row `r` of a V tile: beyond the length it becomes 0; of a node, elements that are not finite do.
// Returns whether there were any.
template <int D, bool kBF16>
__device__ __forceinline__ bool clean_v_row(uint8_t* tile, int r, int key, const Seq& s) {
  constexpr uint32_t kExp = kBF16 ? 0x7F80u : 0x7C00u;
  bool found = false;
#pragma unroll
  for (int a = 0; a < D / 64; ++a)
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      uint4* q = reinterpret_cast<uint4*>(tile + a * 16384 + sw128_offset(r, c));
      if (key >= s.len) {
        *q = make_uint4(0, 0, 0, 0);
        continue;
      }
      uint4 x = *q;
      uint32_t* e = reinterpret_cast<uint32_t*>(&x);
      bool hit = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if ((e[k] & kExp) == kExp) { e[k] &= 0xFFFF0000u; hit = true; }
        if ((e[k] & (kExp << 16)) == (kExp << 16)) { e[k] &= 0x0000FFFFu; hit = true; }
      }
      if (hit) *q = x;
      found |= hit;
    }
  return found;
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

__device__ __forceinline__ bool streams_sync_or(bool x) {  // the 256 threads of both streams
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\t"
      "barrier.cta.red.or.pred b, 1, 256, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(x))
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void streams_sync() { asm volatile("barrier.cta.sync 1, 256;" ::: "memory"); }

// Places in a range's ring sequence of a segment of T tiles: K(0) K(1) V(0) K(2) V(1) ... (single),
// K(0) V(0) K(1) V(1) ... (dual), in the order in which the products need them.
template <bool kDual>
__device__ __forceinline__ uint32_t place_k(int g) {
  return kDual ? 2 * g : (g == 0 ? 0 : 2 * g - 1);
}
template <bool kDual>
__device__ __forceinline__ uint32_t place_v(int g, int T) {
  return kDual ? 2 * g + 1 : (g == T - 1 ? 2 * T - 1 : 2 * g + 2);
}

template <int D, bool kBF16, bool kDual>
__global__ void __launch_bounds__(kTcThreads, 1)
    tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
              const __grid_constant__ Params p) {
  using C = Cfg<D, kDual>;
  using InT = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  constexpr int kRows = C::kRows, kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = base;
  uint8_t* ring = sQ + C::kQTiles * C::kTile;
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(ring + kStages * C::kTile);
  uint64_t* kv_empty = kv_full + kStages;
  uint64_t* s_full = kv_empty + kStages;  // [2] S of stream s is there (and its earlier PV done)
  uint64_t* p_full = s_full + 2;          // [2] P of stream s is there (4 warps)
  uint64_t* q_full = p_full + 2;          // Q of the segment is there (8 warps)
  uint64_t* drain = q_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  int* odd_flag = abort_flag + 1;  // a V tile of the segment held values that are not finite
  int* s_begin = odd_flag + 1;     // first sequence, KV head, group, tile; tiles of the range; flat start
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 32) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
    }
    mbar_init(q_full, 8);
    mbar_init(drain, 1);
    *abort_flag = 0;
    *odd_flag = 0;
    fence_barrier_init();
  }
  if (warp == 2) tmem_alloc(tmem_slot, 512);
  if (warp == 0) {
    const int64_t total = total_tiles<kRows>(p);
    const int ctas = range_ctas(total, gridDim.x, p.least);
    int64_t f0 = 0, f1 = 0, before = 0;
    int b = 0;
    if (static_cast<int>(blockIdx.x) < ctas) {
      f0 = range_start(total, ctas, blockIdx.x);
      f1 = range_start(total, ctas, blockIdx.x + 1);
      find_seq<kRows>(p, f0, &b, &before);
    }
    if (lane == 0) {
      s_begin[0] = b;
      s_begin[1] = static_cast<int>(f0 - before);
      s_begin[2] = static_cast<int>(f1 - f0);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  Walk w;
  w.b = s_begin[0];
  w.left = s_begin[2];
  w.hk = w.grp = w.at = 0;
  w.tiles = 1;
  if (w.left > 0) {
    w.s = load_seq(p, w.b);
    const int per_head = seq_tiles<kRows>(p, w.s);
    int rem = s_begin[1];
    w.hk = rem / per_head;
    rem -= w.hk * per_head;
    for (w.tiles = unit_tiles<kRows>(p, w.s, 0); rem >= w.tiles; w.tiles = unit_tiles<kRows>(p, w.s, ++w.grp)) rem -= w.tiles;
    w.at = rem;
  }

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    const int S = static_cast<int>(p.page_size);
    const int per_tile = S < 128 ? 128 / S : 1;
    const int pi = lane / C::kAtoms, a = lane % C::kAtoms;
    const bool mine = pi < per_tile;
    const uint32_t off = a * 16384 + pi * (S < 128 ? S * 128 : 0);
    uint32_t pos = 0;
    bool ok = true;
    for (; w.left > 0 && ok; walk_next<kRows>(p, w)) {
      const int T = min(w.left, w.tiles - w.at);
      const int held = (w.s.len + S - 1) / S;
      const int32_t* row = p.table + w.s.row * p.table_stride;
      // the page of this lane's box in tile g of the segment (the number past the pool: zeros)
      auto page_of = [&](int g) -> int {
        const int j = (w.at + g) * 128 / S + (S < 128 ? pi : 0);
        if (!mine || g >= T || j >= held) return static_cast<int>(p.pages);
        const int q = row[j];
        return q < 0 || q >= p.pages ? static_cast<int>(p.pages) : q;
      };
      auto load = [&](const CUtensorMap* map, int g, int page) {
        const int st = pos % kStages;
        ok = ok && mbar_wait(&kv_empty[st], ((pos / kStages) & 1) ^ 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], C::kTile);
        __syncwarp();
        const int slot = S < 128 ? 0 : (w.at + g) * 128 % S;
        if (mine) tma_load_4d(ring + st * C::kTile + off, map, &kv_full[st], 64 * a, slot, w.hk, page);
        ++pos;
      };
      int e0 = page_of(0), e1 = page_of(1), e2 = page_of(2);
      if constexpr (!kDual) {
        load(&kmap, 0, e0);
        if (T > 1) load(&kmap, 1, e1);
      }
      for (int g = 0; g < T; ++g) {
        const int e3 = page_of(g + 3);
        if constexpr (kDual) {
          load(&kmap, g, e0);
          load(&vmap, g, e0);
        } else {
          load(&vmap, g, e0);
          if (g + 2 < T) load(&kmap, g + 2, e2);
        }
        e0 = e1;
        e1 = e2;
        e2 = e3;
      }
    }
    if (!ok) {  // copies still in flight land before the CTA ends
      for (uint32_t k = 0; k < kStages && k < pos; ++k) {
        const uint32_t q = pos - 1 - k;
        (void)mbar_wait(&kv_full[q % kStages], (q / kStages) & 1, nullptr);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_idesc_f16(128, 128, kBF16 ? 1 : 0, 0, 0);
      constexpr uint32_t idesc_o = make_idesc_f16(128, D, kBF16 ? 1 : 0, 0, 1);
      const uint64_t dQ = make_smem_desc(smem_u32(sQ), 16, 1024, 2);
      const uint64_t dK = make_smem_desc(smem_u32(ring), 16, 1024, 2);
      const uint64_t dV = make_smem_desc(smem_u32(ring), 16384, 1024, 2);
      uint32_t pos = 0, seg = 0, np[2] = {0, 0};
      bool ok = true;
      for (; w.left > 0 && ok; walk_next<kRows>(p, w), ++seg) {
        const int T = min(w.left, w.tiles - w.at);
        const int rows = min(kRows, p.G * p.T - w.grp * kRows);
        const int n0 = kDual ? T : (T + 1) / 2, n1 = kDual ? (rows > 128 ? T : 0) : T / 2;
        const int last = kDual ? (n1 > 0 ? 1 : 0) : 0;  // the stream after which a shared tile is free
        ok = mbar_wait(q_full, seg & 1, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        auto scores = [&](int s, int g) {
          const uint32_t at = pos + place_k<kDual>(g), st = at % kStages;
          if (!mbar_wait(&kv_full[st], (at / kStages) & 1, abort_flag)) { ok = false; return; }
          tc_fence_after_sync();
          const uint64_t dq = dQ + static_cast<uint64_t>((kDual ? s * C::kTile : 0) >> 4);
          const uint64_t dk = dK + static_cast<uint64_t>((st * C::kTile) >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t o = (kk >> 2) * (16384 >> 4) + (kk & 3) * (32 >> 4);
            mma_f16_ss(tmem + s * 128, dq + o, dk + o, idesc_s, kk > 0 ? 1u : 0u);
          }
          if (!kDual || s == last) mma_commit(&kv_empty[st]);
        };
        scores(0, 0);
        if (ok) mma_commit(&s_full[0]);
        if (ok && n1 > 0) {
          scores(1, kDual ? 0 : 1);
          if (ok) mma_commit(&s_full[1]);
        }
        for (int i = 0; i < n0 && ok; ++i) {
          for (int s = 0; s < 2 && ok; ++s) {
            const int ns = s ? n1 : n0;
            if (i >= ns) continue;
            const int g = kDual ? i : 2 * i + s;
            const uint32_t at = pos + place_v<kDual>(g, T), st = at % kStages;
            if (!mbar_wait(&kv_full[st], (at / kStages) & 1, abort_flag) ||
                !mbar_wait(&p_full[s], np[s] & 1, abort_flag)) { ok = false; break; }
            ++np[s];
            tc_fence_after_sync();
            const uint64_t dv = dV + static_cast<uint64_t>((st * C::kTile) >> 4);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              mma_f16_ts(tmem + kTmemO + s * 128, tmem + s * 128 + kk * 8, dv + static_cast<uint64_t>(kk * (2048 >> 4)), idesc_o,
                         (i > 0 || kk > 0) ? 1u : 0u);
            if (!kDual || s == last) mma_commit(&kv_empty[st]);
            if (i + 1 < ns) scores(s, kDual ? i + 1 : g + 2);
            if (ok) mma_commit(&s_full[s]);  // S(i + 1), or the stream's finished O
          }
        }
        pos += 2 * T;
      }
      mma_commit(drain);
      (void)mbar_wait(drain, 0, nullptr);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- softmax and epilogue
    const int s = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane, st_tid = threadIdx.x - 128;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_s = tmem + lanes + s * 128, t_o = tmem + lanes + kTmemO + s * 128;
    uint32_t pos = 0, ns_done = 0;
    bool first = true;
    for (; w.left > 0; walk_next<kRows>(p, w)) {
      const int T = min(w.left, w.tiles - w.at);
      const Seq q = w.s;
      const int R = p.G * p.T, row0 = w.grp * kRows;
      const int rows = min(kRows, R - row0);
      const int n0 = kDual ? T : (T + 1) / 2, n1 = kDual ? (rows > 128 ? T : 0) : T / 2;
      const int count = s ? n1 : n0;
      const int rr = kDual ? s * 128 + r : r;
      const int t = (row0 + rr) / p.G;
      const bool live = rr < rows && t < q.m;
      const bool any_live = __any_sync(0xffffffffu, live);
      const int key_lo = w.at * 128, keys = unit_keys<kRows>(p, q, w.grp);

      // both streams have left the previous segment (its products are complete, its O is read)
      if (!first) streams_sync();
      first = false;
      if (st_tid == 0) *odd_flag = 0;
      for (int e = st_tid; e < kRows * (D / 8); e += 256) {
        const int x = e / (D / 8), c = e - x * (D / 8);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (x < rows) {
          const int row = row0 + x;
          v = *reinterpret_cast<const uint4*>(static_cast<const InT*>(p.q) + w.b * p.qs[0] +
                                              (w.hk * p.G + row % p.G) * p.qs[1] + (row / p.G) * p.qs[2] + c * 8);
        }
        *reinterpret_cast<uint4*>(sQ + (x >> 7) * C::kTile + (c >> 3) * 16384 + sw128_offset(x & 127, c & 7)) = v;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      bool bad = false;
      {
        const int S = static_cast<int>(p.page_size), j1 = (min(keys, key_lo + T * 128) + S - 1) / S;
        for (int j = key_lo / S + st_tid; j < j1; j += 256) {
          const int pg = p.table[q.row * p.table_stride + j];
          bad |= pg < 0 || pg >= p.pages;
        }
      }
      bad = streams_sync_or(bad);

      float m_run = -INFINITY, l = 0.f;
      for (int i = 0; i < count; ++i) {
        const int g = kDual ? i : 2 * i + s;
        const int key0 = key_lo + g * 128;
        const bool tail = bad || key0 + 128 > q.ctx;
        (void)mbar_wait(&s_full[s], ns_done & 1, abort_flag);
        ++ns_done;
        tc_fence_after_sync();
        if (tail && (!kDual || s == 0)) {
          const uint32_t at = pos + place_v<kDual>(g, T), sg = at % kStages;
          (void)mbar_wait(&kv_full[sg], (at / kStages) & 1, abort_flag);
          const int key = key0 + r;
          if (key >= q.ctx) {
            if (clean_v_row<D, kBF16>(ring + sg * C::kTile, r, key, q)) *reinterpret_cast<volatile int*>(odd_flag) = 1;
            fence_proxy_async_smem();
          }
        }
        if (any_live) {
          Bits see{~0ull, ~0ull};
          if (tail) see = live ? seen_bits(p, q, w.b, t, key0, bad) : Bits{0, 0};
          float mx = -INFINITY;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t x[32];
            tmem_ld32(t_s + 32 * c, x);
            tmem_wait_ld();
            if (tail) {
              const uint32_t word = static_cast<uint32_t>((c < 2 ? see.lo : see.hi) >> (32 * (c & 1)));
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (word >> k & 1u) mx = fmaxf(mx, __uint_as_float(x[k]));
            } else {
              float m4[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int k = 0; k < 32; ++k) m4[k & 3] = fmaxf(m4[k & 3], __uint_as_float(x[k]));
              mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            }
          }
          const float m_tile = mx * p.scale_log2;
          float alpha = 1.f;
          if (m_run == -INFINITY) {
            m_run = m_tile;
          } else if (m_tile > m_run + kRescaleThreshold) {
            alpha = ex2(m_run - m_tile);
            m_run = m_tile;
            l *= alpha;
          }
          if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
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
          const float sub = m_run == -INFINITY ? 0.f : m_run;  // all scores -inf so far: weights 0
          float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t x[32], y[16];
            tmem_ld32(t_s + 32 * c, x);
            tmem_wait_ld();
            const uint32_t word = static_cast<uint32_t>((c < 2 ? see.lo : see.hi) >> (32 * (c & 1)));
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              float p0 = ex2(fmaf(__uint_as_float(x[k]), p.scale_log2, -sub));
              float p1 = ex2(fmaf(__uint_as_float(x[k + 1]), p.scale_log2, -sub));
              if (tail) {
                p0 = word >> k & 1u ? p0 : 0.f;
                p1 = word >> (k + 1) & 1u ? p1 : 0.f;
              }
              l4[(k >> 1) & 3] += p0 + p1;
              y[k >> 1] = pack2<kBF16>(p0, p1);
            }
            tmem_st16(t_s + 16 * c, y);
          }
          l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
          tmem_wait_st();
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[s]);
      }
      if (count > 0) {
        (void)mbar_wait(&s_full[s], ns_done & 1, abort_flag);
        ++ns_done;
        tc_fence_after_sync();
      }
      pos += 2 * T;

      // epilogue: dual: this stream's rows; single: half the columns of the row's two sums
      float m_other = -INFINITY, l_other = 0.f;
      tc_fence_before_sync();
      if constexpr (!kDual) {
        streams_sync();  // all products are complete: Q's memory is free, both O can be read
        float2* xchg = reinterpret_cast<float2*>(sQ);
        xchg[s * 128 + r] = make_float2(m_run, l);
        streams_sync();
        const float2 o = xchg[(s ^ 1) * 128 + r];
        m_other = o.x;
        l_other = o.y;
      } else {
        streams_sync();
      }
      tc_fence_after_sync();
      const bool odd = *reinterpret_cast<volatile int*>(odd_flag) != 0;
      if (any_live || (kDual ? s * 128 + quad * 32 : quad * 32) < rows) {
        const float m_all = fmaxf(m_run, m_other);
        const float m_ref = m_all == -INFINITY ? 0.f : m_all;
        const float w_own = ex2(m_run - m_ref), w_other = ex2(m_other - m_ref);  // 2^-inf = 0
        const float l_all = l * w_own + l_other * w_other;
        const bool whole = T == w.tiles;
        const bool own_used = count > 0 && any_live, other_used = !kDual && (s ? n0 : n1) > 0 && any_live;
        const float inv = l_all != 0.f ? 1.f / l_all : 0.f;
        const int row = row0 + rr;
        InT* orow = static_cast<InT*>(p.out) + w.b * p.os[0] + (w.hk * p.G + row % p.G) * p.os[1] + t * p.os[2];
        const int slot = 2 * static_cast<int>(blockIdx.x) + (w.left == s_begin[2] ? 0 : 1);
        const int64_t prow = static_cast<int64_t>(slot) * p.part_rows + rr;
        constexpr int kCols = kDual ? D : D / 2;
        const int col0 = kDual ? 0 : s * kCols;
#pragma unroll 1
        for (int c = col0; c < col0 + kCols; c += 32) {
          float o[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0.f;
          if (own_used) {
            uint32_t x[32];
            tmem_ld32(t_o + c, x);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __uint_as_float(x[k]) * w_own;
          }
          if (other_used) {
            uint32_t x[32];
            tmem_ld32(tmem + lanes + kTmemO + (s ^ 1) * 128 + c, x);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = fmaf(__uint_as_float(x[k]), w_other, o[k]);
          }
          if (rr < rows) {
            if (odd && live) {
              float more[32];  // rare: kept out of the sum's registers
#pragma unroll
              for (int k = 0; k < 32; ++k) more[k] = 0.f;
              fix_up<InT>(p, q, w.b, w.hk, t, key_lo, key_lo + T * 128, c, more);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] += more[k];
            }
            if (whole) {
              const float f = live ? inv : 0.f;
              if (p.out_vec) {
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                  uint4 v;
                  v.x = live ? pack2<kBF16>(o[k] * f, o[k + 1] * f) : 0u;
                  v.y = live ? pack2<kBF16>(o[k + 2] * f, o[k + 3] * f) : 0u;
                  v.z = live ? pack2<kBF16>(o[k + 4] * f, o[k + 5] * f) : 0u;
                  v.w = live ? pack2<kBF16>(o[k + 6] * f, o[k + 7] * f) : 0u;
                  *reinterpret_cast<uint4*>(orow + c + k) = v;
                }
              } else {
#pragma unroll
                for (int k = 0; k < 32; ++k) orow[c + k] = from_f32<InT>(live ? o[k] * f : 0.f);
              }
            } else {
              float4* po = reinterpret_cast<float4*>(p.part_o + prow * D + c);
#pragma unroll
              for (int k = 0; k < 8; ++k) po[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
            }
          }
        }
        if (rr < rows && (kDual || s == 0)) {
          if (whole) {
            if (p.lse)
              p.lse[(static_cast<int64_t>(w.b) * p.Hq + w.hk * p.G + row % p.G) * p.T + t] =
                  live ? (m_ref + log2f(l_all)) * kLn2 : -INFINITY;
          } else {
            p.part_ml[prow * 2] = live ? m_all : -INFINITY;
            p.part_ml[prow * 2 + 1] = live ? l_all : 0.f;
          }
        }
        tc_fence_before_sync();
      }
    }
  }
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

// Adds a cut unit's partial sums: one warp per row, in key order.
template <int D, bool kBF16, bool kDual>
__global__ void __launch_bounds__(256) join_kernel(const Params p, int ctas_max) {
  using C = Cfg<D, kDual>;
  using InT = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  constexpr int kRows = C::kRows;
  __shared__ int s_c0, s_c1, s_first;
  const int groups = (p.G * p.T + kRows - 1) / kRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = blockIdx.x % groups, hk = blockIdx.x / groups % p.Hkv, b = blockIdx.x / groups / p.Hkv;
  if (warp == 0) {
    int64_t total = 0, before = 0;
    for (int i = lane; i < p.n; i += 32) {
      const int64_t x = static_cast<int64_t>(seq_tiles<kRows>(p, load_seq(p, i))) * p.Hkv;
      total += x;
      if (i < b) before += x;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    const Seq s = load_seq(p, b);
    before += static_cast<int64_t>(hk) * seq_tiles<kRows>(p, s);
    for (int g = 0; g < grp; ++g) before += unit_tiles<kRows>(p, s, g);
    const int64_t end = before + unit_tiles<kRows>(p, s, grp);
    const int64_t ctas = range_ctas(total, ctas_max, p.least);
    // the CTA of flat tile f is the largest c with total * c / ctas <= f
    int64_t c0 = (before * ctas + ctas - 1) / total, c1 = ((end - 1) * ctas + ctas - 1) / total;
    while (range_start(total, ctas, c0) > before) --c0;
    while (c0 + 1 < ctas && range_start(total, ctas, c0 + 1) <= before) ++c0;
    while (range_start(total, ctas, c1) > end - 1) --c1;
    while (c1 + 1 < ctas && range_start(total, ctas, c1 + 1) <= end - 1) ++c1;
    if (lane == 0) {
      s_c0 = static_cast<int>(c0);
      s_c1 = static_cast<int>(c1);
      s_first = range_start(total, ctas, c0) >= before;  // the unit begins CTA c0's range
    }
  }
  __syncthreads();
  const int c0 = s_c0, c1 = s_c1;
  if (c0 == c1) return;
  const int rr = blockIdx.y * 8 + warp, row = grp * kRows + rr;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (rr >= kRows || row >= p.G * p.T) return;
  float m = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) {
    const int slot = 2 * c + (c == c0 && !s_first ? 1 : 0);
    m = fmaxf(m, p.part_ml[(static_cast<int64_t>(slot) * p.part_rows + rr) * 2]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float m_ref = m == -INFINITY ? 0.f : m;
  constexpr int kV = D / 32;
  float acc[kV], l = 0.f;
#pragma unroll
  for (int k = 0; k < kV; ++k) acc[k] = 0.f;
#pragma unroll 4
  for (int c = c0; c <= c1; ++c) {
    const int slot = 2 * c + (c == c0 && !s_first ? 1 : 0);
    const int64_t x = static_cast<int64_t>(slot) * p.part_rows + rr;
    const float wgt = ex2(p.part_ml[x * 2] - m_ref);
    l = fmaf(wgt, p.part_ml[x * 2 + 1], l);
#pragma unroll
    for (int k = 0; k < kV; ++k) acc[k] = fmaf(wgt, p.part_o[x * D + lane * kV + k], acc[k]);
  }
  const int h = hk * p.G + row % p.G, t = row / p.G;
  InT* o = static_cast<InT*>(p.out) + b * p.os[0] + h * p.os[1] + t * p.os[2] + lane * kV;
  const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int k = 0; k < kV; ++k) o[k] = from_f32<InT>(m == -INFINITY && l == 0.f ? 0.f : acc[k] * inv);
  if (p.lse && lane == 0) p.lse[(static_cast<int64_t>(b) * p.Hq + h) * p.T + t] = (m_ref + log2f(l)) * kLn2;
}

// ------------------------------------------------------------------ host side
inline int simt_splits(int64_t units, int64_t tokens) {
  const int64_t want = (static_cast<int64_t>(current_sm_count()) * 6 + units - 1) / units;
  return static_cast<int>(std::max<int64_t>(1, std::min({want, (tokens + kKeysTile - 1) / kKeysTile, (int64_t)64})));
}

struct Layout {
  bool tc, dual;
  int splits, part_rows, ctas;
  int64_t units;
  size_t part_o, part_ml, total;
};

inline bool use_tensor_cores(const cab_page_cache* c) {
  if (c->dtype != CAB_DTYPE_BF16 && c->dtype != CAB_DTYPE_F16) return false;
  if (c->dim != 64 && c->dim != 128) return false;
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
  const int64_t R = Hq / c->heads * T, D = c->dim;
  L.tc = use_tensor_cores(c);
  if (L.tc) {
    // More than 128 rows a KV head: both halves of a 256-row group use each K / V tile.
    L.dual = R > 128;
    const int64_t rows = L.dual ? 256 : 128;
    L.units = n * c->heads * ((R + rows - 1) / rows);
    L.part_rows = static_cast<int>(std::min(R, rows));
    L.ctas = current_sm_count();
    const size_t slots = static_cast<size_t>(L.ctas) * 2 * L.part_rows;
    L.part_ml = slots * D * 4;
    L.total = L.part_ml + slots * 8;
    return L;
  }
  L.units = n * c->heads * ((R + kRowsTile - 1) / kRowsTile);
  L.splits = simt_splits(L.units, c->width * c->page_size);
  if (L.splits > 1) {
    const size_t slots = static_cast<size_t>(L.units) * L.splits * kRowsTile;
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

template <int D, bool kBF16, bool kDual>
int launch_tc(const CUtensorMap& km, const CUtensorMap& vm, const Params& p, const Layout& L, cudaStream_t st) {
  using C = Cfg<D, kDual>;
  cudaFuncSetAttribute(tc_kernel<D, kBF16, kDual>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  tc_kernel<D, kBF16, kDual><<<L.ctas, kTcThreads, C::kSmem, st>>>(km, vm, p);
  if (int rc = check_launch("tree_attn tc_kernel")) return rc;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(static_cast<unsigned>(L.units), static_cast<unsigned>((L.part_rows + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, join_kernel<D, kBF16, kDual>, p, L.ctas);
  return check_launch("tree_attn join_kernel");
}

template <int D, bool kBF16>
int launch_tc_rows(const CUtensorMap& km, const CUtensorMap& vm, const Params& p, const Layout& L, cudaStream_t st) {
  return L.dual ? launch_tc<D, kBF16, true>(km, vm, p, L, st) : launch_tc<D, kBF16, false>(km, vm, p, L, st);
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
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale)) return fail(CAB_ERR_INVALID_ARG, "tree_attn: softmax_scale must be > 0 and finite");
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] < 0 || o_strides[i] < 0) return fail(CAB_ERR_INVALID_ARG, "tree_attn: negative stride");
  const Layout L = layout(cache, n, Hq, T);
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
  if (L.tc) {
    if (!aligned16(q)) return fail(CAB_ERR_INVALID_ARG, "tree_attn: q must be 16-byte aligned");
    p.least = 2;
    p.part_rows = L.part_rows;
    p.out_vec = aligned16(out);
    for (int i = 0; i < 3; ++i) {
      if (q_strides[i] % 8 != 0) return fail(CAB_ERR_INVALID_ARG, "tree_attn: q strides must be multiples of 16 bytes");
      p.out_vec = p.out_vec && o_strides[i] % 8 == 0;
    }
    CUtensorMap km{}, vm{};
    if (int rc = page_map(&km, p.k, cache, cache->k_strides)) return rc;
    if (int rc = page_map(&vm, p.v, cache, cache->v_strides)) return rc;
    if (cache->dtype == CAB_DTYPE_BF16)
      return cache->dim == 128 ? launch_tc_rows<128, true>(km, vm, p, L, st) : launch_tc_rows<64, true>(km, vm, p, L, st);
    return cache->dim == 128 ? launch_tc_rows<128, false>(km, vm, p, L, st) : launch_tc_rows<64, false>(km, vm, p, L, st);
  }
  switch (cache->dtype) {
    case CAB_DTYPE_F32: return launch_simt_d<float>(p, L.units, st);
    case CAB_DTYPE_F16: return launch_simt_d<__half>(p, L.units, st);
    default: return launch_simt_d<__nv_bfloat16>(p, L.units, st);
  }
}
