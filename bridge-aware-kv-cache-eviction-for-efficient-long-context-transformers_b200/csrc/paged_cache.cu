// Paged KV cache: the bookkeeping of its pages (fork, compact, extend, truncate and free are
// one update), the copies of the tokens that change their page, and the write of new tokens.
//
// State (cab_page_cache): K / V pages [layers, pages, heads, page_size, dim], a table of page
// numbers and a length per sequence row, a use count per page, one status word. A page is
// free when its count is 0. A page whose content ends inside it (a row's last one) belongs to
// one row alone, so rows share full pages only and appending never needs a copy.
//
// Update: pair i turns row d into a selection of row s. With n = len[s], a = start[i] and the
// offsets x -> keep[x], x < kn, the new content is [0, a) followed by a + keep[x]; C = a + kn
// tokens, then room for grow[i] more. Let I = a + min{x : keep[x] != x} be the prefix that
// stays in place. Pages 0 .. R-1 with R = floor(I / S) keep their content, so d shares them
// with s (count + 1), or keeps them where s == d; so does the last, partly filled page where
// I == C and s == d uses it alone. The other ceil((C + grow) / S) - R pages are fresh: the
// lowest-numbered pages that were free before the call, in order of pair and position, so the
// result does not depend on timing. Counts go down for d's old pages and up for its new ones;
// a page that drops to 0 can be taken by the next call, never by this one, since this call's
// copies may still read it. Tokens R*S .. C-1 are then copied into the fresh pages.
//
// The update is all or nothing: every check is made before the first write, a refused call
// changes nothing but the status word, and while the status word is set later calls do
// nothing either.

#include "cab_host.h"
#include "cab_ptx.cuh"

#include <algorithm>

namespace cab {
namespace pages {

constexpr int kUpdateThreads = 1024;
constexpr int kMaxPairs = 1024;     // one pair per thread of the prefix sum
constexpr int64_t kMaxRows = 65536;  // three bitmaps of the rows in shared memory
constexpr int kMaxCluster = 8;

struct PairRec {
  int32_t stay, base, start, content;  // R, first rank in the free list, a, C
};

struct UpdateParams {
  cab_page_cache c;
  const int32_t *src, *dst, *start, *keep_num, *grow;
  const void* keep;
  int64_t start_value, grow_value, keep_stride, keep_cols, keep_num_stride;
  int32_t keep64, n, copies;
  int32_t* header;     // [0] accepted, [1] fresh pages
  int32_t* part;       // per CTA of the cluster: first[n] | free | err0 | err1
  PairRec* pair;       // [n]
  int32_t* free_list;  // [cap] page of each rank
  int32_t* rank_pair;  // [cap] pair of each rank
  int32_t* snap;       // [n, width] the source rows' pages before the update
  int64_t cap;
};

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ int64_t keep_at(const void* keep, int keep64, int64_t off) {
  return keep64 ? static_cast<const int64_t*>(keep)[off] : static_cast<const int32_t*>(keep)[off];
}

// Sum over the block of one value per thread; every thread gets it. `tmp` holds 33 words.
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* tmp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) tmp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int64_t s = lane < static_cast<int>(blockDim.x >> 5) ? tmp[lane] : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) tmp[32] = s;
  }
  __syncthreads();
  return tmp[32];
}

// Exclusive prefix sum over the block; *total gets the sum.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* tmp, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();
  if (lane == 31) tmp[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int64_t w = lane < static_cast<int>(blockDim.x >> 5) ? tmp[lane] : 0;
    const int64_t own = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    tmp[lane] = w - own;
    if (lane == 31) tmp[32] = w;
  }
  __syncthreads();
  *total = tmp[32];
  return tmp[warp] + inc - v;
}

// One cluster (1 or 8 CTAs) makes the whole update: the work is a few passes over small
// integer arrays (keep list, use counts, table rows), bound by the latency of its dependent
// passes, so the passes are separated by cluster barriers instead of launches.
__global__ void __launch_bounds__(kUpdateThreads, 1) update_kernel(const UpdateParams p) {
  extern __shared__ int32_t sh[];
  __shared__ int64_t tmp[33];
  __shared__ int32_t s_err;
  grid_launch_dependents();
  const cab_page_cache& c = p.c;
  const int n = p.n, tid = threadIdx.x, nt = kUpdateThreads;
  const int me = static_cast<int>(cluster_rank()), nc = static_cast<int>(cluster_size());
  const int64_t S = c.page_size, W = c.width, P = c.pages;
  int32_t *s_src = sh, *s_dst = sh + n, *s_len = sh + 2 * n, *s_start = sh + 3 * n, *s_content = sh + 4 * n,
          *s_size = sh + 5 * n, *s_first = sh + 6 * n, *s_stay = sh + 7 * n, *s_base = sh + 8 * n, *s_gone = sh + 9 * n;
  const int words = static_cast<int>((c.rows + 31) / 32);
  uint32_t* b_dst = reinterpret_cast<uint32_t*>(sh + 10 * n);
  uint32_t *b_src = b_dst + words, *b_multi = b_src + words;
  const int pstride = n + 3;
  const bool frozen = *reinterpret_cast<volatile int32_t*>(c.status) != 0;

  for (int i = tid; i < 3 * words; i += nt) b_dst[i] = 0u;
  if (tid == 0) s_err = 0;
  __syncthreads();
  // pass 0: the pairs and their checks (every CTA of the cluster does the same)
  for (int i = tid; i < n; i += nt) {
    const int s = p.src ? p.src[i] : i, d = p.dst ? p.dst[i] : s;
    int err = 0;
    int64_t len = 0, start = 0, kn = 0, size = 0, gone = 0;
    if (s < 0 || s >= c.rows || d < 0 || d >= c.rows) {
      err = CAB_PAGES_BAD_ROW;
    } else {
      len = c.seq_lens[s];
      gone = c.seq_lens[d];
      start = p.start ? p.start[i] : (p.start_value < 0 ? len : p.start_value);
      kn = p.keep_num ? p.keep_num[i * p.keep_num_stride] : p.keep_cols;
      const int64_t grow = p.grow ? p.grow[i] : p.grow_value;
      if (len < 0 || len > W * S || gone < 0 || gone > W * S) err |= CAB_PAGES_BAD_TABLE;
      else if (start < 0 || start > len || kn < 0 || kn > p.keep_cols || grow < 0) err |= CAB_PAGES_BAD_ARG;
      else if (start + kn + grow > W * S) err |= CAB_PAGES_TABLE_FULL;
      size = start + kn + grow;
      if (atomicOr(&b_dst[d >> 5], 1u << (d & 31)) >> (d & 31) & 1u) err |= CAB_PAGES_BAD_ROW;
      if (atomicOr(&b_src[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) atomicOr(&b_multi[s >> 5], 1u << (s & 31));
    }
    if (err) atomicOr(&s_err, err);
    s_src[i] = s;
    s_dst[i] = d;
    s_len[i] = static_cast<int32_t>(len);
    s_start[i] = static_cast<int32_t>(start);
    s_content[i] = static_cast<int32_t>(start + kn);
    s_size[i] = static_cast<int32_t>(size);
    s_gone[i] = static_cast<int32_t>(gone);
    s_first[i] = static_cast<int32_t>(kn);
  }
  __syncthreads();
  const int err0 = s_err;
  if (frozen || err0) {  // the same in every CTA: nobody waits for the others
    if (me == 0 && tid == 0) {
      p.header[0] = 0;
      if (err0 && !frozen) atomicOr(c.status, err0);
    }
    return;
  }

  // pass 1: the keep lists (range, and the first entry that moves) and this CTA's free pages
  const int64_t K = p.keep_cols;
  if (K > 0) {
    int bad = 0;
    const int64_t total = K * n;
    for (int64_t e = static_cast<int64_t>(me) * nt + tid; e < total; e += static_cast<int64_t>(nc) * nt) {
      const int i = static_cast<int>(e / K);
      const int64_t x = e - i * K;
      if (x < s_content[i] - s_start[i]) {
        const int64_t v = keep_at(p.keep, p.keep64, i * p.keep_stride + x);
        if (v < 0 || v >= s_len[i] - s_start[i]) bad = 1;
        if (v != x && x < *reinterpret_cast<volatile int32_t*>(&s_first[i])) atomicMin(&s_first[i], static_cast<int32_t>(x));
      }
    }
    if (bad) atomicOr(&s_err, CAB_PAGES_BAD_ARG);
  }
  const int64_t span = (P + nc - 1) / nc;
  const int64_t lo = min(P, span * me), hi = min(P, span * (me + 1));
  int64_t mine = 0;
  for (int64_t q = lo + tid; q < hi; q += nt) mine += c.ref_counts[q] == 0;
  const int64_t free_here = block_sum(mine, tmp);  // its barriers also complete s_first and s_err
  int32_t* part = p.part + static_cast<int64_t>(me) * pstride;
  for (int i = tid; i < n; i += nt) part[i] = s_first[i];
  if (tid == 0) {
    part[n] = static_cast<int32_t>(free_here);
    part[n + 1] = s_err;
    s_err = 0;
  }
  cluster_sync_all();

  // pass 2: what stays, what is fresh (every CTA the same); the free list and the snapshot
  int64_t free_total = 0, free_before = 0;
  int err1 = 0;
  for (int k = 0; k < nc; ++k) {
    const int32_t* q = p.part + static_cast<int64_t>(k) * pstride;
    const int32_t f = __ldcg(q + n);
    if (k < me) free_before += f;
    free_total += f;
    err1 |= __ldcg(q + n + 1);
  }
  int64_t need = 0;
  if (tid < n) {
    const int i = tid;
    int32_t first = s_content[i] - s_start[i];
    for (int k = 0; k < nc; ++k) first = min(first, __ldcg(p.part + static_cast<int64_t>(k) * pstride + i));
    const int64_t intact = static_cast<int64_t>(s_start[i]) + first, held = s_content[i];
    int64_t stay = intact / S;
    const int s = s_src[i];
    if (intact == held && held % S != 0 && s == s_dst[i]) {
      const int32_t tail = c.block_table[s * c.table_stride + held / S];
      const bool alone = tail >= 0 && tail < P && c.ref_counts[tail] == 1 && !(b_multi[s >> 5] >> (s & 31) & 1u);
      if (alone) ++stay;
      else if (!p.copies) atomicOr(&s_err, CAB_PAGES_BAD_TABLE);  // a shared last page and no copy asked for
    }
    s_stay[i] = static_cast<int32_t>(stay);
    need = (static_cast<int64_t>(s_size[i]) + S - 1) / S - stay;
  }
  int64_t total = 0;
  const int64_t base = block_scan(need, tmp, &total);
  if (tid < n) {
    s_base[tid] = static_cast<int32_t>(base);
    if (me == 0) p.pair[tid] = PairRec{s_stay[tid], static_cast<int32_t>(base), s_start[tid], s_content[tid]};
  }
  if (total > free_total) err1 |= CAB_PAGES_FULL;
  if (free_before < total && total <= free_total) {
    int64_t rank0 = free_before;
    for (int64_t q0 = lo; q0 < hi && rank0 < total; q0 += nt) {
      const int64_t q = q0 + tid;
      int64_t got = 0;
      const int64_t is_free = q < hi && c.ref_counts[q] == 0;
      const int64_t r = rank0 + block_scan(is_free, tmp, &got);
      if (is_free && r < total) p.free_list[r] = static_cast<int32_t>(q);
      rank0 += got;
    }
  }
  __syncthreads();
  // Rows are walked in 32-entry chunks by warps of the whole cluster; the same thread later
  // rewrites the entry it has read here.
  const int64_t cpr = (W + 31) / 32, chunks = cpr * n;
  const int lane = tid & 31;
  const int64_t w0 = (static_cast<int64_t>(me) * nt + tid) >> 5, wn = static_cast<int64_t>(nc) * nt / 32;
  for (int64_t ch = w0; ch < chunks; ch += wn) {
    const int i = static_cast<int>(ch / cpr);
    const int64_t j = (ch - i * cpr) * 32 + lane;
    const bool in_place = s_src[i] == s_dst[i];
    const int64_t have = (static_cast<int64_t>(s_len[i]) + S - 1) / S;
    int bad = 0;
    if (j < have && (!in_place || K > 0 || j >= s_stay[i])) {
      const int32_t q = c.block_table[s_src[i] * c.table_stride + j];
      p.snap[static_cast<int64_t>(i) * W + j] = q;
      bad |= q < 0 || q >= P;
    }
    if (!in_place && j < (static_cast<int64_t>(s_gone[i]) + S - 1) / S) {
      const int32_t q = c.block_table[s_dst[i] * c.table_stride + j];
      bad |= q < 0 || q >= P;
    }
    if (bad) atomicOr(&s_err, CAB_PAGES_BAD_TABLE);
  }
  __syncthreads();
  if (tid == 0) part[n + 2] = s_err;
  cluster_sync_all();

  // pass 3: refuse, or apply
  for (int k = 0; k < nc; ++k) err1 |= __ldcg(p.part + static_cast<int64_t>(k) * pstride + n + 2);
  if (err1) {
    if (me == 0 && tid == 0) {
      p.header[0] = 0;
      atomicOr(c.status, err1);
    }
    return;
  }
  if (me == 0 && tid == 0) {
    p.header[0] = 1;
    p.header[1] = static_cast<int32_t>(total);
  }
  for (int64_t ch = w0; ch < chunks; ch += wn) {
    const int i = static_cast<int>(ch / cpr);
    const int64_t j = (ch - i * cpr) * 32 + lane;
    const bool in_place = s_src[i] == s_dst[i];
    const int64_t had = (static_cast<int64_t>(s_gone[i]) + S - 1) / S, now = (static_cast<int64_t>(s_size[i]) + S - 1) / S;
    if (j >= max(had, now) || (in_place && j < s_stay[i])) continue;
    int32_t* entry = c.block_table + s_dst[i] * c.table_stride + j;
    if (j < had) atomicSub(&c.ref_counts[*entry], 1);
    int32_t q = -1;
    if (j < s_stay[i]) {
      q = p.snap[static_cast<int64_t>(i) * W + j];
    } else if (j < now) {
      const int32_t r = s_base[i] + static_cast<int32_t>(j - s_stay[i]);
      q = __ldcg(p.free_list + r);
      p.rank_pair[r] = i;
    }
    if (q >= 0) atomicAdd(&c.ref_counts[q], 1);
    *entry = q;
  }
  if (me == 0)
    for (int i = tid; i < n; i += nt) c.seq_lens[s_dst[i]] = s_size[i];
}

// ------------------------------------------------------------------ token copies
// Moves up to 32 tokens' K and V of one (layer, head) per warp: lane t finds where token t
// comes from and goes to (three dependent small loads for 32 tokens at once), then the warp
// moves the tokens' rows in vectors, kBatch loads of K and of V in flight per lane. Bound by
// HBM: each moved value is read and written once.
struct RowSpan {
  int64_t ksrc, vsrc, kdst, vdst;  // element offsets of a token's row
};

template <typename V>
__device__ __forceinline__ void move_rows(const V* __restrict__ ksrc, const V* __restrict__ vsrc, V* __restrict__ kdst,
                                          V* __restrict__ vdst, const RowSpan& mine, int count, int vecs) {
  constexpr int kBatch = 4;
  const int lane = threadIdx.x & 31;
  const int total = count * vecs;
  for (int e0 = 0; e0 < total; e0 += 32 * kBatch) {
    V rk[kBatch], rv[kBatch];
    int64_t ok[kBatch], ov[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int e = e0 + 32 * u + lane;
      const int t = min(e / vecs, 31), x = e - (e / vecs) * vecs;
      const int64_t a = __shfl_sync(0xffffffffu, mine.ksrc, t), b = __shfl_sync(0xffffffffu, mine.vsrc, t);
      ok[u] = __shfl_sync(0xffffffffu, mine.kdst, t);
      ov[u] = __shfl_sync(0xffffffffu, mine.vdst, t);
      const bool live = e < total && ok[u] >= 0;
      if (live) {
        rk[u] = ksrc[a + x];
        rv[u] = vsrc[b + x];
        ok[u] += x;
        ov[u] += x;
      } else {
        ok[u] = -1;
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (ok[u] >= 0) {
        kdst[ok[u]] = rk[u];
        vdst[ov[u]] = rv[u];
      }
  }
}

template <typename V>
__global__ void __launch_bounds__(256) copy_kernel(const UpdateParams p, int vec_elems, int vecs) {
  grid_dependency_wait();
  if (p.header[0] == 0) return;
  const cab_page_cache& c = p.c;
  const int total = p.header[1];
  const int64_t S = c.page_size, W = c.width;
  const int groups = static_cast<int>((S + 31) / 32);
  const int64_t lh = c.layers * c.heads, tasks = static_cast<int64_t>(total) * groups * lh;
  const int lane = threadIdx.x & 31;
  const int64_t wn = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t task = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); task < tasks; task += wn) {
    const int64_t rg = task / lh;
    const int x = static_cast<int>(task - rg * lh);
    const int l = x / static_cast<int>(c.heads), h = x - l * static_cast<int>(c.heads);
    const int r = static_cast<int>(rg / groups), g = static_cast<int>(rg - static_cast<int64_t>(r) * groups);
    const int i = p.rank_pair[r];
    const PairRec pr = p.pair[i];
    const int64_t pos0 = (static_cast<int64_t>(pr.stay) + r - pr.base) * S + 32 * g;
    const int count = static_cast<int>(min(min(static_cast<int64_t>(32), S - 32 * g), pr.content - pos0));
    if (count <= 0) continue;
    RowSpan m{0, 0, -1, -1};
    if (lane < count) {
      const int64_t pos = pos0 + lane;
      const int64_t from = pos < pr.start ? pos : pr.start + keep_at(p.keep, p.keep64, i * p.keep_stride + pos - pr.start);
      const int64_t pg = p.snap[static_cast<int64_t>(i) * W + from / S], slot = from % S;
      const int64_t to = p.free_list[r], ts = 32 * g + lane;
      const int64_t kb = l * c.k_strides[0] + h * c.k_strides[2], vb = l * c.v_strides[0] + h * c.v_strides[2];
      m.ksrc = (kb + pg * c.k_strides[1] + slot * c.k_strides[3]) / vec_elems;
      m.vsrc = (vb + pg * c.v_strides[1] + slot * c.v_strides[3]) / vec_elems;
      m.kdst = (kb + to * c.k_strides[1] + ts * c.k_strides[3]) / vec_elems;
      m.vdst = (vb + to * c.v_strides[1] + ts * c.v_strides[3]) / vec_elems;
    }
    move_rows<V>(static_cast<const V*>(c.k_pages), static_cast<const V*>(c.v_pages), static_cast<V*>(c.k_pages),
                 static_cast<V*>(c.v_pages), m, count, vecs);
  }
}

struct WriteParams {
  cab_page_cache c;
  const void *k, *v;
  int64_t ks[3], vs[3];
  const int32_t *rows, *num_new;
  int64_t layer, T, num_value;
  int32_t n;
};

template <typename V>
__global__ void __launch_bounds__(256) write_kernel(const WriteParams p, int vec_elems, int vecs) {
  const cab_page_cache& c = p.c;
  if (*reinterpret_cast<volatile int32_t*>(c.status) != 0) return;
  const int64_t S = c.page_size;
  const int64_t groups = (p.T + 31) / 32, tasks = groups * c.heads * p.n;
  const int lane = threadIdx.x & 31;
  const int64_t wn = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t task = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); task < tasks; task += wn) {
    const int64_t ih = task / groups, g = task - ih * groups;
    const int i = static_cast<int>(ih / c.heads), h = static_cast<int>(ih - i * c.heads);
    const int row = p.rows ? p.rows[i] : i;
    int err = 0;
    int64_t len = 0, m = 0;
    if (row < 0 || row >= c.rows) {
      err = CAB_PAGES_BAD_ROW;
    } else {
      bool twice = false;  // a row named before writes nothing again: two writers would race
      if (p.rows)
        for (int k = lane; k < i; k += 32) twice |= p.rows[k] == row;
      if (__any_sync(0xffffffffu, twice)) err = CAB_PAGES_BAD_ROW;
      len = c.seq_lens[row];
      m = p.num_new ? p.num_new[i] : p.num_value;
      if (m < 0 || m > p.T || m > len || len > c.width * S) err |= CAB_PAGES_BAD_ARG;
    }
    const int64_t t = 32 * g + lane;
    RowSpan s{0, 0, -1, -1};
    if (!err && t < m) {
      const int64_t pos = len - m + t, slot = pos % S;
      const int64_t pg = c.block_table[row * c.table_stride + pos / S];
      if (pg < 0 || pg >= c.pages) {
        err = CAB_PAGES_BAD_TABLE;
      } else {
        s.ksrc = (i * p.ks[0] + h * p.ks[1] + t * p.ks[2]) / vec_elems;
        s.vsrc = (i * p.vs[0] + h * p.vs[1] + t * p.vs[2]) / vec_elems;
        s.kdst = (p.layer * c.k_strides[0] + pg * c.k_strides[1] + h * c.k_strides[2] + slot * c.k_strides[3]) / vec_elems;
        s.vdst = (p.layer * c.v_strides[0] + pg * c.v_strides[1] + h * c.v_strides[2] + slot * c.v_strides[3]) / vec_elems;
      }
    }
    if (err) atomicOr(c.status, err);
    const int count = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(32), m - 32 * g)));
    move_rows<V>(static_cast<const V*>(p.k), static_cast<const V*>(p.v), static_cast<V*>(c.k_pages),
                 static_cast<V*>(c.v_pages), s, count, vecs);
  }
}

// ------------------------------------------------------------------ host side
inline int check_cache(const cab_page_cache* c, const char* what, bool data, bool state = true) {
  if (!c) return fail(CAB_ERR_INVALID_ARG, "%s: NULL cache", what);
  if (!c->block_table || !c->seq_lens || (state && (!c->ref_counts || !c->status)))
    return fail(CAB_ERR_INVALID_ARG, "%s: NULL pointer in the cache", what);
  if (c->layers <= 0 || c->pages <= 0 || c->heads <= 0 || c->page_size <= 0 || c->dim <= 0 || c->rows <= 0 || c->width <= 0)
    return fail(CAB_ERR_INVALID_ARG, "%s: non-positive size in the cache", what);
  if (c->pages >= (int64_t)1 << 31 || c->rows > kMaxRows || c->width * c->page_size >= (int64_t)1 << 31 ||
      c->layers * c->heads >= (int64_t)1 << 31)
    return fail(CAB_ERR_UNSUPPORTED, "%s: cache too large (at most 2^31 - 1 pages, 65536 rows, 2^31 - 1 tokens a row)", what);
  if (c->table_stride < c->width && c->rows > 1) return fail(CAB_ERR_INVALID_ARG, "%s: table rows overlap", what);
  if (data) {
    if (!c->k_pages || !c->v_pages) return fail(CAB_ERR_INVALID_ARG, "%s: NULL pages", what);
    if (dtype_size(static_cast<int>(c->dtype)) == 0) return fail(CAB_ERR_UNSUPPORTED, "%s: unknown dtype %d", what, static_cast<int>(c->dtype));
    for (int i = 0; i < 4; ++i)
      if (c->k_strides[i] <= 0 || c->v_strides[i] <= 0) return fail(CAB_ERR_INVALID_ARG, "%s: page strides must be positive", what);
  }
  return CAB_OK;
}

// The widest of 16, 4 and 2 bytes that every row start and the row length allow.
inline int vector_bytes(const cab_page_cache* c, const void* k, const void* v, const int64_t* ks, const int64_t* vs) {
  const int64_t es = static_cast<int64_t>(dtype_size(static_cast<int>(c->dtype)));
  for (int vb : {16, 4}) {
    bool fits = (c->dim * es) % vb == 0;
    for (const void* q : {static_cast<const void*>(c->k_pages), static_cast<const void*>(c->v_pages), k, v})
      fits = fits && reinterpret_cast<uintptr_t>(q) % vb == 0;
    for (int i = 0; i < 4; ++i) fits = fits && (c->k_strides[i] * es) % vb == 0 && (c->v_strides[i] * es) % vb == 0;
    for (int i = 0; i < 3 && ks; ++i) fits = fits && (ks[i] * es) % vb == 0 && (vs[i] * es) % vb == 0;
    if (fits) return vb;
  }
  return 2;
}

struct UpdateLayout {
  size_t part, pair, free_list, rank_pair, snap, total;
  int64_t cap;
};

inline UpdateLayout update_layout(const cab_page_cache* c, int64_t n) {
  auto up = [](size_t x) { return (x + 15) & ~size_t(15); };
  UpdateLayout L{};
  L.cap = std::min(c->pages, n * c->width);
  L.part = 16;
  L.pair = up(L.part + static_cast<size_t>(kMaxCluster) * (n + 3) * 4);
  L.free_list = up(L.pair + static_cast<size_t>(n) * sizeof(PairRec));
  L.rank_pair = up(L.free_list + static_cast<size_t>(L.cap) * 4);
  L.snap = up(L.rank_pair + static_cast<size_t>(L.cap) * 4);
  L.total = up(L.snap + static_cast<size_t>(n) * c->width * 4);
  return L;
}

}  // namespace pages
}  // namespace cab

extern "C" int cab_pages_update_workspace_size(const cab_page_cache* cache, int64_t n, size_t* bytes) {
  using namespace cab;
  using namespace cab::pages;
  if (!bytes) return fail(CAB_ERR_INVALID_ARG, "pages_update_workspace_size: NULL output");
  if (int rc = check_cache(cache, "pages_update_workspace_size", false)) return rc;
  if (n <= 0 || n > kMaxPairs) return fail(CAB_ERR_UNSUPPORTED, "pages_update: 1 to %d pairs a call, got %lld", kMaxPairs, (long long)n);
  *bytes = update_layout(cache, n).total;
  return CAB_OK;
}

extern "C" int cab_pages_update(const cab_page_cache* cache, const int32_t* src, const int32_t* dst, int64_t n,
                                const int32_t* start, int64_t start_value, const void* keep, int keep_bytes,
                                int64_t keep_stride, int64_t keep_cols, const int32_t* keep_num,
                                int64_t keep_num_stride, const int32_t* grow, int64_t grow_value, int copies,
                                void* workspace, size_t workspace_bytes, void* stream) {
  using namespace cab;
  using namespace cab::pages;
  if (int rc = check_cache(cache, "pages_update", copies != 0)) return rc;
  if (n <= 0 || n > kMaxPairs) return fail(CAB_ERR_UNSUPPORTED, "pages_update: 1 to %d pairs a call, got %lld", kMaxPairs, (long long)n);
  if (!src && n > cache->rows) return fail(CAB_ERR_INVALID_ARG, "pages_update: %lld pairs without source rows, %lld rows", (long long)n, (long long)cache->rows);
  if (keep_cols < 0 || keep_cols >= (int64_t)1 << 31) return fail(CAB_ERR_INVALID_ARG, "pages_update: bad number of keep columns");
  if (keep_cols > 0 && (!keep || (keep_bytes != 4 && keep_bytes != 8))) return fail(CAB_ERR_INVALID_ARG, "pages_update: keep must be int32 or int64");
  if (keep_cols > 0 && !copies) return fail(CAB_ERR_INVALID_ARG, "pages_update: a keep list needs copies");
  if (grow_value < 0) return fail(CAB_ERR_INVALID_ARG, "pages_update: negative growth");
  const UpdateLayout L = update_layout(cache, n);
  if (!workspace || workspace_bytes < L.total)
    return fail(CAB_ERR_WORKSPACE, "pages_update: workspace of %zu bytes needed, %zu given", L.total, workspace_bytes);
  if (!aligned16(workspace)) return fail(CAB_ERR_INVALID_ARG, "pages_update: workspace must be 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  UpdateParams p{};
  p.c = *cache;
  p.src = src;
  p.dst = dst;
  p.start = start;
  p.start_value = start_value;
  p.keep = keep;
  p.keep64 = keep_bytes == 8;
  p.keep_stride = keep_stride;
  p.keep_cols = keep_cols;
  p.keep_num = keep_cols > 0 ? keep_num : nullptr;
  p.keep_num_stride = keep_num_stride;
  p.grow = grow;
  p.grow_value = grow_value;
  p.n = static_cast<int32_t>(n);
  p.copies = copies != 0;
  p.header = reinterpret_cast<int32_t*>(ws);
  p.part = reinterpret_cast<int32_t*>(ws + L.part);
  p.pair = reinterpret_cast<PairRec*>(ws + L.pair);
  p.free_list = reinterpret_cast<int32_t*>(ws + L.free_list);
  p.rank_pair = reinterpret_cast<int32_t*>(ws + L.rank_pair);
  p.snap = reinterpret_cast<int32_t*>(ws + L.snap);
  p.cap = L.cap;

  const int64_t words = (cache->rows + 31) / 32;
  const size_t smem = static_cast<size_t>(10 * n + 3 * words) * 4;
  if (smem > 40 * 1024)
    cudaFuncSetAttribute(update_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  const int64_t ints = cache->pages + n * (cache->width + keep_cols);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(ints > 16384 ? kMaxCluster : 1);
  cfg.blockDim = dim3(kUpdateThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cfg.gridDim.x;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, update_kernel, p);
  if (int rc = check_launch("pages update_kernel")) return rc;
  if (!copies) return CAB_OK;

  const int vb = vector_bytes(cache, nullptr, nullptr, nullptr, nullptr);
  const int es = static_cast<int>(dtype_size(static_cast<int>(cache->dtype)));
  const int vecs = static_cast<int>(cache->dim * es / vb), ve = vb >= es ? vb / es : 1;
  // at most keep_cols + page_size tokens of a pair move, or one page where nothing is listed
  const int64_t per = keep_cols > 0 ? (keep_cols + cache->page_size - 1) / cache->page_size + 1 : cache->width;
  const int64_t most = std::min(L.cap, n * std::min(per, cache->width)) * ((cache->page_size + 31) / 32) * cache->layers * cache->heads;
  cudaLaunchConfig_t cc{};
  cudaLaunchAttribute ca[1];
  cc.gridDim = dim3(static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((most + 7) / 8, (int64_t)current_sm_count() * 8))));
  cc.blockDim = dim3(256);
  cc.stream = static_cast<cudaStream_t>(stream);
  ca[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  ca[0].val.programmaticStreamSerializationAllowed = 1;
  cc.attrs = ca;
  cc.numAttrs = 1;
  if (vb == 16) cudaLaunchKernelEx(&cc, copy_kernel<uint4>, p, ve, vecs);
  else if (vb == 4) cudaLaunchKernelEx(&cc, copy_kernel<uint32_t>, p, ve, vecs);
  else cudaLaunchKernelEx(&cc, copy_kernel<uint16_t>, p, ve, vecs);
  return check_launch("pages copy_kernel");
}

extern "C" int cab_pages_write(const cab_page_cache* cache, int64_t layer, const void* k, const void* v, int64_t n,
                               int64_t T, const int64_t* k_strides, const int64_t* v_strides, const int32_t* rows,
                               const int32_t* num_new, int64_t num_value, void* stream) {
  using namespace cab;
  using namespace cab::pages;
  if (int rc = check_cache(cache, "pages_write", true)) return rc;
  if (!k || !v || !k_strides || !v_strides) return fail(CAB_ERR_INVALID_ARG, "pages_write: NULL pointer");
  if (layer < 0 || layer >= cache->layers) return fail(CAB_ERR_INVALID_ARG, "pages_write: layer %lld of %lld", (long long)layer, (long long)cache->layers);
  if (n <= 0 || T <= 0 || T >= (int64_t)1 << 31) return fail(CAB_ERR_INVALID_ARG, "pages_write: non-positive size");
  if (n > kMaxRows) return fail(CAB_ERR_UNSUPPORTED, "pages_write: at most 65536 rows a call");
  if (!rows && n > cache->rows) return fail(CAB_ERR_INVALID_ARG, "pages_write: more sequences than rows");
  if (num_value < 0 || num_value > T) return fail(CAB_ERR_INVALID_ARG, "pages_write: num_new outside [0, T]");
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] < 0 || v_strides[i] < 0) return fail(CAB_ERR_INVALID_ARG, "pages_write: negative stride");
  WriteParams p{};
  p.c = *cache;
  p.k = k;
  p.v = v;
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
  }
  p.rows = rows;
  p.num_new = num_new;
  p.layer = layer;
  p.T = T;
  p.num_value = num_value;
  p.n = static_cast<int32_t>(n);
  const int vb = vector_bytes(cache, k, v, k_strides, v_strides);
  const int es = static_cast<int>(dtype_size(static_cast<int>(cache->dtype)));
  const int vecs = static_cast<int>(cache->dim * es / vb), ve = vb >= es ? vb / es : 1;
  const int64_t tasks = (T + 31) / 32 * cache->heads * n;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((tasks + 7) / 8, (int64_t)current_sm_count() * 8));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (vb == 16) write_kernel<uint4><<<grid, 256, 0, st>>>(p, ve, vecs);
  else if (vb == 4) write_kernel<uint32_t><<<grid, 256, 0, st>>>(p, ve, vecs);
  else write_kernel<uint16_t><<<grid, 256, 0, st>>>(p, ve, vecs);
  return check_launch("pages write_kernel");
}
