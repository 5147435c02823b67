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
// Updates and writes are all or nothing: every check is made before the first store, a refused
// call changes nothing but the status word, and while the status word is set later calls do
// nothing either.

#include "cab_host.h"
#include "cab_ptx.cuh"

#include <algorithm>
#include <atomic>

namespace cab {
namespace pages {

constexpr int kUpdateThreads = 1024;
constexpr int kMaxPairs = 1024;     // one pair per thread of the prefix sum
constexpr int64_t kMaxRows = 65536;  // three bitmaps of the rows in shared memory
constexpr int kMaxCluster = 8;
constexpr int kFrozen = 1 << 30;     // among the passes: the status word was set before

// A fresh page: what the copies into it need.
struct alignas(16) FreshPage {
  int32_t pair, page;       // pair i and the page's number
  int32_t first, content;   // its first position in the row, and the row's tokens
  int32_t start, pad[3];    // a
};

struct UpdateParams {
  cab_page_cache c;
  const int32_t *src, *dst, *start, *keep_num, *grow;
  const void* keep;
  int64_t start_value, grow_value, keep_stride, keep_cols, keep_num_stride;
  int32_t keep64, n, copies;
  uint32_t div_mul, div_shift;  // x / page_size = x * div_mul >> div_shift for x < 2^31
  int32_t* header;      // [0] accepted, [1] fresh pages
  FreshPage* fresh;     // [cap] by rank in the order of taking
  int32_t* free_list;   // [cap] page of each rank
  int32_t* snap;        // [n, width] the source rows' pages before the update
  int64_t cap;
};

// A barrier over the cluster's CTAs (one CTA needs only its own).
__device__ __forceinline__ void cluster_sync(int nc) {
  if (nc == 1) {
    __syncthreads();
    return;
  }
  __syncwarp();  // the aligned form wants the whole warp
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The shared-memory word `p` of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_word(const void* p, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void peer_store(uint32_t a, int32_t v) { asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ int32_t peer_load(uint32_t a) {
  int32_t v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
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

// x / page_size by a multiplication: a hardware-free 32-bit division costs some 150 clocks each time.
__device__ __forceinline__ uint32_t pages_before(const UpdateParams& p, uint32_t x) {
  return static_cast<uint32_t>(static_cast<uint64_t>(x) * p.div_mul >> p.div_shift);
}

__device__ __forceinline__ int64_t keep_at(const void* keep, int keep64, int64_t off) {
  return keep64 ? static_cast<const int64_t*>(keep)[off] : static_cast<const int32_t*>(keep)[off];
}

// Exclusive prefix sum over the first n threads' values (0 beyond); *total gets the sum.
__device__ __forceinline__ int64_t block_scan(int64_t v, int n, int64_t* tmp, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (n <= 32) {  // all in warp 0
    if (threadIdx.x == 31) tmp[32] = inc;
    __syncthreads();
    *total = tmp[32];
    return inc - v;
  }
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

// One cluster (1 or 8 CTAs) makes the whole update. The work is a few passes over small integer
// arrays (use counts, keep lists, table rows), bound by the latency of dependent loads, so the
// passes are separated by cluster barriers instead of launches, what the CTAs tell one another goes through
// distributed shared memory, and each pass has its loads in flight together. About 12,000 clocks with few
// rows, 20,000 with 32 rows of 500 pages; the code runs once a launch, so its size costs as much as its
// loads (unrolling the entry rounds four times instead of two: 20.5 instead of 17.8 us for a fork of 32
// beams with its copies), and one CTA of 1024 threads for everything took twice as long on 32 rows.
constexpr int kWordRounds = 2;  // ballot words of free pages a lane of a warp holds at a time

__global__ void __launch_bounds__(kUpdateThreads, 1) update_kernel(const __grid_constant__ UpdateParams p) {
  extern __shared__ int32_t sh[];
  __shared__ int64_t tmp[33];
  __shared__ int32_t s_err, s_told[2], s_free[kMaxCluster], s_errs[kMaxCluster], s_late[kMaxCluster], s_warp_free[32];
  const cab_page_cache& c = p.c;
  const int n = p.n, tid = threadIdx.x, nt = kUpdateThreads, lane = tid & 31, warp = tid >> 5;
  const int me = static_cast<int>(cluster_rank()), nc = static_cast<int>(cluster_size());
  const int64_t W = c.width, P = c.pages, K = p.keep_cols;
  const uint32_t S = static_cast<uint32_t>(c.page_size);  // lengths and W * S are below 2^31
  int32_t *s_src = sh, *s_dst = sh + n, *s_have = sh + 2 * n, *s_had = sh + 3 * n, *s_start = sh + 4 * n,
          *s_content = sh + 5 * n, *s_size = sh + 6 * n, *s_first = sh + 7 * n, *s_stay = sh + 8 * n, *s_base = sh + 9 * n,
          *s_low = sh + 10 * n, *s_room = sh + 11 * n, *s_alone = sh + 12 * n, *s_now = sh + 13 * n, *s_entry = sh + 14 * n;  // s_entry has n + 1
  const int words = static_cast<int>((c.rows + 31) / 32);
  uint32_t* b_dst = reinterpret_cast<uint32_t*>(sh + 15 * n + 1);
  uint32_t *b_src = b_dst + words, *b_multi = b_src + words;
  grid_launch_dependents();
  grid_dependency_wait();  // the kernel before may have written the state or this call's lists

  // pass 0: the pairs and their checks (the same in every CTA)
  int err = *reinterpret_cast<volatile int32_t*>(c.status) != 0 ? kFrozen : 0;
  for (int i = tid; i < 3 * words; i += nt) b_dst[i] = 0u;
  if (tid == 0) s_err = 0;
  __syncthreads();
  for (int i = tid; i < n; i += nt) {
    const int s = p.src ? p.src[i] : i, d = p.dst ? p.dst[i] : s;
    const int64_t start_i = p.start ? p.start[i] : p.start_value, keep_i = p.keep_num ? p.keep_num[i * p.keep_num_stride] : K,
                  grow = p.grow ? p.grow[i] : p.grow_value;
    int64_t len = 0, start = 0, kn = 0, size = 0, gone = 0;
    bool alone = false;
    if (s < 0 || s >= c.rows || d < 0 || d >= c.rows) {
      err |= CAB_PAGES_BAD_ROW;
    } else {
      len = c.seq_lens[s];
      gone = c.seq_lens[d];
      start = !p.start && start_i < 0 ? len : start_i;
      kn = keep_i;
      int bad = 0;
      if (len < 0 || len > W * S || gone < 0 || gone > W * S) bad = CAB_PAGES_BAD_TABLE;
      else if (start < 0 || start > len || kn < 0 || kn > K || grow < 0) bad = CAB_PAGES_BAD_ARG;
      else if (start + kn + grow > W * S) bad = CAB_PAGES_TABLE_FULL;
      size = start + kn + grow;
      if (atomicOr(&b_dst[d >> 5], 1u << (d & 31)) >> (d & 31) & 1u) bad |= CAB_PAGES_BAD_ROW;
      if (atomicOr(&b_src[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) atomicOr(&b_multi[s >> 5], 1u << (s & 31));
      if (bad) {
        err |= bad;
        len = start = kn = size = gone = 0;
      } else if (const uint32_t held = static_cast<uint32_t>(start + kn), full = pages_before(p, held); s == d && full * S != held) {
        // in place with a partly filled last page: whether it is this row's alone
        const int32_t tail = c.block_table[s * c.table_stride + full];
        alone = tail >= 0 && tail < P && c.ref_counts[tail] == 1;
      }
    }
    s_alone[i] = alone;
    s_src[i] = s;
    s_dst[i] = d;
    s_have[i] = static_cast<int32_t>(pages_before(p, static_cast<uint32_t>(len) + S - 1));
    s_had[i] = static_cast<int32_t>(pages_before(p, static_cast<uint32_t>(gone) + S - 1));
    s_start[i] = static_cast<int32_t>(start);
    s_content[i] = static_cast<int32_t>(start + kn);
    s_size[i] = static_cast<int32_t>(size);
    s_first[i] = static_cast<int32_t>(kn);
    s_room[i] = static_cast<int32_t>(len - start);
  }
  if (err) atomicOr(&s_err, err);

  // pass 1: this CTA's free pages: warp w's are lane k's ballot words, `rounds` at a time
  const int64_t span = ((P + nc - 1) / nc + 31) / 32 * 32, lo = min(P, span * me), hi = min(P, lo + span);
  const int64_t wspan = (span / 32 + 31) / 32 * 32;  // pages of a warp
  const int64_t wlo = min(hi, lo + wspan * warp), whi = min(hi, wlo + wspan);
  uint32_t held_words = 0u;  // lane k: ballot of the warp's pages 32 k .. 32 k + 31 (the first 1024)
  int warp_free = 0;
  for (int64_t q0 = wlo; q0 < whi; q0 += 32 * kWordRounds) {
    int32_t refs[kWordRounds];
#pragma unroll
    for (int u = 0; u < kWordRounds; ++u) {
      const int64_t q = q0 + 32 * u + lane;
      refs[u] = q < whi ? c.ref_counts[q] : 1;
    }
#pragma unroll
    for (int u = 0; u < kWordRounds; ++u) {
      const uint32_t word = __ballot_sync(0xffffffffu, refs[u] == 0);
      if ((q0 - wlo) / 32 + u == lane) held_words = word;
      warp_free += __popc(word);
    }
  }
  if (lane == 0) s_warp_free[warp] = warp_free;
  __syncthreads();  // the pairs and the warps' counts are there
  // the keep lists: range, and the first entry that moves
  if (K > 0) {
    bool bad = false;
    const uint32_t cols = static_cast<uint32_t>(K), listed = cols * n;  // below 2^31
    for (uint32_t e = me * nt + tid; e < listed; e += nc * nt) {
      const int i = static_cast<int>(e / cols), x = static_cast<int>(e - i * cols);
      if (x < s_content[i] - s_start[i]) {
        const int64_t v = keep_at(p.keep, p.keep64, i * p.keep_stride + x);
        bad |= v < 0 || v >= s_room[i];
        if (v != x && x < *reinterpret_cast<volatile int32_t*>(&s_first[i])) atomicMin(&s_first[i], x);
      }
    }
    if (bad) atomicOr(&s_err, CAB_PAGES_BAD_ARG);
    __syncthreads();
  }
  if (warp == 0) {
    int f = s_warp_free[lane];
#pragma unroll
    for (int o = 16; o; o >>= 1) f += __shfl_xor_sync(0xffffffffu, f, o);
    if (lane == 0) {
      s_told[0] = f;
      s_told[1] = s_err;
    }
  }
  cluster_sync(nc);
  if (tid < nc) {
    s_free[tid] = peer_load(peer_word(&s_told[0], tid));
    s_errs[tid] = peer_load(peer_word(&s_told[1], tid));
  }
  int first = tid < n ? s_first[tid] : 0;
  if (K > 0 && tid < n)
    for (int k = 1; k < nc; ++k) first = min(first, peer_load(peer_word(&s_first[tid], (me + k) % nc)));
  __syncthreads();

  // pass 2: what stays, what is fresh (the same in every CTA); the source rows before the update
  int64_t free_total = 0, free_before = 0;
  err = 0;
  for (int k = 0; k < nc; ++k) {
    if (k < me) free_before += s_free[k];
    free_total += s_free[k];
    err |= s_errs[k];
  }
  if (err) {  // the same in every CTA; a peer may still read this one's words
    cluster_sync(nc);
    if (me == 0 && tid == 0) {
      p.header[0] = 0;
      if (!(err & kFrozen)) atomicOr(c.status, err);
    }
    return;
  }
  if (tid == 0) s_err = 0;
  int64_t need = 0, entries = 0;
  bool shared_tail = false;
  if (tid < n) {
    const int i = tid, s = s_src[i];
    const bool in_place = s == s_dst[i];
    const uint32_t held = s_content[i], intact = s_start[i] + first;
    int stay = static_cast<int>(pages_before(p, intact));
    if (intact == held && stay * S != held && in_place) {
      if (s_alone[i] && !(b_multi[s >> 5] >> (s & 31) & 1u)) ++stay;
      else shared_tail = !p.copies;  // a last page in use elsewhere and no copy asked for
    }
    const int now = static_cast<int>(pages_before(p, static_cast<uint32_t>(s_size[i]) + S - 1));
    s_now[i] = now;
    s_stay[i] = stay;
    need = now - stay;
    // entries [low, high) of the rows are looked at: all of the source's where copies or shares need them
    const bool all = !in_place || K > 0;
    const int low = all ? 0 : stay, high = max(max(s_had[i], now), all ? s_have[i] : 0);
    s_low[i] = low;
    entries = max(0, high - low);
  }
  int64_t sums = 0;
  const int64_t at = block_scan(need << 32 | entries, n, tmp, &sums);  // both sums are below 2^31
  const int64_t total = sums >> 32, all_entries = sums & 0x7fffffff;
  if (tid < n) {
    s_base[tid] = static_cast<int32_t>(at >> 32);
    s_entry[tid] = static_cast<int32_t>(at & 0x7fffffff);
  }
  if (tid == 0) s_entry[n] = static_cast<int32_t>(all_entries);
  if (shared_tail) atomicOr(&s_err, CAB_PAGES_BAD_TABLE);
  __syncthreads();
  if (total > free_total) {
    err = CAB_PAGES_FULL;
  } else if (free_before < total) {
    int64_t rank = free_before;
    for (int k = 0; k < warp; ++k) rank += s_warp_free[k];
    for (int64_t q0 = wlo; q0 < whi && rank < total; q0 += 32) {
      const int k = static_cast<int>((q0 - wlo) / 32);
      const uint32_t word = k < 32 ? __shfl_sync(0xffffffffu, held_words, k)
                                   : __ballot_sync(0xffffffffu, q0 + lane < whi && c.ref_counts[q0 + lane] == 0);
      const int64_t r = rank + __popc(word & ((1u << lane) - 1u));
      if (word >> lane & 1u && r < total) p.free_list[r] = static_cast<int32_t>(q0 + lane);
      rank += __popc(word);
    }
  }
  // The entries of all rows, spread over the cluster's threads, kRound of a thread's loads in flight. What a
  // thread has read of its last round (its only one, up to kRound * 8192 entries) it keeps for pass 3.
  constexpr int kRound = 2;
  const int64_t first_entry = static_cast<int64_t>(me) * nt + tid, step = static_cast<int64_t>(nc) * nt;
  const bool one_round = all_entries <= step * kRound;
  int pair[kRound], col[kRound], from[kRound], gone[kRound];
  auto place = [&](int64_t e, int& i, int& j) {  // the pair whose entries hold e, and the column
    int a = 0, b = n;
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (s_entry[m] <= e) a = m;
      else b = m;
    }
    i = e < all_entries ? a : -1;
    j = s_low[a] + static_cast<int>(e) - s_entry[a];
  };
  bool bad = false;
  for (int64_t e0 = first_entry; e0 < all_entries; e0 += step * kRound) {
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      place(e0 + step * u, pair[u], col[u]);
      const int i = pair[u], j = col[u];
      from[u] = gone[u] = 0;
      if (i >= 0) {
        if (j < s_have[i]) from[u] = c.block_table[s_src[i] * c.table_stride + j];
        if (j < s_had[i]) gone[u] = c.block_table[s_dst[i] * c.table_stride + j];
      }
    }
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      if (pair[u] >= 0 && p.copies && col[u] < s_have[pair[u]]) p.snap[static_cast<int64_t>(pair[u]) * W + col[u]] = from[u];
      bad |= from[u] < 0 || from[u] >= P || gone[u] < 0 || gone[u] >= P;
    }
  }
  if (bad) atomicOr(&s_err, CAB_PAGES_BAD_TABLE);
  __syncthreads();
  if (tid < nc) peer_store(peer_word(&s_late[me], tid), s_err | err);
  cluster_sync(nc);

  // pass 3: refuse, or apply
  err = 0;
  for (int k = 0; k < nc; ++k) err |= s_late[k];
  if (err) {
    if (me == 0 && tid == 0) {
      p.header[0] = 0;
      atomicOr(c.status, err);
    }
    return;
  }
  if (me == 0 && tid == 0) {
    p.header[0] = 1;
    p.header[1] = static_cast<int32_t>(total);
  }
  for (int64_t e0 = first_entry; e0 < all_entries; e0 += step * kRound) {
    int32_t page[kRound];
    bool write[kRound];
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      if (!one_round) place(e0 + step * u, pair[u], col[u]);
      const int i = pair[u], j = col[u];
      page[u] = -1;
      write[u] = false;
      if (i >= 0) {
        const int now = s_now[i];
        write[u] = j < max(s_had[i], now) && !(s_src[i] == s_dst[i] && j < s_stay[i]);
        if (!one_round && write[u]) {
          if (j < s_had[i]) gone[u] = c.block_table[s_dst[i] * c.table_stride + j];
          if (j < s_stay[i]) from[u] = p.snap[static_cast<int64_t>(i) * W + j];
        }
        if (write[u] && j < s_stay[i]) page[u] = from[u];
        else if (write[u] && j < now) page[u] = __ldcg(p.free_list + s_base[i] + j - s_stay[i]);
      }
    }
#pragma unroll
    for (int u = 0; u < kRound; ++u)
      if (write[u]) {
        const int i = pair[u], j = col[u];
        // in range unless another stream changes the table during the call, where this is read a second time
        if (j < s_had[i] && gone[u] >= 0 && gone[u] < P) atomicSub(&c.ref_counts[gone[u]], 1);
        if (page[u] >= 0) atomicAdd(&c.ref_counts[page[u]], 1);
        c.block_table[s_dst[i] * c.table_stride + j] = page[u];
        if (p.copies && page[u] >= 0 && j >= s_stay[i]) {
          int4* f = reinterpret_cast<int4*>(p.fresh + s_base[i] + j - s_stay[i]);
          f[0] = make_int4(i, page[u], static_cast<int>(j * S), s_content[i]);
          f[1] = make_int4(s_start[i], 0, 0, 0);
        }
      }
  }
  if (me == 0)
    for (int i = tid; i < n; i += nt) c.seq_lens[s_dst[i]] = s_size[i];
}

// ------------------------------------------------------------------ token copies
// Moves up to 32 tokens' K and V of one (layer, head) per warp: lane t finds where token t
// comes from and goes to (three dependent small loads for 32 tokens at once), then the warp
// moves the tokens' rows in vectors, kBatch loads of K and of V in flight per lane. Bound by
// HBM: each moved value is read and written once. 2 x 6400 tokens of 8 heads of 128 kept out of 128,000:
// 105 MB in 18 us, 5.8 TB/s; writing 2 x 32,768 tokens: 537 MB in 88 us, 6.1 TB/s (copy rate 6.55), of
// which 3 us are the checks before the first store.
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
__global__ void __launch_bounds__(256) copy_kernel(const __grid_constant__ UpdateParams p, int vec_elems, int vecs) {
  const cab_page_cache& c = p.c;
  const int S = static_cast<int>(c.page_size), groups = (S + 31) / 32;
  const int lh = static_cast<int>(c.layers * c.heads), heads = static_cast<int>(c.heads);
  const int lane = threadIdx.x & 31;
  const int64_t wn = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  int64_t task = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t most = p.cap * groups * lh;
  grid_dependency_wait();
  for (; task < most; task += wn) {
    const int64_t rg = task / lh;
    const int x = static_cast<int>(task - rg * lh), l = x / heads, h = x - l * heads;
    const int r = static_cast<int>(rg / groups), g = static_cast<int>(rg - static_cast<int64_t>(r) * groups);
    const int4 f = *reinterpret_cast<const int4*>(p.fresh + r);  // read along with the header: r is within it
    const int start = p.fresh[r].start;
    if (p.header[0] == 0 || r >= p.header[1]) return;
    const int pos0 = f.z + 32 * g, count = min(min(32, S - 32 * g), f.w - pos0);
    if (count <= 0) continue;
    RowSpan m{0, 0, -1, -1};
    if (lane < count) {
      const int pos = pos0 + lane;
      const int64_t from = pos < start ? pos : start + keep_at(p.keep, p.keep64, f.x * p.keep_stride + pos - start);
      // The list is read once more than it was checked: a stream that changes it meanwhile reaches nothing out of range.
      const int64_t col = from >= 0 && from < c.width * S ? static_cast<int64_t>(static_cast<uint32_t>(from) / S) : -1;
      const int64_t pg = col >= 0 ? p.snap[static_cast<int64_t>(f.x) * c.width + col] : -1, slot = from - col * S;
      const int64_t to = pg >= 0 && pg < c.pages ? f.y : -1, ts = 32 * g + lane;
      const int64_t kb = l * c.k_strides[0] + h * c.k_strides[2], vb = l * c.v_strides[0] + h * c.v_strides[2];
      m.ksrc = (kb + pg * c.k_strides[1] + slot * c.k_strides[3]) / vec_elems;
      m.vsrc = (vb + pg * c.v_strides[1] + slot * c.v_strides[3]) / vec_elems;
      m.kdst = to < 0 ? -1 : (kb + to * c.k_strides[1] + ts * c.k_strides[3]) / vec_elems;
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
  uint32_t spans, checks;  // pages that T tokens can reach into, and table entries to check (n * spans)
  int32_t n, check_inline;
};

// The write is all or nothing as well: rows, counts and the table entries of all pages that get tokens are checked
// before the first store. Up to one entry a thread every CTA checks all of them and so comes to the same answer
// without hearing of the others; more are checked by write_check_kernel, spread over the GPU, whose refusal
// write_kernel finds in the status word. One token of 256 rows (256 entries): 4.2 us, 5.4 us with the kernel of its
// own; 1024 rows: 15.0 and 11.1 us; 4 x 2048 tokens (516 entries): 10.8 and 11.0 us. Without checks 3.9, 9.9, 9.4 us.
constexpr int kWriteThreads = 256;

struct WriteRow {
  int row;
  int64_t len, m;
  int err;
};
__device__ __forceinline__ WriteRow write_row(const WriteParams& p, int i) {
  const cab_page_cache& c = p.c;
  WriteRow w{p.rows ? p.rows[i] : i, 0, 0, 0};
  if (w.row < 0 || w.row >= c.rows) {
    w.err = CAB_PAGES_BAD_ROW;
    return w;
  }
  w.len = c.seq_lens[w.row];
  w.m = p.num_new ? p.num_new[i] : p.num_value;
  if (w.m < 0 || w.m > p.T || w.m > w.len || w.len > c.width * c.page_size) w.err = CAB_PAGES_BAD_ARG;
  return w;
}

// CTA `part` of `parts` checks its share: table entries e = (sequence, page) from part on, and part 0 whether a row is
// named twice. The result is the same in all threads of the CTA.
__device__ int write_errors(const WriteParams& p, int part, int parts) {
  extern __shared__ uint32_t named[];  // a bit per row, where rows are listed
  const cab_page_cache& c = p.c;
  const int tid = threadIdx.x;
  int err = 0;
  if (p.rows && part == 0) {
    for (int i = tid; i < static_cast<int>((c.rows + 31) / 32); i += kWriteThreads) named[i] = 0u;
    __syncthreads();
    for (int i = tid; i < p.n; i += kWriteThreads) {
      const int row = p.rows[i];
      if (row >= 0 && row < c.rows && atomicOr(&named[row >> 5], 1u << (row & 31)) >> (row & 31) & 1u) err |= CAB_PAGES_BAD_ROW;
    }
  }
  for (uint32_t e = part * kWriteThreads + tid; e < p.checks; e += parts * kWriteThreads) {  // checks is below 2^31
    const int i = static_cast<int>(e / p.spans);
    const WriteRow w = write_row(p, i);
    err |= w.err;
    if (w.err || w.m == 0) continue;
    const int64_t page = (w.len - w.m) / c.page_size + (e - static_cast<uint32_t>(i) * p.spans);
    if (page * c.page_size >= w.len) continue;
    const int32_t pg = c.block_table[w.row * c.table_stride + page];
    if (pg < 0 || pg >= c.pages) err |= CAB_PAGES_BAD_TABLE;
  }
  if (!__syncthreads_or(err)) return 0;
  int all = 0;
  for (int bit = 1; bit <= CAB_PAGES_BAD_TABLE; bit <<= 1)
    if (__syncthreads_or(err & bit)) all |= bit;
  return all;
}

__global__ void __launch_bounds__(kWriteThreads) write_check_kernel(const __grid_constant__ WriteParams p) {
  grid_dependency_wait();
  if (*reinterpret_cast<volatile int32_t*>(p.c.status) != 0) return;
  const int err = write_errors(p, blockIdx.x, gridDim.x);
  if (err && threadIdx.x == 0) atomicOr(p.c.status, err);
}

template <typename V>
__global__ void __launch_bounds__(kWriteThreads, 3) write_kernel(const __grid_constant__ WriteParams p, int vec_elems, int vecs) {
  const cab_page_cache& c = p.c;
  grid_dependency_wait();
  const int refused = *reinterpret_cast<volatile int32_t*>(c.status);  // on its way along with the checks' loads
  if (p.check_inline) {
    if (const int err = write_errors(p, 0, 1)) {  // the same in every CTA: none stores
      if (refused == 0 && threadIdx.x == 0) atomicOr(c.status, err);
      return;
    }
  }
  if (refused != 0) return;
  const int64_t S = c.page_size;
  const int64_t groups = (p.T + 31) / 32, tasks = groups * c.heads * p.n;
  const int lane = threadIdx.x & 31;
  const int64_t wn = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t task = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); task < tasks; task += wn) {
    const int64_t ih = task / groups, g = task - ih * groups;
    const int i = static_cast<int>(ih / c.heads), h = static_cast<int>(ih - i * c.heads);
    const WriteRow w = write_row(p, i);
    const int64_t t = 32 * g + lane;
    RowSpan s{0, 0, -1, -1};
    if (w.err == 0 && t < w.m) {
      const int64_t pos = w.len - w.m + t, slot = pos % S, col = pos / S;
      const int64_t pg = c.block_table[w.row * c.table_stride + col];
      // The checks have passed. Should another stream change the cache all the same, nothing out of range is touched.
      if (pg >= 0 && pg < c.pages) {
        const bool shared = c.ref_counts[pg] > 1;
        s.ksrc = (i * p.ks[0] + h * p.ks[1] + t * p.ks[2]) / vec_elems;
        s.vsrc = (i * p.vs[0] + h * p.vs[1] + t * p.vs[2]) / vec_elems;
        s.kdst = (p.layer * c.k_strides[0] + pg * c.k_strides[1] + h * c.k_strides[2] + slot * c.k_strides[3]) / vec_elems;
        s.vdst = (p.layer * c.v_strides[0] + pg * c.v_strides[1] + h * c.v_strides[2] + slot * c.v_strides[3]) / vec_elems;
        // Rows share a page in the same column. Of several that write a token of it the last one does.
        for (int j = shared ? i + 1 : p.n; j < p.n; ++j) {
          const WriteRow o = write_row(p, j);
          if (o.err == 0 && pos >= o.len - o.m && pos < o.len && c.block_table[o.row * c.table_stride + col] == pg) s.kdst = -1;
        }
      }
    }
    const int count = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(32), w.m - 32 * g)));
    move_rows<V>(static_cast<const V*>(p.k), static_cast<const V*>(p.v), static_cast<V*>(c.k_pages),
                 static_cast<V*>(c.v_pages), s, count, vecs);
  }
}

// ------------------------------------------------------------------ host side
// A launch whose CTAs may start while the kernel before it on the stream still runs; it waits for that
// kernel's results by griddepcontrol.wait. `cluster` CTAs form a cluster.
template <typename... Args>
void launch_after(void (*kernel)(Args...), dim3 grid, int threads, cudaStream_t st, size_t smem, int cluster, Args... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Raises a kernel's limit of dynamic shared memory, once per device and to the most that any call needs: the limit
// is the device's, not the thread's, so a limit set per call could be lowered by another thread before the launch.
template <auto Kernel>
int allow_smem(size_t most, const char* what) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return CAB_OK;
  const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(CAB_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  }
  done.fetch_or(bit, std::memory_order_relaxed);
  return CAB_OK;
}

inline int check_cache(const cab_page_cache* c, const char* what, bool data, bool state = true) {
  if (!c) return fail(CAB_ERR_INVALID_ARG, "%s: NULL cache", what);
  if (!c->block_table || !c->seq_lens || (state && (!c->ref_counts || !c->status)))
    return fail(CAB_ERR_INVALID_ARG, "%s: NULL pointer in the cache", what);
  if (c->layers <= 0 || c->pages <= 0 || c->heads <= 0 || c->page_size <= 0 || c->dim <= 0 || c->rows <= 0 || c->width <= 0)
    return fail(CAB_ERR_INVALID_ARG, "%s: non-positive size in the cache", what);
  if (c->pages >= (int64_t)1 << 31 || c->rows > kMaxRows || (c->width + 1) * c->page_size >= (int64_t)1 << 31 ||
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
  size_t fresh, free_list, snap, total;
  int64_t cap;
};

inline UpdateLayout update_layout(const cab_page_cache* c, int64_t n) {
  auto up = [](size_t x) { return (x + 15) & ~size_t(15); };
  UpdateLayout L{};
  L.cap = std::min(c->pages, n * c->width);
  L.fresh = 16;
  L.free_list = L.fresh + static_cast<size_t>(L.cap) * sizeof(FreshPage);
  L.snap = up(L.free_list + static_cast<size_t>(L.cap) * 4);
  L.total = up(L.snap + static_cast<size_t>(n) * c->width * 4);
  return L;
}

inline int check_pairs(const cab_page_cache* c, int64_t n) {
  if (n <= 0 || n > kMaxPairs) return fail(CAB_ERR_UNSUPPORTED, "pages_update: 1 to %d pairs a call, got %lld", kMaxPairs, (long long)n);
  if (n * c->width >= (int64_t)1 << 31) return fail(CAB_ERR_UNSUPPORTED, "pages_update: more than 2^31 table entries a call");
  return CAB_OK;
}

}  // namespace pages
}  // namespace cab

extern "C" int cab_pages_update_workspace_size(const cab_page_cache* cache, int64_t n, size_t* bytes) {
  using namespace cab;
  using namespace cab::pages;
  if (!bytes) return fail(CAB_ERR_INVALID_ARG, "pages_update_workspace_size: NULL output");
  if (int rc = check_cache(cache, "pages_update_workspace_size", false)) return rc;
  if (int rc = check_pairs(cache, n)) return rc;
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
  if (int rc = check_pairs(cache, n)) return rc;
  if (!src && n > cache->rows) return fail(CAB_ERR_INVALID_ARG, "pages_update: %lld pairs without source rows, %lld rows", (long long)n, (long long)cache->rows);
  if (keep_cols < 0 || keep_cols >= (int64_t)1 << 31) return fail(CAB_ERR_INVALID_ARG, "pages_update: bad number of keep columns");
  if (n * keep_cols >= (int64_t)1 << 31) return fail(CAB_ERR_UNSUPPORTED, "pages_update: more than 2^31 list entries a call");
  if (keep_cols > 0 && (!keep || (keep_bytes != 4 && keep_bytes != 8))) return fail(CAB_ERR_INVALID_ARG, "pages_update: keep must be int32 or int64");
  if (keep_cols > 0 && !copies) return fail(CAB_ERR_INVALID_ARG, "pages_update: a keep list needs copies");
  // the snapshot of the source rows, which other rows are made from, is taken for the copies alone
  if (dst && !copies) return fail(CAB_ERR_INVALID_ARG, "pages_update: rows that become others need copies");
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
  p.keep_num = keep_num;  // without a list, counts other than 0 are refused
  p.keep_num_stride = keep_num_stride;
  p.grow = grow;
  p.grow_value = std::min(grow_value, (int64_t)INT32_MAX);  // more than any row has room for; sums stay in 64 bits
  p.n = static_cast<int32_t>(n);
  p.copies = copies != 0;
  p.header = reinterpret_cast<int32_t*>(ws);
  p.fresh = reinterpret_cast<FreshPage*>(ws + L.fresh);
  p.free_list = reinterpret_cast<int32_t*>(ws + L.free_list);
  p.snap = reinterpret_cast<int32_t*>(ws + L.snap);
  p.cap = L.cap;
  uint32_t log2s = 0;
  while ((int64_t)1 << log2s < cache->page_size) ++log2s;
  p.div_mul = static_cast<uint32_t>((((uint64_t)1 << (31 + log2s)) + cache->page_size - 1) / cache->page_size);
  p.div_shift = 31 + log2s;

  auto smem_of = [](int64_t pairs, int64_t rows) { return static_cast<size_t>(15 * pairs + 1 + 3 * ((rows + 31) / 32)) * 4; };
  const size_t smem = smem_of(n, cache->rows);
  if (int rc = allow_smem<update_kernel>(smem_of(kMaxPairs, kMaxRows), "pages update_kernel")) return rc;
  // one CTA reads up to 8 values a thread of each array in one go; more are spread over a cluster
  const int64_t ints = std::max(cache->pages, n * std::max(cache->width, keep_cols));
  launch_after(update_kernel, dim3(ints > 8 * kUpdateThreads ? kMaxCluster : 1), kUpdateThreads, static_cast<cudaStream_t>(stream), smem,
               ints > 8 * kUpdateThreads ? kMaxCluster : 1, p);
  if (int rc = check_launch("pages update_kernel")) return rc;
  if (!copies) return CAB_OK;

  const int vb = vector_bytes(cache, nullptr, nullptr, nullptr, nullptr);
  const int es = static_cast<int>(dtype_size(static_cast<int>(cache->dtype)));
  const int vecs = static_cast<int>(cache->dim * es / vb), ve = vb >= es ? vb / es : 1;
  // without a list only a pair's last page is copied, else at most keep_cols + page_size tokens
  const int64_t per = keep_cols > 0 ? (keep_cols + cache->page_size - 1) / cache->page_size + 1 : 1;
  const int64_t most = std::min(L.cap, n * std::min(per, cache->width)) * ((cache->page_size + 31) / 32) * cache->layers * cache->heads;
  const dim3 grid(static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((most + 7) / 8, (int64_t)current_sm_count() * 8))));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (vb == 16) launch_after(copy_kernel<uint4>, grid, 256, st, 0, 1, p, ve, vecs);
  else if (vb == 4) launch_after(copy_kernel<uint32_t>, grid, 256, st, 0, 1, p, ve, vecs);
  else launch_after(copy_kernel<uint16_t>, grid, 256, st, 0, 1, p, ve, vecs);
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
  const int64_t most = (int64_t)current_sm_count() * 8;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((tasks + 7) / 8, most));
  const int64_t spans = std::min((T + cache->page_size - 2) / cache->page_size + 1, cache->width);
  if (n * spans >= (int64_t)1 << 31) return fail(CAB_ERR_UNSUPPORTED, "pages_write: more than 2^31 table entries a call");
  p.spans = static_cast<uint32_t>(spans);
  p.checks = static_cast<uint32_t>(n * spans);
  p.check_inline = p.checks <= kWriteThreads;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t named = rows ? static_cast<size_t>((cache->rows + 31) / 32) * 4 : 0;  // at most 8 KB
  if (!p.check_inline) {
    const unsigned ctas = static_cast<unsigned>(std::min<int64_t>((p.checks + kWriteThreads - 1) / kWriteThreads, most));
    launch_after(write_check_kernel, dim3(ctas), kWriteThreads, st, named, 1, p);
    if (int rc = check_launch("pages write_check_kernel")) return rc;
  }
  const size_t smem = p.check_inline ? named : 0;
  if (vb == 16) launch_after(write_kernel<uint4>, dim3(grid), kWriteThreads, st, smem, 1, p, ve, vecs);
  else if (vb == 4) launch_after(write_kernel<uint32_t>, dim3(grid), kWriteThreads, st, smem, 1, p, ve, vecs);
  else launch_after(write_kernel<uint16_t>, dim3(grid), kWriteThreads, st, smem, 1, p, ve, vecs);
  return check_launch("pages write_kernel");
}
