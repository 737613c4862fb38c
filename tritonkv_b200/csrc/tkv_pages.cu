// Page management of a paged cache (sm_100a): forking and releasing sequences, room for tokens to
// come, and compaction.  All state is the block table and the lengths; what is in use is read off
// the table every time, so nothing can disagree with it, and no call waits for the host.
//
// Fork.  Row b of the new table continues row parents[b] of the old one, n = its length:
//   * full pages (n / page of them) are shared;
//   * a partly filled page is kept by the first row that continues this parent, every other one
//     gets a copy of it in a fresh page;
//   * pages for `reserve` further tokens follow; a parent outside the old table gives an empty row.
// Fresh pages are the lowest ones that no kept entry names, in order of (row, position): the
// outcome does not depend on the order in which threads run.
//
// Compaction.  With n pages in use, the k-th used page at or above n moves to the k-th unused page
// below n.  Pages are only read above n and only written below, so the old table stays valid.
//
// Each is two launches.  The first reads the table -- a bit per used page -- and its last CTA to finish
// (a ticket) ranks and lists what has to be done: everything in order of rows or pages, so the outcome does
// not depend on which CTA that is.  The second, a programmatic dependent, does it: table entries, and
// the copies cut into slices of 16 KB.  The bitmap and the ticket are left zero for the next call.
#include "tkv_common.cuh"

namespace tkv {

constexpr int kMaxPoolTensors = 24;  // of one launch
constexpr int kSlice = 16384;        // bytes that a CTA copies at a time
constexpr int kPlanThreads = 1024;

struct PoolTensors {
  uint8_t* base[kMaxPoolTensors];
  int64_t page_bytes[kMaxPoolTensors];
  int first[kMaxPoolTensors];  // slices of the tensors before
  int n, slices;               // tensors; slices of one page of all of them
  int wide;                    // every page is 16-byte aligned in all of them
};

// One CTA: copy slice `slice` of page `s` to page `d`.
__device__ __forceinline__ void copy_slice(const PoolTensors& t, int slice, int s, int d) {
  int i = 0;
  while (i + 1 < t.n && slice >= t.first[i + 1]) ++i;
  const int64_t at = (int64_t)(slice - t.first[i]) * kSlice, bytes = t.page_bytes[i];
  const int len = (int)min((int64_t)kSlice, bytes - at);
  const uint8_t* from = t.base[i] + s * bytes + at;
  uint8_t* to = t.base[i] + d * bytes + at;
  if (t.wide) {
    constexpr int PER = kSlice / (256 * 16);
    uint4 v[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int o = (k * 256 + threadIdx.x) * 16;
      if (o < len) v[k] = __ldcs(reinterpret_cast<const uint4*>(from + o));
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int o = (k * 256 + threadIdx.x) * 16;
      if (o < len) *reinterpret_cast<uint4*>(to + o) = v[k];
    }
  } else {
    for (int o = threadIdx.x; o < len; o += 256) to[o] = from[o];
  }
}

__device__ __forceinline__ bool page_ok(int id, int num_pages) { return (unsigned)id < (unsigned)num_pages; }

__device__ __forceinline__ uint32_t word_mask(int w, int num_pages) {  // bits of word w that are pages
  const int left = num_pages - w * 32;
  return left >= 32 ? 0xffffffffu : (1u << left) - 1u;
}

// Whether this CTA is the last of the grid to come here; what the others wrote before is then visible.
__device__ __forceinline__ bool last_cta(uint32_t* ticket) {
  __shared__ bool s_last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (s_last) __threadfence();
  return s_last;
}

// Exclusive prefix sum over the CTA's kPlanThreads threads; `total` is the sum.
__device__ __forceinline__ int block_scan(int x, int& total) {
  __shared__ int s_warp[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(kFullMask, incl, off);
    if (lane >= off) incl += y;
  }
  __syncthreads();  // s_warp may still be read from the call before
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int w = s_warp[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(kFullMask, w, off);
      if (lane >= off) w += y;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  total = s_warp[kPlanThreads / 32 - 1];
  return incl - x + (warp > 0 ? s_warp[warp - 1] : 0);
}

// ------------------------------------------------------------------ fork
struct ForkArgs {
  const int32_t *table, *lens, *parents, *reserve;
  int32_t *new_table, *new_lens, *missing;
  uint32_t *ticket, *used;  // bit i of used[w]: page 32 w + i is named by a kept entry
  int32_t* listed;       // fresh pages that are there
  int32_t* src;          // (B) page that the row copies, or -1
  int32_t* start;        // (B) fresh pages of the rows before
  int32_t* fresh;        // (num_pages) unused pages, lowest first
  int64_t table_stride;
  int reserve0, B_old, B, num_pages, page, W;
};

struct ForkRow {
  int full, held, want;  // pages that are filled, touched, and touched with the reserve
};
__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, int b, int n) {
  ForkRow r;
  r.full = n / a.page;
  r.held = r.full + (n - r.full * a.page > 0 ? 1 : 0);
  const int64_t more = max(a.reserve ? a.reserve[b] : a.reserve0, 0);
  r.want = (int)min((int64_t)a.W, (n + more + a.page - 1) / a.page);
  return r;
}

// A warp per new row: entries that stay, and what the row needs besides.  Then, in the last CTA: rank the
// rows' needs and list the lowest unused pages.
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const ForkArgs a) {
  const int tid = threadIdx.x, lane = tid & 31;
  pdl_launch_dependents();
  for (int b = blockIdx.x * (kPlanThreads / 32) + (tid >> 5); b < a.B; b += gridDim.x * (kPlanThreads / 32)) {
    const int par = a.parents[b];
    int32_t* row = a.new_table + (int64_t)b * a.W;
    const bool live = par >= 0 && par < a.B_old;
    // (the loads that hang on the parent alone are on their way while its earlier children are looked for)
    const int32_t* old = a.table + (live ? par : 0) * a.table_stride;
    const int tokens = live ? a.lens[par] : 0;
    int id0 = live && lane < a.W ? old[lane] : -1;
    bool elder = false;
    if (live) {
#pragma unroll 8
      for (int i = lane; i < b; i += 32) elder |= a.parents[i] == par;
    }
    const int n = (int)min((int64_t)max(tokens, 0), (int64_t)a.W * a.page);
    const ForkRow r = fork_row(a, b, n);
    const int last = r.held > r.full ? old[r.full] : -1;  // the partly filled page
    const bool first = !__any_sync(kFullMask, elder);
    const int keep = live ? (first ? r.held : r.full) : 0;
    for (int i = lane; i < a.W; i += 32) {
      int id = -1;
      if (i < keep) {
        id = i < 32 ? id0 : old[i];
        if (!page_ok(id, a.num_pages)) id = -1;
        else atomicOr(a.used + (id >> 5), 1u << (id & 31));
      }
      row[i] = id;
    }
    if (lane == 0) {
      const bool copy = !first && page_ok(last, a.num_pages);
      a.src[b] = copy ? last : -1;
      a.new_lens[b] = n;
      a.start[b] = live ? (copy ? 1 : 0) + max(0, r.want - r.held) : 0;
    }
  }
  if (!last_cta(a.ticket)) return;
  int need = 0, have = 0, total;
  const int words = (a.num_pages + 31) / 32;
  const uint32_t used0 = tid < words ? __ldcg(a.used + tid) : 0;  // (beside the first needs)
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = b0 + tid, x = b < a.B ? __ldcg(a.start + b) : 0;
    const int before = block_scan(x, total);
    if (b < a.B) a.start[b] = need + before;
    need += total;
  }
  for (int w0 = 0; w0 < words; w0 += kPlanThreads) {
    const int w = w0 + tid;
    uint32_t free = 0;
    if (w < words) {
      free = ~(w0 == 0 ? used0 : __ldcg(a.used + w)) & word_mask(w, a.num_pages);
      a.used[w] = 0;
    }
    if (have >= need) continue;  // (the same for all threads) enough: the rest is only wiped
    int rank = have + block_scan(__popc(free), total);
    for (; free && rank < need; free &= free - 1, ++rank) a.fresh[rank] = w * 32 + __ffs(free) - 1;
    have += total;
  }
  if (tid == 0) {
    *a.listed = min(need, have);
    *a.missing = max(0, need - have);
    *a.ticket = 0;
  }
}

// CTA (row, part): fresh pages into the row's entries (part 0 of the first launch), and its slices of the copy.
__global__ void __launch_bounds__(256) fork_apply_kernel(const ForkArgs a, const PoolTensors t, int entries) {
  const int b = blockIdx.x;
  pdl_wait();
  const int src = __ldcg(a.src + b), start = __ldcg(a.start + b), listed = __ldcg(a.listed), par = a.parents[b];
  if (entries && blockIdx.y == 0 && par >= 0 && par < a.B_old) {
    const ForkRow r = fork_row(a, b, __ldcg(a.new_lens + b));
    int32_t* row = a.new_table + (int64_t)b * a.W;
    const int copy = src >= 0 ? 1 : 0, count = copy + max(0, r.want - r.held);
    for (int j = threadIdx.x; j < count; j += 256)
      row[j < copy ? r.full : r.held + j - copy] = start + j < listed ? __ldcg(a.fresh + start + j) : -1;
  }
  if (src < 0 || start >= listed) return;
  const int dst = __ldcg(a.fresh + start);
  for (int slice = blockIdx.y; slice < t.slices; slice += gridDim.y) copy_slice(t, slice, src, dst);
}

// ------------------------------------------------------------------ compact
struct CompactArgs {
  const int32_t* table;
  int32_t *new_table, *live;
  uint32_t *ticket, *used;
  int32_t* n_moves;
  int32_t* before;        // (words) used pages in the words before
  int32_t *src, *dst;     // moves
  int32_t* to;            // (num_pages) where page p >= live goes
  int64_t table_stride;
  int B, W, num_pages;
};

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const CompactArgs a) {
  __shared__ int s_below;
  const int tid = threadIdx.x, lane = tid & 31;
  pdl_launch_dependents();
  for (int b = blockIdx.x * (kPlanThreads / 32) + (tid >> 5); b < a.B; b += gridDim.x * (kPlanThreads / 32))
    for (int i = lane; i < a.W; i += 32) {
      const int id = a.table[b * a.table_stride + i];
      if (page_ok(id, a.num_pages)) atomicOr(a.used + (id >> 5), 1u << (id & 31));
    }
  if (!last_cta(a.ticket)) return;
  const int words = (a.num_pages + 31) / 32;
  int live = 0, total;
  for (int w0 = 0; w0 < words; w0 += kPlanThreads) {
    const int w = w0 + tid;
    const int x = w < words ? __popc(__ldcg(a.used + w)) : 0;
    const int before = block_scan(x, total);
    if (w < words) a.before[w] = live + before;
    live += total;
  }
  __syncthreads();
  if (tid == 0) {  // used pages below `live`: the others have to move
    int below = live;
    if (live < a.num_pages) {
      const int w = live >> 5;
      below = a.before[w] + __popc(__ldcg(a.used + w) & ((1u << (live & 31)) - 1u));
    }
    s_below = below;
    *a.live = live;
    *a.n_moves = live - below;
    *a.ticket = 0;
  }
  __syncthreads();
  const int below = s_below;
  for (int w = tid >> 5; w < words; w += kPlanThreads / 32) {  // a lane per page: its rank says where it goes
    const uint32_t used = __ldcg(a.used + w);
    const int p = w * 32 + lane, u = a.before[w] + __popc(used & ((1u << lane) - 1u));
    if ((used >> lane) & 1u) {
      if (p >= live) a.src[u - below] = p;
    } else if (p < live) {
      a.dst[p - u] = p;
    }
    __syncwarp();
    if (lane == 0) a.used[w] = 0;
  }
  __syncthreads();
  const int moves = live - below;
  for (int i = tid; i < moves; i += kPlanThreads) a.to[a.src[i]] = a.dst[i];
}

__global__ void __launch_bounds__(256) compact_apply_kernel(const CompactArgs a, const PoolTensors t, int entries) {
  pdl_wait();
  const int live = __ldcg(a.live), moves = __ldcg(a.n_moves);
  if (entries) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)a.B * a.W; i += (int64_t)gridDim.x * 256) {
      const int b = (int)(i / a.W);
      int id = a.table[b * a.table_stride + (i - (int64_t)b * a.W)];
      if (!page_ok(id, a.num_pages)) id = -1;
      else if (id >= live) id = __ldcg(a.to + id);
      a.new_table[i] = id;
    }
  }
  const int64_t items = (int64_t)moves * t.slices;
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const int m = (int)(i / t.slices);
    copy_slice(t, (int)(i - (int64_t)m * t.slices), __ldcg(a.src + m), __ldcg(a.dst + m));
  }
}

// ------------------------------------------------------------------ host side
static int check_pools(const char* who, const tkv_page_pool* pools, int n) {
  TKV_REQUIRE(n >= 0 && (n == 0 || pools), TKV_ERR_INVALID, "%s: bad list of %d pools", who, n);
  for (int i = 0; i < n; ++i)
    TKV_REQUIRE(pools[i].base && pools[i].page_bytes > 0 && pools[i].page_bytes < (1LL << 40), TKV_ERR_INVALID,
                "%s: bad pool tensor %d", who, i);
  return TKV_OK;
}

// Tensors [i0, i0 + kMaxPoolTensors) of the list.
static PoolTensors some_pools(const tkv_page_pool* pools, int n, int i0) {
  PoolTensors t{};
  t.n = n - i0 < kMaxPoolTensors ? n - i0 : kMaxPoolTensors;
  t.wide = 1;
  for (int i = 0; i < t.n; ++i) {
    t.base[i] = static_cast<uint8_t*>(pools[i0 + i].base);
    t.page_bytes[i] = pools[i0 + i].page_bytes;
    t.first[i] = t.slices;
    t.slices += (int)((t.page_bytes[i] + kSlice - 1) / kSlice);
    if ((reinterpret_cast<uintptr_t>(t.base[i]) | (uintptr_t)t.page_bytes[i]) & 15) t.wide = 0;
  }
  return t;
}

static int plan_grid(int rows) {  // a warp per row, few CTAs: the last one waits for all
  const int n = (rows + kPlanThreads / 32 - 1) / (kPlanThreads / 32);
  return n < 1 ? 1 : n < 148 ? n : 148;
}

}  // namespace tkv

extern "C" int tkv_pages_workspace(int B, int num_pages, int64_t* words) {
  TKV_REQUIRE(words && B >= 0 && num_pages > 0, TKV_ERR_INVALID, "pages_workspace: bad sizes B=%d num_pages=%d", B,
              num_pages);
  *words = 4 + 2LL * ((num_pages + 31) / 32) + 3LL * num_pages + 2LL * B;
  return TKV_OK;
}

extern "C" int tkv_pages_fork(const tkv_pages_fork_args* args, const tkv_page_pool* pools, int n_pools, void* stream) {
  using namespace tkv;
  TKV_REQUIRE(args, TKV_ERR_INVALID, "fork: null arguments");
  const tkv_pages_fork_args& in = *args;
  TKV_REQUIRE(in.B >= 0 && in.B_old >= 0 && in.max_pages >= 0 && in.num_pages > 0 && in.page_size > 0, TKV_ERR_INVALID,
              "fork: bad sizes B=%d B_old=%d max_pages=%d num_pages=%d page_size=%d", in.B, in.B_old, in.max_pages,
              in.num_pages, in.page_size);
  TKV_REQUIRE((int64_t)in.max_pages * in.page_size < (1LL << 30) && (int64_t)in.B * in.max_pages < (1LL << 30),
              TKV_ERR_INVALID, "fork: a table of %d x %d pages of %d tokens is too large", in.B, in.max_pages, in.page_size);
  TKV_REQUIRE(in.missing && in.workspace, TKV_ERR_INVALID, "fork: null pointer");
  TKV_REQUIRE(in.B == 0 || (in.parents && in.new_lens), TKV_ERR_INVALID, "fork: null pointer");
  TKV_REQUIRE(in.B == 0 || in.max_pages == 0 || in.new_table, TKV_ERR_INVALID, "fork: null pointer");
  TKV_REQUIRE(in.B_old == 0 || ((in.block_table || in.max_pages == 0) && in.seq_lens), TKV_ERR_INVALID, "fork: null pointer");
  const int rc = check_pools("fork", pools, n_pools);
  if (rc != TKV_OK) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  const int B = in.B, words = (in.num_pages + 31) / 32;
  ForkArgs a{};
  a.table = in.block_table;
  a.lens = in.seq_lens;
  a.parents = in.parents;
  a.reserve = in.reserve;
  a.new_table = in.new_table;
  a.new_lens = in.new_lens;
  a.missing = in.missing;
  a.ticket = (uint32_t*)in.workspace;  // [ticket, listed, -, -][bitmap][fresh][src][start]
  a.listed = in.workspace + 1;
  a.used = (uint32_t*)in.workspace + 4;
  a.fresh = in.workspace + 4 + words;
  a.src = a.fresh + in.num_pages;
  a.start = a.src + B;
  a.table_stride = in.table_stride;
  a.reserve0 = in.reserve0;
  a.B_old = in.B_old;
  a.B = B;
  a.num_pages = in.num_pages;
  a.page = in.page_size;
  a.W = in.max_pages;
  fork_plan_kernel<<<plan_grid(B), kPlanThreads, 0, s>>>(a);
  TKV_CUDA(cudaGetLastError());
  if (B == 0) return TKV_OK;
  for (int i0 = 0; i0 == 0 || i0 < n_pools; i0 += kMaxPoolTensors) {
    const PoolTensors t = some_pools(pools, n_pools, i0);
    // CTAs of a row: about four waves in all where every row copies
    int parts = (148 * 32 + B - 1) / B;
    parts = parts < 1 ? 1 : parts > t.slices ? (t.slices > 0 ? t.slices : 1) : parts;
    TKV_CUDA(launch_pdl(fork_apply_kernel, dim3(B, parts), dim3(256), 0, s, a, t, i0 == 0 ? 1 : 0));
  }
  return TKV_OK;
}

extern "C" int tkv_pages_compact(const tkv_pages_compact_args* args, const tkv_page_pool* pools, int n_pools,
                                 void* stream) {
  using namespace tkv;
  TKV_REQUIRE(args, TKV_ERR_INVALID, "compact: null arguments");
  const tkv_pages_compact_args& in = *args;
  TKV_REQUIRE(in.B >= 0 && in.max_pages >= 0 && in.num_pages > 0, TKV_ERR_INVALID,
              "compact: bad sizes B=%d max_pages=%d num_pages=%d", in.B, in.max_pages, in.num_pages);
  TKV_REQUIRE((int64_t)in.B * in.max_pages < (1LL << 30), TKV_ERR_INVALID,
              "compact: a table of %d x %d entries is too large", in.B, in.max_pages);
  TKV_REQUIRE(in.live && in.workspace, TKV_ERR_INVALID, "compact: null pointer");
  TKV_REQUIRE(in.B == 0 || in.max_pages == 0 || (in.block_table && in.new_table), TKV_ERR_INVALID, "compact: null pointer");
  const int rc = check_pools("compact", pools, n_pools);
  if (rc != TKV_OK) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  const int words = (in.num_pages + 31) / 32;
  CompactArgs a{};
  a.table = in.block_table;
  a.new_table = in.new_table;
  a.live = in.live;
  a.ticket = (uint32_t*)in.workspace;  // [ticket, moves, -, -][bitmap][before][src][dst][to]
  a.n_moves = in.workspace + 1;
  a.used = (uint32_t*)in.workspace + 4;
  a.before = in.workspace + 4 + words;
  a.src = a.before + words;
  a.dst = a.src + in.num_pages;
  a.to = a.dst + in.num_pages;
  a.table_stride = in.table_stride;
  a.B = in.B;
  a.W = in.max_pages;
  a.num_pages = in.num_pages;
  compact_plan_kernel<<<plan_grid(in.B), kPlanThreads, 0, s>>>(a);
  TKV_CUDA(cudaGetLastError());
  for (int i0 = 0; i0 == 0 || i0 < n_pools; i0 += kMaxPoolTensors) {
    const PoolTensors t = some_pools(pools, n_pools, i0);
    TKV_CUDA(launch_pdl(compact_apply_kernel, dim3(148 * 8), dim3(256), 0, s, a, t, i0 == 0 ? 1 : 0));
  }
  return TKV_OK;
}
