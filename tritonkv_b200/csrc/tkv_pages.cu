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
#include "tkv_common.cuh"

namespace tkv {

constexpr int kMaxPoolTensors = 24;

struct PoolTensors {
  uint8_t* base[kMaxPoolTensors];
  int64_t page_bytes[kMaxPoolTensors];
  int n;
};

struct ForkArgs {
  const int32_t *table, *lens, *parents, *reserve;
  int32_t *new_table, *new_lens, *missing;
  uint32_t* used;        // bit i of word w: page 32 w + i is named by a kept entry
  int32_t *src, *dst;    // (B) page copies, -1 for none
  int32_t* start;        // (B) fresh pages of the rows before
  int32_t* fresh;        // (num_pages) unused pages, lowest first
  int64_t table_stride;
  int reserve0, B_old, B, num_pages, page, W;
};

__device__ __forceinline__ bool page_ok(int id, int num_pages) { return (unsigned)id < (unsigned)num_pages; }

struct ForkRow {
  int n, full, held, want;  // tokens; pages filled, touched, and touched with the reserve
};
__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, int b, int n) {
  ForkRow r;
  r.n = n;
  r.full = n / a.page;
  r.held = (int)(((int64_t)n + a.page - 1) / a.page);
  const int64_t more = max(a.reserve ? a.reserve[b] : a.reserve0, 0);
  r.want = (int)min((int64_t)a.W, (n + more + a.page - 1) / a.page);
  return r;
}

// One CTA per new row: entries that stay, and what the row needs besides.
__global__ void __launch_bounds__(128) fork_mark_kernel(const ForkArgs a) {
  const int b = blockIdx.x, tid = threadIdx.x, par = a.parents[b];
  int32_t* row = a.new_table + (int64_t)b * a.W;
  const bool live = par >= 0 && par < a.B_old;
  bool elder = false;
  if (live)
    for (int i = tid; i < b; i += 128) elder |= a.parents[i] == par;
  const bool first = !__syncthreads_or(elder);
  const int n = live ? (int)min((int64_t)max(a.lens[par], 0), (int64_t)a.W * a.page) : 0;
  const ForkRow r = fork_row(a, b, n);
  const int32_t* old = a.table + (live ? par : 0) * a.table_stride;
  const int keep = live ? (first ? r.held : r.full) : 0;
  for (int i = tid; i < a.W; i += 128) {
    int id = -1;
    if (i < keep) {
      id = old[i];
      if (!page_ok(id, a.num_pages)) id = -1;
      else atomicOr(a.used + (id >> 5), 1u << (id & 31));
    }
    row[i] = id;
  }
  if (tid == 0) {
    const bool copy = live && r.held > r.full && !first && page_ok(old[r.full], a.num_pages);
    a.src[b] = copy ? old[r.full] : -1;
    a.dst[b] = -1;
    a.new_lens[b] = n;
    a.start[b] = live ? (copy ? 1 : 0) + max(0, r.want - r.held) : 0;
  }
}

// Exclusive prefix sum over the CTA's 1024 threads; `total` is the sum.
__device__ __forceinline__ int block_scan(int x, int* s_warp, int& total) {
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
  total = s_warp[31];
  return incl - x + (warp > 0 ? s_warp[warp - 1] : 0);
}

__device__ __forceinline__ uint32_t word_mask(int w, int num_pages) {  // bits of word w that are pages
  const int left = num_pages - w * 32;
  return left >= 32 ? 0xffffffffu : (1u << left) - 1u;
}

// One CTA: rank the rows' needs, list the lowest unused pages, hand them out.
__global__ void __launch_bounds__(1024) fork_assign_kernel(const ForkArgs a) {
  __shared__ int s_warp[32];
  const int tid = threadIdx.x, words = (a.num_pages + 31) / 32;
  int need = 0, total;
  for (int b0 = 0; b0 < a.B; b0 += 1024) {
    const int b = b0 + tid, x = b < a.B ? a.start[b] : 0;
    const int before = block_scan(x, s_warp, total);
    if (b < a.B) a.start[b] = need + before;
    need += total;
  }
  int have = 0;
  for (int w0 = 0; w0 < words && have < need; w0 += 1024) {
    const int w = w0 + tid;
    uint32_t free = w < words ? ~a.used[w] & word_mask(w, a.num_pages) : 0u;
    int rank = have + block_scan(__popc(free), s_warp, total);
    for (; free && rank < need; free &= free - 1, ++rank) a.fresh[rank] = w * 32 + __ffs(free) - 1;
    have += total;
  }
  if (tid == 0) *a.missing = max(0, need - have);
  __syncthreads();
  for (int b = tid >> 5; b < a.B; b += 32) {
    const int par = a.parents[b];
    if (par < 0 || par >= a.B_old) continue;
    const ForkRow r = fork_row(a, b, a.new_lens[b]);
    int32_t* row = a.new_table + (int64_t)b * a.W;
    const int copy = a.src[b] >= 0 ? 1 : 0, count = copy + max(0, r.want - r.held), start = a.start[b];
    for (int j = tid & 31; j < count; j += 32) {
      const int id = start + j < have ? a.fresh[start + j] : -1;
      if (j < copy) {
        row[r.full] = id;
        a.dst[b] = id;
      } else {
        row[r.held + j - copy] = id;
      }
    }
  }
}

struct CompactArgs {
  const int32_t* table;
  int32_t *new_table, *live;
  uint32_t* used;
  int32_t* before;        // (words) used pages in the words before
  int32_t *src, *dst;     // moves
  int32_t* n_moves;
  int64_t table_stride;
  int B, W, num_pages;
};

__global__ void __launch_bounds__(256) compact_mark_kernel(const CompactArgs a) {
  const int b = blockIdx.y;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < a.W; i += gridDim.x * 256) {
    const int id = a.table[b * a.table_stride + i];
    if (page_ok(id, a.num_pages)) atomicOr(a.used + (id >> 5), 1u << (id & 31));
  }
}

// One CTA: count the used pages, then list the moves.
__global__ void __launch_bounds__(1024) compact_plan_kernel(const CompactArgs a) {
  __shared__ int s_warp[32];
  __shared__ int s_below;
  const int tid = threadIdx.x, words = (a.num_pages + 31) / 32;
  int live = 0, total;
  for (int w0 = 0; w0 < words; w0 += 1024) {
    const int w = w0 + tid;
    const int x = w < words ? __popc(a.used[w]) : 0;
    const int before = block_scan(x, s_warp, total);
    if (w < words) a.before[w] = live + before;
    live += total;
  }
  __syncthreads();
  if (tid == 0) {  // used pages below `live`: the others have to move
    int below = live;
    if (live < a.num_pages) {
      const int w = live >> 5;
      below = a.before[w] + __popc(a.used[w] & ((1u << (live & 31)) - 1u));
    }
    s_below = below;
    *a.live = live;
    *a.n_moves = live - below;
  }
  __syncthreads();
  const int below = s_below;
  for (int w = tid; w < words; w += 1024) {
    const uint32_t used = a.used[w], mask = word_mask(w, a.num_pages);
    const int p0 = w * 32, before = a.before[w];
    for (uint32_t m = mask; m; m &= m - 1) {
      const int i = __ffs(m) - 1, p = p0 + i, u = before + __popc(used & ((1u << i) - 1u));
      if ((used >> i) & 1u) {
        if (p >= live) a.src[u - below] = p;
      } else if (p < live) {
        a.dst[p - u] = p;
      }
    }
  }
}

__global__ void __launch_bounds__(256) compact_table_kernel(const CompactArgs a) {
  const int b = blockIdx.y, live = *a.live, below = live - *a.n_moves;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < a.W; i += gridDim.x * 256) {
    int id = a.table[b * a.table_stride + i];
    if (!page_ok(id, a.num_pages)) id = -1;
    else if (id >= live) {
      const int w = id >> 5;
      id = a.dst[a.before[w] + __popc(a.used[w] & ((1u << (id & 31)) - 1u)) - below];
    }
    a.new_table[(int64_t)b * a.W + i] = id;
  }
}

// Copy page src[i] to dst[i] in every tensor, i < (count ? *count : n); a negative entry is none.
__global__ void __launch_bounds__(256)
    copy_pages_kernel(const PoolTensors t, const int32_t* __restrict__ src, const int32_t* __restrict__ dst,
                      const int32_t* __restrict__ count, int n) {
  const int pairs = count ? *count : n;
  for (int i = blockIdx.x; i < pairs; i += gridDim.x) {
    const int s = src[i], d = dst[i];
    if (s < 0 || d < 0) continue;
    const int64_t bytes = t.page_bytes[blockIdx.y];
    const uint8_t* from = t.base[blockIdx.y] + s * bytes;
    uint8_t* to = t.base[blockIdx.y] + d * bytes;
    if (((bytes | reinterpret_cast<uintptr_t>(from) | reinterpret_cast<uintptr_t>(to)) & 15) == 0) {
      for (int64_t k = threadIdx.x * 16; k < bytes; k += 256 * 16)
        *reinterpret_cast<uint4*>(to + k) = *reinterpret_cast<const uint4*>(from + k);
    } else {
      for (int64_t k = threadIdx.x; k < bytes; k += 256) to[k] = from[k];
    }
  }
}

static int check_pools(const char* who, void* const* pools, const int64_t* page_bytes, int n) {
  TKV_REQUIRE(n >= 0 && (n == 0 || (pools && page_bytes)), TKV_ERR_INVALID, "%s: bad list of %d pools", who, n);
  for (int i = 0; i < n; ++i)
    TKV_REQUIRE(pools[i] && page_bytes[i] > 0, TKV_ERR_INVALID, "%s: bad pool tensor %d", who, i);
  return TKV_OK;
}

// The copies of all tensors, kMaxPoolTensors in a launch.
static int launch_copy(void* const* pools, const int64_t* page_bytes, int n_pools, const int32_t* src,
                       const int32_t* dst, const int32_t* count, int n, cudaStream_t stream) {
  if (n == 0) return TKV_OK;
  for (int i0 = 0; i0 < n_pools; i0 += kMaxPoolTensors) {
    PoolTensors t{};
    t.n = n_pools - i0 < kMaxPoolTensors ? n_pools - i0 : kMaxPoolTensors;
    for (int i = 0; i < t.n; ++i) {
      t.base[i] = static_cast<uint8_t*>(pools[i0 + i]);
      t.page_bytes[i] = page_bytes[i0 + i];
    }
    copy_pages_kernel<<<dim3(n < 2048 ? n : 2048, t.n), 256, 0, stream>>>(t, src, dst, count, n);
    TKV_CUDA(cudaGetLastError());
  }
  return TKV_OK;
}

}  // namespace tkv

extern "C" int tkv_pages_workspace(int B, int num_pages, int64_t* words) {
  TKV_REQUIRE(words && B >= 0 && num_pages > 0, TKV_ERR_INVALID, "pages_workspace: bad sizes B=%d num_pages=%d", B,
              num_pages);
  *words = 2LL * ((num_pages + 31) / 32) + 2LL * num_pages + 3LL * B + 4;
  return TKV_OK;
}

extern "C" int tkv_pages_fork(const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens,
                              int B_old, const int32_t* parents, const int32_t* reserve, int reserve0, int B,
                              int max_pages, int num_pages, int page_size, int32_t* new_table,
                              int32_t* new_lens, int32_t* missing, int32_t* workspace, void* const* pools,
                              const int64_t* page_bytes, int n_pools, void* stream) {
  using namespace tkv;
  TKV_REQUIRE(B >= 0 && B_old >= 0 && max_pages >= 0 && num_pages > 0 && page_size > 0, TKV_ERR_INVALID,
              "fork: bad sizes B=%d B_old=%d max_pages=%d num_pages=%d page_size=%d", B, B_old, max_pages,
              num_pages, page_size);
  TKV_REQUIRE((int64_t)max_pages * page_size < (1LL << 30) && (int64_t)B * max_pages < (1LL << 30), TKV_ERR_INVALID,
              "fork: a table of %d x %d pages of %d tokens is too large", B, max_pages, page_size);
  TKV_REQUIRE(missing && workspace, TKV_ERR_INVALID, "fork: null pointer");
  TKV_REQUIRE(B == 0 || (parents && new_lens), TKV_ERR_INVALID, "fork: null pointer");
  TKV_REQUIRE(B == 0 || max_pages == 0 || new_table, TKV_ERR_INVALID, "fork: null pointer");
  TKV_REQUIRE(B_old == 0 || ((block_table || max_pages == 0) && seq_lens), TKV_ERR_INVALID, "fork: null pointer");
  const int rc = check_pools("fork", pools, page_bytes, n_pools);
  if (rc != TKV_OK) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  const int words = (num_pages + 31) / 32;
  ForkArgs a{};
  a.table = block_table;
  a.lens = seq_lens;
  a.parents = parents;
  a.reserve = reserve;
  a.new_table = new_table;
  a.new_lens = new_lens;
  a.missing = missing;
  a.used = (uint32_t*)workspace;
  a.fresh = workspace + words;
  a.src = a.fresh + num_pages;
  a.dst = a.src + B;
  a.start = a.dst + B;
  a.table_stride = table_stride;
  a.reserve0 = reserve0;
  a.B_old = B_old;
  a.B = B;
  a.num_pages = num_pages;
  a.page = page_size;
  a.W = max_pages;
  TKV_CUDA(cudaMemsetAsync(a.used, 0, (size_t)words * 4, s));
  if (B > 0) {
    fork_mark_kernel<<<B, 128, 0, s>>>(a);
    TKV_CUDA(cudaGetLastError());
  }
  fork_assign_kernel<<<1, 1024, 0, s>>>(a);
  TKV_CUDA(cudaGetLastError());
  return launch_copy(pools, page_bytes, n_pools, a.src, a.dst, nullptr, B, s);
}

extern "C" int tkv_pages_compact(const int32_t* block_table, int64_t table_stride, int B, int max_pages,
                                 int num_pages, int32_t* new_table, int32_t* live, int32_t* workspace,
                                 void* const* pools, const int64_t* page_bytes, int n_pools, void* stream) {
  using namespace tkv;
  TKV_REQUIRE(B >= 0 && B < 65536 && max_pages >= 0 && num_pages > 0, TKV_ERR_INVALID,
              "compact: bad sizes B=%d (below 65536) max_pages=%d num_pages=%d", B, max_pages, num_pages);
  TKV_REQUIRE((int64_t)B * max_pages < (1LL << 30), TKV_ERR_INVALID, "compact: a table of %d x %d entries is too large",
              B, max_pages);
  TKV_REQUIRE(live && workspace, TKV_ERR_INVALID, "compact: null pointer");
  TKV_REQUIRE(B == 0 || max_pages == 0 || (block_table && new_table), TKV_ERR_INVALID, "compact: null pointer");
  const int rc = check_pools("compact", pools, page_bytes, n_pools);
  if (rc != TKV_OK) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  const int words = (num_pages + 31) / 32;
  CompactArgs a{};
  a.table = block_table;
  a.new_table = new_table;
  a.live = live;
  a.used = (uint32_t*)workspace;
  a.before = workspace + words;
  a.src = a.before + words;
  a.dst = a.src + num_pages;
  a.n_moves = a.dst + num_pages;
  a.table_stride = table_stride;
  a.B = B;
  a.W = max_pages;
  a.num_pages = num_pages;
  TKV_CUDA(cudaMemsetAsync(a.used, 0, (size_t)words * 4, s));
  const dim3 grid((max_pages + 255) / 256, B);
  if (B > 0 && max_pages > 0) {
    compact_mark_kernel<<<grid, 256, 0, s>>>(a);
    TKV_CUDA(cudaGetLastError());
  }
  compact_plan_kernel<<<1, 1024, 0, s>>>(a);
  TKV_CUDA(cudaGetLastError());
  if (B > 0 && max_pages > 0) {
    compact_table_kernel<<<grid, 256, 0, s>>>(a);
    TKV_CUDA(cudaGetLastError());
  }
  return launch_copy(pools, page_bytes, n_pools, a.src, a.dst, a.n_moves, num_pages, s);
}
