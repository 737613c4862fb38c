// Decode attention over a paged KV cache (sm_100a): packed 2/4-bit pages and float16 pages.
//
//     o_h = sum_n softmax_n(q_h . k_n * scale) v_n        over the n < seq_lens[b] of the table
//
// Token n of sequence b lies in row (block_table[b][n / page] * HKV + hkv) * page + n % page of a
// pool that has the layout of the contiguous cache with pages in the place of sequences.  Table
// entries outside the pool hold no tokens: theirs are not attended.
//
// The tiles, their arithmetic and the per-warp copy rings are those of the contiguous kernels
// (tkv_fused_policy.cuh, tkv_fp16_policy.cuh); what differs is where a tile comes from and how the
// work is cut.  A tile of 32 packed tokens is one run of rows where the page is a multiple of 32
// tokens, else two runs of 16 (PIECES: 64 sequences at 4 bits 57 us against 53.8 in one).  The lanes of a warp look
// up the pool rows of the warp's next 32 tiles, one each, across the segments to come; an issue takes
// its row by a shuffle, so the table's latency is paid once per 32 tiles, behind tiles in flight, and the
// tile loop holds no cursor (with one, 100 instructions a tile more).
//
// Lengths live on the device, so the plan is made there, by every CTA for itself: the prefix of the
// sequences' work in shared memory, then either
//   * whole (units -- sequence, KV head, 8 query heads -- at most half the CTAs): every unit has CTAs of its
//     own, ceil(t / TC) for t tiles with the smallest TC for which they suffice; or
//   * equal ranges of all work, whatever the lengths are; a range that crosses from one unit to the next is
//     processed segment by segment, and the switch counts as kSwitch tiles when the ranges are cut.
// A unit that one CTA has to itself goes straight to the output.  Else segment (unit u, CTA c) leaves
// its partial (acc, m, l) in slot u + c (whole: c) -- distinct for all segments, since the next unit
// starts no earlier than in the CTA where this one ends.  So the workspace holds units + CTAs partials
// whatever the lengths, and no slot has to be marked empty.  They are merged by the CTA that draws the unit's last
// ticket, or by a kernel of their own: see PagedLaunch::run.
//
// What is rounded: q to f16; the probabilities, formed in f32 against a running maximum, to f16 for
// the second product (on packed pages their sum counts the rounded ones, and they are rounded once
// more when the values' scale is multiplied in, since the codes are exact in f16 and the scales differ
// by token); the output once.  All sums are f32.  Against float64 the output is 3.1e-4 to 5.0e-4 off
// on packed pages and 2.5e-4 on float16 ones (2-norm), where rounding it to f16 alone is 2.0e-4.  The
// larger figure is that of one sequence of 65536: codes run from 0, so the mean of many tokens is a
// difference of two larger sums, of scale * code and of the zero points, and only the first has the
// second rounding in it.  Carrying the second rounding's error through a second product took 8-12 % with
// many tiles (64 sequences at 2 bits: 51.4 -> 57.7 us) for 2.4e-4.  Small weights and small values keep their
// bits (FusedPolicy::kTopMax, Fp16Policy::kTop): 4-bit values of 1/256 are as far off as values of 1, and the
// tokens beside one of weight 0.95 as those of a flat softmax.
//
// What bounds it: with many tiles the instructions of the tile loop (packed; about 600 a tile and warp) or the
// memory (float16: 32 sequences, 338 MB, 60.3 us, 5.6 TB/s); with few, the chain of latencies: lengths, table, first tile
// (3.3 us before it is asked for), 1.2 us a tile, the merge (2.5 us).
#include "tkv_fp16_policy.cuh"
#include "tkv_fused_policy.cuh"

namespace tkv {

constexpr float kNoReference = -1e30f;  // below every score: the softmax reference before the first token
constexpr int kFewUnits = 4;       // up to here the family of 8 warps, see few_units
constexpr int kFewPartials = 10;   // of a unit, about: up to here the CTA that finishes it merges them
constexpr int kTickets = 8192;     // units of a launch that can have a ticket
constexpr int kMaxPagedB = 512;    // sequences whose prefix a CTA holds; larger batches go in parts

struct PagedParams {
  DecodeParams d;         // what the tile policies read; d.B sequences of this launch
  const int32_t* table;
  int64_t table_stride;
  void* out;
  int out_dtype;
  int num_pages, page, HKVc;
  int whole;              // a CTA takes part of one unit only: how many a unit can have; 0: equal ranges of all tiles
  FastDiv dpage, dHch, dHKVc, dHQ, dgroup, dgrid;
  float *acc, *m, *l;     // (slots, 8, D), (slots, 8), (slots, 8)
  int2* info;             // (units): first slot and number of partials; none: the output is there
  uint32_t* tickets;      // (units), zero between calls: partials stored so far -- the last CTA merges; or null
};

__device__ __forceinline__ void store_out4(void* out, int dtype, int64_t i, float4 v) {
  if (dtype == TKV_DTYPE_F32) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + i) = v;
  } else if (dtype == TKV_DTYPE_F16) {
    *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(out) + i) = make_uint2(pack_half2(v.x, v.y), pack_half2(v.z, v.w));
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(out) + i) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
}

// What all lanes of a warp hold, said so that the compiler sees it: ring slots, cursor and barrier
// arithmetic that hangs off it can then go to the uniform datapath.
__device__ __forceinline__ int warp_uniform(int x) { return __shfl_sync(kFullMask, x, 0); }

// floor(a / b) by a float quotient, put right by at most one (a below 2^25, a quotient below 2^23)
__device__ __forceinline__ int small_div(int a, int b) {
  int q = (int)__fdividef((float)a, (float)b);
  const int r = a - q * b;
  if (r < 0) --q;
  else if (r >= b) ++q;
  return q;
}

// The work is cut in steps: a unit of t > 0 tiles takes kSwitch + t of them, since a CTA that goes from one
// unit to the next spends about as long as on kSwitch tiles (the merge of its warps, the next query's
// fragments, the pipeline run down and up again).  With 0 / 4 / 8 / 12 / 20: 40 sequences of 100-2000 tokens 28.8 /
// 23.7 / 22.4 / 22.2 / 22.4 us, 55 of 1000-4096 45.4 / 43.7 / 42.8 / 42.7 / 43.0, 64 at 2 bits 53.8 / 52.9 / 52.2 / 51.4 / 51.9;
// 200 of 20-500 53.3 / 36.0 / 31.9 / 32.1 with up to 12, and 64 of 4096 the same to 1 %.
// `pref`: word b = (steps of one head unit of the sequences before b) << kRemBits | tokens in its last tile - 1.
constexpr int kSwitch = 12;
__device__ __forceinline__ int unit_tiles(int steps) { return max(steps - kSwitch, 0); }
__device__ __forceinline__ int unit_steps(int tiles) { return tiles > 0 ? tiles + kSwitch : 0; }

// The part of a unit that a CTA processes.
struct PagedSegment {
  int b, hk;        // sequence; KV head and head chunk
  int hi, t_b;      // length of the sequence, tiles of the unit
  int lo_tile;      // first tile, within the unit
  int ntiles;
  int g_end;        // the step behind it
};

template <int kTok>
__device__ __forceinline__ void paged_segment_of(PagedSegment& s, const int* pref) {
  const int word = warp_uniform(pref[s.b]);
  s.t_b = unit_tiles(warp_uniform(pref[s.b + 1] >> kRemBits) - (word >> kRemBits));
  s.hi = (s.t_b - 1) * kTok + (word & ((1 << kRemBits) - 1)) + 1;
}
// The segment of steps [g, g1), g being a step of some unit.  By all lanes of a warp: two ballots find the
// sequence (the largest b with HKVc * pref[b] <= g; empty ones are skipped), 32 candidates at a time.
template <int kTok>
__device__ __forceinline__ PagedSegment paged_segment_at(const int* pref, int B, int HKVc, int g, int g1, int lane) {
  PagedSegment s;
  const int step = (B + 31) >> 5;  // at most kMaxPagedB / 32 = 16
  const int i = min(lane * step, B);
  const uint32_t coarse = __ballot_sync(kFullMask, i < B && HKVc * (pref[i] >> kRemBits) <= g);
  int lo = (31 - __clz(coarse)) * step;  // (pref[0] = 0: lane 0 always votes)
  if (step > 1) {
    const int k = min(lo + lane, B);
    lo += 31 - __clz(__ballot_sync(kFullMask, lane < step && k < B && HKVc * (pref[k] >> kRemBits) <= g));
  }
  s.b = warp_uniform(lo);
  paged_segment_of<kTok>(s, pref);
  const int r = g - HKVc * warp_uniform(pref[s.b] >> kRemBits), steps = s.t_b + kSwitch;
  s.hk = small_div(r, steps);
  const int at = r - s.hk * steps, len = min(g1 - g, steps - at);
  s.lo_tile = unit_tiles(at);
  s.ntiles = unit_tiles(at + len) - s.lo_tile;
  s.g_end = g + len;
  return s;
}
// The part of one unit that CTA `cta` takes where every unit has CTAs of its own, ceil(t / TC) of them for a unit
// of t tiles; `first` is the unit's first CTA and `count` how many it has.  false: nothing is left for this CTA.  By
// all lanes of a warp.
template <int kTok>
__device__ __forceinline__ bool paged_segment_whole(PagedSegment& s, const int* pref, int B, int HKVc, int TC, int cta,
                                                    int lane, int& first, int& count) {
  int carry = 0;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int b = min(b0 + lane, B - 1), t = unit_tiles((pref[b + 1] >> kRemBits) - (pref[b] >> kRemBits));
    const int n = b0 + lane < B ? small_div(t + TC - 1, TC) : 0, ctas = n * HKVc;
    int incl = ctas;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(kFullMask, incl, off);
      if (lane >= off) incl += y;
    }
    const uint32_t behind = __ballot_sync(kFullMask, carry + incl > cta);
    if (behind) {
      const int l = __ffs(behind) - 1;
      count = warp_uniform(__shfl_sync(kFullMask, n, l));
      first = carry + warp_uniform(__shfl_sync(kFullMask, incl - ctas, l));
      s.b = warp_uniform(b0 + l);
      s.hk = warp_uniform(small_div(cta - first, count));
      first += s.hk * count;
      paged_segment_of<kTok>(s, pref);
      const int j = cta - first, q = warp_uniform(small_div(s.t_b, count)), rem = s.t_b - q * count;
      s.lo_tile = j * q + min(j, rem);
      s.ntiles = q + (j < rem ? 1 : 0);
      s.g_end = 0;
      return true;
    }
    carry += warp_uniform(__shfl_sync(kFullMask, incl, 31));
  }
  return false;
}
// Whether steps up to g1 reach into the unit behind a segment, and the segment there
__device__ __forceinline__ bool paged_segment_more(const PagedSegment& s, int g1) { return g1 - s.g_end > kSwitch; }
template <int kTok>
__device__ __forceinline__ void paged_segment_next(PagedSegment& s, const int* pref, int HKVc, int g1) {
  s.lo_tile = 0;
  if (++s.hk == HKVc) {
    s.hk = 0;
    do ++s.b;
    while (warp_uniform(pref[s.b + 1] >> kRemBits) == warp_uniform(pref[s.b] >> kRemBits));
    paged_segment_of<kTok>(s, pref);
  }
  s.ntiles = min(g1 - s.g_end - kSwitch, s.t_b);
  s.g_end += s.ntiles + kSwitch;
}

// Where a warp's copies stand, segments ahead of the one being computed.  Kept in shared memory: only
// the look-up of the next 32 tiles needs it.
struct PagedCursor {
  PagedSegment seg;
  int tile;  // the warp's next tile, within the segment
};
// A tile's place as one word: (pool row / 16) << 5 | tokens - 1, or all ones where it has none.
constexpr uint32_t kNoPlace = 0xffffffffu;
__device__ __forceinline__ uint32_t place_word(int row, int tokens) {
  return ((uint32_t)row >> 4) << 5 | (uint32_t)(tokens - 1);
}

// The merge of a unit's n partials (slot rows r0, r0 + 8, ...) by one whole CTA: kMergeAtOnce of them in flight,
// a running maximum over more.
constexpr int kMergeAtOnce = 8;
template <int D, int THREADS>
__device__ __forceinline__ void paged_merge_unit(const PagedParams& pp, int64_t r0, int n, int b, int hk) {
  constexpr int D4 = D / 4, ITEMS = kHeadsPerCta * D4, ROUNDS = (ITEMS + THREADS - 1) / THREADS;
  __shared__ float s_pm[kMergeAtOnce * kHeadsPerCta], s_pl[kMergeAtOnce * kHeadsPerCta];
  const DecodeParams& p = pp.d;
  float4 a[ROUNDS];
  float L[ROUNDS], M[ROUNDS];
#pragma unroll
  for (int it = 0; it < ROUNDS; ++it) {
    a[it] = make_float4(0.f, 0.f, 0.f, 0.f);
    L[it] = 0.f;
    M[it] = -INFINITY;
  }
  for (int s0 = 0; s0 < n; s0 += kMergeAtOnce) {
    float4 x[ROUNDS][kMergeAtOnce];
#pragma unroll
    for (int it = 0; it < ROUNDS; ++it) {
      const int idx = it * THREADS + threadIdx.x;
#pragma unroll
      for (int j = 0; j < kMergeAtOnce; ++j)
        x[it][j] = idx < ITEMS && s0 + j < n
                       ? __ldcg(reinterpret_cast<const float4*>(pp.acc + (r0 + (s0 + j) * kHeadsPerCta) * D) + idx)
                       : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const bool there = threadIdx.x < kMergeAtOnce * kHeadsPerCta && s0 + (int)threadIdx.x / kHeadsPerCta < n;
    const float m = there ? __ldcg(pp.m + r0 + s0 * kHeadsPerCta + threadIdx.x) : -INFINITY;
    const float l = there ? __ldcg(pp.l + r0 + s0 * kHeadsPerCta + threadIdx.x) : 0.f;
    __syncthreads();
    if (threadIdx.x < kMergeAtOnce * kHeadsPerCta) {
      s_pm[threadIdx.x] = m;
      s_pl[threadIdx.x] = l;
    }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < ROUNDS; ++it) {
      const int h = min(it * THREADS + (int)threadIdx.x, ITEMS - 1) / D4;
      float top = M[it];
#pragma unroll
      for (int j = 0; j < kMergeAtOnce; ++j) top = fmaxf(top, s_pm[j * kHeadsPerCta + h]);
      const float old = M[it] > -INFINITY ? ex2(M[it] - top) : 0.f;
      L[it] *= old;
      a[it].x *= old;
      a[it].y *= old;
      a[it].z *= old;
      a[it].w *= old;
      M[it] = top;
#pragma unroll
      for (int j = 0; j < kMergeAtOnce; ++j) {
        const float mj = s_pm[j * kHeadsPerCta + h], w = mj > -INFINITY ? ex2(mj - top) : 0.f;
        L[it] = fmaf(w, s_pl[j * kHeadsPerCta + h], L[it]);
        a[it].x = fmaf(w, x[it][j].x, a[it].x);
        a[it].y = fmaf(w, x[it][j].y, a[it].y);
        a[it].z = fmaf(w, x[it][j].z, a[it].z);
        a[it].w = fmaf(w, x[it][j].w, a[it].w);
      }
    }
  }
  const int hkv = fast_div(hk, pp.dHch), hc = hk - hkv * p.hchunks;
#pragma unroll
  for (int it = 0; it < ROUNDS; ++it) {
    const int idx = it * THREADS + threadIdx.x, h = idx / D4, hg = hc * kHeadsPerCta + h;
    if (idx < ITEMS && hg < p.group) {
      const float inv = L[it] > 0.f ? 1.f / L[it] : 0.f;
      store_out4(pp.out, pp.out_dtype, ((int64_t)b * p.HQ + hkv * p.group + hg) * D + (idx - h * D4) * 4,
                 make_float4(a[it].x * inv, a[it].y * inv, a[it].z * inv, a[it].w * inv));
    }
  }
}

template <class Policy>
__global__ void __launch_bounds__(Policy::WARPS * 32, Policy::MIN_CTAS)
    paged_split_kernel(const __grid_constant__ typename Policy::Maps maps, const PagedParams pp) {
  constexpr int WARPS = Policy::WARPS, STAGES = Policy::STAGES, D = Policy::D, PIECES = Policy::PIECES;
  constexpr int kTok = Policy::TOK, STAGE_BYTES = Policy::STAGE_BYTES;
  constexpr int kLog2D = D == 64 ? 6 : 7;
  static_assert((1 << kLog2D) == D && STAGES >= (Policy::PIPELINED ? 3 : 2) && STAGE_BYTES % 1024 == 0 &&
                    STAGE_BYTES >= kHeadsPerCta * D * 4 && STAGES * 2 <= 32,
                "a ring of whole swizzle atoms that holds a warp's partial, two tiles resident or one");
  const DecodeParams& p = pp.d;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ float s_m[WARPS][kHeadsPerCta];
  __shared__ float s_l[WARPS][kHeadsPerCta];
  __shared__ int s_slot[WARPS], s_tiles[WARPS];
  __shared__ PagedCursor s_cursor[WARPS];
  // units that this CTA shares with others: its first and its last at most
  struct Shared {
    int b, hk, slot, count;  // first slot, number of partials
    uint32_t ticket;
  };
  __shared__ Shared s_shared[2];
  int n_shared = 0;
  uint32_t ticket[2] = {0, 0};  // (thread 0)
  const int warp = __shfl_sync(kFullMask, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int cta = blockIdx.x;
  pdl_launch_dependents();  // the whole grid is resident: the merge may take its place and wait
  if (threadIdx.x == 0) Policy::prefetch_maps(maps);

  uint8_t* ring = smem + (size_t)warp * STAGES * STAGE_BYTES;
  const uint32_t ring_u32 = smem_u32(ring);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (size_t)WARPS * STAGES * STAGE_BYTES);
  const uint32_t bar_u32 = smem_u32(bars + warp * STAGES);
  constexpr int QB = kHeadsPerCta * D * 4;  // query rows of a segment, staged one segment ahead
  uint64_t* qbars = bars + WARPS * STAGES;
  const uint32_t qbar_u32 = smem_u32(qbars);
  uint8_t* qbuf = reinterpret_cast<uint8_t*>(qbars + 2);
  const uint32_t qbuf_u32 = smem_u32(qbuf);
  const uint32_t qfrag_u32 = qbuf_u32 + 2 * QB;
  int* s_pref = reinterpret_cast<int*>(qbuf + 2 * QB + ((Policy::QFRAG_BYTES + 15) & ~15));
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) mbar_init(bar_u32 + 8 * s, Policy::BAR_COUNT);
    if (warp == 0) {
      mbar_init(qbar_u32, WARPS * 32);
      mbar_init(qbar_u32 + 8, WARPS * 32);
    }
    fence_barrier_init();
  }
  const int q_esz = p.q_dtype == TKV_DTYPE_F32 ? 4 : 2;
  auto prefetch_q = [&](int slot, const PagedSegment& s) {
    const int s_hkv = fast_div(s.hk, pp.dHch), s_hc = s.hk - s_hkv * p.hchunks;
    const int row_bytes = D * q_esz, cpr = row_bytes >> 4, cpr_shift = q_esz == 4 ? kLog2D - 2 : kLog2D - 3;
    for (int i = threadIdx.x; i < kHeadsPerCta * cpr; i += WARPS * 32) {
      const int h = i >> cpr_shift, c = i - (h << cpr_shift);
      const int hg = s_hc * kHeadsPerCta + h;
      const bool ok = hg < p.group;
      const uint8_t* src = reinterpret_cast<const uint8_t*>(p.q) +
                           (((int64_t)s.b * p.HQ + (int64_t)s_hkv * p.group + hg) * D) * q_esz + c * 16;
      cp_async16(qbuf_u32 + slot * QB + h * row_bytes + c * 16,
                 ok ? src : reinterpret_cast<const uint8_t*>(p.q), ok ? 16 : 0);
    }
    cp_async_mbar_arrive_noinc(qbar_u32 + 8 * slot);
  };
  typename Policy::IssueState ist;
  Policy::issue_init(ist, p, lane);
  typename Policy::Query qs;
  Policy::lane_init(qs, p, lane);

  // ---- the steps of the sequences, one after the other ----
  pdl_wait();
  int total_tiles = 0;
  {
    constexpr int K = kMaxPagedB / (32 * WARPS);  // blocks of 32 sequences that a warp may have to take
    const int blocks = (p.B + 31) >> 5, per_warp = (blocks + WARPS - 1) / WARPS, b0 = warp * per_warp * 32;
    int len[K], before[K], sum = 0, tiles = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int b = b0 + k * 32 + lane;
      len[k] = k < per_warp && b < p.B ? min(max(p.seq_lens[b], 0), p.S) : 0;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k >= per_warp) break;
      const int t = unit_steps((len[k] + kTok - 1) / kTok);
      int incl = t;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(kFullMask, incl, off);
        if (lane >= off) incl += y;
      }
      before[k] = sum + incl - t;
      sum += __shfl_sync(kFullMask, incl, 31);
      tiles += unit_tiles(t);
    }
    tiles = __reduce_add_sync(kFullMask, (unsigned)tiles);
    if (lane == 0) {
      s_slot[warp] = sum;
      s_tiles[warp] = tiles;
    }
    __syncthreads();
    int base = 0, total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      base += w < warp ? s_slot[w] : 0;
      total += s_slot[w];
      total_tiles += s_tiles[w];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int b = b0 + k * 32 + lane;
      if (k < per_warp && b < p.B)
        s_pref[b] = ((base + before[k]) << kRemBits) | (len[k] > 0 ? (len[k] - 1) % kTok : 0);
    }
    if (threadIdx.x == 0) s_pref[p.B] = total << kRemBits;
  }
  __syncthreads();
  const int T = pp.HKVc * warp_uniform(s_pref[p.B] >> kRemBits);
  int TC = max(1, fast_div(T + (int)gridDim.x - 1, pp.dgrid));
  int g0, g1, whole_first = 0, whole_count = 0;
  PagedSegment seg;
  if (pp.whole) {
    if (p.B == 1) {
      TC = max(1, small_div(unit_tiles(s_pref[1] >> kRemBits) + pp.whole - 1, pp.whole));
    } else {
      // the smallest TC for which the CTAs are enough, of PER * WARPS candidates from an even share up to twice that
      constexpr int PER = 4;
      TC = max(1, fast_div(pp.HKVc * warp_uniform(total_tiles) + (int)gridDim.x - 1, pp.dgrid));
      int mine[PER], ctas[PER], best = 1 << 24;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        mine[k] = TC + small_div(TC * (k * WARPS + warp) + PER * WARPS - 2, PER * WARPS - 1);
        ctas[k] = 0;
      }
      for (int b = lane; b < p.B; b += 32) {
        const int t = unit_tiles((s_pref[b + 1] >> kRemBits) - (s_pref[b] >> kRemBits));
#pragma unroll
        for (int k = 0; k < PER; ++k) ctas[k] += small_div(t + mine[k] - 1, mine[k]);
      }
#pragma unroll
      for (int k = PER - 1; k >= 0; --k)
        if ((int)__reduce_add_sync(kFullMask, (unsigned)ctas[k]) * pp.HKVc <= (int)gridDim.x) best = mine[k];
      __syncthreads();  // (s_slot still holds the warps' sums)
      if (lane == 0) s_slot[warp] = best;
      __syncthreads();
      TC = s_slot[0];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) TC = min(TC, s_slot[w]);
      TC = warp_uniform(TC);
    }
    if (TC <= 4 * WARPS) TC = (TC + WARPS - 1) / WARPS * WARPS;  // no warp without a tile: fewer partials, same time
    g0 = g1 = 0;
    if (!paged_segment_whole<kTok>(seg, s_pref, p.B, pp.HKVc, TC, cta, lane, whole_first, whole_count)) seg.ntiles = 0;
  } else {
    g0 = min(cta * TC, T);
    g1 = min(g0 + TC, T);
    seg.ntiles = 0;
    if (g0 < g1) seg = paged_segment_at<kTok>(s_pref, p.B, pp.HKVc, g0, g1, lane);
  }
  // sequences without tokens are touched by no range
  auto empty_units = [&]() {
    for (int u = cta; u < p.B * pp.HKVc; u += gridDim.x) {
      const int b = fast_div(u, pp.dHKVc), hk = u - b * pp.HKVc;
      if ((s_pref[b + 1] >> kRemBits) != (s_pref[b] >> kRemBits)) continue;
      const int hkv = fast_div(hk, pp.dHch), hc = hk - hkv * p.hchunks;
      for (int idx = threadIdx.x; idx < kHeadsPerCta * D / 4; idx += WARPS * 32) {
        const int h = idx / (D / 4), d = (idx - h * (D / 4)) * 4, hg = hc * kHeadsPerCta + h;
        if (hg < p.group)
          store_out4(pp.out, pp.out_dtype, ((int64_t)b * p.HQ + hkv * p.group + hg) * D + d, make_float4(0.f, 0.f, 0.f, 0.f));
      }
      if (threadIdx.x == 0 && !pp.tickets) pp.info[u] = make_int2(0, 0);
    }
  };
  if (seg.ntiles == 0) {
    empty_units();
    return;
  }

  // ---- the warp's next 32 tiles, across segments: lane i has the place of the i-th ----
  PagedCursor* my_cursor = &s_cursor[warp];
  uint32_t place[PIECES];
  int k_next = 0, n_listed = 0;  // the tile to issue next, and how many there are
  auto look_up = [&](PagedCursor cur) {
    k_next = n_listed = 0;
#pragma unroll
    for (int h = 0; h < PIECES; ++h) place[h] = kNoPlace;
    for (;;) {
      const int cnt = cur.seg.ntiles > cur.tile ? (cur.seg.ntiles - cur.tile + WARPS - 1) / WARPS : 0;
      const int take = min(cnt, 32 - n_listed), i = lane - n_listed;
      if (i >= 0 && i < take) {
        const int tok = (cur.seg.lo_tile + cur.tile + i * WARPS) * kTok, hkv = fast_div(cur.seg.hk, pp.dHch);
#pragma unroll
        for (int h = 0; h < PIECES; ++h) {
          const int n = tok + h * (kTok / PIECES);
          if (n < cur.seg.hi) {
            const int e = fast_div(n, pp.dpage), id = __ldcg(pp.table + cur.seg.b * pp.table_stride + e);
            if ((unsigned)id < (unsigned)pp.num_pages)
              place[h] = place_word((id * p.HKV + hkv) * pp.page + (n - e * pp.page), min(kTok, cur.seg.hi - tok));
          }
        }
      }
      n_listed += take;
      cur.tile += take * WARPS;
      if (n_listed == 32 || !paged_segment_more(cur.seg, g1)) break;
      paged_segment_next<kTok>(cur.seg, s_pref, pp.HKVc, g1);
      cur.tile = warp;
    }
    __syncwarp();
    if (lane == 0) *my_cursor = cur;
  };
  look_up(PagedCursor{seg, warp});
  int iss_slot = 0;          // slot the next issue fills
  uint32_t valid = 0;        // bits [s*PIECES, (s+1)*PIECES): which pieces of slot s name a page
  constexpr uint32_t kAll = (1u << PIECES) - 1u;
  bool need_proxy_fence = false;
  auto issue_next = [&]() {
    if (k_next >= n_listed) return;
    const int slot = iss_slot;
    iss_slot = (slot + 1 == STAGES) ? 0 : slot + 1;
    if (need_proxy_fence) {  // a generic-proxy epilogue touched the ring since the last issue
      fence_proxy_async();
      need_proxy_fence = false;
    }
    int rows[PIECES], tokens = kTok;
    uint32_t ok = 0;
#pragma unroll
    for (int h = 0; h < PIECES; ++h) {
      const uint32_t w = __shfl_sync(kFullMask, place[h], k_next);
      const bool there = w != kNoPlace;
      rows[h] = there ? (int)(w >> 5 << 4) : -1;
      if (there) tokens = (int)(w & 31u) + 1;
      ok |= (there ? 1u : 0u) << h;
    }
    valid = (valid & ~(kAll << (slot * PIECES))) | (ok << (slot * PIECES));
    Policy::issue_pieces(ist, p, maps, rows, tokens, ring_u32 + slot * STAGE_BYTES, bar_u32 + 8 * slot, lane);
    if (++k_next == 32) {
      __syncwarp();
      look_up(*my_cursor);
    }
  };
  prefetch_q(0, seg);
#pragma unroll 1
  for (int s = 0; s < (Policy::PIPELINED ? STAGES - 1 : STAGES); ++s) issue_next();
  empty_units();
  if (paged_segment_more(seg, g1)) {
    PagedSegment s = seg;
    paged_segment_next<kTok>(s, s_pref, pp.HKVc, g1);
    prefetch_q(1, s);
  }
  int seg_k = 0;  // index of the current segment within this CTA
  int c_slot = 0, c_phase = 0;  // slot and barrier phase of the next tile to consume
  bool timed_out = false;
  typename Policy::Accum acc;

  for (;;) {
    // ---- one segment ----
    if (!mbar_wait_bounded(qbar_u32 + 8 * (seg_k & 1), (seg_k >> 1) & 1)) timed_out = true;
    if (Policy::QFRAG_BYTES > 0) {
      Policy::build_query(p, qbuf + (seg_k & 1) * QB, qfrag_u32, warp, lane);
      __syncthreads();
    }
    Policy::load_query(qs, p, qbuf + (seg_k & 1) * QB, qfrag_u32, lane);
    Policy::reset(acc);
    // (finite, so that a first tile without any token is exp2(-inf) = 0 like any other masked one)
    acc.m_ref0 = acc.m_ref1 = acc.p_ref0 = acc.p_ref1 = kNoReference;
    const int my_tiles = seg.ntiles > warp ? (seg.ntiles - warp + WARPS - 1) / WARPS : 0;
    int left = seg.hi - (seg.lo_tile + warp) * kTok;
    auto scores = [&](typename Policy::Scores& sc, int slot, int left_of) {
      Policy::scores(sc, qs, ring_u32 + slot * STAGE_BYTES, ring + slot * STAGE_BYTES, kTok, p.qk_scale, lane);
      const uint32_t v = valid >> (slot * PIECES) & kAll;
      if (left_of < kTok || v != kAll) Policy::mask_tokens(sc, left_of, v, lane);
    };
    auto update = [&](typename Policy::Scores& sc, int slot) {
      Policy::update(acc, qs, sc, ring_u32 + slot * STAGE_BYTES, ring + slot * STAGE_BYTES, left, lane);
    };
    if (!Policy::PIPELINED) {
      // One tile at a time; its stage is refilled as soon as it is finished -- after the segment's
      // last tile, which carries the warp's partial, behind the epilogue.
      for (int i = 0; i < my_tiles; ++i) {
        if (!mbar_wait_bounded(bar_u32 + 8 * c_slot, c_phase)) {
          timed_out = true;
          break;
        }
        __syncwarp();
        typename Policy::Scores sc;
        scores(sc, c_slot, left);
        update(sc, c_slot);
        left -= WARPS * kTok;
        if (++c_slot == STAGES) {
          c_slot = 0;
          c_phase ^= 1;
        }
        __syncwarp();
        if (i + 1 < my_tiles) issue_next();
      }
    } else if (my_tiles > 0 && !timed_out) {
      // Software pipeline: the scores of tile i+1 beside the softmax and output of tile i.
      typename Policy::Scores sc_cur;
      if (!mbar_wait_bounded(bar_u32 + 8 * c_slot, c_phase)) timed_out = true;
      __syncwarp();
      if (!timed_out) scores(sc_cur, c_slot, left);
      for (int i = 1; i < my_tiles && !timed_out; ++i) {
        int n_slot = c_slot + 1, n_phase = c_phase;
        if (n_slot == STAGES) {
          n_slot = 0;
          n_phase ^= 1;
        }
        if (!mbar_wait_bounded(bar_u32 + 8 * n_slot, n_phase)) {
          timed_out = true;
          break;
        }
        __syncwarp();
        issue_next();  // refills the stage whose tile was finished in the previous iteration
        typename Policy::Scores sc_next;
        scores(sc_next, n_slot, left - WARPS * kTok);
        update(sc_cur, c_slot);
        sc_cur = sc_next;
        left -= WARPS * kTok;
        c_slot = n_slot;
        c_phase = n_phase;
      }
      if (!timed_out) {
        __syncwarp();
        issue_next();
        update(sc_cur, c_slot);
        if (++c_slot == STAGES) {
          c_slot = 0;
          c_phase ^= 1;
        }
      }
    }

    // ---- merge the warps, store the partial or the output ----
    bool shared_unit = false;
    const int vals_slot = (c_slot == 0 ? STAGES : c_slot) - 1;  // the stage consumed last
    SoftmaxState st{-INFINITY, -INFINITY, 0.f, 0.f};
    if (my_tiles > 0) Policy::finalize(acc, reinterpret_cast<float*>(ring + vals_slot * STAGE_BYTES), st, lane);
    if ((lane >> 2) == 0) {
      const int t = lane & 3;
      s_m[warp][2 * t] = st.m0;
      s_m[warp][2 * t + 1] = st.m1;
      s_l[warp][2 * t] = st.l0;
      s_l[warp][2 * t + 1] = st.l1;
    }
    if (lane == 0) s_slot[warp] = vals_slot;
    __syncthreads();
    {
      constexpr int D4 = D / 4, ITEMS = kHeadsPerCta * D4;
      uint32_t voff[WARPS];
#pragma unroll
      for (int w = 0; w < WARPS; ++w) voff[w] = (uint32_t)((w * STAGES + s_slot[w]) * STAGE_BYTES);
      const int hkv = fast_div(seg.hk, pp.dHch), hc = seg.hk - hkv * p.hchunks;
      const int unit = seg.b * pp.HKVc + seg.hk;
      // the CTAs of the unit, and the slot of this one's partial: distinct, since the next unit begins no
      // earlier than in the CTA where this one ends, or the CTA's own where it has one unit only
      int first = whole_first, count = whole_count, slot0 = 0;
      if (!pp.whole) {  // (only a unit that crosses a border of this CTA's range takes a division)
        const int u0 = pp.HKVc * (s_pref[seg.b] >> kRemBits) + seg.hk * (seg.t_b + kSwitch), u1 = u0 + kSwitch + seg.t_b;
        first = seg.lo_tile == 0 ? cta : (int)((uint32_t)(u0 + kSwitch) / (uint32_t)TC);
        count = (u1 <= g1 ? cta : (int)((uint32_t)(u1 - 1) / (uint32_t)TC)) - first + 1;
        slot0 = unit;
      }
      const int64_t slot = (int64_t)(slot0 + cta) * kHeadsPerCta;
#pragma unroll
      for (int it = 0; it < (ITEMS + WARPS * 32 - 1) / (WARPS * 32); ++it) {
        const int idx = it * (WARPS * 32) + threadIdx.x;
        if (ITEMS % (WARPS * 32) != 0 && idx >= ITEMS) break;
        const int h = idx / D4, d = (idx - h * D4) * 4, hg = hc * kHeadsPerCta + h;
        if (hg >= p.group) continue;
        float mw[WARPS], M = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          mw[w] = s_m[w][h];
          M = fmaxf(M, mw[w]);
        }
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const bool live = mw[w] != -INFINITY;  // a warp without tiles left its stage unwritten
          const float s = live ? ex2(mw[w] - M) : 0.f;
          const float4 v = *reinterpret_cast<const float4*>(smem + voff[w] + (h * D + d) * 4);
          a.x = fmaf(s, live ? v.x : 0.f, a.x);
          a.y = fmaf(s, live ? v.y : 0.f, a.y);
          a.z = fmaf(s, live ? v.z : 0.f, a.z);
          a.w = fmaf(s, live ? v.w : 0.f, a.w);
          L = fmaf(s, s_l[w][h], L);
        }
        if (count > 1) {
          *reinterpret_cast<float4*>(pp.acc + (slot + h) * D + d) = a;
          if (d == 0) {
            pp.m[slot + h] = M;
            pp.l[slot + h] = L;
          }
        } else {
          const float inv = L > 0.f ? 1.f / L : 0.f;
          store_out4(pp.out, pp.out_dtype, ((int64_t)seg.b * p.HQ + hkv * p.group + hg) * D + d,
                     make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
        }
      }
      if (!pp.tickets) {
        if (threadIdx.x == 0 && first == cta) pp.info[unit] = count > 1 ? make_int2(slot0 + cta, count) : make_int2(0, 0);
      } else if (count > 1 && threadIdx.x == 0) {
        s_shared[n_shared] = Shared{seg.b, seg.hk, slot0 + first, count, 0};
      }
      shared_unit = count > 1;
    }
    __syncthreads();
    // This CTA's partial is stored: draw the unit's ticket.  Nobody waits for it before the end, so that the
    // answer travels while the next segment runs.
    if (pp.tickets && shared_unit) {
      if (threadIdx.x == 0) {
        __threadfence();
        const uint32_t t = atomicAdd(pp.tickets + seg.b * pp.HKVc + seg.hk, 1u);
        if (n_shared == 0) ticket[0] = t;
        else ticket[1] = t;
      }
      ++n_shared;
    }
    need_proxy_fence = true;
    if (!paged_segment_more(seg, g1) || timed_out) break;
    if (!Policy::PIPELINED && my_tiles > 0) issue_next();
    paged_segment_next<kTok>(seg, s_pref, pp.HKVc, g1);
    if (paged_segment_more(seg, g1)) {  // the query slot just released takes the segment after the next
      PagedSegment s = seg;
      paged_segment_next<kTok>(s, s_pref, pp.HKVc, g1);
      prefetch_q(seg_k & 1, s);
    }
    ++seg_k;
  }
  if (timed_out) {
    if (lane == 0) Policy::report_timeout();
    drain_ring<STAGES>(bar_u32, c_slot, c_phase);
  }
  if (n_shared == 0) return;
  if (threadIdx.x == 0) {
    s_shared[0].ticket = ticket[0];
    s_shared[1].ticket = ticket[1];
  }
  __syncthreads();
  for (int i = 0; i < n_shared; ++i) {
    if (s_shared[i].ticket != (uint32_t)s_shared[i].count - 1u) continue;  // others are still to come
    __threadfence();
    if (threadIdx.x == 0) pp.tickets[s_shared[i].b * pp.HKVc + s_shared[i].hk] = 0;
    paged_merge_unit<D, WARPS * 32>(pp, (int64_t)s_shared[i].slot * kHeadsPerCta, s_shared[i].count, s_shared[i].b,
                                    s_shared[i].hk);
  }
}

// ---------------------------------------------------------------- merge of a unit's partials
//     out = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M),   M = max_s m_s
// Bound by latency: where the partials are (one load), then maxima, sums and the first partials in one
// go.  A partial without tokens has m = -inf, weighs 0 and holds zeros.

// Where the partials of row (sequence, query head) are: first slot row and how many; 0: nothing to do.
__device__ __forceinline__ int2 paged_partials(const PagedParams& pp, int row) {
  const DecodeParams& p = pp.d;
  const int b = fast_div(row, pp.dHQ), hq = row - b * p.HQ, hkv = fast_div(hq, pp.dgroup), hg = hq - hkv * p.group;
  const int2 at = __ldcg(pp.info + b * pp.HKVc + hkv * p.hchunks + hg / kHeadsPerCta);
  return make_int2(at.x * kHeadsPerCta + hg % kHeadsPerCta, at.y);
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor_sync(kFullMask, x, off));
  return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) x += __shfl_xor_sync(kFullMask, x, off);
  return x;
}
__device__ __forceinline__ void fma4(float4& a, float w, const float4& x) {
  a.x = fmaf(w, x.x, a.x);
  a.y = fmaf(w, x.y, a.y);
  a.z = fmaf(w, x.z, a.z);
  a.w = fmaf(w, x.w, a.w);
}

// Many rows of few partials each: a warp per row, 128 / D partials at a time.
template <int D>
__global__ void __launch_bounds__(256) paged_merge_rows_kernel(const PagedParams pp, int rows) {
  constexpr int PAR = 128 / D, AHEAD = 4;
  const int lane = threadIdx.x & 31, row = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int sub = lane / (32 / PAR), d = lane % (32 / PAR) * 4;
  pdl_wait();
  if (row < rows) {
    const int2 at = paged_partials(pp, row);
    const int n = at.y;
    if (n > 0) {
      const float* acc = pp.acc + (int64_t)at.x * D + d;
      float4 x[AHEAD], a = make_float4(0.f, 0.f, 0.f, 0.f);
      auto fetch = [&](int s0) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int s = s0 + i * PAR + sub;
          x[i] = s < n ? __ldcg(reinterpret_cast<const float4*>(acc + (int64_t)s * (kHeadsPerCta * D))) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      };
      fetch(0);
      float m = lane < n ? __ldcg(pp.m + at.x + lane * kHeadsPerCta) : -INFINITY;
      float l = lane < n ? __ldcg(pp.l + at.x + lane * kHeadsPerCta) : 0.f;
      float M = m;
      for (int s = 32 + lane; s < n; s += 32) M = fmaxf(M, __ldcg(pp.m + at.x + s * kHeadsPerCta));
      M = warp_max(M);
      float L = 0.f;
      for (int s0 = 0; s0 < n; s0 += 32) {  // weights of 32 partials, a lane each
        if (s0 > 0) {
          m = s0 + lane < n ? __ldcg(pp.m + at.x + (s0 + lane) * kHeadsPerCta) : -INFINITY;
          l = s0 + lane < n ? __ldcg(pp.l + at.x + (s0 + lane) * kHeadsPerCta) : 0.f;
        }
        const float w = m > -INFINITY ? ex2(m - M) : 0.f;
        L = fmaf(w, l, L);
        for (int s1 = s0; s1 < min(n, s0 + 32); s1 += AHEAD * PAR) {
          if (s1 > 0) fetch(s1);
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) fma4(a, __shfl_sync(kFullMask, w, (s1 - s0 + i * PAR + sub) & 31), x[i]);
        }
      }
      L = warp_sum(L);
      if constexpr (PAR == 2) {
        a.x += __shfl_xor_sync(kFullMask, a.x, 16);
        a.y += __shfl_xor_sync(kFullMask, a.y, 16);
        a.z += __shfl_xor_sync(kFullMask, a.z, 16);
        a.w += __shfl_xor_sync(kFullMask, a.w, 16);
      }
      const float inv = L > 0.f ? 1.f / L : 0.f;
      if (sub == 0)
        store_out4(pp.out, pp.out_dtype, (int64_t)row * D + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
    }
  }
  pdl_launch_dependents();  // the balanced kernel of the next step wants its SMs free: only now
}

// Few rows of many partials: a CTA per 32 dims of a row, 32 groups of 8 threads over the partials.
template <int D>
__global__ void __launch_bounds__(256) paged_merge_long_kernel(const PagedParams pp) {
  constexpr int kAtOnce = 256, PER = kAtOnce / 32;  // partials in flight, of a thread
  __shared__ float s_w[kAtOnce], s_red[8], s_sum[8];
  __shared__ float4 s_acc[8][8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x;
  const int g = tid >> 3, d = blockIdx.y * 32 + (tid & 7) * 4;
  pdl_launch_dependents();
  pdl_wait();
  const int2 at = paged_partials(pp, row);
  const int n = at.y;
  if (n == 0) return;
  const float* acc = pp.acc + (int64_t)at.x * D + d;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float L = 0.f, M = -INFINITY;
  for (int s0 = 0; s0 < n; s0 += kAtOnce) {
    float4 x[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = s0 + i * 32 + g;
      x[i] = s < n ? __ldcg(reinterpret_cast<const float4*>(acc + (int64_t)s * (kHeadsPerCta * D))) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float m = s0 + tid < n ? __ldcg(pp.m + at.x + (s0 + tid) * kHeadsPerCta) : -INFINITY;
    const float l = s0 + tid < n ? __ldcg(pp.l + at.x + (s0 + tid) * kHeadsPerCta) : 0.f;
    const float mw = warp_max(m);
    if (lane == 0) s_red[warp] = mw;
    __syncthreads();
    float top = M;
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, s_red[w]);
    const float w = m > -INFINITY ? ex2(m - top) : 0.f;
    s_w[tid] = w;
    const float old = M > -INFINITY ? ex2(M - top) : 0.f;  // (more than kAtOnce partials: a running maximum)
    L = fmaf(L, old, w * l);
    a.x *= old;
    a.y *= old;
    a.z *= old;
    a.w *= old;
    M = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) fma4(a, s_w[i * 32 + g], x[i]);
  }
  L = warp_sum(L);
#pragma unroll
  for (int off = 8; off <= 16; off <<= 1) {  // the 4 groups of a warp
    a.x += __shfl_xor_sync(kFullMask, a.x, off);
    a.y += __shfl_xor_sync(kFullMask, a.y, off);
    a.z += __shfl_xor_sync(kFullMask, a.z, off);
    a.w += __shfl_xor_sync(kFullMask, a.w, off);
  }
  if (lane < 8) s_acc[warp][lane] = a;
  if (lane == 0) s_sum[warp] = L;
  __syncthreads();
  if (tid < 8) {
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      fma4(a, 1.f, s_acc[w][tid]);
      L += s_sum[w];
    }
    L = __shfl_sync(0xffu, L, 0);
    const float inv = L > 0.f ? 1.f / L : 0.f;
    store_out4(pp.out, pp.out_dtype, (int64_t)row * D + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
  }
}

// ------------------------------------------------------------------ host side
struct PagedCall {  // one call, before it is cut into launches
  PagedParams pp;
  int B;
  void* workspace;
  int64_t workspace_bytes;
  uint32_t* tickets;
};

template <class Policy>
struct PagedLaunch {
  static int smem_bytes(int B) {
    return Policy::WARPS * Policy::STAGES * Policy::STAGE_BYTES + Policy::WARPS * Policy::STAGES * 8 + 16 +
           2 * kHeadsPerCta * Policy::D * 4 + ((Policy::QFRAG_BYTES + 15) & ~15) + (B + 1) * 4 +
           1024;  // slack for the 1024-byte alignment of the ring
  }
  // CTAs resident at once with the largest prefix
  static int wave(int* out) {
    static int cached[64] = {};
    int dev = 0;
    TKV_CUDA(cudaGetDevice(&dev));
    if (dev < 64 && cached[dev] > 0) {
      *out = cached[dev];
      return TKV_OK;
    }
    const void* fn = reinterpret_cast<const void*>(&paged_split_kernel<Policy>);
    int n = 0, sms = 0;
    TKV_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(kMaxPagedB)));
    TKV_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, Policy::WARPS * 32, smem_bytes(kMaxPagedB)));
    TKV_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    TKV_REQUIRE(n > 0 && sms > 0, TKV_ERR_CUDA, "paged split kernel does not fit on this device");
    *out = n * sms;
    if (dev < 64) cached[dev] = *out;
    return TKV_OK;
  }
  // partials, then (m, l), then the units' notes
  static int bytes(int B, int HKVc, int64_t* out) {
    int w = 0;
    const int rc = wave(&w);
    if (rc != TKV_OK) return rc;
    const int64_t units = (int64_t)(B < kMaxPagedB ? B : kMaxPagedB) * HKVc;
    *out = (units + w) * kHeadsPerCta * (Policy::D + 2) * 4 + units * 8;
    return TKV_OK;
  }
  static int run(const typename Policy::Maps& maps, const PagedCall& c, cudaStream_t stream) {
    int w = 0;
    int64_t need = 0;
    int rc = wave(&w);
    if (rc == TKV_OK) rc = bytes(c.B, c.pp.HKVc, &need);
    if (rc != TKV_OK) return rc;
    TKV_REQUIRE(c.workspace && c.workspace_bytes >= need, TKV_ERR_INVALID,
                "paged decode: a workspace of %lld bytes is needed, got %lld; size it with tkv_paged_workspace",
                (long long)need, (long long)c.workspace_bytes);
    const int64_t tiles = ((int64_t)c.pp.d.S + Policy::TOK - 1) / Policy::TOK, steps = tiles + kSwitch;  // of one sequence, at most
    int64_t part = kMaxPagedB;  // sequences of a launch: step numbers fit the prefix words and 30 bits
    if (part * steps >= (1 << 25)) part = ((1 << 25) - 1) / steps;
    if (part * steps * c.pp.HKVc >= (1 << 30)) part = ((1 << 30) - 1) / (steps * c.pp.HKVc);
    TKV_REQUIRE(part >= 1, TKV_ERR_INVALID, "paged decode: %lld tiles of %d head units per sequence are too many",
                (long long)tiles, c.pp.HKVc);
    const int64_t units = (int64_t)(c.B < kMaxPagedB ? c.B : kMaxPagedB) * c.pp.HKVc, slots = units + w;
    for (int b0 = 0; b0 < c.B; b0 += (int)part) {
      PagedParams pp = c.pp;
      const int n = c.B - b0 < part ? c.B - b0 : (int)part;
      const int64_t rows0 = (int64_t)b0 * pp.d.HQ * Policy::D;
      pp.d.B = n;
      pp.dgrid = make_fastdiv(w);
      pp.d.q = (const uint8_t*)pp.d.q + rows0 * (pp.d.q_dtype == TKV_DTYPE_F32 ? 4 : 2);
      pp.out = (uint8_t*)pp.out + rows0 * (pp.out_dtype == TKV_DTYPE_F32 ? 4 : 2);
      pp.d.seq_lens += b0;
      pp.table += b0 * pp.table_stride;
      pp.acc = (float*)c.workspace;
      pp.m = pp.acc + slots * kHeadsPerCta * Policy::D;
      pp.l = pp.m + slots * kHeadsPerCta;
      pp.info = (int2*)(pp.l + slots * kHeadsPerCta);
      // How the work is cut.  CTAs of its own for every unit where there are two or more: nobody pays for a
      // second unit (16 sequences of 1024-4096 tokens, 8 KV heads: 19.8 us against 22.2 in equal ranges, 16 of 1000 13.0
      // against 16.2, 27 of 4096 33.3 against 37.5).  With fewer the rounding to whole units costs more (55 of
      // 1000-4096: 52.6 against 47.1).
      const int64_t units_now = (int64_t)n * pp.HKVc;
      pp.whole = units_now * 2 <= w && tiles * Policy::WARPS < (1 << 23) ? (int)(w / units_now) : 0;
      // Who merges.  With at least a CTA per unit and few partials of each, the CTA that finishes a unit:
      // one launch instead of two, 2.3 us of host time (14.4 -> 12.1 us per call), and no more time on the
      // device (1 sequence of 500 tokens 7.9 / 7.9 us, 8 of 4096 18.1 / 18.6, 16 of 4096 25.3 / 26.1).  Else a
      // kernel that spreads the partials over the device: one sequence of 65536 with 2 KV heads (128 partials a
      // unit) 12.8 us against 22.0, of 8000 8.7 against 11.5, and with more units than CTAs, where every CTA would
      // draw two tickets, 51.5 against 52.3 (64 sequences at 2 bits).  The lengths are on the device: what counts here is
      // the width of the table, so a short sequence under a wide table takes the second launch (500 tokens, 2048 pages of
      // 16: 8.3 us against 8.1 on the device, 14.4 against 11.9 per call).
      const int64_t partials = 2 + (w / units_now < tiles / Policy::WARPS ? w / units_now : tiles / Policy::WARPS);
      pp.tickets = units_now <= w && partials <= kFewPartials && units_now <= kTickets ? c.tickets : nullptr;
      TKV_CUDA(launch_pdl(paged_split_kernel<Policy>, dim3(w), dim3(Policy::WARPS * 32), (size_t)smem_bytes(n), stream,
                          maps, pp));
      if (pp.tickets) continue;
      const int rows = n * pp.d.HQ;
      if (rows < kSmallCombineMinRows)
        TKV_CUDA(launch_pdl(paged_merge_long_kernel<Policy::D>, dim3(rows, Policy::D / 32), dim3(256), 0, stream, pp));
      else
        TKV_CUDA(launch_pdl(paged_merge_rows_kernel<Policy::D>, dim3((rows + 7) / 8), dim3(256), 0, stream, pp, rows));
    }
    return TKV_OK;
  }
};

template <class P>
static int packed_run(const PagedCall& c, cudaStream_t stream) {
  using C = typename P::C;
  typename P::Maps maps;
  const DecodeParams& p = c.pp.d;
  // pool rows as 128-byte rows, a box is one piece of a tile
  const int64_t rows = (int64_t)c.pp.num_pages * p.HKV * c.pp.page * C::DP / 128;
  constexpr int box = P::PIECE_BYTES / 128;
  int rc;
  if (p.kv_one) {
    const uint8_t *lo = p.k_second ? p.vp : p.kp, *hi = p.k_second ? p.kp : p.vp;
    rc = make_pair_map(&maps.k, lo, (uint64_t)(hi - lo), rows, box);
    maps.v = maps.k;
  } else {
    rc = make_row_map(&maps.k, p.kp, rows, 128, 128, box);
    if (rc == TKV_OK) rc = make_row_map(&maps.v, p.vp, rows, 128, 128, box);
  }
  if (rc != TKV_OK) return rc;
  return PagedLaunch<P>::run(maps, c, stream);
}

template <class P>
static int f16_run(const PagedCall& c, cudaStream_t stream) {
  typename P::Maps maps;
  maps.unused = 0;
  return PagedLaunch<P>::run(maps, c, stream);
}

// Two families per format, as for contiguous caches (tkv_decode_fused.cu): 4 warps with rings of 3
// stages in a software pipeline, 3 CTAs per SM; and 8 warps with rings of 2, one tile at a time, 2 CTAs per
// SM, where few long units are to be spread thin.  At head_dim 128 some of them spill (bytes stored): of the 4-warp ones
// 2 bits in groups of 32 (16), of the 8-warp ones 2 bits in groups of 64 (68, 80) and 32 (52), 4 bits in groups of 128
// (40) and 16 (16).
template <int NB, int DD, int GG, int PIECES>
using PagedPolicy = FusedPolicy<NB, DD, GG, true, 32, 4, 3, 3, true, false, PIECES>;
template <int NB, int DD, int GG, int PIECES>
using PagedLongPolicy = FusedPolicy<NB, DD, GG, true, 32, 8, 2, 2, false, false, PIECES>;

#define TKV_PAGED_ONE(NB, DD, GG, EXPR)                        \
  if (nbits == NB && D == DD && gs == GG) {                    \
    if (page % 32 == 0) {                                      \
      if (few) {                                               \
        using P = PagedLongPolicy<NB, DD, GG, 1>;              \
        return EXPR;                                           \
      }                                                        \
      using P = PagedPolicy<NB, DD, GG, 1>;                    \
      return EXPR;                                             \
    }                                                          \
    if (few) {                                                 \
      using P = PagedLongPolicy<NB, DD, GG, 2>;                \
      return EXPR;                                             \
    }                                                          \
    using P = PagedPolicy<NB, DD, GG, 2>;                      \
    return EXPR;                                               \
  }
#define TKV_PAGED_ALL(EXPR)          \
  TKV_PAGED_ONE(4, 128, 16, EXPR)    \
  TKV_PAGED_ONE(4, 128, 32, EXPR)    \
  TKV_PAGED_ONE(4, 128, 64, EXPR)    \
  TKV_PAGED_ONE(4, 128, 128, EXPR)   \
  TKV_PAGED_ONE(2, 128, 16, EXPR)    \
  TKV_PAGED_ONE(2, 128, 32, EXPR)    \
  TKV_PAGED_ONE(2, 128, 64, EXPR)    \
  TKV_PAGED_ONE(2, 128, 128, EXPR)   \
  TKV_PAGED_ONE(4, 64, 16, EXPR)     \
  TKV_PAGED_ONE(4, 64, 32, EXPR)     \
  TKV_PAGED_ONE(4, 64, 64, EXPR)     \
  TKV_PAGED_ONE(2, 64, 16, EXPR)     \
  TKV_PAGED_ONE(2, 64, 32, EXPR)     \
  TKV_PAGED_ONE(2, 64, 64, EXPR)

// Few units of work: the family that spreads them thinner.  One sequence of 65536 tokens with 1 / 2 / 4 / 8 KV heads:
// 11.4 / 12.8 / 12.3 / 23.4 us against 13.5 / 13.7 / 12.6 / 24.4; but with 8 heads 4096 tokens are 10.6 against 9.9,
// and 64 sequences are the same to 2 %.
static bool few_units(int B, int HKVc) { return (int64_t)B * HKVc <= kFewUnits; }

static int packed_unsupported(int nbits, int D, int gs) {
  set_error("paged decode: unsupported (nbits=%d, head_dim=%d, group_size=%d); built: nbits in {2,4}, head_dim in "
            "{64,128}, group_size in {16,32,64,128} with group_size <= head_dim", nbits, D, gs);
  return TKV_ERR_UNSUPPORTED;
}

int paged_device_status(int* status) {
  int a = 0, b = 0;
  TKV_CUDA(cudaMemcpyFromSymbol(&a, g_fused_status, sizeof(int)));
  TKV_CUDA(cudaMemcpyFromSymbol(&b, g_fp16_status, sizeof(int)));
  *status = a | b;
  return TKV_OK;
}

int paged_device_status_clear() {
  const int zero = 0;
  TKV_CUDA(cudaMemcpyToSymbol(g_fused_status, &zero, sizeof(int)));
  TKV_CUDA(cudaMemcpyToSymbol(g_fp16_status, &zero, sizeof(int)));
  return TKV_OK;
}

static int paged_fill(PagedCall& c, const tkv_paged_decode_args& a) {
  TKV_REQUIRE(a.nbits == 2 || a.nbits == 4 || a.nbits == 16, TKV_ERR_INVALID,
              "paged decode: nbits must be 2, 4 or 16 (float16 pages), got %d", a.nbits);
  TKV_REQUIRE(a.B > 0 && a.HQ > 0 && a.HKV > 0 && a.HQ % a.HKV == 0, TKV_ERR_INVALID,
              "paged decode: bad sizes B=%d HQ=%d HKV=%d (HQ must be a multiple of HKV)", a.B, a.HQ, a.HKV);
  TKV_REQUIRE(a.num_pages > 0 && a.page_size > 0 && a.max_pages >= 0, TKV_ERR_INVALID,
              "paged decode: bad sizes num_pages=%d page_size=%d max_pages=%d", a.num_pages, a.page_size, a.max_pages);
  TKV_REQUIRE(a.page_size % 16 == 0, TKV_ERR_UNSUPPORTED, "paged decode: unsupported page_size=%d (a multiple of 16 tokens)",
              a.page_size);
  TKV_REQUIRE((int64_t)a.num_pages * a.HKV * a.page_size < (1LL << 31), TKV_ERR_INVALID,
              "paged decode: a pool of %lld token rows exceeds 2^31", (long long)a.num_pages * a.HKV * a.page_size);
  TKV_REQUIRE((int64_t)a.max_pages * a.page_size < (1LL << 30), TKV_ERR_INVALID,
              "paged decode: a table row of %lld tokens exceeds 2^30", (long long)a.max_pages * a.page_size);
  TKV_REQUIRE((int64_t)kMaxPagedB * a.HQ < (1LL << 31), TKV_ERR_INVALID, "paged decode: HQ=%d is too large", a.HQ);
  TKV_REQUIRE(a.q_dtype >= 0 && a.q_dtype <= 2 && a.out_dtype >= 0 && a.out_dtype <= 2, TKV_ERR_INVALID,
              "paged decode: bad dtype codes %d, %d", a.q_dtype, a.out_dtype);
  TKV_REQUIRE(a.q && a.seq_lens && a.out && a.k && a.v && (a.block_table || a.max_pages == 0) &&
                  (a.nbits == 16 || (a.k_scale && a.k_zero && a.v_scale && a.v_zero)),
              TKV_ERR_INVALID, "paged decode: null pointer");
  TKV_REQUIRE(aligned16(a.q) && aligned16(a.out) && aligned16(a.workspace) && aligned16(a.k) && aligned16(a.v) &&
                  (a.nbits == 16 || (aligned16(a.k_scale) && aligned16(a.k_zero) && aligned16(a.v_scale) && aligned16(a.v_zero))),
              TKV_ERR_ALIGN, "paged decode: q, out, the workspace and the pools must be 16-byte aligned");
  c = PagedCall{};
  c.B = a.B;
  c.workspace = a.workspace;
  c.workspace_bytes = a.workspace_bytes;
  c.tickets = a.tickets;
  PagedParams& pp = c.pp;
  DecodeParams& p = pp.d;
  p.q = a.q;
  p.q_dtype = a.q_dtype;
  p.seq_lens = a.seq_lens;
  p.HQ = a.HQ;
  p.HKV = a.HKV;
  p.S = a.max_pages * a.page_size;
  p.group = a.HQ / a.HKV;
  p.hchunks = (p.group + kHeadsPerCta - 1) / kHeadsPerCta;
  p.qk_scale = a.sm_scale * kLog2e;
  p.meta_aligned = 16;
  p.wide = 1;
  pp.table = a.block_table;
  pp.table_stride = a.table_stride;
  pp.out = a.out;
  pp.out_dtype = a.out_dtype;
  pp.num_pages = a.num_pages;
  pp.page = a.page_size;
  pp.HKVc = a.HKV * p.hchunks;
  pp.dpage = make_fastdiv(a.page_size);
  pp.dHch = make_fastdiv(p.hchunks);
  pp.dHKVc = make_fastdiv(pp.HKVc);
  pp.dHQ = make_fastdiv(a.HQ);
  pp.dgroup = make_fastdiv(p.group);
  return TKV_OK;
}

}  // namespace tkv

extern "C" int tkv_paged_workspace(int B, int HQ, int HKV, int page_size, int D, int nbits, int gs, int64_t* bytes) {
  using namespace tkv;
  TKV_REQUIRE(bytes && B > 0 && HQ > 0 && HKV > 0 && HQ % HKV == 0 && page_size > 0, TKV_ERR_INVALID,
              "paged_workspace: bad sizes B=%d HQ=%d HKV=%d page_size=%d", B, HQ, HKV, page_size);
  const int page = page_size, HKVc = HKV * ((HQ / HKV + kHeadsPerCta - 1) / kHeadsPerCta);
  if (nbits == 16) {
    if (D == 128) return PagedLaunch<Fp16Policy<128>>::bytes(B, HKVc, bytes);
    if (D == 64) return PagedLaunch<Fp16Policy<64>>::bytes(B, HKVc, bytes);
    set_error("paged fp16 decode: unsupported head_dim=%d (built: 64, 128)", D);
    return TKV_ERR_UNSUPPORTED;
  }
  const bool few = few_units(B, HKVc);
  TKV_PAGED_ALL(PagedLaunch<P>::bytes(B, HKVc, bytes))
  return packed_unsupported(nbits, D, gs);
}

extern "C" int tkv_paged_decode(const tkv_paged_decode_args* args, void* stream) {
  using namespace tkv;
  TKV_REQUIRE(args, TKV_ERR_INVALID, "paged decode: null arguments");
  const tkv_paged_decode_args& a = *args;
  PagedCall c;
  const int rc = paged_fill(c, a);
  if (rc != TKV_OK) return rc;
  DecodeParams& p = c.pp.d;
  const int nbits = a.nbits, D = a.D, gs = a.gs, page = a.page_size;
  if (nbits == 16) {
    p.k = (const __half*)a.k;
    p.v = (const __half*)a.v;
    if (D == 128) return f16_run<Fp16Policy<128>>(c, (cudaStream_t)stream);
    if (D == 64) return f16_run<Fp16Policy<64>>(c, (cudaStream_t)stream);
    set_error("paged fp16 decode: unsupported head_dim=%d (built: 64, 128)", D);
    return TKV_ERR_UNSUPPORTED;
  }
  p.kp = (const uint8_t*)a.k;
  p.vp = (const uint8_t*)a.v;
  p.ks = (const __half*)a.k_scale;
  p.kz = (const __half*)a.k_zero;
  p.vs = (const __half*)a.v_scale;
  p.vz = (const __half*)a.v_zero;
  {
    // one tensor map over both code pools, where a K and a V run land side by side in whole swizzle
    // atoms (or the stage is laid out for it: two pieces)
    const uint8_t *lo = p.kp < p.vp ? p.kp : p.vp, *hi = p.kp < p.vp ? p.vp : p.kp;
    const uint64_t gap = (uint64_t)(hi - lo);
    const int64_t pool = (int64_t)a.num_pages * a.HKV * page * (D * nbits / 8);
    p.kv_one = (page % 32 != 0 || (32 * (D * nbits / 8)) % 1024 == 0) && gap % 16 == 0 && gap < (1ull << 40) &&
               gap >= (uint64_t)pool;
    p.k_second = p.kv_one && p.kp > p.vp;
  }
  const bool few = few_units(a.B, c.pp.HKVc);
  TKV_PAGED_ALL(packed_run<P>(c, (cudaStream_t)stream))
  return packed_unsupported(nbits, D, gs);
}
