// Decode attention over a paged KV cache (sm_100a): packed 2/4-bit pages and float16 pages.
//
//     o_h = sum_n softmax_n(q_h . k_n * scale) v_n        over the n < seq_lens[b] of the table
//
// Token n of sequence b lies in row (block_table[b][n / page] * HKV + hkv) * page + n % page of a
// pool that has the layout of the contiguous cache with pages in the place of sequences.  Table
// entries outside the pool hold no tokens: theirs are not attended.
//
// One CTA owns one (sequence, query head) and walks the history in blocks of kTokens tokens with
// a running maximum and sum in f32: a thread scores one token, then the threads turn to head dims
// and add the block's weighted values.
#include "tkv_common.cuh"

namespace tkv {

struct PagedArgs {
  const void* q;
  const uint8_t *kp, *vp;             // packed pages, or the float16 pages themselves
  const __half *ks, *kz, *vs, *vz;
  const int32_t* table;
  const int32_t* seq_lens;
  void* out;
  int64_t table_stride;
  int q_dtype, out_dtype;
  int B, HQ, HKV, D, num_pages, page, max_pages, gs;
  float qk_scale;                     // sm_scale * log2(e)
};

constexpr int kTokens = 128;

// Element d of cache row `row` (NBITS == 16: float16 pages)
template <int NBITS>
__device__ __forceinline__ float cache_value(const uint8_t* codes, const __half* scale, const __half* zero,
                                             int64_t row, int d, int D, int gs) {
  if constexpr (NBITS == 16) {
    return __half2float(reinterpret_cast<const __half*>(codes)[row * D + d]);
  } else {
    const int DP = D * NBITS / 8, p = d / DP;
    const int code = (codes[row * DP + (d - p * DP)] >> (NBITS * p)) & ((1 << NBITS) - 1);
    const int64_t g = row * (D / gs) + d / gs;
    return fmaf((float)code, __half2float(scale[g]), __half2float(zero[g]));
  }
}

template <int NBITS>
__global__ void __launch_bounds__(kTokens) paged_attention_kernel(const PagedArgs a) {
  __shared__ float s_q[128], s_p[kTokens], s_red[4];
  __shared__ int64_t s_row[kTokens];
  const int tid = threadIdx.x, b = blockIdx.x / a.HQ, h = blockIdx.x - b * a.HQ;
  const int hkv = h / (a.HQ / a.HKV), D = a.D;
  const int64_t qrow = ((int64_t)b * a.HQ + h) * D;
  if (tid < D) s_q[tid] = __half2float(load_q_half(a.q, a.q_dtype, qrow + tid)) * a.qk_scale;
  const int len = (int)min((int64_t)max(a.seq_lens[b], 0), (int64_t)a.max_pages * a.page);
  float M = -INFINITY, L = 0.f, acc = 0.f;
  for (int n0 = 0; n0 < len; n0 += kTokens) {
    __syncthreads();
    const int n = n0 + tid;
    int64_t row = -1;
    float s = -INFINITY;
    if (n < len) {
      const int i = n / a.page, id = a.table[b * a.table_stride + i];
      if (id >= 0 && id < a.num_pages) row = ((int64_t)id * a.HKV + hkv) * a.page + (n - i * a.page);
    }
    if (row >= 0) {
      s = 0.f;
      for (int d = 0; d < D; ++d)
        s = fmaf(s_q[d], cache_value<NBITS>(a.kp, a.ks, a.kz, row, d, D, a.gs), s);
    }
    float m = s;
    for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, off));
    if ((tid & 31) == 0) s_red[tid >> 5] = m;
    s_row[tid] = row;
    __syncthreads();
    m = fmaxf(M, fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3])));
    if (m == -INFINITY) continue;  // nothing to attend so far
    s_p[tid] = ex2(s - m);
    __syncthreads();
    const float alpha = ex2(M - m);
    M = m;
    L *= alpha;
    acc *= alpha;
    const int count = min(kTokens, len - n0);
    for (int j = 0; j < count; ++j) {
      if (s_row[j] < 0) continue;  // what lies there may be anything
      L += s_p[j];
      if (tid < D) acc = fmaf(s_p[j], cache_value<NBITS>(a.vp, a.vs, a.vz, s_row[j], tid, D, a.gs), acc);
    }
  }
  if (tid < D) {
    const float o = L > 0.f ? acc / L : 0.f;
    if (a.out_dtype == TKV_DTYPE_F32) reinterpret_cast<float*>(a.out)[qrow + tid] = o;
    else if (a.out_dtype == TKV_DTYPE_F16) reinterpret_cast<__half*>(a.out)[qrow + tid] = __float2half_rn(o);
    else reinterpret_cast<__nv_bfloat16*>(a.out)[qrow + tid] = __float2bfloat16_rn(o);
  }
}

static int paged_check(const char* who, const PagedArgs& a, int nbits) {
  TKV_REQUIRE(a.B > 0 && a.HQ > 0 && a.HKV > 0 && a.HQ % a.HKV == 0, TKV_ERR_INVALID,
              "%s: bad sizes B=%d HQ=%d HKV=%d (HQ must be a multiple of HKV)", who, a.B, a.HQ, a.HKV);
  TKV_REQUIRE(a.num_pages > 0 && a.page > 0 && a.max_pages >= 0, TKV_ERR_INVALID,
              "%s: bad sizes num_pages=%d page_size=%d max_pages=%d", who, a.num_pages, a.page, a.max_pages);
  TKV_REQUIRE(a.page % 16 == 0, TKV_ERR_UNSUPPORTED, "%s: unsupported page_size=%d (a multiple of 16 tokens)",
              who, a.page);
  TKV_REQUIRE((int64_t)a.num_pages * a.HKV * a.page < (1LL << 31), TKV_ERR_INVALID,
              "%s: a pool of %lld token rows exceeds 2^31", who, (long long)a.num_pages * a.HKV * a.page);
  TKV_REQUIRE((int64_t)a.max_pages * a.page < (1LL << 30), TKV_ERR_INVALID,
              "%s: a table row of %lld tokens exceeds 2^30", who, (long long)a.max_pages * a.page);
  TKV_REQUIRE((int64_t)a.B * a.HQ < (1LL << 31), TKV_ERR_INVALID, "%s: B*HQ exceeds 2^31", who);
  TKV_REQUIRE(a.q_dtype >= 0 && a.q_dtype <= 2 && a.out_dtype >= 0 && a.out_dtype <= 2, TKV_ERR_INVALID,
              "%s: bad dtype codes %d, %d", who, a.q_dtype, a.out_dtype);
  TKV_REQUIRE(a.D == 64 || a.D == 128, TKV_ERR_UNSUPPORTED, "%s: unsupported head_dim=%d (built: 64, 128)", who, a.D);
  if (nbits != 16) {
    TKV_REQUIRE(nbits == 2 || nbits == 4, TKV_ERR_INVALID, "nbits must be one of (2, 4), got %d", nbits);
    TKV_REQUIRE((a.gs == 16 || a.gs == 32 || a.gs == 64 || a.gs == 128) && a.gs <= a.D, TKV_ERR_UNSUPPORTED,
                "%s: unsupported (nbits=%d, head_dim=%d, group_size=%d); built: group_size in {16,32,64,128} "
                "with group_size <= head_dim", who, nbits, a.D, a.gs);
    TKV_REQUIRE(aligned16(a.ks) && aligned16(a.kz) && aligned16(a.vs) && aligned16(a.vz), TKV_ERR_ALIGN,
                "%s: scale and zero pointers must be 16-byte aligned", who);
  }
  TKV_REQUIRE(a.q && a.kp && a.vp && a.seq_lens && a.out && (a.table || a.max_pages == 0), TKV_ERR_INVALID,
              "%s: null pointer", who);
  TKV_REQUIRE(aligned16(a.q) && aligned16(a.kp) && aligned16(a.vp) && aligned16(a.out), TKV_ERR_ALIGN,
              "%s: q, the pools and out must be 16-byte aligned", who);
  return TKV_OK;
}

}  // namespace tkv

extern "C" int tkv_paged_decode(const void* q, int q_dtype, const uint8_t* k_packed, const void* k_scale,
                                const void* k_zero, const uint8_t* v_packed, const void* v_scale,
                                const void* v_zero, const int32_t* block_table, int64_t table_stride,
                                const int32_t* seq_lens, void* out, int out_dtype, int B, int HQ, int HKV,
                                int num_pages, int page_size, int max_pages, int D, int nbits, int gs,
                                float sm_scale, void* stream) {
  using namespace tkv;
  const PagedArgs a{q, k_packed, v_packed, (const __half*)k_scale, (const __half*)k_zero, (const __half*)v_scale,
                    (const __half*)v_zero, block_table, seq_lens, out, table_stride, q_dtype, out_dtype, B, HQ,
                    HKV, D, num_pages, page_size, max_pages, gs, sm_scale * kLog2e};
  TKV_REQUIRE(k_scale && k_zero && v_scale && v_zero, TKV_ERR_INVALID, "paged decode: null pointer");
  TKV_REQUIRE(nbits == 2 || nbits == 4, TKV_ERR_INVALID, "nbits must be one of (2, 4), got %d", nbits);
  const int rc = paged_check("paged decode", a, nbits);
  if (rc != TKV_OK) return rc;
  if (nbits == 4)
    paged_attention_kernel<4><<<B * HQ, kTokens, 0, (cudaStream_t)stream>>>(a);
  else
    paged_attention_kernel<2><<<B * HQ, kTokens, 0, (cudaStream_t)stream>>>(a);
  TKV_CUDA(cudaGetLastError());
  return TKV_OK;
}

extern "C" int tkv_paged_fp16_decode(const void* q, int q_dtype, const void* k, const void* v,
                                     const int32_t* block_table, int64_t table_stride,
                                     const int32_t* seq_lens, void* out, int out_dtype, int B, int HQ, int HKV,
                                     int num_pages, int page_size, int max_pages, int D, float sm_scale,
                                     void* stream) {
  using namespace tkv;
  const PagedArgs a{q, (const uint8_t*)k, (const uint8_t*)v, nullptr, nullptr, nullptr, nullptr, block_table,
                    seq_lens, out, table_stride, q_dtype, out_dtype, B, HQ, HKV, D, num_pages, page_size,
                    max_pages, 0, sm_scale * kLog2e};
  const int rc = paged_check("paged fp16 decode", a, 16);
  if (rc != TKV_OK) return rc;
  paged_attention_kernel<16><<<B * HQ, kTokens, 0, (cudaStream_t)stream>>>(a);
  TKV_CUDA(cudaGetLastError());
  return TKV_OK;
}
