// Write side of a paged cache (sm_100a): quantise new tokens of K and V into their pages.
//
// Token t < lengths[b] of sequence b goes to position pos = positions[b] + t, which is row
// (block_table[b][pos / page] * HKV + head) * page + pos % page of both pools; positions outside
// the table and table entries outside the pool drop the token.  Per group of gs dims
//     scale = f16((max - min) / (2^nbits - 1))  (1 if that is not positive),   zero = f16(min),
//     code  = clamp(rint((x - zero) / scale), 0, 2^nbits - 1),
// the arithmetic of tkv_quantize_pack, so the bytes are the same.  Every float operation is one
// IEEE operation written with an intrinsic.  With a values tensor the token's code*scale + zero
// goes there too: what the cache now stands for, as a prompt's own attention needs it.
#include <type_traits>

#include "tkv_common.cuh"

namespace tkv {

struct AppendTensor {
  const void* x;                    // (B, HKV, T, D) with strides sb, sh, st (elements)
  uint8_t* packed;                  // (num_pages, HKV, page, D*nbits/8), or float16 pages
  __half *scale, *zero;             // (num_pages, HKV, page, D/gs)
  void* values;                     // (B, HKV, T, D) of x's type with its own strides, or null
  int64_t sb, sh, st, vb, vh, vt;
};

struct AppendArgs {
  AppendTensor t[2];                // K, V
  const int32_t *table, *positions, *lengths;
  int64_t table_stride;
  int pos0, B, HKV, T, D, gs, num_pages, page, max_pages;
};

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else return static_cast<float>(x);
}
__device__ __forceinline__ void from_f32(float* d, float x) { *d = x; }
__device__ __forceinline__ void from_f32(__half* d, float x) { *d = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(__nv_bfloat16* d, float x) { *d = __float2bfloat16_rn(x); }

// The pool row of token t of (sequence b, head h), or -1.
__device__ __forceinline__ int64_t append_row(const AppendArgs& a, int b, int h, int t) {
  if (a.lengths && t >= a.lengths[b]) return -1;
  const int64_t pos = (a.positions ? (int64_t)a.positions[b] : (int64_t)a.pos0) + t;
  if (pos < 0 || pos >= (int64_t)a.max_pages * a.page) return -1;
  const int i = (int)(pos / a.page), id = a.table[b * a.table_stride + i];
  if (id < 0 || id >= a.num_pages) return -1;
  return ((int64_t)id * a.HKV + h) * a.page + (pos - (int64_t)i * a.page);
}

// One CTA of D threads per row; NBITS == 16 copies into float16 pages.
template <typename T, int NBITS>
__global__ void paged_append_kernel(const AppendArgs a) {
  __shared__ float s_x[256];
  __shared__ uint8_t s_code[256];
  const int d = threadIdx.x, D = a.D;
  const AppendTensor& w = a.t[blockIdx.y];
  const int64_t r = blockIdx.x;
  const int t = (int)(r % a.T), h = (int)(r / a.T % a.HKV), b = (int)(r / a.T / a.HKV);
  const int64_t row = append_row(a, b, h, t);
  if (row < 0) return;
  const T raw = reinterpret_cast<const T*>(w.x)[b * w.sb + h * w.sh + t * w.st + d];
  const float x = to_f32(raw);
  float value;
  if constexpr (NBITS == 16) {
    __half y;
    if constexpr (std::is_same<T, __half>::value) y = raw;  // as stored, whatever a NaN holds
    else y = __float2half_rn(x);
    reinterpret_cast<__half*>(w.packed)[row * D + d] = y;
    value = __half2float(y);
  } else {
    constexpr float QMAX = float((1 << NBITS) - 1);
    s_x[d] = x;
    __syncthreads();
    const int g0 = d / a.gs * a.gs;
    float lo = s_x[g0], hi = lo;
    for (int i = 1; i < a.gs; ++i) {  // a NaN stays, as it does in tkv_quantize_pack
      const float y = s_x[g0 + i];
      lo = (y < lo || y != y) ? y : lo;
      hi = (y > hi || y != y) ? y : hi;
    }
    float s = __fdiv_rn(__fsub_rn(hi, lo), QMAX);
    s = s > 0.f ? s : 1.f;
    const __half s16 = __float2half_rn(s), z16 = __float2half_rn(lo);
    const float sf = __half2float(s16), zf = __half2float(z16);
    float c = rintf(__fdiv_rn(__fsub_rn(x, zf), sf));
    c = fminf(fmaxf(c, 0.f), QMAX);
    s_code[d] = (uint8_t)c;
    if (d == g0) {
      const int64_t g = row * (D / a.gs) + d / a.gs;
      w.scale[g] = s16;
      w.zero[g] = z16;
    }
    __syncthreads();
    constexpr int P = 8 / NBITS;
    const int DP = D / P;
    if (d < DP) {
      uint32_t byte = 0;
      for (int p = 0; p < P; ++p) byte |= (uint32_t)s_code[d + p * DP] << (NBITS * p);
      w.packed[row * DP + d] = (uint8_t)byte;
    }
    value = __fadd_rn(__fmul_rn(c, sf), zf);
  }
  if (w.values) from_f32(reinterpret_cast<T*>(w.values) + b * w.vb + h * w.vh + t * w.vt + d, value);
}

template <typename T>
static int launch_append(const AppendArgs& a, int nbits, int tensors, cudaStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.B * a.HKV * a.T), tensors);
  if (nbits == 16) paged_append_kernel<T, 16><<<grid, a.D, 0, stream>>>(a);
  else if (nbits == 4) paged_append_kernel<T, 4><<<grid, a.D, 0, stream>>>(a);
  else paged_append_kernel<T, 2><<<grid, a.D, 0, stream>>>(a);
  TKV_CUDA(cudaGetLastError());
  return TKV_OK;
}

static inline bool pow2(int x) { return x > 0 && (x & (x - 1)) == 0; }

}  // namespace tkv

extern "C" int tkv_paged_append(const void* k, const void* v, int in_dtype, const int64_t* strides,
                                uint8_t* k_packed, void* k_scale, void* k_zero, uint8_t* v_packed,
                                void* v_scale, void* v_zero, void* k_values, void* v_values,
                                const int64_t* value_strides, const int32_t* block_table,
                                int64_t table_stride, const int32_t* positions, int pos0,
                                const int32_t* lengths, int B, int HKV, int T, int num_pages, int page_size,
                                int max_pages, int D, int nbits, int gs, void* stream) {
  using namespace tkv;
  TKV_REQUIRE(nbits == 2 || nbits == 4 || nbits == 16, TKV_ERR_INVALID,
              "paged append: nbits must be 2, 4 or 16 (float16 pages), got %d", nbits);
  TKV_REQUIRE(B >= 0 && HKV > 0 && T >= 0 && num_pages > 0 && page_size > 0 && max_pages >= 0, TKV_ERR_INVALID,
              "paged append: bad sizes B=%d HKV=%d T=%d num_pages=%d page_size=%d max_pages=%d", B, HKV, T,
              num_pages, page_size, max_pages);
  TKV_REQUIRE(in_dtype >= 0 && in_dtype <= 2, TKV_ERR_INVALID, "paged append: bad dtype %d", in_dtype);
  TKV_REQUIRE(pow2(D) && D >= 16 && D <= 256, TKV_ERR_UNSUPPORTED,
              "paged append: unsupported head_dim=%d (a power of two from 16 to 256)", D);
  if (nbits != 16) {
    TKV_REQUIRE(pow2(gs) && gs >= 8 && gs <= D, TKV_ERR_UNSUPPORTED,
                "paged append: unsupported group_size=%d (a power of two from 8 to head_dim)", gs);
    TKV_REQUIRE((D * nbits / 8) % 8 == 0, TKV_ERR_UNSUPPORTED,
                "paged append: packed row of %d bytes is not a multiple of 8", D * nbits / 8);
  }
  if (B == 0 || T == 0 || max_pages == 0) return TKV_OK;
  TKV_REQUIRE(k && v && strides && k_packed && v_packed && block_table, TKV_ERR_INVALID,
              "paged append: null pointer");
  TKV_REQUIRE(nbits == 16 || (k_scale && k_zero && v_scale && v_zero), TKV_ERR_INVALID,
              "paged append: null scale or zero pointer");
  TKV_REQUIRE((k_values == nullptr && v_values == nullptr) || value_strides, TKV_ERR_INVALID,
              "paged append: values need their strides");
  const int al = in_dtype == TKV_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
  for (int i = 0; i < 6; ++i)
    TKV_REQUIRE(strides[i] % al == 0 && ((i < 3 ? k_values : v_values) == nullptr || value_strides[i] % al == 0),
                TKV_ERR_ALIGN, "paged append: rows of the new tokens must start on 16-byte boundaries");
  TKV_REQUIRE(aligned16(k) && aligned16(v) && aligned16(k_packed) && aligned16(v_packed) && aligned16(k_values) &&
                  aligned16(v_values), TKV_ERR_ALIGN, "paged append: pointers must be 16-byte aligned");
  TKV_REQUIRE((int64_t)B * HKV * T < (1LL << 31), TKV_ERR_INVALID, "paged append: B*HKV*T exceeds 2^31");
  AppendArgs a{};
  a.t[0] = {k, k_packed, (__half*)k_scale, (__half*)k_zero, k_values, strides[0], strides[1], strides[2], 0, 0, 0};
  a.t[1] = {v, v_packed, (__half*)v_scale, (__half*)v_zero, v_values, strides[3], strides[4], strides[5], 0, 0, 0};
  if (k_values) a.t[0].vb = value_strides[0], a.t[0].vh = value_strides[1], a.t[0].vt = value_strides[2];
  if (v_values) a.t[1].vb = value_strides[3], a.t[1].vh = value_strides[4], a.t[1].vt = value_strides[5];
  a.table = block_table;
  a.positions = positions;
  a.lengths = lengths;
  a.table_stride = table_stride;
  a.pos0 = pos0;
  a.B = B;
  a.HKV = HKV;
  a.T = T;
  a.D = D;
  a.gs = nbits == 16 ? D : gs;
  a.num_pages = num_pages;
  a.page = page_size;
  a.max_pages = max_pages;
  cudaStream_t s = (cudaStream_t)stream;
  if (in_dtype == TKV_DTYPE_F16) return launch_append<__half>(a, nbits, 2, s);
  if (in_dtype == TKV_DTYPE_BF16) return launch_append<__nv_bfloat16>(a, nbits, 2, s);
  return launch_append<float>(a, nbits, 2, s);
}
