// Write side of a paged cache (sm_100a): quantise new tokens of K and V into their pages.
//
// Token t < lengths[b] of sequence b goes to position pos = positions[b] + t, which is row
// (block_table[b][pos / page] * HKV + head) * page + pos % page of both pools; positions outside
// the table and table entries outside the pool drop the token.  Per group of gs dims
//     scale = f16((max - min) / (2^nbits - 1))  (1 if that is not positive),   zero = f16(min),
//     code  = clamp(rint((x - zero) / scale), 0, 2^nbits - 1),
// with the arithmetic of tkv_quantize_pack (tkv_quant_part.cuh), so the bytes are the same.  With a
// values tensor the token's code*scale + zero goes there too: what the cache now stands for, as a
// prompt's own attention needs it.
//
// K and V go in one launch.  A thread owns E = 16 (8) consecutive elements of a row, in one row of a step and
// four of a prompt.
// Two ways to cut the rows (BLOCK):
//   * prompts: a CTA takes a block of tokens of one head of one sequence, so that where it stands
//     is known from its indexes alone and the codes and metadata it writes are consecutive;
//   * a step (T of at most kStepTokens): a CTA takes rows of several heads and sequences.
// The row's place (two dependent loads: position, then table entry) is looked up beside the element
// loads and needed only by the stores.
#include "tkv_quant_part.cuh"
#include "tkv_splitk_driver.cuh"  // FastDiv

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
  int pos0, B, HKV, T, num_pages, page;
  int limit;                        // tokens that a row of the table has room for
  FastDiv dpage, dT, dHKV;
};

constexpr int kStepTokens = 8;
constexpr int kRowsBlock = 4, kRowsStep = 1;  // rows of a thread

__device__ __forceinline__ float elem_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float elem_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __half*) { return pack_half2(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16*) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 8 consecutive values, 16 or 32 bytes
template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&v)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack2(v[0], v[1], dst), pack2(v[2], v[3], dst),
                                                pack2(v[4], v[5], dst), pack2(v[6], v[7], dst));
  }
}

// The token of a row of the work.  A row that is not there names the nearest one that is, so that
// a whole warp can load and shuffle.
struct AppendRow {
  int b, h, t;
  bool live;
};
template <bool BLOCK>
__device__ __forceinline__ AppendRow append_row(const AppendArgs& a, int rows_per_cta, int i) {
  AppendRow w;
  if constexpr (BLOCK) {
    const int t = blockIdx.x * rows_per_cta + i;
    w.b = blockIdx.z;
    w.h = blockIdx.y >> 1;
    w.live = t < a.T;
    w.t = min(t, a.T - 1);
  } else {
    const int r = blockIdx.x * rows_per_cta + i, q = fast_div(r, a.dT), b = fast_div(q, a.dHKV);
    w.live = b < a.B;
    w.b = min(b, a.B - 1);
    w.h = q - b * a.HKV;
    w.t = r - q * a.T;
  }
  return w;
}
// Its pool row, or -1: nowhere.
__device__ __forceinline__ int append_place(const AppendArgs& a, const AppendRow& w) {
  const int len = a.lengths ? __ldg(a.lengths + w.b) : a.T;
  const int64_t pos = (int64_t)(a.positions ? __ldg(a.positions + w.b) : a.pos0) + w.t;
  if (!w.live || w.t >= len || (uint64_t)pos >= (uint32_t)a.limit) return -1;
  const int k = fast_div((int)pos, a.dpage), id = __ldg(a.table + w.b * a.table_stride + k);
  return (unsigned)id < (unsigned)a.num_pages ? (id * a.HKV + w.h) * a.page + ((int)pos - k * a.page) : -1;
}

// `tpr_shift` = log2(D/E) (threads of a row), `lpg_shift` = log2(gs/E) (lanes of a group).
template <typename T, int NBITS, int E, bool BLOCK>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendArgs a, int tpr_shift, int lpg_shift) {
  constexpr int LOG2P = NBITS == 4 ? 1 : 2, ROWS = BLOCK ? kRowsBlock : kRowsStep;
  const AppendTensor& w = a.t[blockIdx.y & 1];
  const int tpr = 1 << tpr_shift, c = threadIdx.x & (tpr - 1), rstep = 256 >> tpr_shift;
  const int tps_shift = tpr_shift - LOG2P, p = c >> tps_shift, D = E << tpr_shift;
  if (BLOCK && a.lengths && (int)blockIdx.x * ROWS * rstep >= __ldg(a.lengths + blockIdx.z)) return;  // padding
  const AppendRow row0 = append_row<BLOCK>(a, ROWS * rstep, threadIdx.x >> tpr_shift);
  const T* src0 = reinterpret_cast<const T*>(w.x) + row0.b * w.sb + row0.h * w.sh + E * c;
  T* val0 = reinterpret_cast<T*>(w.values) + row0.b * w.vb + row0.h * w.vh + E * c;
#pragma unroll
  for (int it = 0; it < ROWS; ++it) {
    AppendRow row = row0;
    if (BLOCK && it > 0) row = append_row<BLOCK>(a, ROWS * rstep, it * rstep + (threadIdx.x >> tpr_shift));
    const int at = append_place(a, row);
    uint32_t code[E / 4];
    __half sc16, ze16;
    float m[E];
    quantize_part<T, NBITS, E>(src0 + row.t * w.st, 1 << lpg_shift, code, sc16, ze16, m);
    if (w.values && at >= 0) {
      T* dst = val0 + row.t * w.vt;
      const float s = __half2float(sc16), z = __half2float(ze16);
#pragma unroll
      for (int i = 0; i < E / 8; ++i) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = fmaf(__fsub_rn(m[8 * i + k], kMagic), s, z);  // (the product is exact)
        store8(dst + 8 * i, v);
      }
    }
    pack_slices<NBITS, E>(code, p, tps_shift, tpr);
    if (at >= 0) {
      if (p == 0) {
        uint8_t* dst = w.packed + (int64_t)at * (D >> LOG2P) + E * c;
        if constexpr (E == 16) *reinterpret_cast<uint4*>(dst) = make_uint4(code[0], code[1], code[2], code[3]);
        else *reinterpret_cast<uint2*>(dst) = make_uint2(code[0], code[1]);
      }
      if ((c & ((1 << lpg_shift) - 1)) == 0) {
        const int64_t g = ((int64_t)at << (tpr_shift - lpg_shift)) + (c >> lpg_shift);
        w.scale[g] = sc16;
        w.zero[g] = ze16;
      }
    }
  }
}

// Float16 pages: 8 elements of a thread; float16 rows are copied as stored, whatever a NaN holds.
template <typename T, bool BLOCK>
__global__ void __launch_bounds__(256) paged_append_f16_kernel(const AppendArgs a, int tpr_shift) {
  constexpr int ROWS = BLOCK ? kRowsBlock : kRowsStep;
  const AppendTensor& w = a.t[blockIdx.y & 1];
  const int c = threadIdx.x & ((1 << tpr_shift) - 1), rstep = 256 >> tpr_shift, D = 8 << tpr_shift;
#pragma unroll
  for (int it = 0; it < ROWS; ++it) {
    const AppendRow row = append_row<BLOCK>(a, ROWS * rstep, it * rstep + (threadIdx.x >> tpr_shift));
    const int at = append_place(a, row);
    if (at < 0) continue;
    const T* src = reinterpret_cast<const T*>(w.x) + row.b * w.sb + row.h * w.sh + row.t * w.st + 8 * c;
    uint4 y;
    if constexpr (std::is_same<T, float>::value) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(src)), v = __ldg(reinterpret_cast<const float4*>(src) + 1);
      y = make_uint4(pack_half2(u.x, u.y), pack_half2(u.z, u.w), pack_half2(v.x, v.y), pack_half2(v.z, v.w));
    } else {
      y = __ldg(reinterpret_cast<const uint4*>(src));
      if constexpr (!std::is_same<T, __half>::value) {
        const T* e = reinterpret_cast<const T*>(&y);
        const uint4 x = make_uint4(pack_half2(elem_f32(e[0]), elem_f32(e[1])), pack_half2(elem_f32(e[2]), elem_f32(e[3])),
                                   pack_half2(elem_f32(e[4]), elem_f32(e[5])), pack_half2(elem_f32(e[6]), elem_f32(e[7])));
        y = x;
      }
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<__half*>(w.packed) + (int64_t)at * D + 8 * c) = y;
    if (w.values) {
      T* dst = reinterpret_cast<T*>(w.values) + row.b * w.vb + row.h * w.vh + row.t * w.vt + 8 * c;
      if constexpr (std::is_same<T, __half>::value) {
        *reinterpret_cast<uint4*>(dst) = y;
      } else {
        const __half* e = reinterpret_cast<const __half*>(&y);
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __half2float(e[k]);
        store8(dst, v);
      }
    }
  }
}

static inline bool is_pow2(int x) { return x > 0 && (x & (x - 1)) == 0; }
static inline int log2i(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

template <typename T, bool BLOCK>
static void launch_append_as(const AppendArgs& a, dim3 grid, int D, int nbits, int gs, bool wide, cudaStream_t stream) {
  const int E = wide ? 16 : 8, tpr = log2i(D / E), lpg = nbits == 16 ? 0 : log2i(gs / E);
  if (nbits == 16) {
    paged_append_f16_kernel<T, BLOCK><<<grid, 256, 0, stream>>>(a, tpr);
  } else if (wide) {
    if constexpr (!std::is_same<T, float>::value) {
      if (nbits == 4) paged_append_kernel<T, 4, 16, BLOCK><<<grid, 256, 0, stream>>>(a, tpr, lpg);
      else paged_append_kernel<T, 2, 16, BLOCK><<<grid, 256, 0, stream>>>(a, tpr, lpg);
    }
  } else if (nbits == 4) {
    paged_append_kernel<T, 4, 8, BLOCK><<<grid, 256, 0, stream>>>(a, tpr, lpg);
  } else {
    paged_append_kernel<T, 2, 8, BLOCK><<<grid, 256, 0, stream>>>(a, tpr, lpg);
  }
}

template <typename T>
static int launch_append(const AppendArgs& a, int D, int nbits, int gs, cudaStream_t stream) {
  // 16 elements of a thread where a 16-bit row gives every bit slice and every group a whole thread
  const bool wide = !std::is_same<T, float>::value && nbits != 16 && gs >= 16 && D / 16 >= 8 / nbits;
  const int per_pass = 256 >> log2i(D / (wide ? 16 : 8));
  // (65535: the limit of the grid's y and z)
  if (a.T > kStepTokens && a.HKV <= 65535 / 2 && a.B <= 65535) {
    const int per_cta = kRowsBlock * per_pass;
    launch_append_as<T, true>(a, dim3((a.T + per_cta - 1) / per_cta, 2 * a.HKV, a.B), D, nbits, gs, wide, stream);
  } else {
    const int64_t rows = (int64_t)a.B * a.HKV * a.T, per_cta = kRowsStep * per_pass;
    launch_append_as<T, false>(a, dim3((unsigned)((rows + per_cta - 1) / per_cta), 2), D, nbits, gs, wide, stream);
  }
  TKV_CUDA(cudaGetLastError());
  return TKV_OK;
}

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
  TKV_REQUIRE(is_pow2(D) && D >= 16 && D <= 256, TKV_ERR_UNSUPPORTED,
              "paged append: unsupported head_dim=%d (a power of two from 16 to 256)", D);
  if (nbits != 16) {
    TKV_REQUIRE(is_pow2(gs) && gs >= 8 && gs <= D, TKV_ERR_UNSUPPORTED,
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
  TKV_REQUIRE((int64_t)max_pages * page_size < (1LL << 30), TKV_ERR_INVALID,
              "paged append: a table row of %lld tokens exceeds 2^30", (long long)max_pages * page_size);
  TKV_REQUIRE((int64_t)B * HKV * T < (1LL << 31) - 4096, TKV_ERR_INVALID, "paged append: %lld token rows exceed 2^31",
              (long long)B * HKV * T);
  TKV_REQUIRE((int64_t)num_pages * HKV * page_size < (1LL << 31), TKV_ERR_INVALID,
              "paged append: a pool of %lld token rows exceeds 2^31", (long long)num_pages * HKV * page_size);
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
  a.dpage = make_fastdiv(page_size);
  a.dT = make_fastdiv(T);
  a.dHKV = make_fastdiv(HKV);
  a.num_pages = num_pages;
  a.page = page_size;
  a.limit = max_pages * page_size;
  cudaStream_t s = (cudaStream_t)stream;
  if (in_dtype == TKV_DTYPE_F16) return launch_append<__half>(a, D, nbits, gs, s);
  if (in_dtype == TKV_DTYPE_BF16) return launch_append<__nv_bfloat16>(a, D, nbits, gs, s);
  return launch_append<float>(a, D, nbits, gs, s);
}
