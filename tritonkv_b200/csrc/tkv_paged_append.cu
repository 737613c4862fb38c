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
// K and V go in one launch.  A thread owns E = 16 (8) consecutive elements of a row.  Two ways to cut
// the rows:
//   * prompts: a warp takes 32 tokens of one head of one sequence; each lane looks up the place of one
//     of them (two dependent loads: position, then table entry), and the warp walks over them,
//     32 * E / D rows at a time, with the places in a shuffle's reach;
//   * a step (T of at most kStepTokens): a CTA takes rows of several heads and sequences, one a
//     thread, and every thread looks up its own.
#include "tkv_quant_part.cuh"
#include "tkv_splitk_driver.cuh"  // FastDiv

namespace tkv {

struct AppendTensor {
  const void* x;                    // (B, HKV, T, D) with strides sb, sh, st (elements)
  uint8_t* packed;                  // (num_pages, HKV, page, D*nbits/8), or float16 pages
  __half *scale, *zero;             // (num_pages, HKV, page, D/gs)
  void* values;                     // (B, HKV, T, D) of x's type with its own strides, or null
  int64_t sb, sh, st, vb, vh, vt;
  int values32;                     // every row of the values starts on a 32-byte boundary
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
constexpr int kBlockThreads = 128;  // of a CTA of prompt rows: 128 tokens

__device__ __forceinline__ float elem_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float elem_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __half*) { return pack_half2(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16*) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 8 consecutive values, 16 or 32 bytes
template <typename T>
__device__ __forceinline__ void store8(T* dst, const float* v) {
  if constexpr (std::is_same<T, float>::value) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack2(v[0], v[1], dst), pack2(v[2], v[3], dst),
                                                pack2(v[4], v[5], dst), pack2(v[6], v[7], dst));
  }
}

// E consecutive values; 16 of a 16-bit type as one 32-byte store where they start on such a boundary
// (two halves of a sector would travel to L2 apart).
template <typename T, int E>
__device__ __forceinline__ void store_row_part(T* dst, const float (&v)[E], bool aligned32) {
  if constexpr (E == 16) {
    if (aligned32) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = pack2(v[2 * i], v[2 * i + 1], dst);
      asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                   "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                   : "memory");
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < E / 8; ++i) store8(dst + 8 * i, v + 8 * i);
}

// The pool row of token t of (sequence b, head h), or -1: nowhere.
__device__ __forceinline__ int append_place(const AppendArgs& a, int b, int h, int t) {
  const int len = a.lengths ? __ldg(a.lengths + b) : a.T;
  const int64_t pos = (int64_t)(a.positions ? __ldg(a.positions + b) : a.pos0) + t;
  if (t >= min(len, a.T) || (uint64_t)pos >= (uint32_t)a.limit) return -1;
  const int k = fast_div((int)pos, a.dpage), id = __ldg(a.table + b * a.table_stride + k);
  return (unsigned)id < (unsigned)a.num_pages ? (id * a.HKV + h) * a.page + ((int)pos - k * a.page) : -1;
}

// Codes, scale and zero point of a thread's part of a row into pool row `at` (-1: nowhere), and what
// they stand for to `val`.
template <typename T, int NBITS, int E>
__device__ __forceinline__ void append_part(const AppendTensor& w, const T* src, T* val, int at, int c, int tpr_shift,
                                            int lpg_shift) {
  constexpr int LOG2P = NBITS == 4 ? 1 : 2;
  const int tps_shift = tpr_shift - LOG2P, p = c >> tps_shift, D = E << tpr_shift;
  uint32_t code[E / 4];
  __half sc16, ze16;
  float m[E];
  quantize_part<T, NBITS, E>(src, 1 << lpg_shift, code, sc16, ze16, m);
  if (w.values && at >= 0) {
    const float s = __half2float(sc16), z = __half2float(ze16);
#pragma unroll
    for (int i = 0; i < E; ++i) m[i] = fmaf(__fsub_rn(m[i], kMagic), s, z);  // (the product is exact)
    store_row_part<T, E>(val, m, w.values32);
  }
  pack_slices<NBITS, E>(code, p, tps_shift, 1 << tpr_shift);
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

// Float16 pages: 8 elements of a thread; float16 rows are copied as stored, whatever a NaN holds.
template <typename T>
__device__ __forceinline__ void append_part_f16(const AppendTensor& w, const T* src, T* val, int at, int c, int D) {
  if (at < 0) return;
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
    if constexpr (std::is_same<T, __half>::value) {
      *reinterpret_cast<uint4*>(val) = y;
    } else {
      const __half* e = reinterpret_cast<const __half*>(&y);
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = __half2float(e[k]);
      store8(val, v);
    }
  }
}

// `tpr_shift` = log2(D/E) (threads of a row), `lpg_shift` = log2(gs/E) (lanes of a group); NBITS 16: float16
// pages.
template <typename T, int NBITS, int E, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? kBlockThreads : 256)
    paged_append_kernel(const AppendArgs a, int tpr_shift, int lpg_shift) {
  const AppendTensor& w = a.t[blockIdx.y & 1];
  const int tpr = 1 << tpr_shift, c = threadIdx.x & (tpr - 1);
  const T* x = reinterpret_cast<const T*>(w.x) + E * c;
  T* values = reinterpret_cast<T*>(w.values) + E * c;
  auto part = [&](int b, int h, int t, int at) {
    const T* src = x + b * w.sb + h * w.sh + t * w.st;
    T* val = values + b * w.vb + h * w.vh + t * w.vt;
    if constexpr (NBITS == 16) append_part_f16<T>(w, src, val, at, c, E << tpr_shift);
    else append_part<T, NBITS, E>(w, src, val, at, c, tpr_shift, lpg_shift);
  };
  if constexpr (BLOCK) {
    const int lane = threadIdx.x & 31, b = blockIdx.z, h = blockIdx.y >> 1;
    const int t0 = (blockIdx.x * (kBlockThreads / 32) + (threadIdx.x >> 5)) * 32;
    const int len = min(a.T, a.lengths ? __ldg(a.lengths + b) : a.T);
    if (t0 >= len) return;  // padding
    const int place = append_place(a, b, h, t0 + lane);
    const int per_pass = 32 >> tpr_shift, n = min(32, len - t0);
    for (int r0 = 0; r0 < n; r0 += per_pass) {
      const int r = r0 + (lane >> tpr_shift);
      // (a row past the end has place -1 and mirrors the last one: the shuffles stay full-warp)
      part(b, h, t0 + min(r, n - 1), __shfl_sync(kFullMask, place, r));
    }
  } else {
    const int r = blockIdx.x * (256 >> tpr_shift) + (threadIdx.x >> tpr_shift);
    const int q = fast_div(r, a.dT), b = fast_div(q, a.dHKV), h = q - b * a.HKV, t = r - q * a.T;
    const bool live = b < a.B;
    part(min(b, a.B - 1), h, t, live ? append_place(a, b, h, t) : -1);
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
  constexpr int threads = BLOCK ? kBlockThreads : 256;
  if (nbits == 16) {
    paged_append_kernel<T, 16, 8, BLOCK><<<grid, threads, 0, stream>>>(a, tpr, lpg);
  } else if (wide) {
    if constexpr (!std::is_same<T, float>::value) {
      if (nbits == 4) paged_append_kernel<T, 4, 16, BLOCK><<<grid, threads, 0, stream>>>(a, tpr, lpg);
      else paged_append_kernel<T, 2, 16, BLOCK><<<grid, threads, 0, stream>>>(a, tpr, lpg);
    }
  } else if (nbits == 4) {
    paged_append_kernel<T, 4, 8, BLOCK><<<grid, threads, 0, stream>>>(a, tpr, lpg);
  } else {
    paged_append_kernel<T, 2, 8, BLOCK><<<grid, threads, 0, stream>>>(a, tpr, lpg);
  }
}

template <typename T>
static int launch_append(const AppendArgs& a, int D, int nbits, int gs, cudaStream_t stream) {
  // 16 elements of a thread where a 16-bit row gives every bit slice and every group a whole thread
  const bool wide = !std::is_same<T, float>::value && nbits != 16 && gs >= 16 && D / 16 >= 8 / nbits;
  // (65535: the limit of the grid's y and z)
  if (a.T > kStepTokens && a.HKV <= 65535 / 2 && a.B <= 65535) {
    launch_append_as<T, true>(a, dim3((a.T + kBlockThreads - 1) / kBlockThreads, 2 * a.HKV, a.B), D, nbits, gs, wide, stream);
  } else {
    const int64_t rows = (int64_t)a.B * a.HKV * a.T, per_cta = 256 >> log2i(D / (wide ? 16 : 8));
    launch_append_as<T, false>(a, dim3((unsigned)((rows + per_cta - 1) / per_cta), 2), D, nbits, gs, wide, stream);
  }
  TKV_CUDA(cudaGetLastError());
  return TKV_OK;
}

}  // namespace tkv

extern "C" int tkv_paged_append(const tkv_paged_append_args* args, void* stream) {
  using namespace tkv;
  TKV_REQUIRE(args, TKV_ERR_INVALID, "paged append: null arguments");
  const tkv_paged_append_args& in = *args;
  const int nbits = in.nbits, D = in.D, gs = in.gs;
  TKV_REQUIRE(nbits == 2 || nbits == 4 || nbits == 16, TKV_ERR_INVALID,
              "paged append: nbits must be 2, 4 or 16 (float16 pages), got %d", nbits);
  TKV_REQUIRE(in.B >= 0 && in.HKV > 0 && in.T >= 0 && in.num_pages > 0 && in.page_size > 0 && in.max_pages >= 0,
              TKV_ERR_INVALID, "paged append: bad sizes B=%d HKV=%d T=%d num_pages=%d page_size=%d max_pages=%d", in.B,
              in.HKV, in.T, in.num_pages, in.page_size, in.max_pages);
  TKV_REQUIRE(in.in_dtype >= 0 && in.in_dtype <= 2, TKV_ERR_INVALID, "paged append: bad dtype %d", in.in_dtype);
  TKV_REQUIRE(is_pow2(D) && D >= 16 && D <= 256, TKV_ERR_UNSUPPORTED,
              "paged append: unsupported head_dim=%d (a power of two from 16 to 256)", D);
  if (nbits != 16) {
    TKV_REQUIRE(is_pow2(gs) && gs >= 8 && gs <= D, TKV_ERR_UNSUPPORTED,
                "paged append: unsupported group_size=%d (a power of two from 8 to head_dim)", gs);
    TKV_REQUIRE((D * nbits / 8) % 8 == 0, TKV_ERR_UNSUPPORTED,
                "paged append: packed row of %d bytes is not a multiple of 8", D * nbits / 8);
  }
  if (in.B == 0 || in.T == 0 || in.max_pages == 0) return TKV_OK;
  TKV_REQUIRE(in.k && in.v && in.k_pool && in.v_pool && in.block_table, TKV_ERR_INVALID, "paged append: null pointer");
  TKV_REQUIRE(nbits == 16 || (in.k_scale && in.k_zero && in.v_scale && in.v_zero), TKV_ERR_INVALID,
              "paged append: null scale or zero pointer");
  const int al = in.in_dtype == TKV_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
  for (int i = 0; i < 6; ++i)
    TKV_REQUIRE(in.strides[i] % al == 0 && ((i < 3 ? in.k_values : in.v_values) == nullptr || in.value_strides[i] % al == 0),
                TKV_ERR_ALIGN, "paged append: rows of the new tokens must start on 16-byte boundaries");
  TKV_REQUIRE(aligned16(in.k) && aligned16(in.v) && aligned16(in.k_pool) && aligned16(in.v_pool) &&
                  aligned16(in.k_values) && aligned16(in.v_values), TKV_ERR_ALIGN,
              "paged append: pointers must be 16-byte aligned");
  TKV_REQUIRE((int64_t)in.max_pages * in.page_size < (1LL << 30), TKV_ERR_INVALID,
              "paged append: a table row of %lld tokens exceeds 2^30", (long long)in.max_pages * in.page_size);
  TKV_REQUIRE((int64_t)in.B * in.HKV * in.T < (1LL << 31) - 4096, TKV_ERR_INVALID,
              "paged append: %lld token rows exceed 2^31", (long long)in.B * in.HKV * in.T);
  TKV_REQUIRE((int64_t)in.num_pages * in.HKV * in.page_size < (1LL << 31), TKV_ERR_INVALID,
              "paged append: a pool of %lld token rows exceeds 2^31", (long long)in.num_pages * in.HKV * in.page_size);
  AppendArgs a{};
  a.t[0] = {in.k, (uint8_t*)in.k_pool, (__half*)in.k_scale, (__half*)in.k_zero, in.k_values, 0, 0, 0, 0, 0, 0, 0};
  a.t[1] = {in.v, (uint8_t*)in.v_pool, (__half*)in.v_scale, (__half*)in.v_zero, in.v_values, 0, 0, 0, 0, 0, 0, 0};
  for (int i = 0; i < 2; ++i) {
    AppendTensor& t = a.t[i];
    t.sb = in.strides[3 * i], t.sh = in.strides[3 * i + 1], t.st = in.strides[3 * i + 2];
    if (t.values) t.vb = in.value_strides[3 * i], t.vh = in.value_strides[3 * i + 1], t.vt = in.value_strides[3 * i + 2];
    t.values32 = in.in_dtype != TKV_DTYPE_F32 && ((uintptr_t)t.values & 31) == 0 && t.vb % 16 == 0 && t.vh % 16 == 0 &&
                 t.vt % 16 == 0;
  }
  a.table = in.block_table;
  a.positions = in.positions;
  a.lengths = in.lengths;
  a.table_stride = in.table_stride;
  a.pos0 = in.pos0;
  a.B = in.B;
  a.HKV = in.HKV;
  a.T = in.T;
  a.dpage = make_fastdiv(in.page_size);
  a.dT = make_fastdiv(in.T);
  a.dHKV = make_fastdiv(in.HKV);
  a.num_pages = in.num_pages;
  a.page = in.page_size;
  a.limit = in.max_pages * in.page_size;
  cudaStream_t s = (cudaStream_t)stream;
  if (in.in_dtype == TKV_DTYPE_F16) return launch_append<__half>(a, D, nbits, gs, s);
  if (in.in_dtype == TKV_DTYPE_BF16) return launch_append<__nv_bfloat16>(a, D, nbits, gs, s);
  return launch_append<float>(a, D, nbits, gs, s);
}
