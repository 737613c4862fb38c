// Arithmetic of the group-wise quantiser, shared by the whole-tensor and append kernels
// (tkv_quant.cu) and the paged append (tkv_paged_append.cu): one thread's part of a row.
#pragma once

#include <type_traits>

#include "tkv_common.cuh"

namespace tkv {

// Each thread owns E consecutive elements of a row (E = 16 for f16/bf16 rows: two 16-byte loads;
// E = 8 otherwise), in kRowsPerThread rows.  A quantisation group spans GS/E adjacent lanes; min
// and max are butterfly-reduced inside it as the pair (min, -max) with a NaN-propagating
// minimum -- for 16-bit inputs as ONE packed half2 per shuffle.  The codes of a thread are E/4
// 32-bit words (one code per byte); split-P packing ORs the words of the P lanes that hold
// dims j, j+DP, ... shifted by their bit-slice position.  Every size is a power of two, so all
// index arithmetic is shifts.
//
// Codes.  The reference computes round((x - zero) / scale) with an IEEE division.  Here, with y the
// rounded reciprocal of the scale s, q0 = a*y and q = fma(fma(-q0, s, a), y, q0) (Markstein 1990): q0
// is within two ulps of a/s, the inner fma is exact, so q is a/s plus less than 2^-21 ulp, rounded.
// That is the IEEE quotient unless a/s lies as close as that to the middle M of two floats.  M has 25
// bits and s, an f16, at most 11, so a - M*s is a multiple of 2^-36 of a's size: zero, or 2^-13 ulp
// of the quotient or more; and zero it is not, since M*s has an odd part of 25 bits or more and a
// one of 24 at most.  Three operations an element and no branch: where the input is coarse (bf16) exact
// ties of the rounding to a code are frequent, and a form that redid the elements next to one
// with a division spent a third of its instructions there (prompt append, bf16 at 2 bits: 47 us).
// The scale's division by 2^nbits - 1 is q0 = d*R, q1 = fma(fma(-q0, QMAX, d), R, q0) with R the
// rounded reciprocal: the correctly rounded quotient for every finite d (checked against the
// IEEE division over 160 M values of d, all fp16 values among them).
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float rcp_approx(float a) {
  float d;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(a));
  return d;
}

// A thread's E elements as f32 plus their (min, -max); NaN propagates to both (torch's
// amin/amax do; fminf/fmaxf would drop it).  For 16-bit types the pair stays a packed half2.
template <typename T>
struct Pair16;
template <>
struct Pair16<__half> { using type = __half2; };
template <>
struct Pair16<__nv_bfloat16> { using type = __nv_bfloat162; };

template <typename H2>
__device__ __forceinline__ float2 widen2(H2 h);
template <>
__device__ __forceinline__ float2 widen2<__half2>(__half2 h) { return __half22float2(h); }
template <>
__device__ __forceinline__ float2 widen2<__nv_bfloat162>(__nv_bfloat162 h) { return __bfloat1622float2(h); }

// (min over both halves of a, -max over both halves of b) as one packed pair
template <typename H2>
__device__ __forceinline__ H2 fold_minmax(H2 a, H2 b) {
  b = __hneg2(b);
  const uint32_t au = *reinterpret_cast<const uint32_t*>(&a), bu = *reinterpret_cast<const uint32_t*>(&b);
  const uint32_t lo = __byte_perm(au, bu, 0x5410), hi = __byte_perm(au, bu, 0x7632);  // (a.x, b.x), (a.y, b.y)
  return __hmin2_nan(*reinterpret_cast<const H2*>(&lo), *reinterpret_cast<const H2*>(&hi));
}

// (x.lo - z, x.hi - z) in f32 from a packed pair of 16-bit values: the mixed-precision subtract of
// sm_100 widens the 16-bit operand itself, so no conversion instruction is spent per element.
template <typename H2>
__device__ __forceinline__ float2 sub_widen(H2 x, float z);
template <>
__device__ __forceinline__ float2 sub_widen<__half2>(__half2 x, float z) {
  float2 r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tsub.rn.f32.f16 %0, l, %3;\n\tsub.rn.f32.f16 %1, h, %3;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "r"(*reinterpret_cast<const uint32_t*>(&x)), "f"(z));
  return r;
}
template <>
__device__ __forceinline__ float2 sub_widen<__nv_bfloat162>(__nv_bfloat162 x, float z) {
  float2 r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tsub.rn.f32.bf16 %0, l, %3;\n\tsub.rn.f32.bf16 %1, h, %3;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "r"(*reinterpret_cast<const uint32_t*>(&x)), "f"(z));
  return r;
}

constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: x + kMagic holds rint(x) in its low mantissa bits

// The codes (one per byte) of the E elements at `src`, whose quantisation group spans
// `lanes_per_group` adjacent lanes, and the group's scale and zero point; `a` leaves with
// kMagic + code.
template <typename T, int NBITS, int E>
__device__ __forceinline__ void quantize_part(const T* __restrict__ src, int lanes_per_group, uint32_t (&w)[E / 4],
                                              __half& sc16, __half& ze16, float (&a)[E]) {
  constexpr float QMAX = float((1 << NBITS) - 1), TOP = QMAX / (1 << NBITS);
  constexpr bool k16 = !std::is_same<T, float>::value;
  static_assert(E == 8 || (E == 16 && k16), "16 elements per thread are two 16-byte loads of a 16-bit type");
  float mn, nmx;  // (a: the elements of f32 rows, then x - zero, then the quotients)
  [[maybe_unused]] uint32_t raw[k16 ? E / 2 : 1];  // 16-bit rows: the elements as loaded
  if constexpr (k16) {
    using H2 = typename Pair16<T>::type;
    H2 h[E / 2];
#pragma unroll
    for (int i = 0; i < E / 8; ++i)
      *reinterpret_cast<uint4*>(&h[4 * i]) = __ldg(reinterpret_cast<const uint4*>(src) + i);
    H2 lo = h[0], hi = h[0];
#pragma unroll
    for (int i = 1; i < E / 2; ++i) {
      lo = __hmin2_nan(lo, h[i]);
      hi = __hmax2_nan(hi, h[i]);
    }
    H2 pm = fold_minmax<H2>(lo, hi);
    for (int off = 1; off < lanes_per_group; off <<= 1) {
      const uint32_t o = __shfl_xor_sync(kFullMask, *reinterpret_cast<const uint32_t*>(&pm), off);
      pm = __hmin2_nan(pm, *reinterpret_cast<const H2*>(&o));
    }
    const float2 f = widen2<H2>(pm);
    mn = f.x;
    nmx = f.y;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) raw[i] = *reinterpret_cast<const uint32_t*>(&h[i]);
  } else {
    const float4 lo4 = __ldg(reinterpret_cast<const float4*>(src));
    const float4 hi4 = __ldg(reinterpret_cast<const float4*>(src) + 1);
    a[0] = lo4.x; a[1] = lo4.y; a[2] = lo4.z; a[3] = lo4.w;
    a[4] = hi4.x; a[5] = hi4.y; a[6] = hi4.z; a[7] = hi4.w;
    mn = a[0];
    nmx = -a[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      mn = min_nan(mn, a[i]);
      nmx = min_nan(nmx, -a[i]);
    }
    for (int off = 1; off < lanes_per_group; off <<= 1) {
      mn = min_nan(mn, __shfl_xor_sync(kFullMask, mn, off));
      nmx = min_nan(nmx, __shfl_xor_sync(kFullMask, nmx, off));
    }
  }
  // A group that holds a NaN gets zero = NaN, scale = 1 and all codes 0, as the reference produces.
  const float range = __fsub_rn(-nmx, mn);
  const float q0 = __fmul_rn(range, 1.f / QMAX);
  const float q1 = __fmaf_rn(__fmaf_rn(-q0, QMAX, range), 1.f / QMAX, q0);
  float sc = range == INFINITY ? range : q1;  // = __fdiv_rn(range, QMAX)
  sc = (sc > 0.f) ? sc : 1.f;
  sc16 = __float2half_rn(sc);
  ze16 = __float2half_rn(mn);
  const float scf = __half2float(sc16), zef = __half2float(ze16);
  // (scaled by 2^-NBITS and 2^NBITS, both exact: the last fma's saturation to [0, 1] is then the clamp at
  // 0 and at 2^NBITS, and takes NaN to 0)
  const float y = __fmul_rn(__frcp_rn(scf), 1.f / (1 << NBITS)), ss = __fmul_rn(scf, float(1 << NBITS));

  if constexpr (k16) {
    using H2 = typename Pair16<T>::type;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 d = sub_widen<H2>(*reinterpret_cast<const H2*>(&raw[i]), zef);
      a[2 * i] = d.x;
      a[2 * i + 1] = d.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) a[i] = __fsub_rn(a[i], zef);
  }
  // A range below the smallest f16 (a / 0 is an infinity, or NaN for 0 / 0) and a minimum below the
  // lowest f16 (a is infinite): the quotient is an infinity where the scale is not one too.
  if (scf == 0.f || zef == -INFINITY) {
#pragma unroll
    for (int i = 0; i < E; ++i) a[i] = (a[i] > 0.f && scf < INFINITY) ? TOP : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float q = __fmul_rn(a[i], y);
      a[i] = __saturatef(__fmaf_rn(__fmaf_rn(-q, ss, a[i]), y, q));
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) a[i] = __fmaf_rn(fminf(a[i], TOP), float(1 << NBITS), kMagic);
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    const uint32_t lo2 = __byte_perm(__float_as_uint(a[4 * i]), __float_as_uint(a[4 * i + 1]), 0x0040);
    const uint32_t hi2 = __byte_perm(__float_as_uint(a[4 * i + 2]), __float_as_uint(a[4 * i + 3]), 0x0040);
    w[i] = __byte_perm(lo2, hi2, 0x5410);
  }
}

// Split-P packing of a row's codes: bit slice p of the byte block is what lane c = p*TPS + c' holds
// (TPS = 1 << tps_shift lanes per slice, tpr lanes per row); every lane of a block gets the bytes.
template <int NBITS, int E>
__device__ __forceinline__ void pack_slices(uint32_t (&w)[E / 4], int p, int tps_shift, int tpr) {
#pragma unroll
  for (int i = 0; i < E / 4; ++i) w[i] <<= (NBITS * p);
  // split-P: lane c = p*TPS + c' contributes bit slice p of bytes [E*c', E*c' + E)
  for (int off = 1 << tps_shift; off < tpr; off <<= 1) {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) w[i] |= __shfl_xor_sync(kFullMask, w[i], off);
  }
}

}  // namespace tkv
