// Fused split-K decode attention on a packed 2/4-bit KV cache (sm_100a).
//
// Replaces _fused_decode_attn_split of the reference (kernels/fused_decode_attn.py:155-353).
//
// Scheduling, the per-warp copy rings and the epilogue live in tkv_splitk_driver.cuh
// (persistent CTAs over balanced tile ranges; one CTA segment serves one (batch, KV
// head, history split) and up to 8 query heads of the GQA group).  This file is the
// tile policy: how a 32-token tile is fetched and what is computed on it.
//
// Data movement.  A stage holds 32 tokens: K codes, V codes, and the four scale/zero
// arrays.  Lane 0 of the warp fetches the codes with two tiled TMA loads; every lane
// fetches a share of the metadata with 16-byte cp.async copies and posts one arrival
// that fires when they land; all of it completes on one mbarrier per stage.  The tensor maps
// view a packed code tensor as rows of 128 bytes (the 32 tokens of a tile are one
// contiguous run) with the hardware 128B swizzle, or -- when sequences do not start on
// 128-byte boundaries -- as [tokens, bytes-per-token] with the 32B/64B swizzle; either
// way the later 8-row x 16-byte ldmatrix reads hit 8 distinct bank groups.  Ragged
// tails and caches whose metadata rows are not 16-byte aligned fetch the metadata with
// plain loads (tokens past the end get scale = zero = 0).  The query rows of a segment
// are staged in shared memory by the driver, one segment ahead.
//
// Arithmetic.  The packed bytes are never expanded to dequantised values.  With
// code c, group scale s and group zero z, a cache value is c*s + z, so
//     q.k = sum_g s_g * (sum_{d in g} q_d c_d)  +  sum_g z_g * (sum_{d in g} q_d)
//     sum_n p_n v_n[d] = sum_n (p_n s_{n,g(d)}) c_n[d]  +  sum_n p_n z_{n,g(d)}
// The inner sums are tensor-core MMAs (m16n8k16, f16 in, f32 accumulate) whose
// A operand is the raw code field, isolated from the packed word by ONE bitwise AND:
// a 2- or 4-bit field inside the mantissa of an f16 is the subnormal (or scaled)
// number c * 2^(pos-24), exact, and the power of two is folded into the f32 scale
// afterwards.  The zero-point terms are one extra MMA each per 16 tokens.
//
// Fragment mapping (g = lane/4, t = lane%4).  Scores use S^T = K Q^T with 16 tokens
// as MMA rows and the 8 heads as columns; the output uses O^T = V^T P^T with 16
// head-dims as rows.  ldmatrix delivers for K the 4 bytes [16b+4t, 16b+4t+4) of
// tokens g / g+8, and with .trans for V the 2 bytes [16b+2g, 16b+2g+2) of token
// pairs (2t, 2t+1) / (2t+8, 2t+9) -- already the layout of an A fragment once masked.
// Chunk ch = slice*NBLK + b covers head dims [16ch, 16ch+16) because of the split-P
// layout (byte j, bit slice p -> dim j + p*DP).
//
// Softmax.  Probabilities are taken relative to a reference exponent m_ref that is
// only raised (to tile max + 4) when a tile exceeds it, so accumulators are rescaled
// a handful of times per split instead of at almost every tile; the true running
// maximum is tracked separately and the partial is converted to it in the epilogue.  A
// probability at the reference is 2^top, as high as float16 allows beside the value scales
// (FusedPolicy::kTopMax): below 2^-14 an f16 operand loses bits.
#include "tkv_fused_policy.cuh"

namespace tkv {

// ------------------------------------------------------------------ host side
// Two kernel families per (nbits, head_dim, group_size, row alignment):
//  * batched -- 4 warps, ring of 3 stages, software-pipelined tile loop, 3 CTAs per SM: the
//    balanced schedules (modes 1 and 3), where a CTA streams tens of tiles per warp;
//  * long -- 8 warps, ring of 2 stages, one tile at a time, 2 CTAs per SM: few long units
//    (mode 2: small batches, and the static one-CTA-per-unit plan).  The same 16 warps per SM
//    in two thirds of the CTAs: a third fewer partial slots for the merge that follows and a
//    third fewer query loads and epilogues, which is what a step of 2-3 tiles per warp is
//    made of (measured: batch 1, ctx 65536, 4-bit step 12.4 -> 10.8 us).
constexpr int kVariantBatched = 0, kVariantLong = 1;
template <int NB, int DD, int GG, bool A16, bool KCHAN = false>
using BatchedPolicy = FusedPolicy<NB, DD, GG, A16, 32, 4, 3, 3, true, KCHAN>;
template <int NB, int DD, int GG, bool A16, bool KCHAN = false>
using LongPolicy = FusedPolicy<NB, DD, GG, A16, 32, 8, 2, 2, false, KCHAN>;

// Keys quantised per channel (value groups of 32): dense batches only, so mode 1 and mode 2.
#define TKV_KCHAN_DISPATCH(NB, DD, EXPR)                            \
  if (nbits == NB && D == DD && gs == 32) {                         \
    using PB = BatchedPolicy<NB, DD, 32, true, true>;               \
    using PL = LongPolicy<NB, DD, 32, true, true>;                  \
    using LB = SplitLaunch<PB, 0x2>;                                \
    using LL = SplitLaunch<PL, 0x4>;                                \
    return EXPR;                                                    \
  }
#define TKV_KCHAN_ALL(EXPR)        \
  TKV_KCHAN_DISPATCH(4, 128, EXPR) \
  TKV_KCHAN_DISPATCH(2, 128, EXPR) \
  TKV_KCHAN_DISPATCH(4, 64, EXPR)  \
  TKV_KCHAN_DISPATCH(2, 64, EXPR)

#define TKV_FUSED_DISPATCH(NB, DD, GG, EXPR)                        \
  if (nbits == NB && D == DD && gs == GG) {                         \
    if (aligned16_rows) {                                           \
      using PB = BatchedPolicy<NB, DD, GG, true>;                   \
      using PL = LongPolicy<NB, DD, GG, true>;                      \
      using LB = SplitLaunch<PB, 0xA>;                              \
      using LL = SplitLaunch<PL, 0x4>;                              \
      return EXPR;                                                  \
    } else {                                                        \
      using PB = BatchedPolicy<NB, DD, GG, false>;                  \
      using PL = LongPolicy<NB, DD, GG, false>;                     \
      using LB = SplitLaunch<PB, 0xA>;                              \
      using LL = SplitLaunch<PL, 0x4>;                              \
      return EXPR;                                                  \
    }                                                               \
  }

#define TKV_FUSED_ALL(EXPR)             \
  TKV_FUSED_DISPATCH(4, 128, 16, EXPR)  \
  TKV_FUSED_DISPATCH(4, 128, 32, EXPR)  \
  TKV_FUSED_DISPATCH(4, 128, 64, EXPR)  \
  TKV_FUSED_DISPATCH(4, 128, 128, EXPR) \
  TKV_FUSED_DISPATCH(2, 128, 16, EXPR)  \
  TKV_FUSED_DISPATCH(2, 128, 32, EXPR)  \
  TKV_FUSED_DISPATCH(2, 128, 64, EXPR)  \
  TKV_FUSED_DISPATCH(2, 128, 128, EXPR) \
  TKV_FUSED_DISPATCH(4, 64, 16, EXPR)   \
  TKV_FUSED_DISPATCH(4, 64, 32, EXPR)   \
  TKV_FUSED_DISPATCH(4, 64, 64, EXPR)   \
  TKV_FUSED_DISPATCH(2, 64, 16, EXPR)   \
  TKV_FUSED_DISPATCH(2, 64, 32, EXPR)   \
  TKV_FUSED_DISPATCH(2, 64, 64, EXPR)

static int kchan_unsupported(int nbits, int D, int gs) {
  set_error("fused decode with per-channel keys: unsupported (nbits=%d, head_dim=%d, value "
            "group_size=%d); built: nbits in {2,4}, head_dim in {64,128}, value group_size 32",
            nbits, D, gs);
  return TKV_ERR_UNSUPPORTED;
}

static int fused_unsupported(int nbits, int D, int gs) {
  set_error("fused decode: unsupported (nbits=%d, head_dim=%d, group_size=%d); built: nbits in "
            "{2,4}, head_dim in {64,128}, group_size in {16,32,64,128} with group_size <= head_dim",
            nbits, D, gs);
  return TKV_ERR_UNSUPPORTED;
}

template <class L, class P>
static int fused_launch_one(const DecodeParams& p, const SplitSched& sc, cudaStream_t stream) {
  using C = typename P::C;
  typename P::Maps maps;
  const int64_t rows = (int64_t)p.B * p.HKV * p.S;
  int rc;
  if (p.kv_one) {
    const uint8_t* lo = p.k_second ? p.vp : p.kp;
    const uint8_t* hi = p.k_second ? p.kp : p.vp;
    rc = make_pair_map(&maps.k, lo, (uint64_t)(hi - lo), rows * C::DP / 128, C::kTok * C::DP / 128);
    maps.v = maps.k;
  } else if (p.wide) {
    // [bytes/128, 128] view, box = a tile's bytes as 128-byte rows, 128B swizzle
    rc = make_row_map(&maps.k, p.kp, rows * C::DP / 128, 128, 128, C::kTok * C::DP / 128);
    if (rc != TKV_OK) return rc;
    rc = make_row_map(&maps.v, p.vp, rows * C::DP / 128, 128, 128, C::kTok * C::DP / 128);
  } else {
    rc = make_row_map(&maps.k, p.kp, rows, C::DP, C::DP, C::kTok);
    if (rc != TKV_OK) return rc;
    rc = make_row_map(&maps.v, p.vp, rows, C::DP, C::DP, C::kTok);
  }
  if (rc != TKV_OK) return rc;
  return L::launch(maps, p, sc, stream);
}

// The long family plans first: if its plan is a mode-2 one (unit-aligned, or static units for
// ragged batches with explicit splits) it is taken, otherwise the batched family plans.
template <class LB, class LL>
static int fused_plan_both(SplitSched* sc, int B, int HKV, int hchunks, int S, int num_splits,
                           int split_size, bool ragged) {
  int rc = LL::plan(sc, B, HKV, hchunks, S, num_splits, split_size, ragged);
  if (rc != TKV_OK) return rc;
  if (sc->persistent == 2 || sc->persistent == 0) {
    sc->variant = kVariantLong;
    return TKV_OK;
  }
  rc = LB::plan(sc, B, HKV, hchunks, S, num_splits, split_size, ragged);
  sc->variant = kVariantBatched;
  return rc;
}

int fused_plan(int nbits, int D, int gs, SplitSched* sc, int B, int HKV, int hchunks, int S,
               int num_splits, int split_size, bool ragged, bool kchan) {
  if (kchan) {
    TKV_KCHAN_ALL((fused_plan_both<LB, LL>(sc, B, HKV, hchunks, S, num_splits, split_size, ragged)))
    return kchan_unsupported(nbits, D, gs);
  }
  constexpr bool aligned16_rows = true;  // both instantiations have the same resources
  TKV_FUSED_ALL((fused_plan_both<LB, LL>(sc, B, HKV, hchunks, S, num_splits, split_size, ragged)))
  return fused_unsupported(nbits, D, gs);
}

static int fused_launch(int nbits, int D, int gs, const DecodeParams& p, const SplitSched& sc,
                        cudaStream_t stream, bool kchan) {
  if (kchan) {
    TKV_KCHAN_ALL((sc.variant == kVariantLong ? fused_launch_one<LL, PL>(p, sc, stream)
                                              : fused_launch_one<LB, PB>(p, sc, stream)))
    return kchan_unsupported(nbits, D, gs);
  }
  const bool aligned16_rows = p.meta_aligned == 16;
  TKV_FUSED_ALL((sc.variant == kVariantLong ? fused_launch_one<LL, PL>(p, sc, stream)
                                            : fused_launch_one<LB, PB>(p, sc, stream)))
  return fused_unsupported(nbits, D, gs);
}

// Resources of the batched family (the one that runs where bandwidth binds).
int fused_attrs(int nbits, int D, int gs, int* regs, int* smem, int* local, int* ctas) {
  constexpr bool aligned16_rows = true;
  TKV_FUSED_ALL(LB::attrs(regs, smem, local, ctas))
  return fused_unsupported(nbits, D, gs);
}

int fused_device_status_clear() {
  const int zero = 0;
  TKV_CUDA(cudaMemcpyToSymbol(g_fused_status, &zero, sizeof(int)));
  return TKV_OK;
}

int fused_device_status(int* status) {
  int v = 0;
  TKV_CUDA(cudaMemcpyFromSymbol(&v, g_fused_status, sizeof(int)));
  *status = v;
  return TKV_OK;
}

}  // namespace tkv

extern "C" int tkv_fused_decode(const void* q, int q_dtype, const uint8_t* k_packed,
                                const void* k_scale, const void* k_zero, const uint8_t* v_packed,
                                const void* v_scale, const void* v_zero, float* acc, float* m,
                                float* l, float* out, int B, int HQ, int HKV, int S, int D,
                                int nbits, int gs, float sm_scale, int num_splits, int split_size,
                                int nslots, const int32_t* seq_lens, int flags, void* stream) {
  using namespace tkv;
  TKV_REQUIRE(q && k_packed && k_scale && k_zero && v_packed && v_scale && v_zero, TKV_ERR_INVALID,
              "fused decode: null input pointer");
  DecodeParams p{};
  int rc = fill_common(p, "fused decode", q, q_dtype, acc, m, l, out, B, HQ, HKV, S, sm_scale,
                       num_splits, split_size, nslots, seq_lens, flags);
  if (rc != TKV_OK) return rc;
  TKV_REQUIRE(aligned16(k_packed) && aligned16(v_packed), TKV_ERR_ALIGN,
              "fused decode: packed code pointers must be 16-byte aligned");
  p.kp = k_packed;
  p.vp = v_packed;
  p.ks = (const __half*)k_scale;
  p.kz = (const __half*)k_zero;
  p.vs = (const __half*)v_scale;
  p.vz = (const __half*)v_zero;
  const int ng = (gs > 0 && D % gs == 0) ? D / gs : 0;
  // Alignment of the first byte of any scale/zero tile: the pointers' own alignment, that
  // of a sequence's stride when there is more than one, and 32 bytes inside a sequence
  // (tiles start at multiples of 16 tokens).  The copies use the largest unit that fits.
  {
    const int res = (int)(reinterpret_cast<uintptr_t>(k_scale) & 15);
    TKV_REQUIRE((int)(reinterpret_cast<uintptr_t>(k_zero) & 15) == res &&
                    (int)(reinterpret_cast<uintptr_t>(v_scale) & 15) == res &&
                    (int)(reinterpret_cast<uintptr_t>(v_zero) & 15) == res && (res & 1) == 0,
                TKV_ERR_ALIGN,
                "fused decode: the four scale/zero pointers must share their offset within 16 bytes");
    const int64_t seq_bytes = (int64_t)S * ng * 2;
    const int ptr_al = (res | 16) & -(res | 16);
    const int seq_al = ((int64_t)B * HKV > 1) ? (int)((seq_bytes | 16) & -(seq_bytes | 16)) : 16;
    const int al = ptr_al < seq_al ? ptr_al : seq_al;
    p.meta_aligned = al >= 4 ? al : 0;
    p.meta_phase = res & 3;
    TKV_REQUIRE(al >= 4 || ng == 1, TKV_ERR_ALIGN,
                "fused decode: scale/zero rows of %d bytes must start on 4-byte boundaries", ng * 2);
  }
  // 128-byte-row view of the code tensors: every sequence must start on a 128-byte boundary
  p.wide = (((int64_t)S * D * nbits / 8) % 128 == 0) ? 1 : 0;
  {
    // one tensor map over both code tensors when a tile fills whole 1024-byte swizzle atoms
    const uint8_t* lo = k_packed < v_packed ? k_packed : v_packed;
    const uint8_t* hi = k_packed < v_packed ? v_packed : k_packed;
    const uint64_t gap = (uint64_t)(hi - lo);
    const int64_t tensor_bytes = (int64_t)B * HKV * S * (D * nbits / 8);
    const bool ok = p.wide && ((32 * (D * nbits / 8)) % 1024 == 0) && gap % 16 == 0 && gap < (1ull << 40) &&
                    gap >= (uint64_t)tensor_bytes;
    p.kv_one = ok ? 1 : 0;
    p.k_second = (ok && k_packed > v_packed) ? 1 : 0;
  }
  const bool kchan = (flags & TKV_FLAG_K_PER_CHANNEL) != 0;
  if (kchan) {
    // k_scale / k_zero are (B, HKV, S/32, D): one row per block of 32 tokens, so every tile
    // must be one whole block -- a history of whole blocks, one split, no per-sequence lengths
    TKV_REQUIRE(S % 32 == 0 && num_splits == 1 && seq_lens == nullptr, TKV_ERR_INVALID,
                "fused decode with per-channel keys: S=%d must be a multiple of 32, with one split "
                "and no seq_lens (the fp16 tail goes through tkv_fp16_decode)", S);
    TKV_REQUIRE(aligned16(k_scale) && aligned16(v_scale), TKV_ERR_ALIGN,
                "fused decode with per-channel keys: scale/zero pointers must be 16-byte aligned");
    p.meta_aligned = 16;
  }
  SplitSched sc;
  rc = fused_plan(nbits, D, gs, &sc, B, HKV, p.hchunks, S, num_splits, split_size,
                  seq_lens != nullptr, kchan);
  if (rc != TKV_OK) return rc;
  TKV_REQUIRE(sc.nslots == nslots, TKV_ERR_INVALID,
              "fused decode: nslots=%d does not match the plan (%d); size acc/m/l with "
              "tkv_decode_plan", nslots, sc.nslots);
  rc = fused_launch(nbits, D, gs, p, sc, (cudaStream_t)stream, kchan);
  if (rc != TKV_OK) return rc;
  if ((flags & TKV_FLAG_COMBINE) && nslots > 1 && !(flags & TKV_FLAG_PARTIALS_ONLY)) {
    TKV_REQUIRE(out, TKV_ERR_INVALID, "fused decode: TKV_FLAG_COMBINE needs out");
    return tkv_combine(acc, m, l, out, nullptr, nullptr, B, HQ, nslots, D, stream);
  }
  return TKV_OK;
}
