// fp16 control: split-K decode attention on an unquantised f16 cache (sm_100a).
//
// Replaces _fp16_decode_attn_split of the reference (kernels/fp16_decode_attn.py:47-135).
// Scheduling, the per-warp copy rings and the epilogue are the shared driver of
// tkv_splitk_driver.cuh -- identical split, online softmax, GQA grouping and partial
// format as the packed-cache kernel; this file is the tile policy: K and V tiles are
// plain f16 rows, fetched with 16-byte cp.async copies into a 128B-swizzled layout
// (completion posted on the stage's mbarrier) and read with ldmatrix (K as the A operand of S^T = K Q^T, V with .trans as
// the A operand of O^T = V^T P^T).
#include "tkv_fp16_policy.cuh"

namespace tkv {

static int fp16_unsupported(int D) {
  set_error("fp16 decode: unsupported head_dim=%d (built: 64, 128)", D);
  return TKV_ERR_UNSUPPORTED;
}

int fp16_plan(int D, SplitSched* sc, int B, int HKV, int hchunks, int S, int num_splits,
              int split_size, bool ragged) {
  if (D == 128)
    return SplitLaunch<Fp16Policy<128>>::plan(sc, B, HKV, hchunks, S, num_splits, split_size, ragged);
  if (D == 64)
    return SplitLaunch<Fp16Policy<64>>::plan(sc, B, HKV, hchunks, S, num_splits, split_size, ragged);
  return fp16_unsupported(D);
}

int fp16_attrs(int D, int* regs, int* smem, int* local, int* ctas) {
  if (D == 128) return SplitLaunch<Fp16Policy<128>>::attrs(regs, smem, local, ctas);
  if (D == 64) return SplitLaunch<Fp16Policy<64>>::attrs(regs, smem, local, ctas);
  return fp16_unsupported(D);
}

int fp16_device_status_clear() {
  const int zero = 0;
  TKV_CUDA(cudaMemcpyToSymbol(g_fp16_status, &zero, sizeof(int)));
  return TKV_OK;
}

int fp16_device_status(int* status) {
  int v = 0;
  TKV_CUDA(cudaMemcpyFromSymbol(&v, g_fp16_status, sizeof(int)));
  *status = v;
  return TKV_OK;
}

template <int D>
static int fp16_launch_one(const DecodeParams& p, const SplitSched& sc, cudaStream_t stream) {
  using P = Fp16Policy<D>;
  typename P::Maps maps;
  const int64_t rows = (int64_t)p.B * p.HKV * p.S;
  (void)rows;  // the control kernel addresses K and V directly; no tensor maps
  maps.unused = 0;
  return SplitLaunch<P>::launch(maps, p, sc, stream);
}

}  // namespace tkv

extern "C" int tkv_fp16_decode(const void* q, int q_dtype, const void* k, const void* v, float* acc,
                               float* m, float* l, float* out, int B, int HQ, int HKV, int S, int D,
                               float sm_scale, int num_splits, int split_size, int nslots,
                               const int32_t* seq_lens, int flags, void* stream) {
  using namespace tkv;
  TKV_REQUIRE(q && k && v, TKV_ERR_INVALID, "fp16 decode: null input pointer");
  DecodeParams p{};
  int rc = fill_common(p, "fp16 decode", q, q_dtype, acc, m, l, out, B, HQ, HKV, S, sm_scale,
                       num_splits, split_size, nslots, seq_lens, flags);
  if (rc != TKV_OK) return rc;
  TKV_REQUIRE(aligned16(k) && aligned16(v), TKV_ERR_ALIGN,
              "fp16 decode: k and v pointers must be 16-byte aligned");
  p.k = (const __half*)k;
  p.v = (const __half*)v;
  SplitSched sc;
  rc = fp16_plan(D, &sc, B, HKV, p.hchunks, S, num_splits, split_size, seq_lens != nullptr);
  if (rc != TKV_OK) return rc;
  TKV_REQUIRE(sc.nslots == nslots, TKV_ERR_INVALID,
              "fp16 decode: nslots=%d does not match the plan (%d); size acc/m/l with "
              "tkv_decode_plan", nslots, sc.nslots);
  if (D == 128) rc = fp16_launch_one<128>(p, sc, (cudaStream_t)stream);
  else if (D == 64) rc = fp16_launch_one<64>(p, sc, (cudaStream_t)stream);
  else return fp16_unsupported(D);
  if (rc != TKV_OK) return rc;
  if ((flags & TKV_FLAG_COMBINE) && nslots > 1 && !(flags & TKV_FLAG_PARTIALS_ONLY)) {
    TKV_REQUIRE(out, TKV_ERR_INVALID, "fp16 decode: TKV_FLAG_COMBINE needs out");
    return tkv_combine(acc, m, l, out, nullptr, nullptr, B, HQ, nslots, D, stream);
  }
  return TKV_OK;
}
