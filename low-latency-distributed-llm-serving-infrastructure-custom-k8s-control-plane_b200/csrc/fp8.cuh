// Internal interface of the 8-bit cache kernels (fp8_cache.cu, fp8_attention.cu) and their C ABI
// (fp8_api.cu).
//
// An 8-bit cache holds e4m3 numbers (L, NB, BS, Hkv, D) and one fp32 scale per (layer, block, KV
// head), (L, NB, Hkv): an entry stands for code * scale.  The append writes powers of two as
// scales, so dividing by one, and multiplying a code by one, is exact.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace b200 {

// Rows of a call up to which each row's block is looked up by scanning the call's slots (no
// scratch, one launch); above it a marking kernel counts the rows of each block first.  Rows in
// blocks of their own, scanned and marked: 256 rows 6.8 and 10.5 us, 1024 16.6 and 19.0, 2048 36.9
// and 31.8; whole blocks: 1024 rows 18.1 and 17.1, 4096 75 and 26.
constexpr int kAppendScanRows = 1024;

struct AppendFp8Args {
  const void* q_in;  // rotary form: (tokens, hq, D) inside the qkv rows; NULL otherwise
  int64_t q_stok;    // elements
  void* q_out;
  int64_t qo_stok;
  int32_t hq;
  const void* key;
  const void* value;
  int64_t k_stok, k_shead, v_stok, v_shead;  // elements
  const int64_t* positions;                  // rotary form only
  const float* inv_freq;
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  int32_t layer, nb, bs, hkv, head_dim;
  const int64_t* slots;
  int32_t num_tokens;
  int32_t* status;
  // scratch of calls above kAppendScanRows rows: rows per block, num_tokens - (first row of the
  // block), run starts and their number; NULL for the scanning form
  int32_t* count;
  int32_t* first;
  int32_t* num_runs;
  int32_t* runs;
};

size_t append_fp8_scratch_bytes(int nb, int num_tokens);
cudaError_t launch_append_fp8(const AppendFp8Args& a, int dtype, int num_sms, cudaStream_t stream);

struct GatherFp8Args {
  const uint8_t* kc;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  int32_t layer, nb, bs, hkv, head_dim;
  const int64_t* slots;
  int64_t n;
  void* k_out;  // (n, hkv, D), contiguous
  void* v_out;
  int32_t* status;
};

cudaError_t launch_gather_fp8(const GatherFp8Args& a, int dtype, int num_sms, cudaStream_t stream);

struct AttnFp8Args {
  const void* q;
  int64_t q_srow, q_shead;
  const int32_t* query_rows;
  const uint8_t* kc;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  int32_t layer, nb, bs, hkv, head_dim, hq, group;
  const int32_t* bt;
  int32_t bt_stride;
  const int32_t* ctx_lens;
  const int64_t* cu_q;  // NULL: one row per sequence (decode)
  int32_t S;
  float scale;
  void* out;
  int64_t o_srow, o_shead;
  int32_t* status;
};

cudaError_t launch_row_fp8(const AttnFp8Args& a, int dtype, int rows, cudaStream_t stream);

// Copy of the pages of the sequences with more than one new token in 16 bits, for the tensor-core
// prefill: a cache (1, scratch_blocks, BS, Hkv, D) with its block table and clamped lengths.
struct ExpandFp8Args {
  const uint8_t* kc;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  int32_t layer, nb, bs, hkv, head_dim;
  const int32_t* bt;
  int32_t bt_stride;
  const int32_t* ctx_lens;
  const int64_t* cu_q;
  int32_t S, max_ctx;
  int32_t scratch_blocks, scratch_stride;
  int32_t* scratch_ctx;    // (S)
  int32_t* scratch_table;  // (S, scratch_stride)
  void* k16;
  void* v16;
  int32_t* status;
};

cudaError_t launch_expand_fp8(const ExpandFp8Args& a, int dtype, int num_sms, cudaStream_t stream);

// One e4m3 code as fp32 (exact).
__device__ __forceinline__ float e4m3_to_f32(uint8_t c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
  return __half2float(__half(h));
}

// x rounded to the nearest e4m3 number (ties to even); what is not finite becomes NaN, and a
// finite value beyond 448 (a scale that the caller made too small) becomes +-448.
__device__ __forceinline__ uint8_t f32_to_e4m3(float x) {
  return isinf(x) ? 0x7f : __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

}  // namespace b200
