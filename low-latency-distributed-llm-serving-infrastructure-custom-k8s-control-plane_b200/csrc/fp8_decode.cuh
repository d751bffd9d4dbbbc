// Launch interface of the tensor-core decode over an 8-bit cache (fp8_decode.cu).
#pragma once

#include "common.cuh"

namespace b200 {

constexpr int kDecodeFp8MaxSeqs = 1024;  // sequences of one launch (their unit sums sit in shared memory)

// An item that the merge joins: its parts lie at first_slot and at slot + i * slot_step.
struct MergeItem {
  int64_t qrow, slot, first_slot;
  int32_t n, hc, slot_step, pad;
};

struct DecodeFp8Args {
  const void* q;
  int64_t q_srow, q_shead;
  int32_t vec_q;  // query rows and heads are aligned to four elements
  const int32_t* query_rows;
  const int64_t* cu_q;  // mixed batch: only sequences with exactly one new token, row cu_q[s]
  int32_t decodes_only;  // the caller says that there are no others: flagged where there are
  const float* ks;
  const float* vs;
  int32_t layer, nb, bs, hkv, head_dim, group, nchunks;
  const int32_t* bt;
  int32_t bt_stride;
  const int32_t* ctx_lens;
  int32_t S, max_ctx;
  float scale_log2;
  void* out;
  int64_t o_srow, o_shead;
  int32_t* status;
  // workspace: an item to join per warp, and two parts per warp: 8 heads of (m, l) and of D sums
  MergeItem* merge;
  float2* part_ml;
  float* part_o;
};

// CTAs of a launch, and the parts that they may leave behind.
int decode_fp8_grid(int S, int64_t max_ctx, int ips, int num_sms);
int decode_fp8_parts(int grid);
cudaError_t launch_decode_fp8(int dtype, const CUtensorMap& km, const CUtensorMap& vm,
                              const DecodeFp8Args& a, int grid, cudaStream_t stream);

}  // namespace b200
