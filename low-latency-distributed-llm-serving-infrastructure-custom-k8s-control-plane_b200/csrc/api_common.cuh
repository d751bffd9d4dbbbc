// Host helpers that the files of the C ABI share: error reporting, element sizes, the SM count and
// the prefill over a 16-bit cache (api.cu).
#pragma once

#include <atomic>
#include <string>

#include "common.cuh"

namespace b200 {

int cuda_fail(cudaError_t e, const char* where);
int fail(int code, const std::string& msg);
int esize_of(int dtype);
int num_sms();

// Lets a kernel have `bytes` of dynamic shared memory on the current device, asking the runtime
// once per kernel and device.  One instance of the flags per kernel: the kernel is a template
// argument.
template <auto Kern>
cudaError_t allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (bit != 0 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn();

// The tensor-core prefill over a 16-bit cache for the sequences with more than one new token only.
// The workspace size is 0 for parameters that it does not cover.
size_t prefill_chunks_workspace_bytes(const B200PrefillParams& p);
int prefill_chunks(const B200PrefillParams& p, void* workspace, size_t workspace_bytes,
                   cudaStream_t st);

}  // namespace b200
