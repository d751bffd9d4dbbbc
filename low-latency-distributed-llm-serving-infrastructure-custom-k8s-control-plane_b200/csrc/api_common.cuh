// Host helpers that the files of the C ABI share: error reporting, element sizes, the SM count and
// the prefill over a 16-bit cache (api.cu).
#pragma once

#include <string>

#include "common.cuh"

namespace b200 {

int cuda_fail(cudaError_t e, const char* where);
int fail(int code, const std::string& msg);
int esize_of(int dtype);
int num_sms();

}  // namespace b200
