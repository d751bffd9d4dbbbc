// Token sampling: temperature, top-k, top-p and min-p, then a draw by a given uniform number.
//
// For one row with logits x, temperature t and w_i = exp((x_i - max x) / t), tokens ordered by
// decreasing x (ties: the lower index first):
//   top-k keeps the first k;  top-p keeps, of those, each token whose predecessors' sum of w is
//   below p times the sum over the top-k's tokens (so always the first);  min-p keeps tokens with
//   w_i >= min_p (and always the first).  In index order the token drawn is the first one whose
//   cumulative w exceeds u times the kept sum.
// What a draw and a top-p border are decided by are sums of up to 10^5 weights, so w is computed
// in 64 bits and summed in fixed point (64-bit integers): exact sums, in any order.
#include "api_common.cuh"
#include "cache_ops.cuh"
#include "nvtx.cuh"

namespace b200 {

namespace {

struct SampleArgs {
  const void* logits;
  int64_t stride;
  int32_t rows, vocab;
  const float* uniform;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* tokens;
  float* logprobs;
  int32_t* status;
  int32_t shift;  // w is held as round(w * 2^shift)
};

constexpr int kSampleThreads = 1024;

// Row parameters; ok is false where one of them is no number or out of its range.
struct RowParams {
  float u, t, p, mp;
  int32_t k;
  bool ok, greedy;
};

__device__ __forceinline__ RowParams row_params(const SampleArgs& a, int row) {
  RowParams r;
  r.u = a.uniform[row];
  r.t = a.temperature ? a.temperature[row] : 1.f;
  r.k = a.top_k ? a.top_k[row] : 0;
  r.p = a.top_p ? a.top_p[row] : 1.f;
  r.mp = a.min_p ? a.min_p[row] : 0.f;
  r.ok = r.u >= 0.f && r.u < 1.f && r.t >= 0.f && r.t < INFINITY && r.p == r.p && r.mp == r.mp;
  r.greedy = r.t == 0.f;
  if (r.greedy || r.p <= 0.f) r.k = 1;
  if (r.k <= 0 || r.k > a.vocab) r.k = a.vocab;
  r.mp = fminf(r.mp, 1.f);
  return r;
}

// A logit; NaN counts as masked, -0 as 0.
template <typename T>
__device__ __forceinline__ float logit(T v) {
  const float x = to_f32<T>(v) + 0.f;
  return x == x ? x : -INFINITY;
}

// Unsigned key with the order of the floats.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float float_of(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// w of a logit x in a row with maximum mx; it = 1 / temperature is applied by division to stay
// within a rounding of the definition.
__device__ __forceinline__ double weight(float x, float mx, double t) {
  if (x == mx) return 1.0;
  return exp((static_cast<double>(x) - static_cast<double>(mx)) / t);
}

// One CTA per row; the row is read from memory once per pass.
template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_row_kernel(SampleArgs a) {
  __shared__ unsigned long long hist[256];
  __shared__ uint32_t count[256];
  __shared__ int64_t warp_buf[32];
  __shared__ int64_t block_total;
  __shared__ uint32_t sel_prefix;
  __shared__ unsigned long long sel_above;
  __shared__ uint32_t sel_count;
  __shared__ float red_x[32];
  __shared__ int32_t red_i[32];
  __shared__ int32_t found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x, V = a.vocab;
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  const RowParams rp = row_params(a, row);
  const double one = static_cast<double>(1ull << a.shift);

  // maximum, and the lowest index that has it
  float mx = -INFINITY;
  int mi = V;
  for (int i = tid; i < V; i += kSampleThreads) {
    const float v = logit<T>(x[i]);
    if (v > mx) {
      mx = v;
      mi = i;
    }
  }
  const auto better = [&](float v, int i) {
    if (v > mx || (v == mx && i < mi)) {
      mx = v;
      mi = i;
    }
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    better(__shfl_xor_sync(0xffffffffu, mx, o), __shfl_xor_sync(0xffffffffu, mi, o));
  if (lane == 0) {
    red_x[warp] = mx;
    red_i[warp] = mi;
  }
  __syncthreads();
  for (int w = 0; w < 32; ++w) better(red_x[w], red_i[w]);
  if (!rp.ok || mx == -INFINITY) {
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = nanf("");
      flag_status(a.status, B200_DEVICE_BAD_SAMPLE);
    }
    return;
  }
  const double t = rp.greedy ? 1.0 : static_cast<double>(rp.t);
  const auto fixed = [&](double w) { return static_cast<unsigned long long>(__double2ll_rn(w * one)); };

  // the whole vocabulary's sum, for the log probability
  unsigned long long mine = 0;
  for (int i = tid; i < V; i += kSampleThreads) mine += fixed(weight(logit<T>(x[i]), mx, t));
  block_exclusive_scan_1024(static_cast<int64_t>(mine), warp_buf, &block_total);
  const unsigned long long sum_all = block_total;
  __syncthreads();

  uint32_t thr = 0;           // kept: keys above thr, and the first `ties` of the keys equal to it
  int64_t ties = V;
  // ---- top-k: the k-th largest key ---------------------------------------------------------
  if (rp.k < V) {
    uint32_t prefix = 0;
    uint32_t left = rp.k;
    for (int bits = 24; bits >= 0; bits -= 8) {
      if (tid < 256) count[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kSampleThreads) {
        const uint32_t key = key_of(logit<T>(x[i]));
        if (bits == 24 || (key >> (bits + 8)) == prefix) atomicAdd(&count[(key >> bits) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t above = 0;
        int b = 255;
        while (b > 0 && above + count[b] < left) above += count[b--];
        sel_prefix = (prefix << 8) | b;
        sel_count = left - above;
      }
      __syncthreads();
      prefix = sel_prefix;
      left = sel_count;
      __syncthreads();
    }
    thr = prefix;
    ties = left;
  }
  // ---- top-p: where the sum from the top reaches p times the sum ----------------------------
  if (rp.p < 1.f && rp.k > 1) {
    const unsigned long long w_thr = fixed(weight(float_of(thr), mx, t));
    const bool limited = rp.k < V;
    mine = 0;
    for (int i = tid; i < V; i += kSampleThreads) {
      const float v = logit<T>(x[i]);
      if (!limited || key_of(v) > thr) mine += fixed(weight(v, mx, t));
    }
    block_exclusive_scan_1024(static_cast<int64_t>(mine), warp_buf, &block_total);
    unsigned long long total = block_total;
    __syncthreads();
    if (limited) total += w_thr * static_cast<unsigned long long>(ties);
    const double target = static_cast<double>(rp.p) * static_cast<double>(total);
    uint32_t prefix = 0;
    unsigned long long above = 0;
    for (int bits = 24; bits >= 0; bits -= 8) {
      if (tid < 256) {
        hist[tid] = 0;
        count[tid] = 0;
      }
      __syncthreads();
      for (int i = tid; i < V; i += kSampleThreads) {
        const float v = logit<T>(x[i]);
        const uint32_t key = key_of(v);
        if (limited && key <= thr) continue;
        if (bits == 24 || (key >> (bits + 8)) == prefix) {
          atomicAdd(&hist[(key >> bits) & 255u], fixed(weight(v, mx, t)));
          atomicAdd(&count[(key >> bits) & 255u], 1u);
        }
      }
      if (tid == 0 && limited && (bits == 24 || (thr >> (bits + 8)) == prefix)) {
        atomicAdd(&hist[(thr >> bits) & 255u], w_thr * static_cast<unsigned long long>(ties));
        atomicAdd(&count[(thr >> bits) & 255u], static_cast<uint32_t>(ties));
      }
      __syncthreads();
      if (tid == 0) {
        unsigned long long s = above;
        int b = 255, last = -1;
        for (; b >= 0; --b) {
          if (count[b] == 0) continue;
          last = b;
          if (static_cast<double>(s + hist[b]) >= target) break;
          s += hist[b];
        }
        if (b < 0) {  // the sum's rounding: keep everything
          b = last;
          s -= hist[b];
        }
        sel_prefix = (prefix << 8) | b;
        sel_above = s;
        sel_count = count[b];
      }
      __syncthreads();
      prefix = sel_prefix;
      above = sel_above;
      __syncthreads();
    }
    thr = prefix;
    const double w = static_cast<double>(fixed(weight(float_of(thr), mx, t)));
    int64_t n = sel_count;
    if (w > 0) n = min(n, static_cast<int64_t>(ceil((target - static_cast<double>(above)) / w)));
    ties = max(n, static_cast<int64_t>(1));
  }

  // ---- draw: cumulative sums in index order, 1024 tokens at a time ---------------------------
  int token = mi;
  if (!rp.greedy && rp.k > 1) {
    unsigned long long total = 0;
    const double mp = static_cast<double>(rp.mp);
    for (int pass = 0; pass < 2; ++pass) {
      const unsigned long long goal =
          static_cast<unsigned long long>(static_cast<double>(rp.u) * static_cast<double>(total));
      unsigned long long cum = 0;
      int64_t tied = 0;
      if (tid == 0) found = V;
      __syncthreads();
      for (int i0 = 0; i0 < V; i0 += kSampleThreads) {
        const int i = i0 + tid;
        const float v = i < V ? logit<T>(x[i]) : -INFINITY;
        const uint32_t key = key_of(v);
        const bool tie = i < V && key == thr;
        const int64_t rank = block_exclusive_scan_1024(tie ? 1 : 0, warp_buf, &block_total) + tied;
        tied += block_total;
        __syncthreads();
        unsigned long long w = 0;
        if (i < V && (key > thr || (tie && rank < ties))) {
          const double wd = weight(v, mx, t);
          if (wd >= mp) w = fixed(wd);
        }
        const unsigned long long before =
            static_cast<unsigned long long>(block_exclusive_scan_1024(static_cast<int64_t>(w), warp_buf,
                                                                      &block_total)) + cum;
        cum += static_cast<unsigned long long>(block_total);
        if (pass == 1 && w > 0 && before + w > goal) atomicMin(&found, i);
        __syncthreads();
        if (pass == 1 && cum > goal) break;
      }
      total = cum;
    }
    __syncthreads();
    if (found < V) token = found;
  }
  if (tid == 0) {
    a.tokens[row] = token;
    if (a.logprobs) {
      const float v = logit<T>(x[token]);
      const double z = v == mx ? 0.0 : (static_cast<double>(v) - static_cast<double>(mx)) / t;
      a.logprobs[row] = static_cast<float>(z - log(static_cast<double>(sum_all) / one));
    }
  }
}

}  // namespace

}  // namespace b200

extern "C" int b200_sample(const void* logits, int32_t dtype, int64_t stride_row, int32_t rows,
                           int32_t vocab, const float* uniform, const float* temperature,
                           const int32_t* top_k, const float* top_p, const float* min_p,
                           int64_t* tokens, float* logprobs, int32_t* status_word, void* stream) {
  using namespace b200;
  NvtxRange nvtx_range("b200_sample");
  if (esize_of(dtype) == 0) return fail(B200_ERR_UNSUPPORTED, "unsupported dtype");
  if (rows < 0 || vocab <= 0) return fail(B200_ERR_INVALID_ARGUMENT, "rows < 0 or vocab <= 0");
  if (vocab > (1 << 24)) return fail(B200_ERR_UNSUPPORTED, "vocab > 2^24");
  if (rows == 0) return B200_OK;
  if (!logits || !uniform || !tokens) return fail(B200_ERR_INVALID_ARGUMENT, "null pointer");
  SampleArgs a{logits, stride_row, rows,   vocab,  uniform,  temperature, top_k,
               top_p,  min_p,      tokens, logprobs, status_word, 0};
  int bits = 0;
  while ((1 << bits) < vocab) ++bits;
  a.shift = 62 - bits < 46 ? 62 - bits : 46;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200_DTYPE_F32: sample_row_kernel<float><<<rows, kSampleThreads, 0, st>>>(a); break;
    case B200_DTYPE_BF16: sample_row_kernel<__nv_bfloat16><<<rows, kSampleThreads, 0, st>>>(a); break;
    default: sample_row_kernel<__half><<<rows, kSampleThreads, 0, st>>>(a); break;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "sample");
  return B200_OK;
}
