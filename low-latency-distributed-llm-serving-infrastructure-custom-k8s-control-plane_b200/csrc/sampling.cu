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
#include <cooperative_groups.h>

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

// A logit; NaN counts as masked, an infinite one as the largest number.
template <typename T>
__device__ __forceinline__ float logit(T v) {
  const float x = to_f32<T>(v);
  return x == x ? fminf(x, 3.402823466e38f) : -INFINITY;
}

// Unsigned key with the order of the floats; -0 and 0 are one number.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float float_of(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// w of a logit in a row with maximum mx, from a table of 2^(j/64) and four terms of the exponential
// series: with y = 64 (x - mx) log2(e) / t = n + r, w = 2^(n/64) e^(r ln2 / 64), |r ln2 / 64| <=
// 0.0055, remainder below 5e-14.
struct Weights {
  const double* table;  // 2^(j/64), j < 64, in shared memory
  double mx, c;         // maximum; 64 log2(e) / t
  double bias;          // 2^(52 - shift): adding it leaves round(w 2^shift) in the mantissa's low bits

  __device__ __forceinline__ void set(const double* tab, float m, double t, int shift) {
    table = tab;
    mx = static_cast<double>(m);
    c = 64.0 * 1.4426950408889634 / t;
    bias = static_cast<double>(1ull << (52 - shift));
  }
  // No branches, so that several run in flight.  y is clamped at -3968 (w = 2^-62, which rounds to
  // 0) by its high word: among negative numbers the larger word is the lower number.
  __device__ __forceinline__ double operator()(float x) const {
    double y = (static_cast<double>(x) - mx) * c;
    y = __hiloint2double(static_cast<int>(umin(static_cast<uint32_t>(__double2hiint(y)), 0xC0AF0000u)), __double2loint(y));
    const double v = y + 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are round(y)
    const int n = __double2loint(v);
    const double r = y - (v - 6755399441055744.0);
    constexpr double k = 0.6931471805599453 / 64.0;
    double p = fma(r, k * k * k * k / 24.0, k * k * k / 6.0);
    p = fma(p, r, k * k / 2.0);
    p = fma(p, r, k);
    p = fma(p, r, 1.0);
    const double w = table[n & 63] * p;
    return __hiloint2double(__double2hiint(w) + ((n >> 6) << 20), __double2loint(w));
  }
  __device__ __forceinline__ unsigned long long fixed(double w) const {
    return static_cast<unsigned long long>(__double_as_longlong(w + bias)) & 0xfffffffffffffull;
  }
};

__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 64) table[threadIdx.x] = exp2(static_cast<double>(threadIdx.x) / 64.0);
}

// One CTA per row; the row is read from memory once per pass.  Takes the rows that the cluster
// kernel below has left (their token is kTodo), or every row of a vocabulary that is too large for it.
constexpr int64_t kTodo = -2;

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_row_kernel(SampleArgs a, bool todo_only) {
  __shared__ double table[64];
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
  if (todo_only) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (a.tokens[row] != kTodo) return;
  }
  fill_table(table);
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
  Weights weight;
  weight.set(table, mx, t, a.shift);
  const auto fixed = [&](double w) { return weight.fixed(w); };

  // the whole vocabulary's sum, for the log probability
  unsigned long long mine = 0;
  for (int i = tid; i < V; i += kSampleThreads) mine += fixed(weight(logit<T>(x[i])));
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
    const unsigned long long w_thr = fixed(weight(float_of(thr)));
    const bool limited = rp.k < V;
    mine = 0;
    for (int i = tid; i < V; i += kSampleThreads) {
      const float v = logit<T>(x[i]);
      if (!limited || key_of(v) > thr) mine += fixed(weight(v));
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
          atomicAdd(&hist[(key >> bits) & 255u], fixed(weight(v)));
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
    const double w = static_cast<double>(fixed(weight(float_of(thr))));
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
          const double wd = weight(v);
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

// ---- a cluster of CTAs per row ----------------------------------------------------------------------
//
// Bound by instructions: an exact weight takes some 20, 12 of them on the 64-bit pipe.  256 rows of
// 128256: temperature alone 79 us in bf16 (64 % of the issue slots, 12 % of the copy rate) and 122 in
// fp32, top-k 50 113 and 156, top-p 0.95 188 and 262; one CTA per row that reads it once per pass took
// 933 us for temperature alone and 2963 for all filters (186 before the draw lost its pass after
// top-p, 168 now).  One row of 128256: 13, 18 and 28 us.
//
// The CTAs of a cluster hold a row in their shared memory, each a slice, so it is read from memory
// once; what follows are passes over shared memory, joined through the cluster's.
//   1. the maximum, while the slice is loaded
//   2. top-k and top-p: counts of tokens by (max - x) in 2048 steps of 1/64 (of 1/64 t for top-p).
//      Steps that narrow make the probability of a step known to 0.8 % from its count alone.
//   3. top-p: the exact sum over all tokens and above the few steps that can hold the border, and of
//      each of these steps
//   4. the tokens of the border's step, sorted: the border itself, a token
//   5. exact sums of the kept tokens in index order, by warp; the warp that holds the draw finds it
// Where at most kList tokens can be kept after step 2 (top-k), these alone are sorted and 3 to 5
// done on them.  Rows whose border step holds more than kList tokens (many equal logits) are left
// to sample_row_kernel.
constexpr int kMaxClWarps = 16;
constexpr int kBins = 2048;
constexpr int kList = 1024;
// Entries up to which a list's order is counted out instead of sorted: lists of 240 take 10,600 cycles
// counted and 7,700 sorted; with top-k 50 (lists of about 60) bounds of 64 and 128 are alike.
constexpr int kCounted = 128;
constexpr int kBracket = 512;       // steps that can hold a top-p border
constexpr float kBinScale = 64.f;
constexpr int kFine = 128;          // parts that few steps are divided into (32 and 512: the same time)

struct ClusterShared {
  union {  // the counts are read before the sums are written
    uint32_t hist[kBins];
    unsigned long long sums[kList];
  };
  union {  // and the exact sums of the border's steps before the list
    unsigned long long bins[kBracket];
    unsigned long long list[kList];  // key << 32 | ~index (descending: larger logit, lower index first)
  };
  unsigned long long red[3][kMaxClWarps];
  unsigned long long warp_kept[kMaxClWarps];  // top-p: each warp's kept sum
  uint64_t loaded[4];  // barriers of the slice's quarters
  double table[64];
  float warp_x[kMaxClWarps];
  // of this CTA, for its peers
  float mx;
  unsigned long long total, kept;
  // rank 0's: sums over the cluster
  unsigned long long all_total, all_above, sum32;
  // what rank 0 decides
  int32_t bin, lo, hi, list_n, state, token;
  unsigned long long above_bin;
  double last;  // the open step's share
  uint32_t cut_key;
  uint32_t cut_idx;
};

// Sum of a 64-bit integer over the CTA, known to all threads.  `slot`: which of the scratch rows.
template <int kClThreads>
__device__ __forceinline__ unsigned long long cta_sum(unsigned long long v, unsigned long long* red) {
  constexpr int kClWarps = kClThreads / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kClWarps; ++w) v += red[w];
  return v;
}

// Descending bitonic sort of n <= kList entries, padded with zeros to a power of two.  Exchanges over
// less than 32 places are done in registers, a warp per 32 entries; only longer ones go through shared
// memory with a barrier each (512 entries: 15 barriers instead of 45).
template <int kClThreads>
__device__ void sort_list(unsigned long long* v, int n) {
  const int tid = threadIdx.x;
  int size = 32;
  while (size < n) size <<= 1;
  for (int i = n + tid; i < size; i += kClThreads) v[i] = 0;
  __syncthreads();
  const auto within_warps = [&](int k_first, int k_last) {
    for (int i = tid; i < size; i += kClThreads) {  // size is a multiple of 32: whole warps
      unsigned long long own = v[i];
      for (int k = k_first; k <= k_last; k <<= 1)
        for (int j = k < 32 ? k >> 1 : 16; j > 0; j >>= 1) {
          const unsigned long long other = __shfl_xor_sync(0xffffffffu, own, j);
          const bool larger = ((i & j) == 0) == ((i & k) == 0);
          own = (other > own) == larger ? other : own;
        }
      v[i] = own;
    }
    __syncthreads();
  };
  within_warps(2, 32);
  for (int k = 64; k <= size; k <<= 1) {
    for (int j = k >> 1; j >= 32; j >>= 1) {
      for (int p = tid; p < size / 2; p += kClThreads) {
        const int lo = 2 * p - (p & (j - 1)), hi = lo + j;
        const bool down = (lo & k) == 0;
        const unsigned long long a = v[lo], b = v[hi];
        if ((a < b) == down) {
          v[lo] = b;
          v[hi] = a;
        }
      }
      __syncthreads();
    }
    within_warps(k, k);
  }
}

// Exclusive prefix sums of n <= kList entries in place; returns their sum.  Whole CTA.
template <int kClThreads>
__device__ unsigned long long scan_list(unsigned long long* v, int n, unsigned long long* red) {
  constexpr int kClWarps = kClThreads / 32, kPer = kList / kClThreads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned long long a[kPer], own = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    a[j] = kPer * tid + j < n ? v[kPer * tid + j] : 0;
    own += a[j];
  }
  unsigned long long x = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long t = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += t;
  }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  unsigned long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kClWarps; ++w) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  before += x - own;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (kPer * tid + j < n) v[kPer * tid + j] = before;
    before += a[j];
  }
  __syncthreads();
  return all;
}

// The largest logit of 16 bytes, NaN apart (-inf where there is none).
template <typename T>
__device__ __forceinline__ float largest_of(uint4 u);
template <>
__device__ __forceinline__ float largest_of<float>(uint4 u) {
  return fmaxf(fmaxf(logit<float>(__uint_as_float(u.x)), logit<float>(__uint_as_float(u.y))),
               fmaxf(logit<float>(__uint_as_float(u.z)), logit<float>(__uint_as_float(u.w))));
}
template <>
__device__ __forceinline__ float largest_of<__nv_bfloat16>(uint4 u) {
  const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(&u);
  const __nv_bfloat162 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
  return fmaxf(logit<__nv_bfloat16>(m.x), logit<__nv_bfloat16>(m.y));
}
template <>
__device__ __forceinline__ float largest_of<__half>(uint4 u) {
  const __half2* v = reinterpret_cast<const __half2*>(&u);
  const __half2 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
  return fmaxf(logit<__half>(m.x), logit<__half>(m.y));
}

// kClThreads: 256 for 16-bit logits (four CTAs an SM) and 512 for fp32 (two, as their slices are
// twice the size): when it was chosen, 256 x 128256 with every row's own parameters took 170 us with
// 256 threads and 205 with 512 in bf16, 255 (32 KB slices, 16 CTAs a row) and 234 in fp32.
template <typename T, int kClThreads>
__global__ void __launch_bounds__(kClThreads, 1024 / kClThreads) sample_cluster_kernel(SampleArgs a) {
  constexpr int kClWarps = kClThreads / 32;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) uint8_t dyn[];
  ClusterShared& sh = *reinterpret_cast<ClusterShared*>(dyn);
  uint8_t* buf = dyn + (sizeof(ClusterShared) + 15) / 16 * 16;
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / C, V = a.vocab;
  const int per = (V + C - 1) / C;
  const int begin = min(V, rank * per), n = min(V, begin + per) - begin;
  ClusterShared* head = cluster.map_shared_rank(&sh, 0);
  asm volatile("griddepcontrol.launch_dependents;");

  // ---- 1. load: whole 16-byte pieces where they lie inside the row, single elements at its ends -----
  const T* x0 = static_cast<const T*>(a.logits) + row * a.stride;
  const T* src = x0 + begin;
  const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(src) & 15u);
  const T* s = reinterpret_cast<const T*>(buf + shift);  // s[i]: token begin + i
  fill_table(sh.table);
  for (int i = tid; i < kBins; i += kClThreads) sh.hist[i] = 0;
  for (int i = tid; i < kBracket; i += kClThreads) sh.bins[i] = 0;
  if (tid == 0) {
    sh.list_n = 0;
    sh.state = 0;
    sh.token = 0x7fffffff;
    sh.all_total = sh.all_above = sh.sum32 = 0;
  }
  float mx = -INFINITY;
  {
    // the pieces that lie inside the row come by bulk copy, a quarter at a time (a piece at the
    // slice's end may hold tokens of the next one's)
    constexpr int E = 16 / sizeof(T);
    const uint8_t* aligned = reinterpret_cast<const uint8_t*>(src) - shift;
    const int pieces = n > 0 ? static_cast<int>((shift + n * sizeof(T) + 15) / 16) : 0;
    const int first = begin - static_cast<int>(shift / sizeof(T));  // token of the first piece's first
    const int p0 = pieces > 0 && first < 0 ? 1 : 0;
    const int p1 = pieces > p0 && first + pieces * E > V ? pieces - 1 : pieces;
    const int quarter = (p1 - p0 + 3) / 4;
    if (tid == 0) {
      for (int q = 0; q < 4; ++q) mbar_init(&sh.loaded[q], 1);
      fence_proxy_async_smem();
      for (int q = 0; q < 4; ++q) {
        const int b = p0 + q * quarter, e = min(p1, b + quarter);
        if (e <= b) continue;
        mbar_arrive_expect_tx(&sh.loaded[q], (e - b) * 16);
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                smem_u32(buf + 16 * b)),
            "l"(aligned + 16 * static_cast<int64_t>(b)), "r"((e - b) * 16), "r"(smem_u32(&sh.loaded[q]))
            : "memory");
      }
    }
    // the pieces at the row's ends, by element
    const auto edge = [&](int p) {
      const int i = first + p * E + tid;
      if (tid < E && i >= begin && i < begin + n) {
        const T v = x0[i];
        reinterpret_cast<T*>(buf)[p * E + tid] = v;
        mx = fmaxf(mx, logit<T>(v));
      }
    };
    if (p0 == 1) edge(0);
    if (p1 < pieces) edge(p1);
    __syncthreads();
    for (int q = 0; q < 4; ++q) {
      const int b = p0 + q * quarter, e = min(p1, b + quarter);
      if (e <= b) break;
      if (!mbar_wait_bounded(&sh.loaded[q], 0) && lane == 0) flag_status(a.status, B200_DEVICE_TIMEOUT);
#pragma unroll 2
      for (int p = b + tid; p < e; p += kClThreads)
        mx = fmaxf(mx, largest_of<T>(*reinterpret_cast<const uint4*>(buf + 16 * p)));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) sh.warp_x[warp] = mx;
  __syncthreads();
  for (int w = 0; w < kClWarps; ++w) mx = fmaxf(mx, sh.warp_x[w]);
  if (tid == 0) sh.mx = mx;
  cluster.sync();
  if (lane < C) mx = cluster.map_shared_rank(&sh, lane)->mx;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  mx = __shfl_sync(0xffffffffu, mx, 0);

  const RowParams rp = row_params(a, row);
  if (!rp.ok || mx == -INFINITY) {
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = nanf("");
      flag_status(a.status, B200_DEVICE_BAD_SAMPLE);
    }
    cluster.sync();  // no CTA leaves while its peers read from it
    return;
  }
  // Differences of logits are taken in fp32 below.  One that passes its range stands for a weight of
  // e^-256 or less up to this temperature, and for one that counts beyond: left to sample_row_kernel.
  if (rp.t > 0x1p+120f) {
    if (rank == 0 && tid == 0) a.tokens[row] = kTodo;
    cluster.sync();
    return;
  }
  const double t = rp.greedy ? 1.0 : static_cast<double>(rp.t);
  Weights weight;
  weight.set(sh.table, mx, t, a.shift);
  const double one = static_cast<double>(1ull << a.shift);
  const bool top_k = rp.k < V && rp.k > 1, top_p = rp.p < 1.f && rp.k > 1;
  const double mp = static_cast<double>(rp.mp);
  // each warp's tokens of the slice: [w0, w1), in index order over warps and ranks
  const auto warp_tokens = [](int n) { return ((n + kClWarps - 1) / kClWarps + 31) & ~31; };
  const int wper = warp_tokens(n);
  const int w0 = min(n, warp * wper), w1 = min(n, w0 + wper);

  uint32_t cut_key = 0, cut_idx = 0xffffffffu;  // kept: larger keys, and this key up to this index
  const auto kept = [&](uint32_t key, uint32_t idx) { return key > cut_key || (key == cut_key && idx <= cut_idx); };
  // f(logit, token of the slice) for the warp's tokens; four are read before the first is worked on
  const auto each = [&](auto f) {
    constexpr int U = 4;
    int i = w0 + lane;
    for (; i + 32 * (U - 1) < w1; i += 32 * U) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = logit<T>(s[i + 32 * u]);
#pragma unroll
      for (int u = 0; u < U; ++u) f(v[u], i + 32 * u);
    }
    for (; i < w1; i += 32) f(logit<T>(s[i]), i);
  };
  // f(logit, w in fixed point, token) likewise; the four weights are worked out side by side
  const auto each_weight = [&](auto f) {
    constexpr int U = 4;
    int i = w0 + lane;
    for (; i + 32 * (U - 1) < w1; i += 32 * U) {
      float v[U];
      unsigned long long w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = logit<T>(s[i + 32 * u]);
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = weight.fixed(weight(v[u]));
#pragma unroll
      for (int u = 0; u < U; ++u) f(v[u], w[u], i + 32 * u);
    }
    for (; i < w1; i += 32) {
      const float v = logit<T>(s[i]);
      f(v, weight.fixed(weight(v)), i);
    }
  };
  // Sum of w where only the log probability asks for it: exact for the terms above 2^-10, in fp32 for
  // the many small ones behind them.  A term 2^y of those is off by 3 roundings of y, 2^-24 |y| each, and
  // the exponential's 2^-22: 2.7e-6 of it at the most down to y = -20, below which even 2^20 terms add up
  // to less than the maximum's; measured 2.7e-7 where they hold nearly all of the sum.
  // finite at subnormal temperatures too: the maximum's own term is 2^(0 * c32) = 1
  const float c32 = fminf(static_cast<float>(1.4426950408889634 / t), 3.402823466e38f);
  double sum_large = 0.0;
  float sum_small = 0.f;
  const auto sum32 = [&](float v) {
    const float y = (v - mx) * c32;
    if (y > -10.f) sum_large += weight(v);
    else sum_small += fast_exp2(y);
  };
  // the warps' sums into rank 0's, in fixed point (so their order does not matter); whole CTA
  const auto add_sum32 = [&]() {
    double part = sum_large + static_cast<double>(sum_small);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (lane == 0) atomicAdd(&head->sum32, static_cast<unsigned long long>(part * 0x1p+38));
  };
  const auto sum32_all = [&]() { return static_cast<double>(head->sum32) * 0x1p-38; };
  const auto finish = [&](int token, double sum_all) {
    if (token < 0 || token >= V) {  // none was found: left to sample_row_kernel
      a.tokens[row] = kTodo;
      return;
    }
    a.tokens[row] = token;
    if (a.logprobs) {
      const float v = logit<T>(x0[token]);
      const double z = v == mx ? 0.0 : (static_cast<double>(v) - static_cast<double>(mx)) / t;
      a.logprobs[row] = static_cast<float>(z - log(sum_all));
    }
  };
  // the place of a logit below the maximum, in steps; its step is the place's whole part, the last
  // one being open
  const auto place_of = [&](float v, float scale) { return (mx - v) * scale; };
  const auto bin_of = [&](float v, float scale) {
    return static_cast<int>(fminf(place_of(v, scale), static_cast<float>(kBins - 1)));
  };
  // counts by step, summed over the cluster into rank 0's; `f` is given every logit
  const auto histogram = [&](float scale, bool all, auto f) {
    each([&](float v, int i) {
      f(v);
      if (all || kept(key_of(v), begin + i)) atomicAdd(&sh.hist[bin_of(v, scale)], 1u);
    });
    __syncthreads();
    if (rank != 0)
      for (int i = tid; i < kBins; i += kClThreads)
        if (sh.hist[i]) atomicAdd(&head->hist[i], sh.hist[i]);
  };
  // tokens of steps [lo, hi] that are kept, into rank 0's list
  const auto gather = [&](float scale, int lo, int hi) {
    const float from = static_cast<float>(lo), to = hi >= kBins - 1 ? INFINITY : static_cast<float>(hi + 1);
    each([&](float v, int i) {
      const float at_step = place_of(v, scale);
      if (at_step >= from && (at_step < to || to == INFINITY)) {
        const uint32_t key = key_of(v), idx = begin + i;
        if (kept(key, idx)) {
          const int at = atomicAdd(&head->list_n, 1);
          if (at < kList) head->list[at] = (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - idx);
        }
      }
    });
    cluster.sync();
  };

  if (rp.greedy || rp.k == 1) {
    int best = V;
    each([&](float v, int i) {
      sum32(v);
      if (v == mx) best = min(best, begin + i);
    });
    if (best < V) atomicMin(&head->token, best);
    add_sum32();
    cluster.sync();  // rank 0 goes on with what it holds; its peers are done
    if (rank == 0 && tid == 0) finish(sh.token, sum32_all());
    return;
  }

  // Sums over the entries of the list that `before` puts ahead of an entry, for each of its m <=
  // kCounted entries: a warp takes four entries at a time, its lanes side by side through the list.
  // What is counted and summed goes to take(entry, count, sum), in lane 0.  Whole CTA.
  const auto compare_all = [&](int m, auto before, auto take) {
    constexpr int E = 4;
    for (int e0 = warp * E; e0 < m; e0 += kClWarps * E) {
      unsigned long long own[E], sum[E];
      uint32_t count[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        own[e] = sh.list[min(e0 + e, m - 1)];
        sum[e] = 0;
        count[e] = 0;
      }
#pragma unroll 2
      for (int o = lane; o < m; o += 32) {
        const unsigned long long other = sh.list[o], w = sh.sums[o];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const bool ahead = before(other, own[e]);
          count[e] += ahead ? 1 : 0;
          sum[e] += ahead ? w : 0;
        }
      }
      // a lane's sum is at most 2^48 (kCounted / 32 = 4 weights of at most 2^46): in two parts of 26 bits
      static_assert(kCounted <= 32 * 63, "a lane's sum stays below 2^52");
#pragma unroll
      for (int e = 0; e < E; ++e) {
        count[e] = __reduce_add_sync(0xffffffffu, count[e]);
        const uint32_t low = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(sum[e]) & 0x3ffffffu);
        const uint32_t high = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(sum[e] >> 26));
        if (lane == 0 && e0 + e < m) take(e0 + e, static_cast<int>(count[e]), (static_cast<unsigned long long>(high) << 26) + low);
      }
    }
    __syncthreads();
  };
  // Order of the list's entries: each one's weight into sums, how many are ahead of it into place, and
  // their weights' sum into ahead (behind the entries that the two arrays hold).
  unsigned long long* const ahead = sh.sums + kCounted;
  unsigned long long* const place = sh.list + kCounted;
  const auto order_list = [&](int m) {
    for (int i = tid; i < m; i += kClThreads)
      sh.sums[i] = weight.fixed(weight(float_of(static_cast<uint32_t>(sh.list[i] >> 32))));
    __syncthreads();
    compare_all(m, [](unsigned long long other, unsigned long long own) { return other > own; },
                [&](int e, int count, unsigned long long sum) {
                  place[e] = count;
                  ahead[e] = sum;
                });
  };

  if (top_k) {
    histogram(kBinScale, true, sum32);
    add_sum32();
    cluster.sync();
    if (rank == 0) {
      // the step that holds the k-th token, and how many tokens lie up to it
      const int per_t = kBins / kClThreads;
      unsigned long long mine = 0;
      for (int j = 0; j < per_t; ++j) mine += sh.hist[tid * per_t + j];
      unsigned long long x = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long u = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += u;
      }
      if (lane == 31) sh.red[0][warp] = x;
      __syncthreads();
      unsigned long long before = x - mine;
      for (int w = 0; w < warp; ++w) before += sh.red[0][w];
      const unsigned long long k = static_cast<unsigned long long>(rp.k);
      for (int j = 0; j < per_t; ++j) {
        const unsigned long long h = sh.hist[tid * per_t + j];
        if (before < k && before + h >= k) {
          sh.bin = tid * per_t + j;
          sh.above_bin = before;
          // 1: all tokens up to the step fit in the list; 2: the step's tokens do; 3: neither
          sh.state = before + h <= kList ? 1 : h <= kList ? 2 : 3;
        }
        before += h;
      }
    }
    cluster.sync();
    const int state = head->state, bin = head->bin;  // 3: left to sample_row_kernel
    if (state == 3) {
      if (rank == 0 && tid == 0) a.tokens[row] = kTodo;
      cluster.sync();
      return;
    }
    gather(kBinScale, state == 1 ? 0 : bin, bin);
    if (state == 1 && rank != 0) return;  // rank 0 has all that is left
    if (rank == 0) {
      const int m = sh.list_n;
      if (state == 1) {
        // everything else on the list: its first k tokens, of these top-p's, and the draw
        if (m <= kCounted) {
          order_list(m);
          unsigned long long total = 0, sum = 0;
          for (int i = tid; i < m; i += kClThreads)
            if (static_cast<int>(place[i]) < rp.k) total += sh.sums[i];
          total = cta_sum<kClThreads>(total, sh.red[0]);
          const double target = static_cast<double>(rp.p) * static_cast<double>(total);
          for (int i = tid; i < m; i += kClThreads) {
            const bool in = static_cast<int>(place[i]) < rp.k &&
                            (!top_p || place[i] == 0 || static_cast<double>(ahead[i]) < target) &&
                            weight(float_of(static_cast<uint32_t>(sh.list[i] >> 32))) >= mp;
            if (!in) sh.sums[i] = 0;
            sum += sh.sums[i];
          }
          sum = cta_sum<kClThreads>(sum, sh.red[0]);
          const unsigned long long goal =
              static_cast<unsigned long long>(static_cast<double>(rp.u) * static_cast<double>(sum));
          // the low words are ~index: larger for lower ones
          compare_all(m,
                      [](unsigned long long other, unsigned long long own) {
                        return static_cast<uint32_t>(other) > static_cast<uint32_t>(own);
                      },
                      [&](int e, int, unsigned long long before) {
                        if (before <= goal && goal < before + sh.sums[e])
                          sh.token = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(sh.list[e]));
                      });
        } else {
          sort_list<kClThreads>(sh.list, m);
          const int keep_k = min(m, rp.k);
          for (int i = tid; i < kList; i += kClThreads)
            sh.sums[i] = i < keep_k ? weight.fixed(weight(float_of(static_cast<uint32_t>(sh.list[i] >> 32)))) : 0;
          __syncthreads();
          const unsigned long long total = scan_list<kClThreads>(sh.sums, keep_k, sh.red[0]);
          const double target = static_cast<double>(rp.p) * static_cast<double>(total);
          for (int i = tid; i < m; i += kClThreads) {
            const unsigned long long e = sh.list[i];
            const double w = weight(float_of(static_cast<uint32_t>(e >> 32)));
            const bool in = i < keep_k && (!top_p || i == 0 || static_cast<double>(sh.sums[i]) < target) && w >= mp;
            // by index; a token that is not kept sorts behind as 0
            sh.list[i] = in ? (e << 32) | (e >> 32) : 0;
          }
          __syncthreads();
          sort_list<kClThreads>(sh.list, m);
          for (int i = tid; i < kList; i += kClThreads)
            sh.sums[i] = i < m && sh.list[i] != 0 ? weight.fixed(weight(float_of(static_cast<uint32_t>(sh.list[i])))) : 0;
          __syncthreads();
          const unsigned long long sum = scan_list<kClThreads>(sh.sums, m, sh.red[0]);
          const unsigned long long goal =
              static_cast<unsigned long long>(static_cast<double>(rp.u) * static_cast<double>(sum));
          for (int i = tid; i < m; i += kClThreads) {
            const unsigned long long after = i + 1 < m ? sh.sums[i + 1] : sum;
            if (sh.sums[i] <= goal && goal < after)
              sh.token = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(sh.list[i] >> 32));
          }
        }
        __syncthreads();
        if (tid == 0) finish(sh.token, sum32_all());
      } else {
        sort_list<kClThreads>(sh.list, m);
        if (tid == 0) {
          const unsigned long long e = sh.list[rp.k - static_cast<int>(sh.above_bin) - 1];
          sh.cut_key = static_cast<uint32_t>(e >> 32);
          sh.cut_idx = 0xffffffffu - static_cast<uint32_t>(e);
        }
      }
    }
    if (state == 1) return;
    cluster.sync();
    cut_key = head->cut_key;
    cut_idx = head->cut_idx;
    cluster.sync();
  }

  if (top_p) {
    const float scale = kBinScale / static_cast<float>(t);
    if (top_k) {  // a second set of counts
      for (int i = tid; i < kBins; i += kClThreads) sh.hist[i] = 0;
      for (int i = tid; i < kBracket; i += kClThreads) sh.bins[i] = 0;
      if (tid == 0) {
        sh.list_n = 0;
        sh.state = 0;
      }
      cluster.sync();
    }
    histogram(scale, !top_k, [](float) {});
    cluster.sync();
    if (rank == 0) {
      // the border's steps: where p times the sum can lie, with a step's sum known to e^(1/64)
      const int per_t = kBins / kClThreads;
      constexpr double kStep = 0.9844964370054085;  // e^(-1/64)
      double mine[per_t], sum = 0.0, most_w = exp(-static_cast<double>(tid * per_t) / 64.0), last_w = 0.0;
      for (int j = 0; j < per_t; ++j) {
        mine[j] = sh.hist[tid * per_t + j] * most_w;  // at most this
        sum += mine[j];
        last_w = mine[j];
        most_w *= kStep;
      }
      if (tid == kClThreads - 1) sh.last = last_w;
      double x = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += u;
      }
      if (lane == 31) sh.red[0][warp] = static_cast<unsigned long long>(__double_as_longlong(x));
      if (tid == 0) {
        sh.lo = kBins - 1;
        sh.hi = kBins - 1;
      }
      __syncthreads();
      double before = x - sum, all = 0.0;
      for (int w = 0; w < kClWarps; ++w) {
        const double v = __longlong_as_double(static_cast<long long>(sh.red[0][w]));
        if (w < warp) before += v;
        all += v;
      }
      // A step's true sum lies between e^(-1/64) and 1 times what is counted, but for the last step,
      // which is open; kLow and kUp leave 1e-5 for bin_of's rounding.  The border is the first step
      // where the sum from the top reaches p times the whole, and where the sum behind it is at most
      // 1 - p times the whole: for p near 1 the latter says far more.
      constexpr double kLow = 0.98447, kUp = 1.00001;
      const double last = sh.last;
      const double p = static_cast<double>(rp.p), most = all * kUp, least = (all - last) * kLow;
      int first_may = kBins - 1, first_must = kBins - 1;
      for (int j = 0; j < per_t; ++j) {
        const int b = tid * per_t + j;
        const double after = before + mine[j], tail = fmax(all - after, 0.0);
        const bool may = after * kUp >= p * least && (tail - last) * kLow <= (1.0 - p) * most;
        const bool must = (b == kBins - 1 ? 0.0 : after * kLow) >= p * most || tail * kUp + 1e-12 * all <= (1.0 - p) * least;
        if (may) first_may = min(first_may, b);
        if (must) first_must = min(first_must, b);
        before = after;
      }
      first_may = __reduce_min_sync(0xffffffffu, first_may);
      first_must = __reduce_min_sync(0xffffffffu, first_must);
      if (lane == 0) {
        atomicMin(&sh.lo, first_may);
        atomicMin(&sh.hi, first_must);
      }
    }
    cluster.sync();
    const int lo = head->lo, hi = max(lo, head->hi);
    // exact sums: all kept tokens, those above the border's steps, each of these steps
    unsigned long long total = 0, above = 0;
    const bool few = hi - lo < kBracket;
    // the steps in parts, so that few tokens share one with the border
    int split = 1;
    while (split < kFine && (hi - lo + 1) * split * 2 <= kFine) split *= 2;
    const float parts = static_cast<float>(split);
    if (few) {
      const float from = static_cast<float>(lo), last_part = static_cast<float>(kBins * split - 1);
      const float behind = hi == kBins - 1 ? INFINITY : static_cast<float>(hi + 1);
      each_weight([&](float v, unsigned long long w, int i) {
        if (top_k && !kept(key_of(v), begin + i)) w = 0;
        total += w;
        const float at_step = place_of(v, scale);
        above += at_step < from ? w : 0;
        if (!(at_step < from) && !(at_step >= behind && behind < INFINITY))
          atomicAdd(&sh.bins[static_cast<int>(fminf(at_step * parts, last_part)) - lo * split], w);
      });
    }
    unsigned long long mine = mp > 0.0 ? 0 : above;  // of the kept tokens above the border's step
    total = cta_sum<kClThreads>(total, sh.red[1]);
    above = cta_sum<kClThreads>(above, sh.red[2]);  // its barriers order the steps' sums too
    if (tid == 0) {
      atomicAdd(&head->all_total, total);
      atomicAdd(&head->all_above, above);
    }
    if (rank != 0 && few)
      for (int i = tid; i < (hi - lo + 1) * split; i += kClThreads)
        if (sh.bins[i]) atomicAdd(&head->bins[i], sh.bins[i]);
    cluster.sync();
    if (rank == 0) {
      // the border's part: the first one that reaches the target; each thread looks at kPer parts in a
      // row
      constexpr int kPer = kBracket / kClThreads;
      const int steps = few ? (hi - lo + 1) * split : 0;
      unsigned long long h[kPer], own = 0;
      for (int j = 0; j < kPer; ++j) {
        const int b = kPer * tid + j;
        h[j] = b < steps ? sh.bins[b] : 0;
        own += h[j];
      }
      unsigned long long x = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long u = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += u;
      }
      if (lane == 31) sh.red[0][warp] = x;
      if (tid == 0) sh.state = 3;
      __syncthreads();
      const double target = static_cast<double>(rp.p) * static_cast<double>(sh.all_total);
      unsigned long long up = sh.all_above + x - own;
      for (int w = 0; w < warp; ++w) up += sh.red[0][w];
      for (int j = 0; j < kPer; ++j) {
        const int b = kPer * tid + j;
        if (b < steps && static_cast<double>(up) < target && static_cast<double>(up + h[j]) >= target) {
          sh.bin = lo * split + b;
          sh.above_bin = up;
          sh.state = 2;
        }
        up += h[j];
      }
    }
    cluster.sync();
    const int state = head->state, bin = head->bin;
    if (state == 3) {
      if (rank == 0 && tid == 0) a.tokens[row] = kTodo;
      cluster.sync();
      return;
    }
    // The border part's tokens into rank 0's list.  What the draw needs of the others is the sum of
    // each warp's tokens above it: the exact pass has it but for the steps from lo on, few of
    // the tokens (with min-p, which the exact pass leaves out, all are looked at again).
    {
      const float from = mp > 0.0 ? -1.f : static_cast<float>(lo), at_bin = static_cast<float>(bin) / parts;
      const float to = bin == kBins * split - 1 ? INFINITY : static_cast<float>(bin + 1) / parts;
      each([&](float v, int i) {
        const float at_step = place_of(v, scale);
        if (at_step < from || (at_step >= to && to < INFINITY)) return;
        const uint32_t key = key_of(v), idx = begin + i;
        if (!kept(key, idx)) return;
        if (at_step < at_bin) {
          const double w = weight(v);
          if (w >= mp) mine += weight.fixed(w);
        } else {
          const int at = atomicAdd(&head->list_n, 1);
          if (at < kList) head->list[at] = (static_cast<unsigned long long>(key) << 32) | (0xffffffffu - idx);
        }
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
      if (lane == 0) sh.warp_kept[warp] = mine;
    }
    cluster.sync();
    if (head->list_n > kList) {  // left to sample_row_kernel
      if (rank == 0 && tid == 0) a.tokens[row] = kTodo;
      cluster.sync();
      return;
    }
    if (rank == 0) {
      const int m = sh.list_n;
      const double target = static_cast<double>(rp.p) * static_cast<double>(sh.all_total);
      if (m <= kCounted) {
        order_list(m);
        for (int i = tid; i < m; i += kClThreads) {
          // the last token that is kept: the sum ahead of it is short of the target, with it it is not
          const unsigned long long up = sh.above_bin + ahead[i];
          if (static_cast<double>(up) < target && (static_cast<double>(up + sh.sums[i]) >= target || static_cast<int>(place[i]) == m - 1)) {
            sh.cut_key = static_cast<uint32_t>(sh.list[i] >> 32);
            sh.cut_idx = 0xffffffffu - static_cast<uint32_t>(sh.list[i]);
          }
        }
      } else {
        sort_list<kClThreads>(sh.list, m);
        for (int i = tid; i < kList; i += kClThreads)
          sh.sums[i] = i < m ? weight.fixed(weight(float_of(static_cast<uint32_t>(sh.list[i] >> 32)))) : 0;
        __syncthreads();
        scan_list<kClThreads>(sh.sums, m, sh.red[0]);
        for (int i = tid; i < m; i += kClThreads) {
          const bool in = static_cast<double>(sh.above_bin + sh.sums[i]) < target;
          const bool next = i + 1 < m && static_cast<double>(sh.above_bin + sh.sums[i + 1]) < target;
          if (in && !next) {
            sh.cut_key = static_cast<uint32_t>(sh.list[i] >> 32);
            sh.cut_idx = 0xffffffffu - static_cast<uint32_t>(sh.list[i]);
          }
        }
      }
      __syncthreads();
      // what is kept of the list, to the sums of the warps that hold it
      for (int i = tid; i < m; i += kClThreads) {
        const uint32_t key = static_cast<uint32_t>(sh.list[i] >> 32), idx = 0xffffffffu - static_cast<uint32_t>(sh.list[i]);
        if (key < sh.cut_key || (key == sh.cut_key && idx > sh.cut_idx)) continue;
        const double w = weight(float_of(key));
        if (w < mp) continue;
        const int r = static_cast<int>(idx) / per, at = static_cast<int>(idx) - r * per;
        atomicAdd(&cluster.map_shared_rank(&sh, r)->warp_kept[at / warp_tokens(min(V - r * per, per))], weight.fixed(w));
      }
    }
    cluster.sync();
    cut_key = head->cut_key;
    cut_idx = head->cut_idx;
  }

  // ---- 5. draw -----------------------------------------------------------------------------------
  const bool filtered = top_k || top_p;
  unsigned long long mine = 0, all = 0;
  if (top_p) {
    mine = sh.warp_kept[warp];
  } else if (!filtered && mp <= 0.0) {
    each_weight([&](float, unsigned long long w, int) { mine += w; });
    all = mine;
  } else {
    each([&](float v, int i) {
      if (top_k && !kept(key_of(v), begin + i)) return;
      const double w = weight(v);
      const unsigned long long f = weight.fixed(w);
      all += f;
      if (w >= mp) mine += f;
    });
  }
  if (!top_p) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  }
  __syncthreads();
  if (lane == 0) sh.red[0][warp] = mine;
  all = cta_sum<kClThreads>(all, sh.red[1]);
  if (tid == 0) {
    unsigned long long sum = 0;
    for (int w = 0; w < kClWarps; ++w) sum += sh.red[0][w];
    sh.kept = sum;
    sh.total = all;
  }
  cluster.sync();
  unsigned long long before = 0, sum = 0, sum_all = 0;
  if (lane < C) {
    const ClusterShared* o = cluster.map_shared_rank(&sh, lane);
    sum = o->kept;
    sum_all = o->total;
    before = lane < rank ? sum : 0;
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    sum_all += __shfl_xor_sync(0xffffffffu, sum_all, o);
  }
  before = __shfl_sync(0xffffffffu, before, 0);
  sum = __shfl_sync(0xffffffffu, sum, 0);
  sum_all = __shfl_sync(0xffffffffu, sum_all, 0);
  const unsigned long long goal = static_cast<unsigned long long>(static_cast<double>(rp.u) * static_cast<double>(sum));
  // the whole vocabulary's sum: of this pass, or of the top-p's, or (top-k) of the first
  const double z = top_k ? sum32_all() : static_cast<double>(top_p ? head->all_total : sum_all) / one;
  cluster.sync();  // from here on each CTA reads its own memory only, and may end
  // the warp's part that holds the draw, if it is one of this CTA's: all threads look through it
  int part = -1;
  for (int w = 0; w < kClWarps; ++w) {
    const unsigned long long m = sh.red[0][w];
    if (part < 0) {
      if (before <= goal && goal < before + m) part = w;
      else before += m;
    }
  }
  if (part >= 0) {
    const int p0 = min(n, part * wper), p1 = min(n, p0 + wper);
    const int each = (p1 - p0 + kClThreads - 1) / kClThreads;
    const int i0 = min(p1, p0 + tid * each), i1 = min(p1, i0 + each);
    const auto counts = [&](int i) -> unsigned long long {
      const float v = logit<T>(s[i]);
      if (filtered && !kept(key_of(v), begin + i)) return 0;
      const double w = weight(v);
      return w >= mp ? weight.fixed(w) : 0;
    };
    unsigned long long own = 0;
    for (int i = i0; i < i1; ++i) own += counts(i);
    unsigned long long x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += u;
    }
    if (lane == 31) sh.red[1][warp] = x;
    __syncthreads();
    before += x - own;
    for (int w = 0; w < warp; ++w) before += sh.red[1][w];
    if (before <= goal && goal < before + own) {
      int token = V;
      for (int i = i0; i < i1; ++i) {
        before += counts(i);
        if (before > goal) {
          token = begin + i;
          break;
        }
      }
      finish(token, z);
    }
  }
}

// CTAs a row: enough to make a slice at most 16384 tokens, but 8 at most (192 KB of tokens each);
// more where the rows would leave SMs idle.  0: the vocabulary does not fit.
// Slices of up to 16384 tokens against 32768, rows of 128256: 256 in bf16 with top-p 303 and 373 us,
// top-k 111 and 131, unfiltered 74 and 78; fp32 unfiltered 122 and 117.  Spread over idle SMs or not,
// 8 bf16 rows of 32000: top-p 27 and 50 us, top-k 14 and 23; 16 fp32 rows with top-p 27 and 36.
int cluster_size(int rows, int vocab, int es, int num_sms) {
  const int64_t bytes = static_cast<int64_t>(vocab) * es;
  if ((bytes + 7) / 8 > 192 * 1024) return 0;
  int c = 1;
  while (c < 8 && (vocab / c > 16384 || bytes / c > 192 * 1024 || (rows * c * 2 <= num_sms && vocab / c > 1024))) c *= 2;
  return c;
}

template <typename T>
cudaError_t launch_sample(const SampleArgs& a, cudaStream_t stream) {
  constexpr int kClThreads = sizeof(T) == 2 ? 256 : 512;
  const int C = cluster_size(a.rows, a.vocab, sizeof(T), num_sms());
  if (C == 0) {
    sample_row_kernel<T><<<a.rows, kSampleThreads, 0, stream>>>(a, false);
    return cudaGetLastError();
  }
  const int slice = (a.vocab + C - 1) / C;
  const size_t smem = (sizeof(ClusterShared) + 15) / 16 * 16 + (static_cast<size_t>(slice) * sizeof(T) + 47) / 16 * 16;
  cudaError_t e = allow_smem<sample_cluster_kernel<T, kClThreads>>(227 * 1024);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.rows * C);
  cfg.blockDim = dim3(kClThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, sample_cluster_kernel<T, kClThreads>, a);
  if (e != cudaSuccess) return e;
  // the rows that are left; its launch overlaps the cluster kernel's end
  attr[0] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(a.rows);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, sample_row_kernel<T>, a, true);
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
  const cudaError_t e = dtype == B200_DTYPE_F32    ? launch_sample<float>(a, st)
                        : dtype == B200_DTYPE_BF16 ? launch_sample<__nv_bfloat16>(a, st)
                                                   : launch_sample<__half>(a, st);
  if (e != cudaSuccess) return cuda_fail(e, "sample");
  return B200_OK;
}
