// Attention over an 8-bit paged cache:  o = sum_j softmax_j(scale * q.k_j) v_j  with
// k_j = code * key scale of the block, v_j = code * value scale of the block.
#include <type_traits>

#include "api_common.cuh"
#include "fp8.cuh"

namespace b200 {

namespace {

constexpr int kRowWarps = 8;

// For what the tensor-core kernels do not take (fp32 prefill, head dims other than 64 and 128, odd block
// sizes).  One CTA per (query row, KV head, up to 8 query heads): each warp takes every kRowWarps-th
// position, the running (max, sum, output) of the warps are merged at the end.
template <typename T, int NPL>
__global__ void __launch_bounds__(kRowWarps * 32) row_fp8_kernel(AttnFp8Args a, int nchunks) {
  extern __shared__ float rsm[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x;
  const int h = blockIdx.y / nchunks, cch = blockIdx.y - h * nchunks;
  const int nh = min(8, a.group - cch * 8);
  const int hq0 = h * a.group + cch * 8;
  const int D = a.head_dim;
  float* o_w = rsm;                     // [warps][8][D]
  float* m_w = o_w + kRowWarps * 8 * D;  // [warps][8]
  float* l_w = m_w + kRowWarps * 8;      // [warps][8]

  int64_t qrow = row;
  int32_t seq = row, n_ctx;
  if (a.cu_q == nullptr) {
    qrow = a.query_rows ? a.query_rows[row] : row;
    n_ctx = a.ctx_lens[seq];
  } else {
    int lo = 0, hi = a.S - 1;  // last s with cu_q[s] <= row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.cu_q[mid] <= row) lo = mid; else hi = mid - 1;
    }
    seq = lo;
    if (row < a.cu_q[seq] || row >= a.cu_q[seq + 1]) return;  // behind the last sequence
    n_ctx = a.ctx_lens[seq] - static_cast<int32_t>(a.cu_q[seq + 1] - row) + 1;
  }
  // pages that the table row holds
  n_ctx = static_cast<int32_t>(min(static_cast<int64_t>(n_ctx),
                                   static_cast<int64_t>(a.bt_stride) * a.bs));
  const int32_t* bt_row = a.bt + static_cast<int64_t>(seq) * a.bt_stride;

  float q[8][NPL], acc[8][NPL], m[8], l[8];
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const int d = lane + 32 * i;
      acc[g][i] = 0.f;
      q[g][i] = g < nh && d < D ? to_f32<T>(static_cast<const T*>(a.q)[qrow * a.q_srow +
                                                static_cast<int64_t>(hq0 + g) * a.q_shead + d])
                                : 0.f;
    }
  }
  const int64_t row_bytes = static_cast<int64_t>(a.hkv) * D;
  for (int pos = warp; pos < n_ctx; pos += kRowWarps) {
    const int32_t blk = bt_row[pos / a.bs];
    if (blk < 0 || blk >= a.nb) {
      if (lane == 0) flag_status(a.status, B200_DEVICE_BAD_BLOCK);
      continue;
    }
    const int64_t b = static_cast<int64_t>(a.layer) * a.nb + blk;
    const int64_t at = (b * a.bs + pos % a.bs) * row_bytes + h * D;
    const float ks = a.ks[b * a.hkv + h] * a.scale, vs = a.vs[b * a.hkv + h];
    float kv[NPL], vv[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const int d = lane + 32 * i;
      kv[i] = d < D ? e4m3_to_f32(a.kc[at + d]) : 0.f;
      vv[i] = d < D ? e4m3_to_f32(a.vc[at + d]) * vs : 0.f;
    }
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      if (g >= nh) break;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NPL; ++i) s = fmaf(q[g][i], kv[i], s);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      s *= ks;
      if (s == -INFINITY) continue;
      const float mx = fmaxf(m[g], s == s ? s : -3.0e38f);  // a NaN score reaches the sums
      const float alpha = m[g] == -INFINITY ? 0.f : expf(m[g] - mx);
      const float pw = expf(s - mx);
      l[g] = l[g] * alpha + pw;
#pragma unroll
      for (int i = 0; i < NPL; ++i) acc[g][i] = fmaf(pw, vv[i], acc[g][i] * alpha);
      m[g] = mx;
    }
  }
  if (lane == 0) {
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      m_w[warp * 8 + g] = m[g];
      l_w[warp * 8 + g] = l[g];
    }
  }
#pragma unroll
  for (int g = 0; g < 8; ++g)
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const int d = lane + 32 * i;
      if (d < D) o_w[(warp * 8 + g) * D + d] = acc[g][i];
    }
  __syncthreads();
  for (int idx = tid; idx < nh * D; idx += kRowWarps * 32) {
    const int g = idx / D, d = idx - g * D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) M = fmaxf(M, m_w[w * 8 + g]);
    float o = 0.f, L = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      if (m_w[w * 8 + g] == -INFINITY) continue;
      const float wt = expf(m_w[w * 8 + g] - M);
      o += wt * o_w[(w * 8 + g) * D + d];
      L += wt * l_w[w * 8 + g];
    }
    T* op = static_cast<T*>(a.out) + qrow * a.o_srow + static_cast<int64_t>(hq0 + g) * a.o_shead;
    op[d] = from_f32<T>(L != 0.f ? o / L : 0.f);
  }
}

template <typename T>
cudaError_t launch_row_t(const AttnFp8Args& a, int rows, cudaStream_t stream) {
  const int nchunks = (a.group + 7) / 8;
  const dim3 grid(rows, a.hkv * nchunks);
  const int npl = (a.head_dim + 31) / 32;
  const size_t smem = (kRowWarps * 8 * a.head_dim + 2 * kRowWarps * 8) * sizeof(float);
  if (npl <= 1) row_fp8_kernel<T, 1><<<grid, kRowWarps * 32, smem, stream>>>(a, nchunks);
  else if (npl <= 2) row_fp8_kernel<T, 2><<<grid, kRowWarps * 32, smem, stream>>>(a, nchunks);
  else if (npl <= 4) row_fp8_kernel<T, 4><<<grid, kRowWarps * 32, smem, stream>>>(a, nchunks);
  else if (npl <= 8) {
    const cudaError_t e = allow_smem<row_fp8_kernel<T, 8>>(68 * 1024);
    if (e != cudaSuccess) return e;
    row_fp8_kernel<T, 8><<<grid, kRowWarps * 32, smem, stream>>>(a, nchunks);
  } else {
    return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

// ---- the 16-bit copy of a prefill's pages -----------------------------------------------------

// 16 codes at scale s in 16 bits: exact for bf16 with power-of-two scales; f16 values beyond its
// range become +-65504.
template <typename T>
__device__ __forceinline__ void widen16(uint4 c, float s, uint4 (&out)[2]) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((w[i >> 1] >> (16 * (i & 1))) & 0xffffu), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    float x = f.x * s, y = f.y * s;
    if (std::is_same<T, __half>::value) {
      x = fabsf(x) > 65504.f ? copysignf(65504.f, x) : x;
      y = fabsf(y) > 65504.f ? copysignf(65504.f, y) : y;
    }
    o[i] = MmaOp<T>::pack(x, y);
  }
  out[0] = make_uint4(o[0], o[1], o[2], o[3]);
  out[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

// Each CTA copies an equal share of the scratch blocks, 16 codes per thread and step.  Every CTA
// sums up the sequences' blocks by itself, 256 sequences at a time (1 us for a few hundred; a
// kernel of its own for the sums took 4 us and a launch).  Bound by memory: 1 byte read and 2
// written per entry; 67 MB of codes take 44 us, of which 30 at the copy rate.
template <typename T>
__global__ void __launch_bounds__(256) expand_kernel(ExpandFp8Args a) {
  __shared__ int32_t warp_n[8];
  __shared__ int32_t found_s, before_s;  // the sequence of the share's first block, its own first
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const auto blocks_of = [&](int s) -> int32_t {
    const int32_t ctx = min(a.ctx_lens[s], a.max_ctx);
    return a.cu_q[s + 1] - a.cu_q[s] > 1 && ctx > 0 ? (ctx + a.bs - 1) / a.bs : 0;
  };
  int64_t total = 0;
  for (int s = tid; s < a.S; s += 256) {
    total += blocks_of(s);
    if (blockIdx.x == 0) {
      if (a.ctx_lens[s] > a.max_ctx) flag_status(a.status, B200_DEVICE_BAD_OP);
      a.scratch_ctx[s] = min(a.ctx_lens[s], a.max_ctx);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  __shared__ int64_t warp_total[8];
  if (lane == 0) warp_total[warp] = total;
  if (tid == 0) found_s = -1;
  __syncthreads();
  total = 0;
  for (int w = 0; w < 8; ++w) total += warp_total[w];
  if (total > a.scratch_blocks) {
    if (blockIdx.x == 0 && tid == 0) flag_status(a.status, B200_DEVICE_BAD_STEP);
    total = a.scratch_blocks;
  }
  const int per = static_cast<int>((total + gridDim.x - 1) / gridDim.x);
  const int b0 = static_cast<int>(min(total, static_cast<int64_t>(blockIdx.x) * per));
  const int b1 = static_cast<int>(min(total, static_cast<int64_t>(b0) + per));
  if (b0 >= b1) return;
  // the sequence of block b0
  int64_t carry = 0;
  for (int base = 0; base < a.S; base += 256) {
    const int s = base + tid;
    const int32_t n = s < a.S ? blocks_of(s) : 0;
    int32_t x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t t = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += t;
    }
    if (lane == 31) warp_n[warp] = x;
    __syncthreads();
    int64_t before = carry + x - n;
    for (int w = 0; w < 8; ++w) {
      if (w < warp) before += warp_n[w];
      carry += warp_n[w];
    }
    if (n > 0 && before <= b0 && b0 < before + n) {
      found_s = s;
      before_s = static_cast<int32_t>(before);
    }
    __syncthreads();
    if (found_s >= 0) break;
  }
  int seq = found_s, first = before_s, held = blocks_of(seq);
  const int64_t block_bytes = static_cast<int64_t>(a.bs) * a.hkv * a.head_dim;
  const int chunks = static_cast<int>(block_bytes / 16);
  const int head_chunks = a.head_dim / 16;
  for (int b = b0; b < b1; ++b) {
    while (b >= first + held) {
      first += held;
      held = blocks_of(++seq);
    }
    const int j = b - first;
    int32_t src = a.bt[static_cast<int64_t>(seq) * a.bt_stride + j];
    const bool good = src >= 0 && src < a.nb;
    if (threadIdx.x == 0) {
      a.scratch_table[static_cast<int64_t>(seq) * a.scratch_stride + j] = b;
      if (!good) flag_status(a.status, B200_DEVICE_BAD_BLOCK);
    }
    if (!good) src = 0;
    const int64_t at = static_cast<int64_t>(a.layer) * a.nb + src;
    const uint4* k = reinterpret_cast<const uint4*>(a.kc + at * block_bytes);
    const uint4* v = reinterpret_cast<const uint4*>(a.vc + at * block_bytes);
    uint4* ko = static_cast<uint4*>(a.k16) + static_cast<int64_t>(b) * chunks * 2;
    uint4* vo = static_cast<uint4*>(a.v16) + static_cast<int64_t>(b) * chunks * 2;
#pragma unroll 4
    for (int c = threadIdx.x; c < chunks; c += 256) {
      const int h = (c / head_chunks) % a.hkv;
      uint4 kc = k[c], vc = v[c];
      float ks = a.ks[at * a.hkv + h], vs = a.vs[at * a.hkv + h];
      if (!good) {  // a page outside the pool: zeros
        kc = vc = make_uint4(0u, 0u, 0u, 0u);
        ks = vs = 0.f;
      }
      uint4 o[2];
      widen16<T>(kc, ks, o);
      ko[2 * c] = o[0];
      ko[2 * c + 1] = o[1];
      widen16<T>(vc, vs, o);
      vo[2 * c] = o[0];
      vo[2 * c + 1] = o[1];
    }
  }
}

}  // namespace

cudaError_t launch_expand_fp8(const ExpandFp8Args& a, int dtype, int num_sms, cudaStream_t stream) {
  const int grid = a.scratch_blocks < num_sms * 8 ? a.scratch_blocks : num_sms * 8;
  if (dtype == B200_DTYPE_BF16) expand_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a);
  else if (dtype == B200_DTYPE_F16) expand_kernel<__half><<<grid, 256, 0, stream>>>(a);
  else return cudaErrorInvalidValue;
  return cudaGetLastError();
}

cudaError_t launch_row_fp8(const AttnFp8Args& a, int dtype, int rows, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  switch (dtype) {
    case B200_DTYPE_F32: return launch_row_t<float>(a, rows, stream);
    case B200_DTYPE_BF16: return launch_row_t<__nv_bfloat16>(a, rows, stream);
    case B200_DTYPE_F16: return launch_row_t<__half>(a, rows, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace b200
