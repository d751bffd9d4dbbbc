// Attention over an 8-bit paged cache:  o = sum_j softmax_j(scale * q.k_j) v_j  with
// k_j = code * key scale of the block, v_j = code * value scale of the block.
#include "fp8.cuh"

namespace b200 {

namespace {

constexpr int kRowWarps = 8;

// One CTA per (query row, KV head, up to 8 query heads): each warp takes every kRowWarps-th
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
  const auto launch = [&](auto kern) -> cudaError_t {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 68 * 1024);
    if (e != cudaSuccess) return e;
    kern<<<grid, kRowWarps * 32, smem, stream>>>(a, nchunks);
    return cudaGetLastError();
  };
  if (npl <= 1) return launch(row_fp8_kernel<T, 1>);
  if (npl <= 2) return launch(row_fp8_kernel<T, 2>);
  if (npl <= 4) return launch(row_fp8_kernel<T, 4>);
  if (npl <= 8) return launch(row_fp8_kernel<T, 8>);
  return cudaErrorInvalidValue;
}

}  // namespace

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
