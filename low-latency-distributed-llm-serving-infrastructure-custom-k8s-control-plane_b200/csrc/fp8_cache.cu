// Append to, and read back from, an 8-bit paged cache (e4m3 numbers, one power-of-two scale per
// layer, block and KV head).
//
// For block b and head h let R be the call's rows with a slot in b and m the largest finite |x| of
// those rows (after rotation, for keys).  need = the smallest power of two s with m <= 448 s.
//   new scale = need                    if R writes the block's first slot (the block begins anew)
//             = max(old scale, need)    otherwise
//   a held code c becomes rn(c * old / new) where the scale grew; a row's entry becomes rn(x / new).
// Powers of two make both divisions exact, so each entry is rounded to its code once (a held one again
// only where it falls below e4m3's smallest normal number).
//
// One CTA owns a block: it lists the block's rows in the call, takes the maxima, rescales what the
// block holds and writes the rows, so no two CTAs touch one scale.  In calls of up to
// kAppendScanRows rows every row's CTA scans the call's slots for its block (the CTA of the first
// such row goes on, the others leave); larger calls first count the rows of each block and list
// the rows where a run of rows of one block starts.
//
// Bound: HBM.  A step of 16 prompt chunks and 240 single rows (14,200 rows, GQA 32/8, D 128, bf16, with
// rotation): 76 us for rows, codes and rotated queries (275 MB move: 55 % of the copy rate),
// 22 us for the read-back; one element per thread and memory pass took 427 us for both, against 108.  256
// decode rows take 6.3 us, of which a launch and the chain slot -> block -> scale -> codes are the most.
// Rows that have a block to themselves are what keeps a large call from the copy rate: 8192 of them take
// 115 us, 8192 rows of whole blocks 48.
#include "fp8.cuh"

namespace b200 {

namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kChunkRows = 16;    // rows of a block handled per pass
constexpr int kMaxBlockSize = 1024;

// cos and sin of pos * inv_freq in 64 bits.  The product is formed and reduced to [-pi/4, pi/4] in
// 64 bits (at position 30,000 a 32-bit product alone is off by 1e-3 rad) and the Taylor series there
// end with a remainder below 2e-14.  Keys are rotated in 64 bits too and rounded to fp32 (an error of
// 2^-24, against a code's 2^-4): two products an element, less than fp32 arithmetic in two parts
// (12 operations).
struct __align__(16) Turn {
  double c, s;
};
__device__ __forceinline__ Turn turn_of(int64_t pos, float inv_freq) {
  const double a = static_cast<double>(pos) * static_cast<double>(inv_freq);
  const double k = rint(a * 0.6366197723675814);                    // 2 / pi
  double r = fma(-k, 1.5707963267948966, a);                        // pi / 2 in two parts
  r = fma(-k, 6.123233995736766e-17, r);
  const double z = r * r;
  double s = 1.0 / 6227020800.0;                                    // 1 / 13!
  s = fma(s, z, -1.0 / 39916800.0);
  s = fma(s, z, 1.0 / 362880.0);
  s = fma(s, z, -1.0 / 5040.0);
  s = fma(s, z, 1.0 / 120.0);
  s = fma(s, z, -1.0 / 6.0);
  s = fma(s * z, r, r);
  double c = -1.0 / 87178291200.0;                                  // -1 / 14!
  c = fma(c, z, 1.0 / 479001600.0);
  c = fma(c, z, -1.0 / 3628800.0);
  c = fma(c, z, 1.0 / 40320.0);
  c = fma(c, z, -1.0 / 720.0);
  c = fma(c, z, 1.0 / 24.0);
  c = fma(c, z, -0.5);
  c = fma(c, z, 1.0);
  const int quarter = static_cast<int>(static_cast<int64_t>(k) & 3);
  if (quarter & 1) {
    const double t = s;
    s = c;
    c = -t;
  }
  if (quarter & 2) {
    s = -s;
    c = -c;
  }
  return Turn{c, s};
}

// Rotates the pair (x, y) and rounds it once to fp32.
__device__ __forceinline__ void rotate(const Turn& t, float& x, float& y) {
  const double u = x, v = y;
  x = static_cast<float>(u * t.c - v * t.s);
  y = static_cast<float>(v * t.c + u * t.s);
}

// Smallest power of two s with amax <= 448 s (448 = 1.75 * 2^8), at least 2^-100.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = static_cast<int>(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(e, 27);
  return __uint_as_float(static_cast<uint32_t>(e) << 23);
}

__device__ __forceinline__ bool is_pow2(float s) {
  return (__float_as_uint(s) & 0x7fffffu) == 0;
}

struct RowList {
  int32_t row[kChunkRows];
  int32_t off[kChunkRows];
  bool last[kChunkRows];  // the last of the list's rows with its slot
  int32_t n;
  int32_t next;  // row to go on from
};

// The next rows (at most kChunkRows) of block slots [s0, s0 + bs) at or after row `pos`, in order;
// stops once `want` rows have been found.  want < 0: all rows from `pos` on are looked at, and the
// number found is returned (the first kChunkRows of them are listed).  Called by the whole CTA.
__device__ int next_rows(const AppendFp8Args& a, int64_t s0, int pos, int want, RowList& list,
                         int32_t* warp_n) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int found = 0;
  while (pos < a.num_tokens && (want < 0 || (found < want && found < kChunkRows))) {
    const int r = pos + tid;
    const int64_t slot = r < a.num_tokens ? a.slots[r] : -1;
    const bool in = slot >= s0 && slot < s0 + a.bs;
    const uint32_t m = __ballot_sync(0xffffffffu, in);
    if (lane == 0) warp_n[warp] = __popc(m);
    __syncthreads();
    int before = found, total = 0;
#pragma unroll
    for (int w = 0; w < kAppendWarps; ++w) {
      if (w < warp) before += warp_n[w];
      total += warp_n[w];
    }
    const int at = before + __popc(m & ((1u << lane) - 1u));
    if (in && at < kChunkRows) {
      list.row[at] = r;
      list.off[at] = static_cast<int32_t>(slot - s0);
      if (at == kChunkRows - 1) list.next = r + 1;
    }
    if (found + total < kChunkRows && tid == 0) list.next = pos + kAppendThreads;
    found += total;
    pos += kAppendThreads;
    __syncthreads();
  }
  if (tid == 0) list.n = min(found, kChunkRows);
  __syncthreads();
  return found;
}

template <typename T, bool ROPE>
__global__ void __launch_bounds__(kAppendThreads) append_fp8_kernel(AppendFp8Args a, int q_ctas,
                                                                    int q_rows) {
  extern __shared__ __align__(16) float sm[];
  __shared__ RowList list;
  __shared__ int32_t warp_n[kAppendWarps];
  __shared__ uint32_t written[kMaxBlockSize / 32];
  __shared__ int32_t fresh_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int D = a.head_dim, half = D / 2;

  // ---- queries: rotated and rounded to the call's type ---------------------------------------
  if (ROPE && static_cast<int>(blockIdx.x) < q_ctas) {
    const int r0 = blockIdx.x * q_rows, r1 = min(a.num_tokens, r0 + q_rows);
    float2* cs = reinterpret_cast<float2*>(sm);  // [q_rows][half]: cos, sin
    for (int w = tid; w < (r1 - r0) * half; w += kAppendThreads) {
      const int r = w / half, i = w - r * half;
      const Turn t = turn_of(a.positions[r0 + r], a.inv_freq[i]);
      cs[w] = make_float2(static_cast<float>(t.c), static_cast<float>(t.s));
    }
    __syncthreads();
    const int per_row = a.hq * half;
    for (int w = tid; w < (r1 - r0) * per_row; w += kAppendThreads) {
      const int r = w / per_row, rem = w - r * per_row;
      const int h = rem / half, i = rem - h * half;
      const T* src = static_cast<const T*>(a.q_in) + (r0 + r) * a.q_stok + h * D;
      T* dst = static_cast<T*>(a.q_out) + (r0 + r) * a.qo_stok + h * D;
      const float x1 = to_f32<T>(src[i]), x2 = to_f32<T>(src[i + half]);
      const float2 cv = cs[r * half + i];
      dst[i] = from_f32<T>(x1 * cv.x - x2 * cv.y);
      dst[i + half] = from_f32<T>(x2 * cv.x + x1 * cv.y);
    }
    return;
  }

  // ---- keys and values, block by block -------------------------------------------------------
  const int64_t total_slots = static_cast<int64_t>(a.nb) * a.bs;
  Turn* cs = reinterpret_cast<Turn*>(sm);              // [kChunkRows][half]
  float* amax = sm + (ROPE ? kChunkRows * 2 * D : 0);  // [2 * hkv]
  const bool scan = a.runs == nullptr;
  const int unit0 = static_cast<int>(blockIdx.x) - q_ctas;
  const int step = static_cast<int>(gridDim.x) - q_ctas;
  const int units = scan ? a.num_tokens : *a.num_runs;
  for (int unit = unit0; unit < units; unit += step) {
    const int t = scan ? unit : a.runs[unit];
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= total_slots) {
      if (slot >= total_slots && tid == 0) flag_status(a.status, B200_DEVICE_BAD_SLOT);
      continue;
    }
    const int64_t blk = slot / a.bs, s0 = blk * a.bs;
    int want;
    if (scan) {
      want = next_rows(a, s0, 0, -1, list, warp_n);
      if (list.row[0] != t) continue;  // the block's first row owns it
    } else {
      if (a.num_tokens - a.first[blk] != t) continue;
      want = a.count[blk];
    }

    // maxima over all of the block's rows, kChunkRows at a time
    for (int i = tid; i < 2 * a.hkv; i += kAppendThreads) amax[i] = 0.f;
    for (int i = tid; i < (a.bs + 31) / 32; i += kAppendThreads) written[i] = 0u;
    if (tid == 0) fresh_s = 0;
    __syncthreads();
    int pos = t, seen = 0, chunks = 0;
    const auto load_chunk = [&]() {
      next_rows(a, s0, pos, want - seen, list, warp_n);
      pos = list.next;
      seen += list.n;
      if (ROPE) {
        for (int w = tid; w < list.n * half; w += kAppendThreads) {
          const int r = w / half, i = w - r * half;
          cs[w] = turn_of(a.positions[list.row[r]], a.inv_freq[i]);
        }
      }
      __syncthreads();
    };
    // entry d and (rotary keys) d + half of row r of the chunk, head h
    const auto entry = [&](int task, int r, int d, float& x1, float& x2) {
      const int h = task >> 1;
      if (task & 1) {
        const T* v = static_cast<const T*>(a.value) + list.row[r] * a.v_stok + h * a.v_shead;
        x1 = to_f32<T>(v[d]);
      } else {
        const T* k = static_cast<const T*>(a.key) + list.row[r] * a.k_stok + h * a.k_shead;
        x1 = to_f32<T>(k[d]);
        if (ROPE) {
          x2 = to_f32<T>(k[d + half]);
          rotate(cs[r * half + d], x1, x2);
        }
      }
    };
    do {
      load_chunk();
      ++chunks;
      if (tid < list.n) {
        atomicOr(&written[list.off[tid] >> 5], 1u << (list.off[tid] & 31));
        if (list.off[tid] == 0) fresh_s = 1;
      }
      for (int task = warp; task < 2 * a.hkv; task += kAppendWarps) {
        const bool pair = ROPE && !(task & 1);
        float m = 0.f;
        for (int r = 0; r < list.n; ++r)
          for (int d = lane; d < (pair ? half : D); d += 32) {
            float x1, x2 = 0.f;
            entry(task, r, d, x1, x2);
            x1 = fabsf(x1);
            x2 = pair ? fabsf(x2) : 0.f;
            if (x1 < INFINITY) m = fmaxf(m, x1);  // false for NaN too
            if (x2 < INFINITY) m = fmaxf(m, x2);
          }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) amax[task] = fmaxf(amax[task], m);
      }
      __syncthreads();
    } while (seen < want);

    const bool fresh = fresh_s != 0;
    const bool one_chunk = chunks == 1;
    const int64_t cache_blk = static_cast<int64_t>(a.layer) * a.nb + blk;
    pos = t;
    seen = 0;
    for (int ch = 0; ch < chunks; ++ch) {
      if (!one_chunk) load_chunk();
      for (int task = warp; task < 2 * a.hkv; task += kAppendWarps) {
        const int h = task >> 1;
        const bool is_v = task & 1;
        float* sp = (is_v ? a.vs : a.ks) + cache_blk * a.hkv + h;
        uint8_t* codes = (is_v ? a.vc : a.kc) + (cache_blk * a.bs * a.hkv + h) * D;
        const int64_t row_bytes = static_cast<int64_t>(a.hkv) * D;
        float s_new;
        if (ch == 0) {
          float old = *sp;
          if (!(old > 0.f) || isinf(old)) old = 0.f;  // never written
          s_new = scale_for(amax[task]);
          if (!fresh) {
            s_new = fmaxf(s_new, old);
            if (s_new != old) {
              const float ratio = old / s_new;
              for (int o = 0; o < a.bs; ++o) {
                if ((written[o >> 5] >> (o & 31)) & 1u) continue;
                for (int d = lane; d < D; d += 32) {
                  uint8_t* c = codes + o * row_bytes + d;
                  *c = f32_to_e4m3(e4m3_to_f32(*c) * ratio);
                }
              }
            }
          }
          __syncwarp();
          if (lane == 0) *sp = s_new;
          if (lane == 0) amax[task] = s_new;  // for the chunks that follow
        } else {
          s_new = amax[task];
        }
        __syncwarp();
        const bool pow2 = is_pow2(s_new);
        const float inv = 1.f / s_new;
        const bool pair = ROPE && !is_v;
        for (int r = 0; r < list.n; ++r) {
          uint8_t* c = codes + list.off[r] * row_bytes;
          for (int d = lane; d < (pair ? half : D); d += 32) {
            float x1, x2 = 0.f;
            entry(task, r, d, x1, x2);
            c[d] = f32_to_e4m3(pow2 ? x1 * inv : x1 / s_new);
            if (pair) c[d + half] = f32_to_e4m3(pow2 ? x2 * inv : x2 / s_new);
          }
        }
      }
      __syncthreads();
    }
  }
}

// ---- head dims 64 and 128, 16-byte aligned rows ---------------------------------------------------

// Eight adjacent elements as fp32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(e[i]);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const float4 u = reinterpret_cast<const float4*>(p)[0], v = reinterpret_cast<const float4*>(p)[1];
  x[0] = u.x;
  x[1] = u.y;
  x[2] = u.z;
  x[3] = u.w;
  x[4] = v.x;
  x[5] = v.y;
  x[6] = v.z;
  x[7] = v.w;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint4 u;
  T* e = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
  *reinterpret_cast<uint4*>(p) = u;
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// Two values' codes (no infinities among them).
__device__ __forceinline__ uint32_t codes2(float x, float y) {
  return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
}

// Four held codes rescaled.
__device__ __forceinline__ uint32_t rescale4(uint32_t c, float ratio) {
  const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(c & 0xffffu, __NV_E4M3)));
  const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(c >> 16, __NV_E4M3)));
  return codes2(a.x * ratio, a.y * ratio) | (codes2(b.x * ratio, b.y * ratio) << 16);
}

// A warp takes one head's keys (or values) of up to 8 rows into registers: LPR lanes a row, each
// with 8 elements of the row's first half and the 8 that they rotate with.  They are read once,
// and the maximum, the scale and the codes follow without touching memory again.  Of more than 8
// rows two warps take half each and exchange their maxima.
template <typename T, bool ROPE, int D>
__global__ void __launch_bounds__(kAppendThreads, 4)
    append_vec_kernel(AppendFp8Args a, int kv_ctas, int q_rows) {
  constexpr int kHalf = D / 2, LPR = kHalf / 8, RPP = 32 / LPR, P = kChunkRows / 2 / RPP;
  extern __shared__ __align__(16) float sm[];
  __shared__ RowList list;
  __shared__ int32_t warp_n[kAppendWarps];
  __shared__ uint32_t written[kMaxBlockSize / 32];
  __shared__ int32_t fresh_s;
  __shared__ float half_max[kAppendWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // pair i of a row (elements i and i + D/2) in shared memory: the pairs that the LPR lanes of a row
  // read together lie side by side
  const auto place = [](int i) { return (i % 8) * LPR + i / 8; };

  // ---- queries: every thread keeps the angles of its 8 pairs for all its heads --------------------
  if (ROPE && static_cast<int>(blockIdx.x) >= kv_ctas) {
    const int r0 = (blockIdx.x - kv_ctas) * q_rows, rows = min(a.num_tokens - r0, q_rows);
    float2* cs = reinterpret_cast<float2*>(sm);  // [q_rows][kHalf]
    for (int w = tid; w < rows * kHalf; w += kAppendThreads) {
      const Turn t = turn_of(a.positions[r0 + w / kHalf], a.inv_freq[w % kHalf]);
      cs[w / kHalf * kHalf + place(w % kHalf)] = make_float2(static_cast<float>(t.c), static_cast<float>(t.s));
    }
    __syncthreads();
    const int c = tid % LPR, row = (tid / LPR) % q_rows, groups = kAppendThreads / (LPR * q_rows);
    if (row >= rows) return;
    float cv[8], sv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = cs[row * kHalf + i * LPR + c];
      cv[i] = v.x;
      sv[i] = v.y;
    }
    const T* src = static_cast<const T*>(a.q_in) + (r0 + row) * a.q_stok + c * 8;
    T* dst = static_cast<T*>(a.q_out) + (r0 + row) * a.qo_stok + c * 8;
#pragma unroll 4
    for (int h = tid / (LPR * q_rows); h < a.hq; h += groups) {
      float x[8], y[8];
      load8<T>(src + h * D, x);
      load8<T>(src + h * D + kHalf, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = x[i] * cv[i] - y[i] * sv[i];
        y[i] = y[i] * cv[i] + x[i] * sv[i];
        x[i] = u;
      }
      store8<T>(dst + h * D, x);
      store8<T>(dst + h * D + kHalf, y);
    }
    return;
  }

  // ---- keys and values, block by block -------------------------------------------------------
  const int64_t total_slots = static_cast<int64_t>(a.nb) * a.bs;
  Turn* cs = reinterpret_cast<Turn*>(sm);                  // [kChunkRows][kHalf]
  float* amax = sm + (ROPE ? kChunkRows * 2 * D : 0);      // [2 * hkv], calls with longer lists only
  const int c = lane % LPR, rs = lane / LPR;
  const bool scan = a.runs == nullptr;
  const int units = scan ? a.num_tokens : *a.num_runs;
  for (int unit = blockIdx.x; unit < units; unit += kv_ctas) {
    const int t = scan ? unit : a.runs[unit];
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= total_slots) {
      if (slot >= total_slots && tid == 0) flag_status(a.status, B200_DEVICE_BAD_SLOT);
      continue;
    }
    // 32-bit division where it does: 64-bit division takes some hundred cycles
    const int64_t blk = (slot >> 32) == 0 ? static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.bs) : slot / a.bs;
    const int64_t s0 = blk * a.bs;
    __syncthreads();  // the list of the unit before is no longer read
    int want;
    if (scan) {
      want = next_rows(a, s0, 0, -1, list, warp_n);
      if (list.row[0] != t) continue;  // the block's first row owns it
    } else {
      if (a.num_tokens - a.first[blk] != t) continue;
      want = a.count[blk];
      next_rows(a, s0, t, want, list, warp_n);
    }
    if (tid == 0) fresh_s = 0;
    for (int i = tid; i < (a.bs + 31) / 32; i += kAppendThreads) written[i] = 0u;
    __syncthreads();

    const auto turns = [&]() {  // of the list's rows; what the list says goes into written, fresh_s
      if (tid < list.n) {
        atomicOr(&written[list.off[tid] >> 5], 1u << (list.off[tid] & 31));
        if (list.off[tid] == 0) fresh_s = 1;
        bool last = true;
        for (int k = tid + 1; k < list.n; ++k) last &= list.off[k] != list.off[tid];
        list.last[tid] = last;
      }
      if (ROPE) {
        for (int w = tid; w < list.n * kHalf; w += kAppendThreads)
          cs[w / kHalf * kHalf + place(w % kHalf)] = turn_of(a.positions[list.row[w / kHalf]], a.inv_freq[w % kHalf]);
      }
      __syncthreads();
    };
    // rows [r0, r0 + 8) of the list
    const auto load = [&](int task, int r0, float (&x)[P][2][8]) {
      const bool is_v = task & 1;
      const T* base = static_cast<const T*>(is_v ? a.value : a.key) + (task >> 1) * (is_v ? a.v_shead : a.k_shead) + c * 8;
      const int64_t stok = is_v ? a.v_stok : a.k_stok;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int r = r0 + p * RPP + rs;
        if (r < list.n) {
          load8<T>(base + list.row[r] * stok, x[p][0]);
          load8<T>(base + list.row[r] * stok + kHalf, x[p][1]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[p][0][i] = x[p][1][i] = 0.f;
        }
      }
      if (ROPE && !is_v) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const int r = r0 + p * RPP + rs;
          if (r < list.n) {
#pragma unroll
            for (int i = 0; i < 8; ++i) rotate(cs[r * kHalf + i * LPR + c], x[p][0][i], x[p][1][i]);
          }
        }
      }
    };
    // the warp's largest finite |x|; infinities become NaN on the way, which is what they are held as
    const auto largest = [&](float (&x)[P][2][8]) {
      float m = 0.f;
      for (int again = 0; again < 2; ++again) {
        m = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int i = 0; i < 8; ++i) m = fmaxf(m, fmaxf(fabsf(x[p][0][i]), fabsf(x[p][1][i])));  // NaN apart
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (m < INFINITY) break;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[p][0][i] = fabsf(x[p][0][i]) < INFINITY ? x[p][0][i] : NAN;
            x[p][1][i] = fabsf(x[p][1][i]) < INFINITY ? x[p][1][i] : NAN;
          }
      }
      return m;
    };
    const int64_t cache_blk = static_cast<int64_t>(a.layer) * a.nb + blk;
    const int64_t row_bytes = static_cast<int64_t>(a.hkv) * D;
    const auto codes_of = [&](int task) {
      return ((task & 1) ? a.vc : a.kc) + (cache_blk * a.bs * a.hkv + (task >> 1)) * D;
    };
    // the block's new scale for this head; rescales what it holds where the scale grows
    // (part `part` of `parts` of its rows; part 0 writes the scale)
    const auto settle = [&](int task, float old, float m, int part, int parts) {
      if (!(old > 0.f) || isinf(old)) old = 0.f;  // never written
      float s = scale_for(m);
      if (!fresh_s) {
        s = fmaxf(s, old);
        if (s != old) {
          const float ratio = old / s;
          uint8_t* codes = codes_of(task);
          constexpr int kRowLanes = D / 16;
          for (int o = part * (32 / kRowLanes) + lane / kRowLanes; o < a.bs; o += parts * (32 / kRowLanes)) {
            if ((written[o >> 5] >> (o & 31)) & 1u) continue;
            uint4* q = reinterpret_cast<uint4*>(codes + o * row_bytes) + lane % kRowLanes;
            uint4 v = *q;
            v.x = rescale4(v.x, ratio);
            v.y = rescale4(v.y, ratio);
            v.z = rescale4(v.z, ratio);
            v.w = rescale4(v.w, ratio);
            *q = v;
          }
        }
      }
      if (lane == 0 && part == 0) ((task & 1) ? a.vs : a.ks)[cache_blk * a.hkv + (task >> 1)] = s;
      return s;
    };
    const auto store = [&](int task, int r0, float s, float (&x)[P][2][8]) {
      uint8_t* codes = codes_of(task) + c * 8;
      const bool pow2 = is_pow2(s);
      const float inv = 1.f / s;
      if (!pow2) {  // a scale that a caller wrote
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[p][0][i] /= s;
            x[p][1][i] /= s;
          }
      }
      const float f = pow2 ? inv : 1.f;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int r = r0 + p * RPP + rs;
        if (r >= list.n || !list.last[r]) continue;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const float(&y)[8] = x[p][hf];
          uint2 v;
          v.x = codes2(y[0] * f, y[1] * f) | (codes2(y[2] * f, y[3] * f) << 16);
          v.y = codes2(y[4] * f, y[5] * f) | (codes2(y[6] * f, y[7] * f) << 16);
          *reinterpret_cast<uint2*>(codes + list.off[r] * row_bytes + hf * kHalf) = v;
        }
      }
    };

    turns();
    const auto scale_at = [&](int task) { return ((task & 1) ? a.vs : a.ks) + cache_blk * a.hkv + (task >> 1); };
    if (want <= kChunkRows / 2) {
      for (int task = warp; task < 2 * a.hkv; task += kAppendWarps) {
        const float old = *scale_at(task);
        float x[P][2][8];
        load(task, 0, x);
        const float s = settle(task, old, largest(x), 0, 1);
        store(task, 0, s, x);
      }
      continue;
    }
    const int part = warp & 1, r0 = part * (kChunkRows / 2);
    if (want <= kChunkRows) {
      for (int task = warp >> 1; task < 2 * a.hkv; task += kAppendWarps / 2) {
        const float old = *scale_at(task);
        float x[P][2][8];
        load(task, r0, x);
        const float m = largest(x);
        if (lane == 0) half_max[warp] = m;
        // the two warps of the task: both maxima written and both old scales read
        asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp >> 1)) : "memory");
        const float s = settle(task, old, fmaxf(m, half_max[warp ^ 1]), part, 2);
        store(task, r0, s, x);
        asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp >> 1)) : "memory");
      }
      continue;
    }
    // more rows than the registers hold: the maxima over all chunks of rows first, then the codes
    for (int i = tid; i < 2 * a.hkv; i += kAppendThreads) amax[i] = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      if (pass == 1) {
        __syncthreads();
        for (int task = warp; task < 2 * a.hkv; task += kAppendWarps) {
          const float old = *scale_at(task);
          __syncwarp();
          const float s = settle(task, old, amax[task], 0, 1);
          __syncwarp();
          if (lane == 0) amax[task] = s;
        }
      }
      int pos = t, seen = 0;
      while (seen < want) {
        __syncthreads();
        next_rows(a, s0, pos, want - seen, list, warp_n);
        turns();
        for (int task = warp; task < 2 * a.hkv; task += kAppendWarps) {
          for (int h0 = 0; h0 < kChunkRows; h0 += kChunkRows / 2) {
            float x[P][2][8];
            load(task, h0, x);
            const float m = largest(x);
            if (pass == 0) {
              if (lane == 0) amax[task] = fmaxf(amax[task], m);
            } else {
              store(task, h0, amax[task], x);
            }
          }
        }
        __syncthreads();
        seen += list.n;
        pos = list.next;
        if (list.n == 0) break;
      }
    }
  }
}

// Rows per block, the first row of each block and the starts of runs of rows of one block.
__global__ void __launch_bounds__(256) append_mark_kernel(AppendFp8Args a) {
  const int64_t total_slots = static_cast<int64_t>(a.nb) * a.bs;
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= a.num_tokens) return;
  const int64_t slot = a.slots[r];
  if (slot < 0) return;
  if (slot >= total_slots) {
    flag_status(a.status, B200_DEVICE_BAD_SLOT);
    return;
  }
  const int64_t blk = slot / a.bs;
  atomicAdd(&a.count[blk], 1);
  const int64_t prev = r > 0 ? a.slots[r - 1] : -1;
  if (prev < blk * a.bs || prev >= (blk + 1) * a.bs) {
    atomicMax(&a.first[blk], a.num_tokens - r);
    a.runs[atomicAdd(a.num_runs, 1)] = r;
  }
}

// ---- read back -------------------------------------------------------------------------------
// code * scale in the output's type; what an f16 cannot hold becomes +-65504.
template <typename T>
__device__ __forceinline__ T value_of(uint8_t c, float scale) {
  return from_f32<T>(e4m3_to_f32(c) * scale);
}
template <>
__device__ __forceinline__ __half value_of<__half>(uint8_t c, float scale) {
  const float x = e4m3_to_f32(c) * scale;
  return __float2half_rn(fabsf(x) > 65504.f ? copysignf(65504.f, x) : x);
}

template <typename T>
__global__ void __launch_bounds__(256) gather_fp8_kernel(GatherFp8Args a) {
  const int64_t per_row = static_cast<int64_t>(a.hkv) * a.head_dim;
  const int64_t total = per_row * a.n;
  const int64_t slots = static_cast<int64_t>(a.nb) * a.bs;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = i / per_row, e = i - r * per_row;
    const int64_t slot = a.slots[r];
    if (slot < 0 || slot >= slots) {
      if (slot >= slots && e == 0) flag_status(a.status, B200_DEVICE_BAD_SLOT);
      static_cast<T*>(a.k_out)[i] = from_f32<T>(0.f);
      static_cast<T*>(a.v_out)[i] = from_f32<T>(0.f);
      continue;
    }
    const int64_t blk = static_cast<int64_t>(a.layer) * a.nb + slot / a.bs;
    const int64_t at = (static_cast<int64_t>(a.layer) * slots + slot) * per_row + e;
    const int64_t sc = blk * a.hkv + e / a.head_dim;
    static_cast<T*>(a.k_out)[i] = value_of<T>(a.kc[at], a.ks[sc]);
    static_cast<T*>(a.v_out)[i] = value_of<T>(a.vc[at], a.vs[sc]);
  }
}

// Rows of 16-byte multiples: 16 codes per thread and step.
template <typename T>
__global__ void __launch_bounds__(256) gather_vec_kernel(GatherFp8Args a) {
  const uint32_t per_row = a.hkv * a.head_dim / 16, per_head = a.head_dim / 16;
  const int64_t slots = static_cast<int64_t>(a.nb) * a.bs;
  const uint32_t rows = 256 / per_row > 0 ? 256 / per_row : 1;  // of a CTA, side by side
  const uint32_t r_in = threadIdx.x / per_row;
  if (r_in >= rows) return;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * rows + r_in; r < a.n; r += static_cast<int64_t>(gridDim.x) * rows) {
    const int64_t slot = a.slots[r];
    const bool in = slot >= 0 && slot < slots;
    if (slot >= slots && threadIdx.x % per_row == 0) flag_status(a.status, B200_DEVICE_BAD_SLOT);
    const int64_t s = in ? slot : 0;
    const int64_t blk = static_cast<int64_t>(a.layer) * a.nb +
                        ((s >> 32) == 0 ? static_cast<uint32_t>(s) / static_cast<uint32_t>(a.bs) : s / a.bs);
    const int64_t row = (static_cast<int64_t>(a.layer) * slots + s) * per_row;
    for (uint32_t e = threadIdx.x - r_in * per_row; e < per_row; e += 256) {
      const int64_t sc = blk * a.hkv + e / per_head;
      uint4 kc = reinterpret_cast<const uint4*>(a.kc)[row + e], vc = reinterpret_cast<const uint4*>(a.vc)[row + e];
      float ks = a.ks[sc], vs = a.vs[sc];
      if (!in) {
        kc = vc = make_uint4(0u, 0u, 0u, 0u);
        ks = vs = 0.f;
      }
      const auto put = [&](uint4 code, float scale, void* out) {
        const uint8_t* b = reinterpret_cast<const uint8_t*>(&code);
        alignas(16) T v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = value_of<T>(b[i], scale);
        uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(out) + (r * per_row + e) * 16);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) o[i] = reinterpret_cast<const uint4*>(v)[i];
      };
      put(kc, ks, a.k_out);
      put(vc, vs, a.v_out);
    }
  }
}

template <typename T, bool ROPE, int D>
cudaError_t launch_append_vec(const AppendFp8Args& a, int num_sms, cudaStream_t stream) {
  // Query rows per CTA: four, whose threads reuse their angles for several heads (8192 rows of
  // whole blocks 48 us against 55 with one row, 256 rows 6.3 against 6.8, one row the same).
  constexpr int q_rows = 4;
  const int q_ctas = ROPE ? (a.num_tokens + q_rows - 1) / q_rows : 0;
  int kv_ctas = a.num_tokens;
  if (a.runs != nullptr && kv_ctas > num_sms * 8) kv_ctas = num_sms * 8;
  const size_t smem = ((ROPE ? kChunkRows * 2 * D : 0) + 2 * a.hkv) * sizeof(float);
  append_vec_kernel<T, ROPE, D><<<kv_ctas + q_ctas, kAppendThreads, smem, stream>>>(a, kv_ctas, q_rows);
  return cudaGetLastError();
}

// Every row, head and page starts on a 16-byte boundary.
template <typename T>
bool aligned_rows(const AppendFp8Args& a) {
  const int64_t es = sizeof(T);
  uint64_t all = reinterpret_cast<uintptr_t>(a.key) | reinterpret_cast<uintptr_t>(a.value) |
                 reinterpret_cast<uintptr_t>(a.kc) | reinterpret_cast<uintptr_t>(a.vc);
  all |= static_cast<uint64_t>((a.k_stok | a.k_shead | a.v_stok | a.v_shead) * es);
  if (a.positions != nullptr)
    all |= reinterpret_cast<uintptr_t>(a.q_in) | reinterpret_cast<uintptr_t>(a.q_out) |
           static_cast<uint64_t>((a.q_stok | a.qo_stok) * es);
  return all % 16 == 0;
}

template <typename T>
cudaError_t launch_append_t(const AppendFp8Args& a, int num_sms, cudaStream_t stream) {
  const bool rope = a.positions != nullptr;
  if ((a.head_dim == 128 || a.head_dim == 64) && aligned_rows<T>(a)) {
    if (a.head_dim == 128)
      return rope ? launch_append_vec<T, true, 128>(a, num_sms, stream) : launch_append_vec<T, false, 128>(a, num_sms, stream);
    return rope ? launch_append_vec<T, true, 64>(a, num_sms, stream) : launch_append_vec<T, false, 64>(a, num_sms, stream);
  }
  // as above, four (8192 rows of D 96 147 us; 156 with one row, 149 with eight, which are late with
  // few rows: 64 rows 13.8 us against 7.8)
  constexpr int q_rows = 4;
  const int q_ctas = rope ? (a.num_tokens + q_rows - 1) / q_rows : 0;
  int kv_ctas = a.num_tokens;
  if (a.runs != nullptr && kv_ctas > num_sms * 8) kv_ctas = num_sms * 8;
  const size_t smem = ((rope ? kChunkRows * 2 * a.head_dim : 0) + 2 * a.hkv) * sizeof(float);
  if (rope)
    append_fp8_kernel<T, true><<<q_ctas + kv_ctas, kAppendThreads, smem, stream>>>(a, q_ctas, q_rows);
  else
    append_fp8_kernel<T, false><<<kv_ctas, kAppendThreads, smem, stream>>>(a, 0, 1);
  return cudaGetLastError();
}

}  // namespace

size_t append_fp8_scratch_bytes(int nb, int num_tokens) {
  if (num_tokens <= kAppendScanRows) return 0;
  return (2 * static_cast<size_t>(nb) + 1 + num_tokens) * sizeof(int32_t);
}

cudaError_t launch_append_fp8(const AppendFp8Args& a, int dtype, int num_sms,
                              cudaStream_t stream) {
  if (a.num_tokens <= 0) return cudaSuccess;
  if (a.runs != nullptr) {
    // count, first and num_runs are adjacent
    cudaError_t e = cudaMemsetAsync(a.count, 0, (2 * static_cast<size_t>(a.nb) + 1) * 4, stream);
    if (e != cudaSuccess) return e;
    append_mark_kernel<<<(a.num_tokens + 255) / 256, 256, 0, stream>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  switch (dtype) {
    case B200_DTYPE_BF16: return launch_append_t<__nv_bfloat16>(a, num_sms, stream);
    case B200_DTYPE_F16: return launch_append_t<__half>(a, num_sms, stream);
    case B200_DTYPE_F32: return launch_append_t<float>(a, num_sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_gather_fp8(const GatherFp8Args& a, int dtype, int num_sms,
                              cudaStream_t stream) {
  if (a.n <= 0) return cudaSuccess;
  const uintptr_t all = reinterpret_cast<uintptr_t>(a.kc) | reinterpret_cast<uintptr_t>(a.vc) |
                        reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out);
  if (a.head_dim % 16 == 0 && all % 16 == 0) {
    const int per_row = a.hkv * a.head_dim / 16, rows = 256 / per_row > 0 ? 256 / per_row : 1;
    const int64_t need = (a.n + rows - 1) / rows, most = static_cast<int64_t>(num_sms) * 16;
    const int grid = static_cast<int>(need < most ? need : most);
    switch (dtype) {
      case B200_DTYPE_BF16: gather_vec_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a); break;
      case B200_DTYPE_F16: gather_vec_kernel<__half><<<grid, 256, 0, stream>>>(a); break;
      case B200_DTYPE_F32: gather_vec_kernel<float><<<grid, 256, 0, stream>>>(a); break;
      default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
  }
  const int64_t total = a.n * a.hkv * a.head_dim;
  int64_t blocks = (total + 255) / 256;
  const int64_t cap = static_cast<int64_t>(num_sms) * 8;
  if (blocks > cap) blocks = cap;
  const int grid = static_cast<int>(blocks);
  switch (dtype) {
    case B200_DTYPE_BF16: gather_fp8_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a); break;
    case B200_DTYPE_F16: gather_fp8_kernel<__half><<<grid, 256, 0, stream>>>(a); break;
    case B200_DTYPE_F32: gather_fp8_kernel<float><<<grid, 256, 0, stream>>>(a); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace b200
