// Decode over an 8-bit paged cache on the tensor cores (mma.sync; one new token per sequence).
//
// The batch's work is one line of units of 32 tokens: sequence by sequence, KV head by KV head (and
// tile of 8 query heads by tile).  Every warp of a persistent grid takes an equal share of that
// line, so the shares differ by one unit at most however the context lengths are spread, and runs
// by itself: its own TMA ring, its own softmax, no CTA-wide synchronisation.  A warp writes an
// item (sequence, KV head, tile of query heads) that lies inside its share straight to the output;
// of the first and the last item of its share it may hold only a part, which it leaves in the
// workspace for the merge kernel that follows.
//
// Per 16 tokens: K (16 x D codes) by ldmatrix, four codes of a row per lane and register, widened to
// f16 in registers (exact).  The order of the dims inside a k-step of 16 is free as long as Q has
// it too, so a lane's four adjacent codes serve two k-columns each.  V by transposing ldmatrix on
// pairs of codes (two adjacent dims as one 16-bit element) and one byte permutation.
//   S^T = K Q^T and O^T += V^T P^T, m16n8k16 with f16 operands and fp32 sums.
// Q is scaled to f16 by a power of two per head (exact for bf16 and f16 queries); fp32 queries and
// weights are split in two f16 parts (22 bits), each with its own product.
// The weights of P: p = 2^(x - m) with a reference m that moves in units with a page whose value scale is
// near the largest so far (nearly all) or with a score that passes it by more than 8 (p <= 2^8).  A
// row's largest weight is then mostly 1, exact in f16; a reference that moves at scores alone takes 131 us
// for 256 sequences against 134, with the rounding of the largest weights in every output.  P is stored for the
// product as p * vs * F: vs is the page's value scale and F a power of two per head that keeps the
// head's largest product between 1 and 2^15 whatever the scales are, also where the scores move on to
// pages of far smaller values (11 bits of every product within 2^-14 of the largest, an error of at
// most 2^-25 of the largest for smaller ones).
//
// Bound: HBM (4 * G flop per byte).  A unit is 64 * D bytes.  Measured with GQA 32/8, D 128, bf16
// queries: 256 sequences of 16 to 4096 tokens (677 MB) 134-140 us, 4.8-5.1 TB/s; 14 of 8192 to 32768
// (616 MB) 121-125 us, the merge (8 and 13 us) included.  While the warps run: 5.3 and 5.5 TB/s, 81 and
// 84 % of the copy rate, and 43 % of the issue slots, so what bounds it now is how many loads the 12
// consumers an SM (128 registers a thread) keep in flight beside their conversions and products.
// What the parts brought (256 sequences | 14 long ones, us): a CTA per row on the CUDA cores 2337 | 6022;
// tensor cores and equal shares of 16-token units 173 | 148; the warps of a CTA on adjacent heads 151 |
// 135; 32-token units, 12 warps an SM with 16 KB rings 133 | 125; a loading warp per CTA 134 | 118.
#include <cuda.h>

#include "api_common.cuh"
#include "fp8.cuh"
#include "fp8_decode.cuh"
#include "tc05.cuh"

namespace b200 {

namespace {

constexpr int kWarps = 4;  // consumer warps
constexpr int kCtasPerSm = 3;
constexpr int kThreads = 32 * (kWarps + 1);  // the last warp loads for the others
constexpr int kUnit = 32;      // tokens
// Places on the line per warp at least.  In us, for 1 | 2 | 4: one sequence of 512 tokens 11.0 | 10.7 |
// 12.5, of 4096 28 | 14 | 17, four of 1000 16 | 12.4 | 14.4; large batches are not affected.
constexpr int kMinShare = 2;
// What beginning an item costs, in units: part of its length on the line (256 sequences of 16 to 4096
// tokens take 145 us with 1, 140 with 3 and 140.5 with 6; eight of up to 512 13.3, 11.9 and 11.9).
constexpr int kItemCost = 3;
// F before a page with a nonzero value scale: any of 2^-111 or more moves it.  Set ones are smaller, so p * F
// stays finite for p <= 2^8, and times a scale it is 0 where the weight or the scale is.
constexpr float kUnset = 0x1p+118f;
constexpr float kLazy = 8.f;   // log2 of how far p may exceed 1 before the reference moves

template <int D>
struct Ring {
  static constexpr int kTile = kUnit * D;    // codes of one unit of K (or V)
  static constexpr int kStage = 2 * kTile;
  static constexpr int kStages = 16384 / kStage;  // 16 KB per warp: 2 stages of D 128, 4 of D 64
  static constexpr int kWarpBytes = kStages * kStage;
};

__device__ __forceinline__ uint32_t cvt_e4m3x2(uint32_t v) {  // low 16 bits -> f16x2
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t cvt_e4m3x2_hi(uint32_t v) {  // high 16 bits -> f16x2
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) { return MmaOp<__half>::pack(lo, hi); }

// 16-byte chunk `c` of row `r` in a tile of rows of D bytes, as TMA swizzles it (128 B rows with
// the 128 B pattern, 64 B rows with the 64 B pattern).
template <int D>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  if (D == 128) return r * 128 + ((c ^ (r & 7)) << 4);
  return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

// Four adjacent elements of a query row (aligned to four elements).
template <typename T>
__device__ __forceinline__ void load4(const T* p, bool take, float (&v)[4]) {
  uint2 u = take ? *reinterpret_cast<const uint2*>(p) : make_uint2(0u, 0u);
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = to_f32<T>(e[j]);
}
template <>
__device__ __forceinline__ void load4<float>(const float* p, bool take, float (&v)[4]) {
  const float4 u = take ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
  v[0] = u.x;
  v[1] = u.y;
  v[2] = u.z;
  v[3] = u.w;
}

// 2^(up - e) with mx in [1, 2) * 2^e: an exact power of two, within fp32's normal range.
__device__ __forceinline__ float pow2_inverse(float mx, int up) {
  int e = static_cast<int>(__float_as_uint(mx) >> 23);
  e = min(max(254 - e + up, 1), 253);
  return __uint_as_float(static_cast<uint32_t>(e) << 23);
}

// Inclusive prefix sums of the lengths of the sequences' items (units and kItemCost) into cu[1..S], cu[0] = 0.  Whole CTA.
__device__ void prefix_units(const DecodeFp8Args& a, int32_t* cu, int32_t* warp_sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t carry = 0;
  if (tid == 0) cu[0] = 0;
  for (int base = 0; base < a.S; base += kThreads) {
    const int s = base + tid;
    int32_t n = 0;
    if (s < a.S) {
      const int32_t ctx = min(a.ctx_lens[s], a.max_ctx);
      const bool decoded = a.cu_q == nullptr || a.cu_q[s + 1] - a.cu_q[s] == 1;
      if (decoded && ctx > 0) n = (ctx + kUnit - 1) / kUnit + kItemCost;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t t = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += t;
    }
    if (lane == 31) warp_sums[warp] = n;
    __syncthreads();
#pragma unroll
    for (int w = 0; w <= kWarps; ++w) {
      if (w < warp) n += warp_sums[w];
    }
    if (s < a.S) cu[s + 1] = carry + n;
#pragma unroll
    for (int w = 0; w <= kWarps; ++w) carry += warp_sums[w];
    __syncthreads();
  }
}

// Items (KV heads, or tiles of query heads) that a team takes side by side.  A page's rows hold
// the heads of a token one after another, so the warps of a team read adjacent pieces at about the
// same time.
__device__ __forceinline__ int team_of(int items) {
  return items % 4 == 0 ? 4 : items % 2 == 0 ? 2 : 1;
}

// a / b (64-bit division only where it is needed: it costs some hundred cycles)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

__device__ __forceinline__ int64_t share_of(int64_t total, int warps) {
  const int64_t w = quotient(total + warps - 1, warps);
  return w > kMinShare ? w : kMinShare;
}

// Non-blocking form of mbar_try_wait: the producer looks at several barriers in turn.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t phase) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(phase)
      : "memory");
  return ok != 0;
}

// What the producer tells a consumer about a unit: scales of its NP pieces (halves of 16 tokens, or
// quarters of 8 where a page holds 8) and a bit for each piece that does not take part (behind the
// context, or on a page outside the pool).
struct UnitMeta {
  float ks[4], vs[4];
  uint32_t bad;
  uint32_t pad[3];
};

constexpr uint32_t kBad = 0x80000000u;

// One warp's walk along its share of the line.
struct Walk {
  int64_t at, end;          // next unit and the end of the share
  int seq, hc, u;           // where `at` is: sequence, team's item, place in the item
};

__device__ __forceinline__ Walk start_walk(const int32_t* cu, int S, int ips, int64_t at, int64_t end) {
  Walk w{at, end, 0, 0, 0};
  if (at >= end) return w;
  int lo = 0, hi = S - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (static_cast<int64_t>(cu[mid + 1]) * ips > at) hi = mid; else lo = mid + 1;
  }
  w.seq = lo;
  const int64_t rem = at - static_cast<int64_t>(cu[lo]) * ips;
  const int length = cu[lo + 1] - cu[lo];
  w.hc = static_cast<int>(rem / length);
  w.u = static_cast<int>(rem - static_cast<int64_t>(w.hc) * length);
  return w;
}

// Takes up to `most` units of one item: sequence, item, first unit and count (0 at the share's end).
// The first kItemCost places of an item hold no unit.
__device__ __forceinline__ int next_piece(Walk& w, const int32_t* cu, int ips, int most, int& s, int& hc,
                                          int& u0) {
  for (;;) {
    if (w.at >= w.end) return 0;
    const int length = cu[w.seq + 1] - cu[w.seq];
    if (length == 0) {
      ++w.seq;
      continue;
    }
    if (w.u < kItemCost) {
      const int skip = static_cast<int>(min(static_cast<int64_t>(kItemCost - w.u), w.end - w.at));
      w.at += skip;
      w.u += skip;
      if (w.at >= w.end) return 0;
    }
    s = w.seq;
    hc = w.hc;
    u0 = w.u - kItemCost;
    const int n = static_cast<int>(min(min(static_cast<int64_t>(length - w.u), w.end - w.at), static_cast<int64_t>(most)));
    w.at += n;
    w.u += n;
    if (w.u == length) {
      w.u = 0;
      if (++w.hc == ips) {
        w.hc = 0;
        ++w.seq;
      }
    }
    return n;
  }
}

template <typename T, int D, int NP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    decode_fp8_kernel(const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, DecodeFp8Args a) {
  using R = Ring<D>;
  constexpr int NS = R::kStages;
  constexpr int KS = D / 16;
  constexpr int kPiece = kUnit / NP;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t base_u32 = (raw_u32 + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base_u32 - raw_u32);
  UnitMeta* meta = reinterpret_cast<UnitMeta*>(smem + kWarps * R::kWarpBytes);  // [kWarps][NS]
  uint64_t* full = reinterpret_cast<uint64_t*>(meta + kWarps * NS);             // [kWarps][NS]
  uint64_t* empty = full + kWarps * NS;
  int32_t* warp_sums = reinterpret_cast<int32_t*>(empty + kWarps * NS);
  volatile int32_t* abort_s = warp_sums + kWarps + 1;
  int32_t* cu = warp_sums + kWarps + 2;  // [S + 1]

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    *abort_s = 0;
    for (int i = 0; i < kWarps * NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    fence_proxy_async_smem();
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  prefix_units(a, cu, warp_sums);  // its barriers publish the mbarriers too
  __syncthreads();
  // decoded sequences without context: zeros
  for (int s = blockIdx.x; s < a.S; s += gridDim.x) {
    if (tid == 0 && a.ctx_lens[s] > a.max_ctx) flag_status(a.status, B200_DEVICE_BAD_OP);
    if (tid == 0 && a.decodes_only && a.cu_q[s + 1] - a.cu_q[s] > 1) flag_status(a.status, B200_DEVICE_BAD_STEP);
    if (cu[s + 1] != cu[s] || (a.cu_q != nullptr && a.cu_q[s + 1] - a.cu_q[s] != 1)) continue;
    const int64_t row = a.cu_q ? a.cu_q[s] : (a.query_rows ? a.query_rows[s] : s);
    const int hq = a.hkv * a.group;
    for (int i = tid; i < hq * D; i += kThreads)
      static_cast<T*>(a.out)[row * a.o_srow + static_cast<int64_t>(i / D) * a.o_shead + i % D] = from_f32<T>(0.f);
  }

  asm volatile("griddepcontrol.launch_dependents;");
  // teams of ts warps walk the line side by side, each warp with an item of its own
  const int ts = team_of(a.hkv * a.nchunks), ips = a.hkv * a.nchunks / ts;
  const int64_t total = static_cast<int64_t>(cu[a.S]) * ips;
  const int64_t share = share_of(total, static_cast<int>(gridDim.x) * (kWarps / ts));
  // this warp's share, or (producer) that of the consumer warp which this lane serves
  const int who = warp < kWarps ? warp : lane >> 3;
  const int gw = blockIdx.x * kWarps + who;
  const int64_t begin = min(total, gw / ts * share), end = min(total, begin + share);
  Walk walk = start_walk(cu, a.S, ips, begin, end);

  if (warp == kWarps) {
    // ======== producer: 8 lanes for each consumer warp ========================================
    // Lane sl holds unit sl of the consumer's current 8 units (rows, scales) and of its next 8,
    // whose page ids are asked for when the current 8 begin and whose scales two units later.
    const int sl = lane & 7;
    uint32_t row[NP], nrow[NP];
    float ks[NP], vs[NP], nks[NP], nvs[NP];
    int32_t nid[NP];
    int h = 0, n = 0, i = 0;                       // current units: head, count, next to issue
    int ns = 0, nhc = 0, nu0 = 0, nn = 0, nh = 0;  // next units
    int nstate = 0;                                // 1: ids asked for, 2: scales asked for
    uint8_t* ring = smem + who * R::kWarpBytes;
    UnitMeta* my_meta = meta + who * NS;
    uint64_t* my_full = full + who * NS;
    uint64_t* my_empty = empty + who * NS;
    int stage = 0;
    uint32_t phase = 0, fills = 0;

    const auto ask_ids = [&]() {
      nn = next_piece(walk, cu, ips, 8, ns, nhc, nu0);
      nstate = 1;
      const int hc = nhc * ts + who % ts;
      nh = hc / a.nchunks;
      const int32_t ctx = nn > 0 ? min(a.ctx_lens[ns], a.max_ctx) : 0;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int t = (nu0 + sl) * kUnit + p * kPiece;
        nid[p] = sl < nn && t < ctx ? a.bt[static_cast<int64_t>(ns) * a.bt_stride + t / a.bs] : -1;
        if (sl < nn && t < ctx && (nid[p] < 0 || nid[p] >= a.nb)) flag_status(a.status, B200_DEVICE_BAD_BLOCK);
      }
      if (nn > 0 && (nu0 == 0 || fills == 0)) {
        // the item's queries, on their way to L2 before the consumer asks for them
        const int cch = hc - nh * a.nchunks;
        const int64_t qrow = a.cu_q ? a.cu_q[ns] : (a.query_rows ? a.query_rows[ns] : ns);
        if (cch * 8 + sl < a.group) {
          const T* q = static_cast<const T*>(a.q) + qrow * a.q_srow +
                       static_cast<int64_t>(nh * a.group + cch * 8 + sl) * a.q_shead;
          asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
          asm volatile("prefetch.global.L2 [%0];" ::"l"(q + D - 1));
        }
      }
    };
    const auto ask_scales = [&]() {
      nstate = 2;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const bool good = nid[p] >= 0 && nid[p] < a.nb;
        const int32_t b = good ? nid[p] : 0;
        const int t = (nu0 + sl) * kUnit + p * kPiece;
        const int64_t sc = (static_cast<int64_t>(a.layer) * a.nb + b) * a.hkv + nh;
        nks[p] = good ? a.ks[sc] : 0.f;
        nvs[p] = good ? a.vs[sc] : 0.f;
        nrow[p] = static_cast<uint32_t>((a.layer * a.nb + b) * a.bs + t % a.bs) | (good ? 0u : kBad);
      }
    };

    ask_ids();
    uint64_t idle_since = globaltimer_ns();
    for (;;) {
      if (i == n) {
        if (nn > 0) {
          if (nstate == 1) ask_scales();
          n = nn;
          h = nh;
          i = 0;
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            row[p] = nrow[p];
            ks[p] = nks[p];
            vs[p] = nvs[p];
          }
          ask_ids();
        }
      } else if (nstate == 1 && i >= 2) {
        ask_scales();
      }
      const bool left = i < n;
      if (!__any_sync(0xffffffffu, left)) break;
      const bool can = left && (fills < NS || mbar_test(&my_empty[stage], phase ^ 1u));
      // one decision for the consumer's 8 lanes
      const bool go = __shfl_sync(0xffffffffu, can ? 1 : 0, 0, 8) != 0;
      uint32_t irow[NP], bad = 0, bytes = 0;
      float iks[NP], ivs[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        irow[p] = __shfl_sync(0xffffffffu, row[p], i & 7, 8);
        iks[p] = __shfl_sync(0xffffffffu, ks[p], i & 7, 8);
        ivs[p] = __shfl_sync(0xffffffffu, vs[p], i & 7, 8);
        bad |= (irow[p] >> 31) << p;
        if (!(irow[p] & kBad)) bytes += 2 * kPiece * D;
      }
      if (go) {
        if (sl == 0) {
          UnitMeta& m = my_meta[stage];
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            m.ks[p] = iks[p];
            m.vs[p] = ivs[p];
          }
          m.bad = bad;
          uint8_t* dst = ring + stage * R::kStage;
          mbar_arrive_expect_tx(&my_full[stage], bytes);
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            if (irow[p] & kBad) continue;
            tma_load_3d(dst + p * kPiece * D, &kmap, &my_full[stage], 0, h, static_cast<int32_t>(irow[p]));
            tma_load_3d(dst + R::kTile + p * kPiece * D, &vmap, &my_full[stage], 0, h, static_cast<int32_t>(irow[p]));
          }
        }
        ++i;
        ++fills;
        if (++stage == NS) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (__any_sync(0xffffffffu, go)) {
        idle_since = globaltimer_ns();
      } else if (*abort_s || globaltimer_ns() - idle_since > kWaitLimitNs) {
        if (!*abort_s && lane == 0) flag_status(a.status, B200_DEVICE_TIMEOUT);
        break;
      }
    }
    // no load may land after the CTA is gone: wait (bounded) for the last fill of each stage
    for (uint32_t k = 0; k < NS; ++k) {
      if (stage == 0) phase ^= 1u;
      stage = stage == 0 ? NS - 1 : stage - 1;
      if (k < fills) mbar_wait_bounded(&my_full[stage], phase);
    }
    return;
  }

  // ======== consumers ==========================================================================
  const int r = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * R::kWarpBytes;
  const uint32_t ring_u32 = base_u32 + warp * R::kWarpBytes;
  const UnitMeta* my_meta = meta + warp * NS;
  uint64_t* my_full = full + warp * NS;
  uint64_t* my_empty = empty + warp * NS;
  int stage = 0;
  uint32_t phase = 0;
  MergeItem joined{};  // what the merge is to do for this warp
  // ldmatrix: lane's row of 16 tokens and 16-byte chunk 0 or 1, swizzled; chunk k is at ^ (k << 4)
  const int krow = (lane & 7) + 8 * ((lane >> 3) & 1);
  const uint32_t lane_at = tile_at<D>(krow, lane >> 4);

  for (;;) {
    int seq, hct, u0;
    const int n = next_piece(walk, cu, ips, 0x7fffffff, seq, hct, u0);
    if (n == 0) {
      if (lane == 0) a.merge[gw] = joined;
      break;
    }
    const int hc = hct * ts + warp % ts;
    const int h = hc / a.nchunks, cch = hc - h * a.nchunks;
    const int units = cu[seq + 1] - cu[seq] - kItemCost;
    const int ctx = min(a.ctx_lens[seq], a.max_ctx);
    const int nh = min(8, a.group - cch * 8);
    const int hq0 = h * a.group + cch * 8;
    const int64_t qrow = a.cu_q ? a.cu_q[seq] : (a.query_rows ? a.query_rows[seq] : seq);

    // ---- Q of head r, scaled to f16; |q| below 2^11: the parts that matter stay normal numbers ----
    uint32_t qf[KS][2], ql[SPLIT ? KS : 1][2];
    float qscale0, qscale1;
    {
      float qv[KS][4];
      float mx = 0.f;
      const T* q = static_cast<const T*>(a.q) + qrow * a.q_srow + static_cast<int64_t>(hq0 + r) * a.q_shead + 4 * c;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if (a.vec_q) {
          load4<T>(q + 16 * k, r < nh, qv[k]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) qv[k][j] = r < nh ? to_f32<T>(q[16 * k + j]) : 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, fabsf(qv[k][j]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float inv = pow2_inverse(mx, 10);
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float x = qv[k][2 * j] * inv, y = qv[k][2 * j + 1] * inv;
          qf[k][j] = pack_f16(x, y);
          if (SPLIT) {
            const __half2 hi = *reinterpret_cast<__half2*>(&qf[k][j]);
            ql[k][j] = pack_f16(x - __low2float(hi), y - __high2float(hi));
          }
        }
      const float back = a.scale_log2 / inv;  // head r's; the scores are laid out by 2c, 2c + 1
      qscale0 = __shfl_sync(0xffffffffu, back, 8 * c);
      qscale1 = __shfl_sync(0xffffffffu, back, 8 * c + 4);
    }
    float acc[KS][4];
#pragma unroll
    for (int k = 0; k < KS; ++k) acc[k][0] = acc[k][1] = acc[k][2] = acc[k][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, F0 = kUnset, F1 = kUnset;

    for (int i = 0; i < n; ++i) {
      if (!mbar_wait_bounded(&my_full[stage], phase)) {
        if (lane == 0) flag_status(a.status, B200_DEVICE_TIMEOUT);
        *abort_s = 1;  // the producer sees to what is in flight
        if (lane == 0) a.merge[gw] = MergeItem{};
        return;
      }
      const uint32_t kb = ring_u32 + stage * R::kStage + lane_at;
      const uint32_t vb = kb + R::kTile;
      const UnitMeta& m = my_meta[stage];
      const uint32_t bad = m.bad;
      float ks[NP], vs[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        ks[p] = m.ks[p];
        vs[p] = m.vs[p];
      }
      const int valid = ctx - (u0 + i) * kUnit;  // tokens of the unit inside the context
      const bool whole = valid >= kUnit && bad == 0;
      // token t of the unit takes part
      const auto takes_part = [&](int t) { return t < valid && !((bad >> (t / kPiece)) & 1u); };
      if (!whole) {
        // rows that do not take part may hold anything, NaN codes among it: their V is zeroed
        uint8_t* v = ring + stage * R::kStage + R::kTile;
        for (int idx = lane; idx < kUnit * (D / 16); idx += 32) {
          const int rr = idx / (D / 16), ch = idx % (D / 16);
          if (!takes_part(rr))
            *reinterpret_cast<uint4*>(v + tile_at<D>(rr, ch)) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();  // before the stage's next fill
        __syncwarp();
      }

      // ---- S^T = K Q^T: s[j] has tokens 16j + r (elements 0, 1) and 16j + r + 8 (2, 3) -----------
      float s[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sb[4] = {0.f, 0.f, 0.f, 0.f};
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          uint32_t x0, x1, x2, x3;
          ldmatrix_x4((kb ^ (k << 4)) + j * 16 * D, x0, x1, x2, x3);
          {
            const uint32_t a0 = cvt_e4m3x2(x0), a1 = cvt_e4m3x2(x1), a2 = cvt_e4m3x2_hi(x0), a3 = cvt_e4m3x2_hi(x1);
            MmaOp<__half>::run(s[j], a0, a1, a2, a3, qf[k][0], qf[k][1]);
            if (SPLIT) MmaOp<__half>::run(s[j], a0, a1, a2, a3, ql[k][0], ql[k][1]);
          }
          {
            const uint32_t a0 = cvt_e4m3x2(x2), a1 = cvt_e4m3x2(x3), a2 = cvt_e4m3x2_hi(x2), a3 = cvt_e4m3x2_hi(x3);
            MmaOp<__half>::run(sb, a0, a1, a2, a3, qf[k + 1][0], qf[k + 1][1]);
            if (SPLIT) MmaOp<__half>::run(sb, a0, a1, a2, a3, ql[k + 1][0], ql[k + 1][1]);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] += sb[e];
      }

      // ---- softmax relative to the reference: y = score - m, in log2 units ----------------------
      float y[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float ka = ks[j * NP / 2], kc = ks[(j + 1) * NP / 2 - 1];  // of rows r and r + 8
        y[j][0] = fmaf(s[j][0], ka * qscale0, -m0);
        y[j][1] = fmaf(s[j][1], ka * qscale1, -m1);
        y[j][2] = fmaf(s[j][2], kc * qscale0, -m0);
        y[j][3] = fmaf(s[j][3], kc * qscale1, -m1);
        if (!whole) {
          if (!takes_part(16 * j + r)) y[j][0] = y[j][1] = -INFINITY;
          if (!takes_part(16 * j + r + 8)) y[j][2] = y[j][3] = -INFINITY;
        }
      }
      float vmax = vs[0], top = y[0][0];
#pragma unroll
      for (int p = 1; p < NP; ++p) vmax = fmaxf(vmax, vs[p]);
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, y[e >> 2][e & 3]);
      // (a unit fitted to F has p * vs * F in [2^8, 2^9); without a move p is up to 2^8, the product to 2^15)
      const bool move = top > kLazy || vmax * fmaxf(F0, F1) > 128.f;
      if (__any_sync(0xffffffffu, move)) {
        float t0 = m0, t1 = m1;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float ka = ks[j * NP / 2], kc = ks[(j + 1) * NP / 2 - 1];
          y[j][0] = s[j][0] * (ka * qscale0);
          y[j][1] = s[j][1] * (ka * qscale1);
          y[j][2] = s[j][2] * (kc * qscale0);
          y[j][3] = s[j][3] * (kc * qscale1);
          if (!takes_part(16 * j + r)) y[j][0] = y[j][1] = -INFINITY;
          if (!takes_part(16 * j + r + 8)) y[j][2] = y[j][3] = -INFINITY;
          t0 = fmaxf(t0, fmaxf(y[j][0], y[j][2]));
          t1 = fmaxf(t1, fmaxf(y[j][1], y[j][3]));
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
          t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
        }
        const float u0 = t0 == -INFINITY ? 0.f : t0, u1 = t1 == -INFINITY ? 0.f : t1;
        float al0 = fast_exp2(m0 - u0), al1 = fast_exp2(m1 - u1);
        l0 *= al0;
        l1 *= al1;
        m0 = t0;
        m1 = t1;
        // the largest product p * vs of the unit, per head
        float w0 = 0.f, w1 = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float va = vs[j * NP / 2], vc = vs[(j + 1) * NP / 2 - 1];
          y[j][0] -= u0;
          y[j][1] -= u1;
          y[j][2] -= u0;
          y[j][3] -= u1;
          w0 = fmaxf(w0, fmaxf(fast_exp2(y[j][0]) * va, fast_exp2(y[j][2]) * vc));
          w1 = fmaxf(w1, fmaxf(fast_exp2(y[j][1]) * va, fast_exp2(y[j][3]) * vc));
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          w0 = fmaxf(w0, __shfl_xor_sync(0xffffffffu, w0, o));
          w1 = fmaxf(w1, __shfl_xor_sync(0xffffffffu, w1, o));
        }
        // F changes when unset, when a product would pass 2^15, and when the unit's largest one falls below
        // 1: the reference may have moved to pages of smaller values, whose products f16 would hold in
        // fewer bits.  What raises F leaves the sums held so far below 2^101; the products of a unit
        // that would need more are 2^-90 of them at most.
        const auto low = [](float w, float F) { return w > 0.f && F != kUnset && w * F < 1.f; };
        float held0 = 0.f, held1 = 0.f;
        if (__any_sync(0xffffffffu, low(w0, F0) || low(w1, F1))) {
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            held0 = fmaxf(held0, fmaxf(fabsf(acc[k][0]), fabsf(acc[k][2])));
            held1 = fmaxf(held1, fmaxf(fabsf(acc[k][1]), fabsf(acc[k][3])));
          }
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            held0 = fmaxf(held0, __shfl_xor_sync(0xffffffffu, held0, o));
            held1 = fmaxf(held1, __shfl_xor_sync(0xffffffffu, held1, o));
          }
        }
        const auto exponent = [](float x) { return static_cast<int>(__float_as_uint(x) >> 23); };
        const auto refit = [&](float w, float held, float& F, float& al) {
          if (!(w > 0.f) || (F != kUnset && w * F >= 1.f && w * F <= 32768.f)) return;
          const float f = fminf(pow2_inverse(w, 8), 0.5f * kUnset);  // p * vs * F in [2^8, 2^9)
          int by = exponent(f) - exponent(F);
          if (by > 0) by = min(by, max(227 - exponent(held * al), 0));
          F = __uint_as_float(__float_as_uint(F) + (static_cast<uint32_t>(by) << 23));
          al = ldexpf(al, by);
        };
        refit(w0, held0, F0, al0);
        refit(w1, held1, F1, al1);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          acc[k][0] *= al0;
          acc[k][1] *= al1;
          acc[k][2] *= al0;
          acc[k][3] *= al1;
        }
      }
      uint32_t pb[2][2], pl[SPLIT ? 2 : 1][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float va = vs[j * NP / 2], vc = vs[(j + 1) * NP / 2 - 1];
        float p0 = fast_exp2(y[j][0]), p1 = fast_exp2(y[j][1]), p2 = fast_exp2(y[j][2]), p3 = fast_exp2(y[j][3]);
        l0 += p0 + p2;
        l1 += p1 + p3;
        p0 = p0 * F0 * va;
        p1 = p1 * F1 * va;
        p2 = p2 * F0 * vc;
        p3 = p3 * F1 * vc;
        const uint32_t ph0 = pack_f16(p0, p1), ph1 = pack_f16(p2, p3);
        pb[j][0] = movmatrix_trans(ph0);
        pb[j][1] = movmatrix_trans(ph1);
        if (SPLIT) {
          const __half2 h0 = *reinterpret_cast<const __half2*>(&ph0);
          const __half2 h1 = *reinterpret_cast<const __half2*>(&ph1);
          pl[j][0] = movmatrix_trans(pack_f16(p0 - __low2float(h0), p1 - __high2float(h0)));
          pl[j][1] = movmatrix_trans(pack_f16(p2 - __low2float(h1), p3 - __high2float(h1)));
        }
      }

      // ---- O^T += V^T P^T: row r of a 16-dim tile is dim 2r, row r + 8 dim 2r + 1 ------------
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          uint32_t z0, z1, z2, z3;
          ldmatrix_x4_trans((vb ^ (k << 4)) + j * 16 * D, z0, z1, z2, z3);
          z0 = __byte_perm(z0, 0, 0x3120);
          z1 = __byte_perm(z1, 0, 0x3120);
          z2 = __byte_perm(z2, 0, 0x3120);
          z3 = __byte_perm(z3, 0, 0x3120);
          {
            const uint32_t a0 = cvt_e4m3x2(z0), a1 = cvt_e4m3x2_hi(z0), a2 = cvt_e4m3x2(z1), a3 = cvt_e4m3x2_hi(z1);
            MmaOp<__half>::run(acc[k], a0, a1, a2, a3, pb[j][0], pb[j][1]);
            if (SPLIT) MmaOp<__half>::run(acc[k], a0, a1, a2, a3, pl[j][0], pl[j][1]);
          }
          {
            const uint32_t a0 = cvt_e4m3x2(z2), a1 = cvt_e4m3x2_hi(z2), a2 = cvt_e4m3x2(z3), a3 = cvt_e4m3x2_hi(z3);
            MmaOp<__half>::run(acc[k + 1], a0, a1, a2, a3, pb[j][0], pb[j][1]);
            if (SPLIT) MmaOp<__half>::run(acc[k + 1], a0, a1, a2, a3, pl[j][0], pl[j][1]);
          }
        }
      __syncwarp();
      if (lane == 0) tc05::mbar_arrive(&my_empty[stage]);
      if (++stage == NS) {
        stage = 0;
        phase ^= 1u;
      }
    }

    // ---- the item's end, or the share's ---------------------------------------------------
    const bool done = u0 + n == units;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }
    const int64_t item0 = walk.at - n - u0;  // the line's place of the item's first unit
    if (done && item0 >= begin) {
      const float f0 = 1.f / F0, f1 = 1.f / F1;
      const float i0 = l0 != 0.f ? 1.f / l0 : 0.f, i1 = l1 != 0.f ? 1.f / l1 : 0.f;
      T* o0 = static_cast<T*>(a.out) + qrow * a.o_srow + static_cast<int64_t>(hq0 + 2 * c) * a.o_shead;
      T* o1 = o0 + a.o_shead;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int d = 16 * k + 2 * r;
        if (2 * c < nh) {
          o0[d] = from_f32<T>(acc[k][0] * f0 * i0);
          o0[d + 1] = from_f32<T>(acc[k][2] * f0 * i0);
        }
        if (2 * c + 1 < nh) {
          o1[d] = from_f32<T>(acc[k][1] * f1 * i1);
          o1[d + 1] = from_f32<T>(acc[k][3] * f1 * i1);
        }
      }
    } else {
      // a part of an item: sums relative to 2^m, the output sum as the values' (without F)
      if (done) {
        const int64_t w0 = quotient(item0, share);
        joined.n = gw / ts - static_cast<int>(w0) + 1;
        joined.hc = hc;
        joined.qrow = qrow;
        joined.slot = 2 * (w0 * ts + warp % ts);
        joined.slot_step = 2 * ts;
        joined.first_slot = joined.slot + (item0 > w0 * share ? 1 : 0);
      }
      const int64_t slot = 2 * static_cast<int64_t>(gw) + (item0 <= begin ? 0 : 1);
      float* po = a.part_o + slot * 8 * D;
      float2* ml = a.part_ml + slot * 8;
      const float i0 = 1.f / F0, i1 = 1.f / F1;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int d = 16 * k + 2 * r;
        if (2 * c < nh)
          *reinterpret_cast<float2*>(po + (2 * c) * D + d) = make_float2(acc[k][0] * i0, acc[k][2] * i0);
        if (2 * c + 1 < nh)
          *reinterpret_cast<float2*>(po + (2 * c + 1) * D + d) = make_float2(acc[k][1] * i1, acc[k][3] * i1);
      }
      if (r == 0) {
        ml[2 * c] = make_float2(m0, l0);
        ml[2 * c + 1] = make_float2(m1, l1);
      }
    }
  }
}

// The merge: joins the parts of an item that several warps shared, in the order of the warps.  One
// CTA per warp of the decode, for the item that ended in that warp's share after beginning in an
// earlier one; the warp has left what there is to know about it.  Launched while the decode still
// runs: its first statement waits for the decode's results.
//
// W warps (at least as many as an item has heads) with U parts in flight each.  Most items of a
// large batch have two or three parts, and what counts is how many CTAs an SM holds: 4 warps and 4
// parts (8 warps for more than 4 heads).  Up to kFewItems items have many (222 for one sequence of
// 32768 tokens with 8 KV heads): 16 warps and 8 parts.  Decode and merge with 4 heads an item:
//   4 / 4:   256 sequences of 512 61 us, 16 of 1000 16.2, 4 of 1000 14.2, 1 of 32768 52
//   16 / 8:  256 sequences of 512 71 us, 16 of 1000 18.3, 4 of 1000 12.6, 1 of 32768 29
constexpr int kFewItems = 64;

template <typename T, int D, int W, int U>
__global__ void __launch_bounds__(32 * W) merge_fp8_kernel(DecodeFp8Args a) {
  __shared__ float4 o_s[W][D / 4];
  __shared__ float2 ml_s[W];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const MergeItem it = a.merge[blockIdx.x];
  if (it.n == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = it.hc / a.nchunks, cch = it.hc - h * a.nchunks;
  const int nh = min(8, a.group - cch * 8), hq0 = h * a.group + cch * 8;
  // warps: heads first, then groups that take every groups-th part; with D = 64 a warp's halves
  // are groups of their own
  constexpr int kVec = D / 4, kPer = 32 / kVec;
  const int hh = warp % nh, grp = warp / nh, groups = W / nh;
  const int e = lane % kVec;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = -INFINITY, L = 0.f;
  const auto add = [&](float2 ml, float4 v) {
    const float N = fmaxf(M, ml.x);
    const float Nu = N == -INFINITY ? 0.f : N;
    const float wa = fast_exp2(M - Nu), wb = fast_exp2(ml.x - Nu);
    o.x = o.x * wa + v.x * wb;
    o.y = o.y * wa + v.y * wb;
    o.z = o.z * wa + v.z * wb;
    o.w = o.w * wa + v.w * wb;
    L = L * wa + ml.y * wb;
    M = N;
  };
  if (grp < groups) {
    // U parts at a time, all their loads in flight together
    const int step = groups * kPer;
    for (int i0 = grp * kPer + lane / kVec; i0 < it.n; i0 += U * step) {
      float2 ml[U];
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * step;
        const int64_t sl = i == 0 ? it.first_slot : it.slot + static_cast<int64_t>(i) * it.slot_step;
        ml[u] = i < it.n ? a.part_ml[sl * 8 + hh] : make_float2(-INFINITY, 0.f);
        v[u] = i < it.n ? *reinterpret_cast<const float4*>(a.part_o + (sl * 8 + hh) * D + e * 4)
                        : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float N = M;
#pragma unroll
      for (int u = 0; u < U; ++u) N = fmaxf(N, ml[u].x);
      const float Nu = N == -INFINITY ? 0.f : N;
      const float wa = fast_exp2(M - Nu);
      o.x *= wa;
      o.y *= wa;
      o.z *= wa;
      o.w *= wa;
      L *= wa;
      M = N;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = fast_exp2(ml[u].x - Nu);
        o.x += v[u].x * w;
        o.y += v[u].y * w;
        o.z += v[u].z * w;
        o.w += v[u].w * w;
        L += ml[u].y * w;
      }
    }
    if (kPer == 2)
      add(make_float2(__shfl_xor_sync(0xffffffffu, M, 16), __shfl_xor_sync(0xffffffffu, L, 16)),
          make_float4(__shfl_xor_sync(0xffffffffu, o.x, 16), __shfl_xor_sync(0xffffffffu, o.y, 16),
                      __shfl_xor_sync(0xffffffffu, o.z, 16), __shfl_xor_sync(0xffffffffu, o.w, 16)));
    if (lane < kVec) o_s[warp][lane] = o;
    if (lane == 0) ml_s[warp] = make_float2(M, L);
  }
  __syncthreads();
  if (grp == 0 && lane < kVec) {
    for (int g = 1; g < groups; ++g) add(ml_s[g * nh + hh], o_s[g * nh + hh][lane]);
    const float inv = L != 0.f ? 1.f / L : 0.f;
    T* d = static_cast<T*>(a.out) + it.qrow * a.o_srow + static_cast<int64_t>(hq0 + hh) * a.o_shead + e * 4;
    d[0] = from_f32<T>(o.x * inv);
    d[1] = from_f32<T>(o.y * inv);
    d[2] = from_f32<T>(o.z * inv);
    d[3] = from_f32<T>(o.w * inv);
  }
}

template <int D>
int smem_bytes(int S) {
  using R = Ring<D>;
  return 1024 + kWarps * R::kWarpBytes + kWarps * R::kStages * (sizeof(UnitMeta) + 16) + (kWarps + 2) * 4 +
         (S + 1) * 4;
}

template <typename T, int D, int NP, bool SPLIT>
cudaError_t launch_t(const CUtensorMap& km, const CUtensorMap& vm, const DecodeFp8Args& a, int grid,
                     cudaStream_t stream) {
  const int smem = smem_bytes<D>(a.S);
  auto kern = decode_fp8_kernel<T, D, NP, SPLIT>;
  cudaError_t e = allow_smem<decode_fp8_kernel<T, D, NP, SPLIT>>(smem_bytes<D>(kDecodeFp8MaxSeqs));
  if (e != cudaSuccess) return e;
  kern<<<grid, kThreads, smem, stream>>>(km, vm, a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // the merge's launch overlaps the decode's end
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(grid * kWarps);
  if (static_cast<int64_t>(a.S) * a.hkv * a.nchunks <= kFewItems) {
    cfg.blockDim = dim3(32 * 16);
    return cudaLaunchKernelEx(&cfg, merge_fp8_kernel<T, D, 16, 8>, a);
  }
  if (a.group > 4) {
    cfg.blockDim = dim3(32 * 8);
    return cudaLaunchKernelEx(&cfg, merge_fp8_kernel<T, D, 8, 4>, a);
  }
  cfg.blockDim = dim3(32 * 4);
  return cudaLaunchKernelEx(&cfg, merge_fp8_kernel<T, D, 4, 4>, a);
}

template <typename T, bool SPLIT>
cudaError_t launch_d(const CUtensorMap& km, const CUtensorMap& vm, const DecodeFp8Args& a, int grid,
                     cudaStream_t stream) {
  if (a.head_dim == 128)
    return a.bs == 8 ? launch_t<T, 128, 4, SPLIT>(km, vm, a, grid, stream)
                     : launch_t<T, 128, 2, SPLIT>(km, vm, a, grid, stream);
  return a.bs == 8 ? launch_t<T, 64, 4, SPLIT>(km, vm, a, grid, stream)
                   : launch_t<T, 64, 2, SPLIT>(km, vm, a, grid, stream);
}

}  // namespace

int decode_fp8_grid(int S, int64_t max_ctx, int ips, int num_sms) {
  const int64_t line = static_cast<int64_t>(S) * ((max_ctx + kUnit - 1) / kUnit + kItemCost) * ips;
  const int64_t need = (line + kMinShare * kWarps - 1) / (kMinShare * kWarps);
  const int64_t most = static_cast<int64_t>(num_sms) * kCtasPerSm;
  return static_cast<int>(need < 1 ? 1 : need < most ? need : most);
}

int decode_fp8_parts(int grid) { return 2 * kWarps * grid; }

cudaError_t launch_decode_fp8(int dtype, const CUtensorMap& km, const CUtensorMap& vm,
                              const DecodeFp8Args& a, int grid, cudaStream_t stream) {
  switch (dtype) {
    case B200_DTYPE_F32: return launch_d<float, true>(km, vm, a, grid, stream);
    case B200_DTYPE_BF16: return launch_d<__nv_bfloat16, false>(km, vm, a, grid, stream);
    case B200_DTYPE_F16: return launch_d<__half, false>(km, vm, a, grid, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace b200
