// The kernels around the experts' products: the router (top-k, softmax weights, rows sorted by expert), the
// row-wise quantizer that also places each token's codes in expert order, and the weighted sum that brings
// the experts' results back to their tokens.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "common.cuh"

namespace lc {
namespace {

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// 16 bytes as floats
template <typename T>
struct Vec16 {
  static constexpr int kN = 16 / sizeof(T);
  T v[kN];
  __device__ __forceinline__ void load(const T* p) { *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void load_stream(const T* p) {
    *reinterpret_cast<uint4*>(v) = __ldcs(reinterpret_cast<const uint4*>(p));
  }
};

// =============================================================================================
// Router.  For each token: the top_k largest logits (equal logits: lowest expert first), their softmax
// weights, and each choice's place in the order "by expert, then by token".
//
// A logit of -inf or NaN is never chosen and carries no weight (masked experts, padded tokens); what is not
// chosen has expert -1, position -1 and weight 0.  +inf shares the weight with the other +inf of its row.
//
// One warp per token: lane l holds the EPL values l*EPL .. l*EPL + EPL-1 in registers and their maximum.  A round is
// one warp-wide integer maximum (order-preserving bits of the value) and a vote: of several lanes with the largest
// value the lowest has the lowest expert, and that lane moves on to its next one.  Up to eight values a
// lane are sorted first, in lists of up to four, so that moving on is a shift (16384 tokens of 256 experts, 8 of them
// chosen: 24.1 -> 21.3 us with nothing else changed, now 17.1); more are searched.  The kernel is bound by the instructions of a token
// (16384 tokens of 128 experts, 8 of them chosen: 480, three quarters of the issue slots), 13.8 us together with the
// second kernel's latency.  The winning lane leaves its choice in shared memory: broadcast by shuffle it was 14.8 us.
// A warp walks a contiguous run of tokens and counts its choices per expert in shared memory; a choice's
// count is its rank inside the run.  Small batches (one CTA) finish in the same kernel; otherwise each CTA
// leaves its counts and its ranks, and the second kernel adds what precedes them.  Every sum is an integer
// one over a fixed order, so the result does not depend on scheduling.
// =============================================================================================
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopK = 32;

// unsigned order = float order; NaN and -inf map to 0 (never chosen), -0 and +0 are equal
__device__ __forceinline__ uint32_t order_bits(float v) {
  if (!(v > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t b) {
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}

struct RouteParams {
  const void* logits;
  int64_t tokens, ld;
  int experts, top_k, renormalize;
  float* weights;      // [tokens, top_k]
  int32_t* chosen;     // [tokens, top_k]
  int32_t* positions;  // [tokens, top_k]
  int32_t* offsets;    // [experts + 1]
  uint16_t* counts;    // [CTAs, count_pitch(experts)], several CTAs only; a CTA has at most 65535 tokens
  int per_cta, run;    // tokens per CTA and per warp
  int vec;             // rows may be read in vectors
};

__host__ __device__ constexpr int64_t count_pitch(int64_t experts) { return (experts + 7) / 8 * 8; }  // 16-byte loads

// inclusive sum over the block of one int per thread; `tmp` holds 32 ints
__device__ __forceinline__ int block_scan(int v, int* tmp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) tmp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = lane < warps ? tmp[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    tmp[lane] = w;
  }
  __syncthreads();
  return v + (warp ? tmp[warp - 1] : 0);
}

template <typename T, int EPL>
__device__ __forceinline__ void load_row(const T* row, int E, int lane, int vec, T (&v)[EPL]) {
  if (vec) {  // E is 32 * EPL and rows start on a boundary of the lane's bytes
    constexpr int kBytes = EPL * sizeof(T) < 16 ? EPL * sizeof(T) : 16, kPer = kBytes / sizeof(T);
#pragma unroll
    for (int i = 0; i < EPL; i += kPer) {
      const T* src = row + lane * EPL + i;
      if constexpr (kBytes == 16)
        *reinterpret_cast<uint4*>(v + i) = __ldg(reinterpret_cast<const uint4*>(src));
      else if constexpr (kBytes == 8)
        *reinterpret_cast<uint2*>(v + i) = __ldg(reinterpret_cast<const uint2*>(src));
      else if constexpr (kBytes == 4)
        *reinterpret_cast<uint32_t*>(v + i) = __ldg(reinterpret_cast<const uint32_t*>(src));
      else
        v[i] = src[0];
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane * EPL + i < E) v[i] = row[lane * EPL + i];
  }
}

template <typename T, int EPL, bool ONE_CTA>
__global__ void __launch_bounds__(1024) route_kernel(const RouteParams p) {
  extern __shared__ int s_counts[];  // [warps][experts]; one CTA: then [experts] bases
  __shared__ int s_tmp[32];
  __shared__ uint2 s_pick[32][kRouteMaxTopK];  // a token's choices: value, expert
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t below = (1u << lane) - 1u;
  const int E = p.experts, K = p.top_k;
  int* mine = s_counts + warp * E;
  for (int i = threadIdx.x; i < warps * E; i += blockDim.x) s_counts[i] = 0;
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();

  const int64_t begin = static_cast<int64_t>(blockIdx.x) * p.per_cta;
  const int64_t end = begin + p.per_cta < p.tokens ? begin + p.per_cta : p.tokens;
  const int64_t first = begin + warp * p.run;
  const int64_t last = first + p.run < end ? first + p.run : end;
  T next[EPL];
  if (first < last) load_row<T, EPL>(static_cast<const T*>(p.logits) + first * p.ld, E, lane, p.vec, next);
  for (int64_t t = first; t < last; ++t) {
    uint32_t key[EPL], top = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      key[i] = lane * EPL + i < E ? order_bits(to_float<T>(next[i])) : 0u;
      top = max(top, key[i]);
    }
    if (t + 1 < last) load_row<T, EPL>(static_cast<const T*>(p.logits) + (t + 1) * p.ld, E, lane, p.vec, next);
    uint32_t mine_max = top;
    top = __reduce_max_sync(0xffffffffu, top);
    const float largest = order_value(top);
    const bool finite = largest < INFINITY;
    // exp(v - largest); with an infinite largest value 1 for those equal to it and 0 for the rest
    auto mass = [&](uint32_t k) {
      return k == 0u ? 0.0f : finite ? expf(order_value(k) - largest) : (k == top ? 1.0f : 0.0f);
    };
    float total = 0.0f;
    if (!p.renormalize) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) total += mass(key[i]);
    }
    // lane j keeps the j-th choice
    uint32_t my_key = 0, best = top;
    int my_e = -1;
    if constexpr (EPL <= 8) {
      // lists of up to four: descending, equal values in the order of their experts; two bits per value say where it
      // came from.  Of a lane's two lists with the same head the first has the lower expert.
      constexpr int LEN = EPL < 4 ? EPL : 4, LISTS = EPL / LEN;
      uint32_t from[LISTS];
#pragma unroll
      for (int l = 0; l < LISTS; ++l) {
        uint32_t* k = key + l * LEN;
        from[l] = 0xe4u;  // 3, 2, 1, 0
#pragma unroll
        for (int n = LEN - 1; n > 0; --n)
#pragma unroll
          for (int i = 0; i < n; ++i) {
            const bool swap = k[i + 1] > k[i];
            const uint32_t hi = max(k[i], k[i + 1]), lo = min(k[i], k[i + 1]);
            k[i] = hi;
            k[i + 1] = lo;
            const uint32_t bits = ((from[l] >> 2 * i) ^ (from[l] >> 2 * (i + 1))) & 3u;
            if (swap) from[l] ^= bits << 2 * i | bits << 2 * (i + 1);
          }
      }
      int j = 0;
      for (; j < K && best; ++j) {
        const bool second = LISTS > 1 && key[0] != best;
        const uint32_t head = second ? key[EPL - LEN] : key[0];
        const bool equal = head == best;
        const uint32_t who = __ballot_sync(0xffffffffu, equal);
        if (equal && !(who & below)) {  // the lowest lane of several
          const int at = second ? LEN + static_cast<int>(from[LISTS - 1] & 3u) : static_cast<int>(from[0] & 3u);
          s_pick[warp][j] = make_uint2(best, lane * EPL + at);
#pragma unroll
          for (int l = 0; l < LISTS; ++l) {
            if (second != (l == 1)) continue;
#pragma unroll
            for (int i = 0; i < LEN; ++i) key[l * LEN + i] = i + 1 < LEN ? key[l * LEN + i + 1] : 0u;
            from[l] >>= 2;
          }
        }
        best = __reduce_max_sync(0xffffffffu, LISTS > 1 ? max(key[0], key[EPL - LEN]) : key[0]);
      }
      __syncwarp();
      if (lane < j) {
        const uint2 pick = s_pick[warp][lane];
        my_key = pick.x;
        my_e = static_cast<int>(pick.y);
      }
    } else {
      for (int j = 0; j < K && best; ++j) {
        const int winner = __ffs(__ballot_sync(0xffffffffu, mine_max == best)) - 1;
        int at = 0;
        if (lane == winner) {
#pragma unroll
          for (int i = EPL - 1; i >= 0; --i)
            if (key[i] == best) at = i;
          mine_max = 0;
#pragma unroll
          for (int i = 0; i < EPL; ++i) {
            if (i == at) key[i] = 0u;
            mine_max = max(mine_max, key[i]);
          }
        }
        at = __shfl_sync(0xffffffffu, at, winner);
        if (lane == j) {
          my_key = best;
          my_e = winner * EPL + at;
        }
        best = __reduce_max_sync(0xffffffffu, mine_max);
      }
    }
    const float my_p = mass(my_key);
    if (p.renormalize) total = my_p;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane < K) {
      int rank = -1;
      if (my_e >= 0) rank = mine[my_e]++;  // a token's choices are distinct experts: no two lanes meet
      p.weights[t * K + lane] = my_e >= 0 ? __fdiv_rn(my_p, total) : 0.0f;
      p.chosen[t * K + lane] = my_e;
      p.positions[t * K + lane] = rank;  // rank inside this warp's run; completed below or by the second kernel
    }
    __syncwarp();
  }
  __syncthreads();

  // counts of the CTA, and each warp's start inside them
  int* base = s_counts + warps * E;
  const int counted = ONE_CTA ? E : static_cast<int>(count_pitch(E));
  for (int e0 = 0; e0 < counted; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    int sum = 0;
    if (e < E) {
      for (int w = 0; w < warps; w += 8) {  // (a multiple of 8 warps)
        int c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = s_counts[(w + i) * E + e];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s_counts[(w + i) * E + e] = sum;
          sum += c[i];
        }
      }
    }
    if (!ONE_CTA && e < counted) p.counts[static_cast<int64_t>(blockIdx.x) * counted + e] = static_cast<uint16_t>(sum);
    if (ONE_CTA) {  // (1024 threads: one round covers all experts)
      const int end = block_scan(sum, s_tmp);
      if (e < E) {
        base[e] = end - sum;
        p.offsets[e + 1] = end;
        if (e == 0) p.offsets[0] = 0;
      }
    }
  }
  __syncthreads();
  for (int64_t i = first * K + lane; i < last * K; i += 32) {
    const int e = p.chosen[i];
    if (e >= 0) p.positions[i] += mine[e] + (ONE_CTA ? base[e] : 0);
  }
}

// Second kernel of a large batch: CTA b adds to its tokens' ranks the rows of the experts before and the counts of the
// CTAs before it.  Every CTA reads every count (148 x 128: 38 KB), so what costs is latency: 16 bits a count, eight
// counts a load, and a warp for each 16th or 32nd of the CTAs leave some five loads a thread, which are in flight
// together with those of the choices.  Before and behind CTA b only whole warps' sums differ, but for the warp that b is
// in.  512 threads of up to 64 registers share an SM with a CTA of the first kernel (up to 128 experts), so that the next
// call's begins while this one ends (16384 tokens of 128, 8 of them chosen: 22.1 us a call with 1024 threads, then 14.8).  The
// first kernel for more experts leaves no room in any case, and then more threads read many CTAs' counts sooner (16384
// tokens of 256: 17.7 us, with 512 threads 19.5; but 128 tokens, four CTAs: 8.3 and 7.6 us).
template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
route_place_kernel(const RouteParams p, int ctas, int64_t tokens_per_cta, int lanes_log2) {
  constexpr int WARPS = THREADS / 32;
  constexpr int kSpan = 256;  // experts at a time: 8 a lane
  __shared__ __align__(16) int s_rows[WARPS][kSpan];
  __shared__ __align__(16) int s_own[kSpan];
  __shared__ int s_sum[kRouteMaxExperts], s_before[kRouteMaxExperts], s_tmp[32];
  const int E = p.experts, pitch = static_cast<int>(count_pitch(E));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < kRouteMaxExperts; e += THREADS) s_sum[e] = s_before[e] = 0;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t first = blockIdx.x * tokens_per_cta;
  const int64_t last = first + tokens_per_cta < p.tokens ? first + tokens_per_cta : p.tokens;
  int64_t item = first * p.top_k + threadIdx.x;
  const int64_t items_end = last * p.top_k;
  int at = item < items_end ? p.chosen[item] : -1;
  int rank = item < items_end ? p.positions[item] : -1;

  const int lanes = 1 << lanes_log2, col = lane & (lanes - 1);
  const int each = (ctas + WARPS - 1) / WARPS, begin = warp * each, end = min(begin + each, ctas);
  const int own_warp = static_cast<int>(blockIdx.x) / each;
  for (int e0 = 0; e0 < pitch; e0 += kSpan) {
    const int e = e0 + col * 8;
    int sum[8] = {}, before[8] = {};
    if (e < pitch) {
#pragma unroll 5
      for (int b = begin + (lane >> lanes_log2); b < end; b += 32 >> lanes_log2) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.counts + static_cast<int64_t>(b) * pitch + e));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        const bool precedes = b < static_cast<int>(blockIdx.x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = static_cast<int>(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
          sum[i] += c;
          before[i] += precedes ? c : 0;
        }
      }
    }
    for (int o = lanes; o < 32; o <<= 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
        before[i] += __shfl_xor_sync(0xffffffffu, before[i], o);
      }
    }
    if (lane < lanes) {
      int4* row = reinterpret_cast<int4*>(&s_rows[warp][col * 8]);
      row[0] = make_int4(sum[0], sum[1], sum[2], sum[3]);
      row[1] = make_int4(sum[4], sum[5], sum[6], sum[7]);
      if (warp == own_warp) {
        int4* own = reinterpret_cast<int4*>(&s_own[col * 8]);
        own[0] = make_int4(before[0], before[1], before[2], before[3]);
        own[1] = make_int4(before[4], before[5], before[6], before[7]);
      }
    }
    __syncthreads();
    const int x = threadIdx.x & (kSpan - 1), share = threadIdx.x / kSpan;  // (integer sums: any order)
    if (e0 + x < E) {
      int all = 0, some = share == 0 ? s_own[x] : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int w = share * 8 + i, c = s_rows[w][x];
        all += c;
        some += w < own_warp ? c : 0;
      }
      atomicAdd(&s_sum[e0 + x], all);
      atomicAdd(&s_before[e0 + x], some);
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.offsets[0] = 0;
  int preceding = 0;
  for (int e0 = 0; e0 < E; e0 += THREADS) {
    const int e = e0 + threadIdx.x, sum = s_sum[e];
    const int behind = preceding + block_scan(sum, s_tmp);
    s_before[e] += behind - sum;
    if (blockIdx.x == 0 && e < E) p.offsets[e + 1] = behind;
    if (e0 + THREADS < E) {
      __syncthreads();
      preceding += s_tmp[WARPS - 1];
    }
  }
  __syncthreads();
  while (item < items_end) {
    if (at >= 0) p.positions[item] = rank + s_before[at];
    item += THREADS;
    if (item < items_end) {
      at = p.chosen[item];
      rank = p.positions[item];
    }
  }
}

constexpr int kRouteWarps = 32;
constexpr int64_t kRouteOneCta = 32;   // tokens (one a warp) that one CTA routes and places in one kernel: 128 tokens of
                                       // 128 experts take 11.5 us that way, on four CTAs and a second kernel 6.2 us
constexpr int64_t kRouteCtas = 148;    // CTAs of a larger batch: one for each SM, more behind 9.7 million tokens

// shared memory of which an SM has no two: where the previous kernel's CTAs leave one by one, two CTAs of the next could
// meet on one SM while another has none
constexpr int kRouteOnePerSm = 116 * 1024;

int64_t route_per_cta(int64_t tokens) {  // at least one token per warp, and counts of 16 bits
  const int64_t n = (tokens + kRouteCtas - 1) / kRouteCtas;
  return n < kRouteWarps ? kRouteWarps : n < 65535 ? n : 65535;
}

template <typename T, int EPL>
cudaError_t launch_route(RouteParams p, cudaStream_t st) {
  static std::once_flag flags[64][2];
  static cudaError_t results[64][2];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  const int one = p.tokens <= kRouteOneCta;
  constexpr int kLaneBytes = EPL * sizeof(T) < 16 ? EPL * sizeof(T) : 16;
  p.vec = p.experts == 32 * EPL && aligned(p.logits, kLaneBytes) && (p.ld * sizeof(T)) % kLaneBytes == 0;
  std::call_once(flags[dev][one], [dev, one]() {
    const int bytes = std::max((kRouteWarps + 1) * EPL * 32 * 4, one ? 0 : kRouteOnePerSm);
    results[dev][one] =
        one ? cudaFuncSetAttribute(route_kernel<T, EPL, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)
            : cudaFuncSetAttribute(route_kernel<T, EPL, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  });
  if (results[dev][one] != cudaSuccess) return results[dev][one];
  const size_t smem = std::max<size_t>(static_cast<size_t>(kRouteWarps + 1) * p.experts * 4, one ? 0 : kRouteOnePerSm);
  const int64_t per_cta = one ? p.tokens : route_per_cta(p.tokens);
  p.per_cta = static_cast<int>(per_cta);
  p.run = static_cast<int>((per_cta + kRouteWarps - 1) / kRouteWarps);
  if (one) return launch_overlapped(route_kernel<T, EPL, true>, dim3(1), dim3(1024), smem, st, p);
  const int ctas = static_cast<int>((p.tokens + per_cta - 1) / per_cta);
  cudaError_t err = launch_overlapped(route_kernel<T, EPL, false>, dim3(ctas), dim3(1024), smem, st, p);
  if (err != cudaSuccess) return err;
  int lanes_log2 = 0;
  while (lanes_log2 < 5 && (8 << lanes_log2) < p.experts) ++lanes_log2;
  if (EPL > 4 && ctas > 32)
    return launch_overlapped(route_place_kernel<1024>, dim3(ctas), dim3(1024), 0, st, p, ctas, per_cta, lanes_log2);
  return launch_overlapped(route_place_kernel<512>, dim3(ctas), dim3(512), 0, st, p, ctas, per_cta, lanes_log2);
}

template <typename T>
cudaError_t dispatch_route(const RouteParams& p, cudaStream_t st) {
  if (p.experts <= 32) return launch_route<T, 1>(p, st);
  if (p.experts <= 64) return launch_route<T, 2>(p, st);
  if (p.experts <= 128) return launch_route<T, 4>(p, st);
  if (p.experts <= 256) return launch_route<T, 8>(p, st);
  return launch_route<T, 32>(p, st);
}

// =============================================================================================
// Row-wise symmetric int8 quantization of fp32 / bf16 / f16 rows:
//   s = max(max|x| / 127.5, 1e-8), code = clamp(rint(x * (1/s)), -128, 127), NaN -> 0,
// every step one IEEE fp32 operation (the per-row grid of lucid/nn/quantized/dynamic/linear.py's weights;
// lucid/quantization/_qparams.py:186-205).  With `positions`, the codes and the scale of token t go to the
// rows positions[t, 0..copies) (negative: nowhere); otherwise to row t.  `valid` (device): rows of x.
//
// The row stays in registers between the maximum and the codes, so x is read once.  The kernel lets its
// successor start only after its own wait, so a successor may assume that whatever preceded this kernel is
// complete.
// =============================================================================================
struct TokenParams {
  const void* x;
  int64_t rows, cols, ldx;
  const int32_t* positions;
  int copies;
  int64_t out_rows;
  const int32_t* valid;
  int8_t* codes;
  int64_t ldq;
  float* scale;
};

// largest |x| of 16 bytes (fmaxf and __hmax2 drop NaN); 16-bit types two at a time
__device__ __forceinline__ float largest_of(const Vec16<float>& v) {
  return fmaxf(fmaxf(fabsf(v.v[0]), fabsf(v.v[1])), fmaxf(fabsf(v.v[2]), fabsf(v.v[3])));
}
template <typename T, typename T2>
__device__ __forceinline__ float largest_of_pairs(const T* v) {
  const T2* w = reinterpret_cast<const T2*>(v);
  const T2 m = __hmax2(__hmax2(__habs2(w[0]), __habs2(w[1])), __hmax2(__habs2(w[2]), __habs2(w[3])));
  return fmaxf(to_float<T>(m.x), to_float<T>(m.y));
}
__device__ __forceinline__ float largest_of(const Vec16<__nv_bfloat16>& v) {
  return largest_of_pairs<__nv_bfloat16, __nv_bfloat162>(v.v);
}
__device__ __forceinline__ float largest_of(const Vec16<__half>& v) { return largest_of_pairs<__half, __half2>(v.v); }

__device__ __forceinline__ float token_scale(float largest) { return fmaxf(__fdiv_rn(largest, 127.5f), 1e-8f); }

// The 16 bytes of a row's aligned vector `at` (VN elements from index at * VN - skew of the row on); elements outside
// the row are zero and not read.
template <typename T>
__device__ __forceinline__ void load_skewed(Vec16<T>& v, const T* aligned_row, int at, int skew, int cols) {
  constexpr int VN = Vec16<T>::kN;
  const int first = at * VN;
  if (first >= skew && first + VN <= skew + cols) {
    v.load(aligned_row + first);
  } else {
#pragma unroll
    for (int j = 0; j < VN; ++j)
      v.v[j] = first + j >= skew && first + j < skew + cols ? aligned_row[first + j] : from_float<T>(0.0f);
  }
}

// TPR threads hold a row of up to TPR * ITEMS vectors; 256 / TPR rows (at least one) per CTA.
// SKEWED: rows begin anywhere and have any length (an odd number of 16-bit elements puts every row elsewhere).  They
// are read in aligned vectors all the same, and a thread's codes are shifted into place with its neighbour's: the
// codes' rows are aligned.  8192 rows of 1001 bf16 in 7.0 us against 19.8 element
// by element, of 5001 in 36.9 against 48.6.
template <typename T, int TPR, int ITEMS, bool SKEWED>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) quantize_tokens_kernel(const TokenParams p) {
  constexpr int VN = Vec16<T>::kN, THREADS = TPR < 256 ? 256 : TPR, ROWS = THREADS / TPR, WPR = TPR / 32;
  using Codes = std::conditional_t<VN == 8, unsigned long long, uint32_t>;  // of one vector, first element lowest
  __shared__ float s_max[THREADS / 32];
  __shared__ Codes s_edge[SKEWED ? THREADS / 32 : 1][ITEMS + 1];  // what the lane before a warp's first one needs
  pdl_wait();
  pdl_launch_dependents();
  const int sub = threadIdx.x % TPR, warp = threadIdx.x >> 5, w0 = warp / WPR * WPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / TPR;
  const bool there = row < p.rows;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const int cols = static_cast<int>(p.cols);
  const int skew = SKEWED ? static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)) : 0;
  const int vectors = SKEWED ? (skew + cols + VN - 1) / VN : cols / VN, copies = p.positions ? p.copies : 1;
  Vec16<T> v[ITEMS];
  float largest = 0.0f;
  // the row, where it goes and whether it counts are requested together
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int at = i * TPR + sub;
    if (there && at < vectors) {
      if constexpr (SKEWED)
        load_skewed<T>(v[i], x - skew, at, skew, cols);
      else
        v[i].load(x + static_cast<int64_t>(at) * VN);
    }
  }
  int64_t to = row;
  if (there && p.positions) to = __ldg(p.positions + row * copies);
  const bool live = there && (!p.valid || row < __ldg(p.valid));
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (there && i * TPR + sub < vectors) largest = fmaxf(largest, largest_of(v[i]));
  }
  largest = warp_max(largest);
  if (TPR > 32) {
    if ((threadIdx.x & 31) == 0) s_max[warp] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WPR; ++w) largest = fmaxf(largest, s_max[w0 + w]);
  }
  const float s = token_scale(largest), inv = __fdiv_rn(1.0f, s);
  Codes packed[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    packed[i] = 0;
    if (!SKEWED || (there && i * TPR + sub < vectors)) {
#pragma unroll
      for (int j = 0; j < VN; j += 4)
        packed[i] |= static_cast<Codes>(pack4_sat<false>(
                         __fmul_rn(to_float<T>(v[i].v[j]), inv), __fmul_rn(to_float<T>(v[i].v[j + 1]), inv),
                         __fmul_rn(to_float<T>(v[i].v[j + 2]), inv), __fmul_rn(to_float<T>(v[i].v[j + 3]), inv), 0.0f, false))
                     << (8 * j);
    }
  }
  if constexpr (SKEWED) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) s_edge[warp][i] = packed[i];
      s_edge[warp][ITEMS] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      Codes next = __shfl_down_sync(0xffffffffu, packed[i], 1);
      if (lane == 31) next = warp - w0 + 1 < WPR ? s_edge[warp + 1][i] : s_edge[w0][i + 1];
      if (skew) packed[i] = packed[i] >> (8 * skew) | next << (8 * (VN - skew));
    }
  }
  if (!live) return;
  for (int c = 0; c < copies; ++c) {
    const int64_t row_out = to;
    if (c + 1 < copies) to = __ldg(p.positions + row * copies + c + 1);
    if (row_out < 0 || row_out >= p.out_rows) continue;
    if (sub == 0) p.scale[row_out] = s;
    int8_t* q = p.codes + row_out * p.ldq;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int first = (i * TPR + sub) * VN;
      if (first + VN <= cols) {
        *reinterpret_cast<Codes*>(q + first) = packed[i];
      } else if (SKEWED) {
        for (int j = 0; first + j < cols; ++j) q[first + j] = static_cast<int8_t>(packed[i] >> (8 * j));
      }
    }
  }
}

// rows too long for that: 256 threads read the row twice, the second time from the L2 (six rows a SM are 50 MB)
template <typename T>
__global__ void __launch_bounds__(256) quantize_tokens_long_kernel(const TokenParams p) {
  constexpr int VN = Vec16<T>::kN, UNROLL = 4;
  __shared__ float s_max[8];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  if (p.valid && row >= __ldg(p.valid)) return;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const int vectors = static_cast<int>(p.cols / VN);
  float largest = 0.0f;
  for (int i = threadIdx.x; i < vectors; i += UNROLL * 256) {
    Vec16<T> v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (i + u * 256 < vectors) v[u].load(x + static_cast<int64_t>(i + u * 256) * VN);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (i + u * 256 < vectors) largest = fmaxf(largest, largest_of(v[u]));
  }
  largest = warp_max(largest);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = largest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) largest = fmaxf(largest, s_max[w]);
  const float s = token_scale(largest), inv = __fdiv_rn(1.0f, s);
  const int copies = p.positions ? p.copies : 1;
  for (int c = 0; c < copies; ++c) {
    const int64_t to = p.positions ? __ldg(p.positions + row * copies + c) : row;
    if (to < 0 || to >= p.out_rows) continue;
    if (threadIdx.x == 0) p.scale[to] = s;
    int8_t* q = p.codes + to * p.ldq;
    for (int i = threadIdx.x; i < vectors; i += UNROLL * 256) {
      Vec16<T> v[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
        if (i + u * 256 < vectors) v[u].load(x + static_cast<int64_t>(i + u * 256) * VN);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if (i + u * 256 >= vectors) continue;
        uint32_t packed[VN / 4];
#pragma unroll
        for (int j = 0; j < VN; j += 4)
          packed[j / 4] = pack4_sat<false>(__fmul_rn(to_float<T>(v[u].v[j]), inv), __fmul_rn(to_float<T>(v[u].v[j + 1]), inv),
                                           __fmul_rn(to_float<T>(v[u].v[j + 2]), inv),
                                           __fmul_rn(to_float<T>(v[u].v[j + 3]), inv), 0.0f, false);
        int8_t* dst = q + static_cast<int64_t>(i + u * 256) * VN;
        if (VN == 8)
          *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[VN / 4 - 1]);
        else
          *reinterpret_cast<uint32_t*>(dst) = packed[0];
      }
    }
  }
}

// any length and alignment: one CTA per row, which is read twice (the second time from L1 / L2)
template <typename T>
__global__ void __launch_bounds__(256) quantize_tokens_any_kernel(const TokenParams p) {
  __shared__ float s_max[8];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x;
  if (p.valid && row >= __ldg(p.valid)) return;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  float largest = 0.0f;
  for (int64_t i = threadIdx.x; i < p.cols; i += 256) largest = fmaxf(largest, fabsf(to_float<T>(x[i])));
  largest = warp_max(largest);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = largest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) largest = fmaxf(largest, s_max[w]);
  const float s = token_scale(largest), inv = __fdiv_rn(1.0f, s);
  const int copies = p.positions ? p.copies : 1;
  for (int c = 0; c < copies; ++c) {
    const int64_t to = p.positions ? __ldg(p.positions + row * copies + c) : row;
    if (to < 0 || to >= p.out_rows) continue;
    if (threadIdx.x == 0) p.scale[to] = s;
    for (int64_t i = threadIdx.x; i < p.cols; i += 256)
      p.codes[to * p.ldq + i] = static_cast<int8_t>(code_to_int(grid_code(to_float<T>(x[i]), inv, 0.0f), -128.0f, 127.0f));
  }
}

template <typename T, bool SKEWED>
cudaError_t launch_rows(const TokenParams& p, int64_t vectors, cudaStream_t st) {
  auto grid = [&](int rows_per_cta) { return dim3(static_cast<unsigned>((p.rows + rows_per_cta - 1) / rows_per_cta)); };
  if (vectors <= 32) return launch_overlapped(quantize_tokens_kernel<T, 32, 1, SKEWED>, grid(8), dim3(256), 0, st, p);
  if (vectors <= 128) return launch_overlapped(quantize_tokens_kernel<T, 32, 4, SKEWED>, grid(8), dim3(256), 0, st, p);
  if (vectors <= 256) return launch_overlapped(quantize_tokens_kernel<T, 64, 4, SKEWED>, grid(4), dim3(256), 0, st, p);
  if (vectors <= 512) return launch_overlapped(quantize_tokens_kernel<T, 128, 4, SKEWED>, grid(2), dim3(256), 0, st, p);
  if (vectors <= 1024) return launch_overlapped(quantize_tokens_kernel<T, 256, 4, SKEWED>, grid(1), dim3(256), 0, st, p);
  return launch_overlapped(quantize_tokens_kernel<T, 512, 4, SKEWED>, grid(1), dim3(512), 0, st, p);
}

template <typename T>
cudaError_t launch_tokens(const TokenParams& p, cudaStream_t st) {
  constexpr int VN = Vec16<T>::kN;
  const bool dense = p.cols % VN == 0 && (p.ldx * sizeof(T)) % 16 == 0 && aligned(p.x, 16);
  const bool out_ok = p.ldq % VN == 0 && aligned(p.codes, VN);
  const int64_t vectors = dense ? p.cols / VN : p.cols / VN + 2;  // skewed: a partial one at either end
  if (out_ok && vectors <= 2048) return dense ? launch_rows<T, false>(p, vectors, st) : launch_rows<T, true>(p, vectors, st);
  const dim3 grid(static_cast<unsigned>(p.rows));
  if (out_ok && dense) return launch_overlapped(quantize_tokens_long_kernel<T>, grid, dim3(256), 0, st, p);
  return launch_overlapped(quantize_tokens_any_kernel<T>, grid, dim3(256), 0, st, p);
}

// =============================================================================================
// out[t] = sum_j weights[t,j] * y[positions[t,j]] + residual[t], the terms added in the order of j in fp32,
// rounded once.  Positions of -1 contribute nothing.  HBM-bound: a thread owns 16 bytes of a row and has the
// loads of four experts in flight.
// =============================================================================================
struct CombineParams {
  const void* y;
  int64_t rows, cols, ldy, tokens;
  int top_k;
  const float* weights;
  const int32_t* positions;
  const void* residual;
  int64_t ldr;
  void* out;
  int64_t ldo;
};

template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p, int vectors) {
  constexpr int VN = Vec16<T>::kN;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t t = at / vectors;
  if (t >= p.tokens) return;
  const int64_t col = (at - t * vectors) * VN;
  float acc[VN];
#pragma unroll
  for (int i = 0; i < VN; ++i) acc[i] = 0.0f;
  Vec16<T> res;
  if (p.residual) res.load_stream(static_cast<const T*>(p.residual) + t * p.ldr + col);
  for (int j0 = 0; j0 < p.top_k; j0 += 4) {
    Vec16<T> v[4];
    float w[4];
    int32_t from[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      from[j] = j0 + j < p.top_k ? __ldg(p.positions + t * p.top_k + j0 + j) : -1;
      if (from[j] >= p.rows) from[j] = -1;
      w[j] = from[j] >= 0 ? __ldg(p.weights + t * p.top_k + j0 + j) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (from[j] >= 0) v[j].load_stream(static_cast<const T*>(p.y) + from[j] * p.ldy + col);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (from[j] >= 0) {
#pragma unroll
        for (int i = 0; i < VN; ++i) acc[i] = fmaf(w[j], to_float<T>(v[j].v[i]), acc[i]);
      }
    }
  }
  if (p.residual) {
#pragma unroll
    for (int i = 0; i < VN; ++i) acc[i] += to_float<T>(res.v[i]);
  }
  Vec16<T> o;
#pragma unroll
  for (int i = 0; i < VN; ++i) o.v[i] = from_float<T>(acc[i]);
  *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + t * p.ldo + col) = *reinterpret_cast<const uint4*>(o.v);
}

// rows that are not made of aligned vectors: TPR threads share a piece of a row, four elements each, TPR apart
// (8192 x 8 rows of 2001 bf16: 92 us, 3.6 TB/s; with 2000 the vectors take 49 us)
template <typename T, int TPR>
__global__ void __launch_bounds__(256) combine_any_kernel(const CombineParams p, int chunks) {
  constexpr int U = 4;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t piece = static_cast<int64_t>(blockIdx.x) * (256 / TPR) + threadIdx.x / TPR, t = piece / chunks;
  if (t >= p.tokens) return;
  const int64_t col = (piece - t * chunks) * (U * TPR) + threadIdx.x % TPR;
  float acc[U] = {};
  T res[U];
  if (p.residual) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (col + u * TPR < p.cols) res[u] = static_cast<const T*>(p.residual)[t * p.ldr + col + u * TPR];
  }
  for (int j0 = 0; j0 < p.top_k; j0 += 4) {
    T v[4][U];
    float w[4];
    int32_t from[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      from[j] = j0 + j < p.top_k ? __ldg(p.positions + t * p.top_k + j0 + j) : -1;
      if (from[j] >= p.rows) from[j] = -1;
      w[j] = from[j] >= 0 ? __ldg(p.weights + t * p.top_k + j0 + j) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (from[j] >= 0) {
        const T* src = static_cast<const T*>(p.y) + from[j] * p.ldy + col;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (col + u * TPR < p.cols) v[j][u] = src[u * TPR];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (from[j] >= 0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (col + u * TPR < p.cols) acc[u] = fmaf(w[j], to_float<T>(v[j][u]), acc[u]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (col + u * TPR < p.cols) {
      if (p.residual) acc[u] += to_float<T>(res[u]);
      static_cast<T*>(p.out)[t * p.ldo + col + u * TPR] = from_float<T>(acc[u]);
    }
  }
}

template <typename T, int TPR>
cudaError_t launch_combine_any(const CombineParams& p, cudaStream_t st) {
  const int64_t chunks = (p.cols + 4 * TPR - 1) / (4 * TPR), pieces = p.tokens * chunks;
  const dim3 grid(static_cast<unsigned>((pieces + 256 / TPR - 1) / (256 / TPR)));
  return launch_overlapped(combine_any_kernel<T, TPR>, grid, dim3(256), 0, st, p, static_cast<int>(chunks));
}

template <typename T>
cudaError_t launch_combine(const CombineParams& p, cudaStream_t st) {
  constexpr int VN = Vec16<T>::kN;
  auto row_ok = [](const void* base, int64_t ld) { return aligned(base, 16) && (ld * sizeof(T)) % 16 == 0; };
  const bool vec = p.cols % VN == 0 && row_ok(p.y, p.ldy) && row_ok(p.out, p.ldo) &&
                   (!p.residual || row_ok(p.residual, p.ldr));
  if (vec) {
    const dim3 grid(static_cast<unsigned>((p.tokens * (p.cols / VN) + 255) / 256));
    return launch_overlapped(combine_kernel<T>, grid, dim3(256), 0, st, p, static_cast<int>(p.cols / VN));
  }
  if (p.cols <= 128) return launch_combine_any<T, 32>(p, st);
  if (p.cols <= 512) return launch_combine_any<T, 128>(p, st);
  return launch_combine_any<T, 256>(p, st);
}

int32_t finish_launch(const char* what, cudaError_t err) {
  if (err != cudaSuccess) return fail(LC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
  return check_launch(what);
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" int64_t lc_route_experts_workspace_bytes(int64_t tokens, int64_t experts) {
  if (tokens <= kRouteOneCta || experts <= 0) return 0;
  const int64_t per_cta = route_per_cta(tokens);
  return (tokens + per_cta - 1) / per_cta * count_pitch(experts) * 2;
}

extern "C" int32_t lc_route_experts(const void* logits, int32_t dtype, int64_t tokens, int64_t experts, int64_t ld,
                                    int64_t top_k, int32_t renormalize, float* weights, int32_t* chosen,
                                    int32_t* offsets, int32_t* positions, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  if (tokens < 0 || experts < 1 || top_k < 1 || top_k > experts || ld < experts)
    return fail(LC_ERR_INVALID_ARG, "route_experts: bad shape (1 <= top_k <= experts is required)");
  if (experts > kRouteMaxExperts || top_k > kRouteMaxTopK)
    return fail(LC_ERR_UNSUPPORTED, "route_experts: at most %d experts and top_k %d", kRouteMaxExperts, kRouteMaxTopK);
  if (tokens * top_k > 0x7fffffffLL - 512) return fail(LC_ERR_UNSUPPORTED, "route_experts: too many tokens");
  if (dtype != LC_F32 && dtype != LC_BF16 && dtype != LC_F16)
    return fail(LC_ERR_UNSUPPORTED, "route_experts: dtype %d not supported", dtype);
  if (!offsets) return fail(LC_ERR_INVALID_ARG, "route_experts: null pointer");
  if (tokens == 0) {  // no token, no row: all offsets are zero
    if (cudaMemsetAsync(offsets, 0, static_cast<size_t>(experts + 1) * 4, as_stream(stream)) != cudaSuccess)
      return fail(LC_ERR_CUDA, "route_experts: %s", cudaGetErrorString(cudaGetLastError()));
    return LC_OK;
  }
  if (!logits || !weights || !chosen || !positions) return fail(LC_ERR_INVALID_ARG, "route_experts: null pointer");
  const int64_t need = lc_route_experts_workspace_bytes(tokens, experts);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(LC_ERR_WORKSPACE, "route_experts: workspace of %lld bytes required", (long long)need);
  RouteParams p = {};
  p.logits = logits;
  p.tokens = tokens;
  p.ld = ld;
  p.experts = static_cast<int>(experts);
  p.top_k = static_cast<int>(top_k);
  p.renormalize = renormalize;
  p.weights = weights;
  p.chosen = chosen;
  p.positions = positions;
  p.offsets = offsets;
  p.counts = static_cast<uint16_t*>(workspace);
  cudaStream_t st = as_stream(stream);
  return finish_launch("route_experts", dtype == LC_F32    ? dispatch_route<float>(p, st)
                                        : dtype == LC_BF16 ? dispatch_route<__nv_bfloat16>(p, st)
                                                           : dispatch_route<__half>(p, st));
}

extern "C" int32_t lc_quantize_tokens(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ldx,
                                      const int32_t* positions, int64_t copies, int64_t out_rows, const int32_t* valid,
                                      int8_t* codes, int64_t ldq, float* scale, void* stream) {
  if (rows < 0 || cols < 0 || ldx < cols || ldq < cols || (positions && copies < 1))
    return fail(LC_ERR_INVALID_ARG, "quantize_tokens: bad shape");
  if (!positions && out_rows < rows) return fail(LC_ERR_INVALID_ARG, "quantize_tokens: fewer output rows than rows");
  if (dtype != LC_F32 && dtype != LC_BF16 && dtype != LC_F16)
    return fail(LC_ERR_UNSUPPORTED, "quantize_tokens: dtype %d not supported", dtype);
  if (rows == 0 || cols == 0) return LC_OK;
  if (!x || !codes || !scale) return fail(LC_ERR_INVALID_ARG, "quantize_tokens: null pointer");
  if (rows > 0x7fffffffLL || copies > 0x7fffffffLL) return fail(LC_ERR_UNSUPPORTED, "quantize_tokens: too many rows");
  const TokenParams p = {x, rows, cols, ldx, positions, static_cast<int>(copies), out_rows, valid, codes, ldq, scale};
  cudaStream_t st = as_stream(stream);
  return finish_launch("quantize_tokens", dtype == LC_F32    ? launch_tokens<float>(p, st)
                                          : dtype == LC_BF16 ? launch_tokens<__nv_bfloat16>(p, st)
                                                             : launch_tokens<__half>(p, st));
}

extern "C" int32_t lc_combine_experts(const void* y, int32_t dtype, int64_t rows, int64_t cols, int64_t ldy,
                                      const float* weights, const int32_t* positions, int64_t tokens, int64_t top_k,
                                      const void* residual, int64_t ldr, void* out, int64_t ldo, void* stream) {
  if (rows < 0 || cols < 0 || tokens < 0 || top_k < 1 || ldy < cols || ldo < cols || (residual && ldr < cols))
    return fail(LC_ERR_INVALID_ARG, "combine_experts: bad shape");
  if (dtype != LC_F32 && dtype != LC_BF16 && dtype != LC_F16)
    return fail(LC_ERR_UNSUPPORTED, "combine_experts: dtype %d not supported", dtype);
  if (tokens == 0 || cols == 0) return LC_OK;
  if (!weights || !positions || !out || (!y && rows > 0)) return fail(LC_ERR_INVALID_ARG, "combine_experts: null pointer");
  if (top_k > 0x7fffffffLL || cols > 0x7fffffffLL || tokens > 0x7fffffffLL || tokens * ((cols + 255) / 256) > 0x7fffffffLL)
    return fail(LC_ERR_UNSUPPORTED, "combine_experts: too many elements");
  const CombineParams p = {y, rows, cols, ldy, tokens, static_cast<int>(top_k), weights, positions, residual, ldr, out, ldo};
  cudaStream_t st = as_stream(stream);
  return finish_launch("combine_experts", dtype == LC_F32    ? launch_combine<float>(p, st)
                                          : dtype == LC_BF16 ? launch_combine<__nv_bfloat16>(p, st)
                                                             : launch_combine<__half>(p, st));
}
