// int8 Linear of one or many groups with bias, activation and residual in its epilogue, for B200:
//
//   acc[m,n] = sum_k q[m,k] * w[e,n,k]                     e = group (expert) that owns row m
//   out[m,n] = act(f32(acc - zx*wsum[e,n]) * (sx[m] * sw[e,n]) + bias[e,n]) + residual[m,n]
//
// The rows of q are sorted by group; offsets[e] .. offsets[e+1] are the rows of group e and live on the
// device, so nothing of the routing is read on the host.  One group without offsets is the dense Linear.
//
// The WEIGHT is the 128-row (256-row in a CTA pair) operand of tcgen05.mma kind::i8 and the activation
// codes are its N side, whose width follows the rows a tile really has (a multiple of 16, or 32 in a
// pair): a group of three rows costs a 16-column product instead of a 128-row one, and one kernel serves
// every group size.  The accumulator then has one output column per lane: scale, bias and zero-point
// term of a lane are registers, the gate and up rows of a SwiGLU (interleaved in blocks of eight) sit
// eight lanes apart in one warp, and a warp stores 32 adjacent outputs of a row at a time, so the
// epilogue needs no transpose through shared memory.
//
// Two forms:
//  * pair (cta_group::2): 256 weight rows x up to 256 rows of q per tile, each CTA of the pair loading
//    its own 128 weight rows and half of the q rows; for groups that fill such tiles.
//  * split (cta_group::1): 128 weight rows x up to 64 rows of q, K cut over the CTAs of a cluster.
//    Decode batches have few tiles (a [4096, 14336] layer: 32), and a cluster of up to eight gives every
//    SM a share of the weight's bytes.  The partial sums are int32, so adding them in rank 0's shared
//    memory in any order gives the same bits.
//
// CTA = 320 threads: TMA warp, MMA warp, eight epilogue warps; the accumulator is double-buffered in
// TMEM.  Every wait on an mbarrier is bounded: on expiry the role records a code in the status word and
// leaves its loop, the CTA waits (bounded) for its own copies in flight, frees its TMEM and returns.
#include <cuda.h>

#include <cmath>
#include <mutex>

#include "tcgen05.cuh"

namespace lc {
namespace grouped {

using namespace tc;

constexpr int BK = 128;               // bytes of K per stage = one 128B swizzle atom
constexpr int UMMA_K = 32;
constexpr int WROWS = 128;            // weight rows a CTA loads per tile
constexpr int A_BYTES = WROWS * BK;
constexpr int EPI_WARPS = 8;          // two per TMEM lane quadrant (four: the same times, decode batches 4 % slower)
constexpr int EPI_THREADS = EPI_WARPS * 32;
constexpr int NUM_THREADS = 64 + EPI_THREADS;
constexpr int MAX_GROUPS = 1024;

// kTokens: most rows of q per tile; kStep: granularity of the instruction's N; kBox: rows of q per TMA box of a tile
// that is not full; kRing: bytes of the operand ring (its stages are 16 KB of weights and the tile's codes); kRed:
// bytes of rank 0's buffer for the other ranks' partial sums, [column][lane]
template <int CG>
struct Cfg;
template <>
struct Cfg<1> {
  static constexpr int kTokens = 64, kStep = 16, kBox = 16;
  static constexpr int kRing = 7 * (A_BYTES + kTokens * BK), kRed = kTokens * WROWS * 4;
};
template <>
struct Cfg<2> {
  static constexpr int kTokens = 256, kStep = 32, kBox = 32;
  static constexpr int kRing = 6 * (A_BYTES + kTokens / 2 * BK), kRed = 0;
};
constexpr int MAX_STAGES = 12;
template <int CG>
__host__ __device__ constexpr int smem_bytes() {
  return 1024 + Cfg<CG>::kRing + 256 + Cfg<CG>::kRed + 2 * Cfg<CG>::kTokens * 4 + 2 * (MAX_GROUPS + 1) * 4;
}
static_assert(smem_bytes<1>() <= 232448 && smem_bytes<2>() <= 232448, "shared memory of a CTA");
static_assert(2 * MAX_STAGES * 8 + 6 * 8 <= 256 && MAX_STAGES + 3 <= 31, "barrier area; a lane sets each pair up");

enum : int { ST_PRODUCER = 1, ST_MMA = 2, ST_EPILOGUE = 3 };

struct Params {
  int64_t R, N, K;          // rows of q, weight rows of a group, contraction length
  int E;
  const int32_t* offsets;   // [E + 1] or null (one group of R rows)
  const float* sx;          // 1 or R
  int sx_per_row;
  const float* zx;          // device scalar holding an integer value, or null
  const int32_t* wsum;      // [E, N], with zx
  const float* sw;          // [E, N]
  const float* bias;        // [E, N] or null
  int act;
  const void* residual;     // [R, out columns] of out's type, or null
  int64_t ldr;
  void* out;
  int out_dtype;
  int64_t ldo;
  int32_t* status;
  int wait_test;
  int tokens;               // rows of q per tile, at most the form's kTokens
  int tile_rows;            // weight rows per tile: 128 (256 in a pair) or fewer, a multiple of 8 for each CTA
  int stages, stage_bytes;  // of the operand ring
  int split;                // CTAs of a cluster that share a tile's K (CG == 1)
  int early_weights;        // the weight and offsets were complete before the previous kernel began
  uint32_t idesc;           // instruction descriptor without its N field
};

__device__ __forceinline__ void report(int32_t* status, int code) {
  if (status) atomicCAS(status, 0, code);
}

// ---- cluster-scope synchronisation of the split form -------------------------------------
__device__ __forceinline__ bool mbar_try_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, long long budget) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait_cluster(bar, parity)) {
    if (clock64() - t0 > budget) return false;
  }
  return true;
}
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// adds to a word of another CTA's shared memory and counts four bytes on that CTA's mbarrier once it is there
__device__ __forceinline__ void red_add_async(uint32_t cluster_addr, uint32_t v, uint32_t cluster_bar) {
  asm volatile("red.async.relaxed.cluster.shared::cluster.mbarrier::complete_tx::bytes.add.u32 [%0], %1, [%2];" ::"r"(
                   cluster_addr),
               "r"(v), "r"(cluster_bar)
               : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                                 uint32_t cluster_bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(cluster_bar)
      : "memory");
}
__device__ __forceinline__ void tc_ld(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// barrier over the epilogue threads that also ANDs a predicate
__device__ __forceinline__ bool epilogue_all(bool ok) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred pin, pout;\n\t"
      "setp.ne.u32 pin, %1, 0;\n\t"
      "bar.red.and.pred pout, 1, %2, pin;\n\t"
      "selp.u32 %0, 1, 0, pout;\n\t}"
      : "=r"(out)
      : "r"(static_cast<uint32_t>(ok)), "n"(EPI_THREADS)
      : "memory");
  return out != 0;
}

// ---- which tile ---------------------------------------------------------------------------
struct Tile {
  int e, m0, rows;  // group, first row of q, rows
  int64_t n0;       // first weight row inside the group
};

// Tiles are numbered group by group; within a group, bands of 16 row tiles share the weight tiles.  The walk only
// moves forward, because a CTA's tile numbers grow: to this group's next tile or, by bisection, to a later group (a
// token among 128 experts leaves 122 empty groups to step over).
struct TileWalk {
  const int* start;  // [E + 1] first tile of each group
  const int* off;    // [E + 1] first row of each group
  int tiles_n, tokens, tile_rows, groups, e;
  __device__ __forceinline__ TileWalk(const int* s, const int* o, int tn, const Params& p)
      : start(s), off(o), tiles_n(tn), tokens(p.tokens), tile_rows(p.tile_rows), groups(p.E), e(0) {}
  __device__ __forceinline__ Tile at(int t) {
    if (t >= start[e + 1]) {  // the first group behind whose tiles t does not lie
      int lo = e + 1, hi = groups - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (t >= start[mid + 1])
          lo = mid + 1;
        else
          hi = mid;
      }
      e = lo;
    }
    const int rows = off[e + 1] - off[e];
    const int tiles_m = (rows + tokens - 1) / tokens;
    const int local = t - start[e];
    constexpr int kBand = 16;
    const int band = kBand * tiles_n;
    const int g = local / band, first = g * kBand;
    const int gm = tiles_m - first < kBand ? tiles_m - first : kBand;
    const int r = local - g * band;
    const int tm = first + r % gm, tn = r / gm;
    Tile tile;
    tile.e = e;
    tile.m0 = off[e] + tm * tokens;
    const int left = off[e + 1] - tile.m0;
    tile.rows = left < tokens ? left : tokens;
    tile.n0 = static_cast<int64_t>(tn) * tile_rows;
    return tile;
  }
};

// ---- epilogue arithmetic -------------------------------------------------------------------
// Sigmoids take the hardware exponential and the approximate division: with z = -arg, ex2's argument carries a
// relative rounding of 2^-23, so exp(z) is off by (2 + 1.2 |z|) 2^-23, which sigma (1 - sigma) turns into less than
// 2^-23 of v, next to the division's 2 ulp.
__device__ __forceinline__ float sigmoid_times(float v, float arg) { return __fdividef(v, 1.0f + __expf(-arg)); }

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// two fp32 values in one register pair: one instruction multiplies or multiply-adds both
struct Pair {
  unsigned long long v;
};
__device__ __forceinline__ Pair pack(float lo, float hi) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack(Pair a, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v));
}
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// v * Phi(v) = max(v, 0) - |v| Phi(-|v|), Phi the normal distribution function, for two values.  Phi(n) = 2^p(n) for
// n = -|v|, p a polynomial of degree 9 fitted to log2 Phi on [-6, 0] (least squares over Chebyshev nodes, reweighted
// towards the smallest largest error in n * Phi): n * Phi(n) is off by at most 3.5e-8, and by 2e-12 beyond -6.  20
// instructions a pair where the library's erff takes about 80: an 8192 x 2048 x 512 product, whose time is the
// epilogue's, 24.0 us against 32.3 us.
__device__ __forceinline__ void gelu(float& v0, float& v1) {
  const float n0 = fmaxf(-fabsf(v0), -10.0f), n1 = fmaxf(-fabsf(v1), -10.0f);
  const Pair n = pack(n0, n1);
  constexpr float kCoeff[10] = {-2.9685912750210264e-07f, -6.425118044717237e-06f, -5.635188063024543e-05f,
                                -0.00022571126464754343f, 9.095141285797581e-05f,  0.007042091339826584f,
                                0.052499450743198395f,    -0.4592026472091675f,    1.151106357574463f,
                                -0.9999999403953552f};
  Pair p = pack(kCoeff[0], kCoeff[0]);
#pragma unroll
  for (int i = 1; i < 10; ++i) p = fma(p, n, pack(kCoeff[i], kCoeff[i]));
  float p0, p1;
  unpack(p, p0, p1);
  unpack(fma(n, pack(exp2_approx(p0), exp2_approx(p1)), pack(max_nan(v0, 0.0f), max_nan(v1, 0.0f))), v0, v1);
}

template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if constexpr (ACT == LC_ACT_RELU) return v < 0.0f ? 0.0f : v;  // NaN compares false and stays
  if constexpr (ACT == LC_ACT_GELU_TANH)  // 0.5 v (1 + tanh(u)) = v / (1 + exp(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3)
    return sigmoid_times(v, 1.5957691216057307f * (v + 0.044715f * v * v * v));
  if constexpr (ACT == LC_ACT_SILU) return sigmoid_times(v, v);
  return v;
}

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

// What an epilogue warp knows of its tile: its lane's weight row and the columns it drains.
struct Lane {
  uint32_t t_row;   // TMEM address of this warp's quadrant of the accumulator
  int64_t m0;       // first row of q
  int rows;
  int64_t n;        // this lane's weight row inside the group
  bool in;          // there is such a row in this tile
  float sw, bias;
  int corr;         // zx * wsum
  const float* sx;  // scales of the tile's rows
  int first;        // first column this warp takes; every second chunk from there
  int slot;         // this lane's word in a row of the partial-sum buffer
  int* red;         // rank 0 of a split tile: the other ranks' sums, cleared as they are read; else null
};

// Drains the accumulator in chunks of 16 columns: 16 rows of q, 32 adjacent outputs of each per warp.  The
// activation and the type are compiled in and the loop over the chunks is not unrolled: with all of them in one
// unrolled body (5000 instructions and more) the epilogue ran at the speed of instruction fetch, 30 us per
// 256 x 256 tile.
constexpr int CH = 16;
template <typename T, int ACT>
__device__ __forceinline__ void drain(const Params& p, const Lane& l) {
  const int up = (static_cast<int>(l.n) >> 3) & 1;  // SwiGLU: this lane's weight row is an up row
  const int64_t col = ACT == LC_ACT_SWIGLU ? (((l.n >> 4) << 3) | (l.n & 7)) : l.n;
  const int64_t row0 = l.m0 + (ACT == LC_ACT_SWIGLU ? up : 0);
  const T* const res = static_cast<const T*>(p.residual);
  const Pair sw2 = pack(l.sw, l.sw), bias2 = pack(l.bias, l.bias);
#pragma unroll 1
  for (int c = l.first; c < l.rows; c += EPI_WARPS / 4 * CH) {
    const int left = l.in ? l.rows - c : 0;
    constexpr int kStep = ACT == LC_ACT_SWIGLU ? 2 : 1;  // a lane finishes every row, or every second one
    T rv[CH / kStep];
    if (res) {
      const T* src = res + (row0 + c) * p.ldr + col;
#pragma unroll
      for (int j = 0; j < CH; j += kStep) {
        if (j + (kStep == 2 ? up : 0) < left) rv[j / kStep] = *src;
        src += kStep * p.ldr;
      }
    }
    uint32_t r[CH];
    tc_ld(l.t_row + static_cast<uint32_t>(c), r);
    tc_wait_ld();
    if (l.red) {
      int* mine = l.red + c * WROWS + l.slot;
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        if (c + j < l.rows) {
          r[j] += static_cast<uint32_t>(mine[j * WROWS]);
          mine[j * WROWS] = 0;
        }
      }
    }
    if (p.zx) {
#pragma unroll
      for (int j = 0; j < CH; ++j) r[j] -= static_cast<uint32_t>(l.corr);
    }
    float f[CH];
#pragma unroll
    for (int j = 0; j < CH; j += 4) {
      const float4 s = *reinterpret_cast<const float4*>(l.sx + c + j);
      auto value = [&](int i) { return static_cast<float>(static_cast<int>(r[i])); };
      unpack(fma(pack(value(j), value(j + 1)), mul(pack(s.x, s.y), sw2), bias2), f[j], f[j + 1]);
      unpack(fma(pack(value(j + 2), value(j + 3)), mul(pack(s.z, s.w), sw2), bias2), f[j + 2], f[j + 3]);
    }
    if constexpr (ACT == LC_ACT_GELU) {
#pragma unroll
      for (int j = 0; j < CH; j += 2) gelu(f[j], f[j + 1]);
    }
    T* o = static_cast<T*>(p.out) + (row0 + c) * p.ldo + col;
    auto finish = [&](int j) {  // the result of row c + j
      float v;
      if constexpr (ACT == LC_ACT_SWIGLU) {
        // lanes 8 apart hold the gate and the up value of one unit: each finishes every other row
        const float got = __shfl_xor_sync(0xffffffffu, up ? f[j] : f[j + 1], 8);
        const float gate = up ? got : f[j], lin = up ? f[j + 1] : got;
        v = sigmoid_times(gate, gate) * lin;
      } else {
        v = activate<ACT>(f[j]);
      }
      if (res) v += widen<T>(rv[j / kStep]);
      return narrow<T>(v);
    };
    if (__all_sync(0xffffffffu, left >= CH)) {
#pragma unroll
      for (int j = 0; j < CH; j += kStep, o += kStep * p.ldo) *o = finish(j);
    } else {
#pragma unroll
      for (int j = 0; j < CH; j += kStep, o += kStep * p.ldo) {
        const T v = finish(j);
        if (j + (kStep == 2 ? up : 0) < left) *o = v;
      }
    }
  }
}

template <int CG, typename T, int ACT>
__global__ void __launch_bounds__(NUM_THREADS, 1)
grouped_linear_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_q,
                      const __grid_constant__ CUtensorMap tmap_q_full, const Params p) {
  using C = Cfg<CG>;
  const int stages = p.stages, stage_bytes = p.stage_bytes;
  constexpr int TMEM_COLS = 2 * C::kTokens;  // 128 or 512
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint32_t s_tmem_base;

  pdl_launch_dependents();
  const uint32_t tiles_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar_base = tiles_base + C::kRing;
  const uint32_t red_base = bar_base + 256;
  uint8_t* const after = smem_raw + (red_base - smem_u32(smem_raw));
  int* const s_red = reinterpret_cast<int*>(after);
  float* const s_sx = reinterpret_cast<float*>(after + C::kRed);  // two accumulator stages
  int* const s_off = reinterpret_cast<int*>(s_sx + 2 * C::kTokens);
  int* const s_start = s_off + (MAX_GROUPS + 1);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (MAX_STAGES + s); };
  auto acc_full_bar = [&](int s) { return bar_base + 8u * (2 * MAX_STAGES + s); };
  auto acc_empty_bar = [&](int s) { return bar_base + 8u * (2 * MAX_STAGES + 2 + s); };
  const uint32_t part_bar = bar_base + 8u * (2 * MAX_STAGES + 4);  // rank 0: the other ranks' sums have been added
  const uint32_t free_bar = part_bar + 8u;                     // other ranks: rank 0's buffer is zero again

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long budget = p.wait_test ? 20000LL : kWaitCycles;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster = CG == 2 ? 2 : p.split;
  const int unit = static_cast<int>(blockIdx.x) / cluster, units = static_cast<int>(gridDim.x) / cluster;
  const int tiles_n = static_cast<int>((p.N + p.tile_rows - 1) / p.tile_rows);
  const int num_kb = static_cast<int>((p.K + BK - 1) / BK);
  const int kb0 = CG == 2 ? 0 : static_cast<int>(static_cast<int64_t>(num_kb) * rank / p.split);
  const int kb1 = CG == 2 ? num_kb : static_cast<int>(static_cast<int64_t>(num_kb) * (rank + 1) / p.split);

  // Warp 0 sets up the barriers and the tile table and requests the first weights: with early_weights before the
  // codes are there, and in the split form before the rest of the CTA is ready (its copies touch no barrier but this
  // CTA's own).  Warp 1 allocates TMEM meanwhile.
  uint32_t armed = 0, armed_parity = 0;  // producer: stages with copies in flight, one bit each
  int ahead = 0;                         // producer: stages whose weights have been requested
  auto request_first = [&]() {
    if (unit >= s_start[p.E] || p.wait_test) return;
    TileWalk walk(s_start, s_off, tiles_n, p);
    const Tile tile = walk.at(unit);
    const int mine = (tile.rows + C::kStep - 1) / C::kStep * C::kStep / CG;
    const int boxed = mine == p.tokens / CG ? mine : (mine + C::kBox - 1) / C::kBox * C::kBox;
    const int n0 = static_cast<int>(tile.n0) + (CG == 2 ? static_cast<int>(rank) * (p.tile_rows / 2) : 0);
    ahead = min(stages, kb1 - kb0);
    if (elect_one())
      for (int s = 0; s < ahead; ++s) {
        if (CG == 1 || leader) mbar_expect_tx(full_bar(s), static_cast<uint32_t>((p.tile_rows + CG * boxed) * BK));
        if constexpr (CG == 2)
          tma_load_3d_pair(tiles_base + s * stage_bytes, &tmap_w, (kb0 + s) * BK, n0, tile.e, map_to_cta(full_bar(s), 0));
        else
          tma_load_3d(tiles_base + s * stage_bytes, &tmap_w, (kb0 + s) * BK, n0, tile.e, full_bar(s));
      }
    __syncwarp();
    if (CG == 1 || leader) armed = (1u << ahead) - 1;
  };
  if (warp == 0) {
    if (lane < MAX_STAGES) {
      mbar_init(full_bar(lane), 1);
      mbar_init(empty_bar(lane), 1);
    } else if (lane < MAX_STAGES + 2) {
      mbar_init(acc_full_bar(lane - MAX_STAGES), 1);
      mbar_init(acc_empty_bar(lane - MAX_STAGES), CG * EPI_WARPS);
    } else if (lane == MAX_STAGES + 2) {
      mbar_init(part_bar, 1);
      mbar_init(free_bar, EPI_WARPS);
    } else if (lane == 31) {
      prefetch_map(&tmap_w);
      prefetch_map(&tmap_q);
      prefetch_map(&tmap_q_full);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the copies below count on them at once
    __syncwarp();
    if (!p.early_weights) pdl_wait();
    // first row and first tile of every group.  Offsets come from the caller: they are clamped to the rows there are
    // and made ascending (a running maximum), so that no tile lies outside and the tiles are as many as launched for.
    if (!p.offsets) {
      if (lane == 0) {
        s_off[0] = 0;
        s_off[1] = static_cast<int>(p.R);
        s_start[0] = 0;
        s_start[1] = static_cast<int>((p.R + p.tokens - 1) / p.tokens) * tiles_n;
      }
    } else {
      const int R = static_cast<int>(p.R);
      int base = 0, top = min(max(p.offsets[0], 0), R);  // tiles and end of the groups so far
      if (lane == 0) {
        s_off[0] = top;
        s_start[0] = 0;
      }
      constexpr int kAtOnce = 4;  // chunks of 32 offsets requested together
      for (int e1 = 0; e1 < p.E; e1 += 32 * kAtOnce) {
        int raw[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          const int e = e1 + i * 32 + lane;
          raw[i] = e < p.E ? p.offsets[e + 1] : 0;
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          const int e = e1 + i * 32 + lane;
          int end = min(max(raw[i], top), R);
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end = max(end, v);
          }
          const int before = __shfl_up_sync(0xffffffffu, end, 1);
          int sum = (end - (lane ? before : top) + p.tokens - 1) / p.tokens * tiles_n;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
          }
          if (e < p.E) {
            s_off[e + 1] = end;
            s_start[e + 1] = base + sum;
          }
          base += __shfl_sync(0xffffffffu, sum, 31);
          top = __shfl_sync(0xffffffffu, end, 31);
        }
      }
    }
    // arrive before the copies are issued: the release of the arrival waits for them otherwise (measured: 4 us)
    __syncwarp();
    cluster_arrive();
    if (CG == 1) request_first();
  } else if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)),
                   "r"(static_cast<uint32_t>(TMEM_COLS))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)),
                   "r"(static_cast<uint32_t>(TMEM_COLS))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  } else if (CG == 1 && p.split > 1 && leader) {
    for (int i = threadIdx.x - 64; i < C::kRed / 4; i += EPI_THREADS) s_red[i] = 0;
  }
  if (warp != 0) {
    tc_fence_before();
    __syncwarp();
    cluster_arrive();
  }
  cluster_wait();  // this CTA's set-up and the other CTAs' barriers (and rank 0's zeroed buffer) are complete
  tc_fence_after();
  const uint32_t tmem_base = s_tmem_base;
  const int total = s_start[p.E];

  if (warp == 0) {
    // ===================== TMA producer =====================
    // The whole warp walks the loop and one elected lane issues: in code that only lane 0 reaches, every operand of
    // a copy or an MMA is moved to a uniform register first, 70 clocks an instruction.
    int stage = 0;
    uint32_t phase = 0, slot = tiles_base;
    bool ok = true;
    if (CG == 2) request_first();     // (signals the leader's barriers: not before the cluster has set them up)
    if (p.early_weights) pdl_wait();  // the codes are the previous kernel's
    TileWalk walk(s_start, s_off, tiles_n, p);
    for (int t = unit; t < total && ok && !p.wait_test; t += units) {
      const Tile tile = walk.at(t);
      const int cols = (tile.rows + C::kStep - 1) / C::kStep * C::kStep;
      const int mine = cols / CG;  // q rows this CTA loads
      const bool full = mine == p.tokens / CG;  // one box; else as many of kBox rows as it takes
      const int boxes = (mine + C::kBox - 1) / C::kBox;
      const uint32_t bytes = static_cast<uint32_t>((p.tile_rows + CG * (full ? mine : boxes * C::kBox)) * BK);
      const int n0 = static_cast<int>(tile.n0) + (CG == 2 ? static_cast<int>(rank) * (p.tile_rows / 2) : 0);
      const int m0 = tile.m0 + (CG == 2 ? static_cast<int>(rank) * mine : 0);
      const int e = tile.e;
      auto load_q = [&](int s, uint32_t dst, int kb) {
        if (full) {
          if constexpr (CG == 2)
            tma_load_2d_pair(dst, &tmap_q_full, kb * BK, m0, map_to_cta(full_bar(s), 0));
          else
            tma_load_2d(dst, &tmap_q_full, kb * BK, m0, full_bar(s));
          return;
        }
        for (int b = 0; b < boxes; ++b) {
          if constexpr (CG == 2)
            tma_load_2d_pair(dst + b * C::kBox * BK, &tmap_q, kb * BK, m0 + b * C::kBox, map_to_cta(full_bar(s), 0));
          else
            tma_load_2d(dst + b * C::kBox * BK, &tmap_q, kb * BK, m0 + b * C::kBox, full_bar(s));
        }
      };
      int kb = kb0;
      if (t == unit && ahead) {  // the first stages have their weights under way
        if (elect_one())
          for (int s = 0; s < ahead; ++s) load_q(s, tiles_base + s * stage_bytes + A_BYTES, kb0 + s);
        __syncwarp();
        kb = kb0 + ahead;
        stage = ahead % stages;
        phase = ahead == stages ? 1u : 0u;
        slot = tiles_base + stage * stage_bytes;
      }
      for (; kb < kb1; ++kb) {
        if (!__all_sync(0xffffffffu, mbar_wait(empty_bar(stage), phase ^ 1u, budget))) {
          if (lane == 0) report(p.status, ST_PRODUCER);
          ok = false;
          break;
        }
        if (elect_one()) {
          if (CG == 1 || leader) mbar_expect_tx(full_bar(stage), bytes);
          if constexpr (CG == 2)
            tma_load_3d_pair(slot, &tmap_w, kb * BK, n0, e, map_to_cta(full_bar(stage), 0));
          else
            tma_load_3d(slot, &tmap_w, kb * BK, n0, e, full_bar(stage));
          load_q(stage, slot + A_BYTES, kb);
        }
        __syncwarp();
        if (CG == 1 || leader) {
          armed |= 1u << stage;
          armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
        }
        slot += stage_bytes;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
          slot = tiles_base;
        }
      }
    }
    // do not leave while a bulk copy may still be landing (a pair's leader counts the bytes of both CTAs)
    for (int s = 0; s < stages; ++s)
      if (armed >> s & 1) mbar_wait(full_bar(s), armed_parity >> s & 1);
    __syncwarp();
  } else if (warp == 1) {
    // ===================== MMA issuer (a pair's leader only) =====================
    if (CG == 1 || leader) {
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      // descriptors of the first stage; a stage further on is stage_bytes / 16 more (the start address is below 2^18)
      const uint64_t w_first = make_smem_desc(tiles_base), q_off = A_BYTES >> 4;
      uint64_t w_desc = w_first;
      TileWalk walk(s_start, s_off, tiles_n, p);
      for (int t = unit; t < total && ok; t += units, ++it) {
        const Tile tile = walk.at(t);
        const uint32_t cols = (tile.rows + C::kStep - 1) / C::kStep * C::kStep;
        const uint32_t idesc = p.idesc | ((cols >> 3) << 17);
        const int as = it & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(acc_empty_bar(as), ((it >> 1) & 1) ^ 1u, budget))) {
          if (lane == 0) report(p.status, ST_MMA);
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(as * C::kTokens);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, budget))) {
            if (lane == 0) report(p.status, ST_MMA);
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t q_desc = w_desc + q_off;
#pragma unroll
            for (int j = 0; j < BK / UMMA_K; ++j) {
              const uint64_t koff = static_cast<uint64_t>((j * UMMA_K) >> 4);
              const uint32_t accumulate = (kb != kb0 || j != 0) ? 1u : 0u;
              if constexpr (CG == 2)
                tc_mma_i8_pair(d_tmem, w_desc + koff, q_desc + koff, idesc, accumulate);
              else
                tc_mma_i8(d_tmem, w_desc + koff, q_desc + koff, idesc, accumulate);
            }
            if constexpr (CG == 2)
              tc_commit_pair(empty_bar(stage));
            else
              tc_commit(empty_bar(stage));
          }
          __syncwarp();
          w_desc += static_cast<uint32_t>(stage_bytes) >> 4;
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
            w_desc = w_first;
          }
        }
        if (ok && elect_one()) {
          if constexpr (CG == 2)
            tc_commit_pair(acc_full_bar(as));
          else
            tc_commit(acc_full_bar(as));
        }
        __syncwarp();
      }
    }
  } else {
    // ===================== epilogue (eight warps of every CTA) =====================
    const int q = warp & 3;  // TMEM lane quadrant this warp may read
    const int group = (warp - 2) >> 2;
    const int et = threadIdx.x - 64;
    if (p.early_weights) pdl_wait();
    const int zx = p.zx ? __float2int_rn(__ldg(p.zx)) : 0;
    TileWalk walk(s_start, s_off, tiles_n, p);
    const int cta_rows = p.tile_rows / CG, local = q * 32 + lane;  // this lane's weight row among the CTA's
    // a tile's scales and biases, fetched while the tile before it is drained
    struct Side {
      Tile tile;
      int64_t n;
      bool in;
      float sx, sw, bias;
      int corr;
    };
    auto fetch = [&](int t) {
      Side s;
      s.tile = walk.at(t);
      s.n = s.tile.n0 + (CG == 2 ? static_cast<int64_t>(rank) * cta_rows : 0) + local;
      s.in = s.n < p.N && local < cta_rows;  // lanes beyond a narrow tile hold nothing
      const int64_t at = static_cast<int64_t>(s.tile.e) * p.N + s.n;
      s.sx = et < s.tile.rows ? __ldg(p.sx + (p.sx_per_row ? s.tile.m0 + et : 0)) : 0.0f;
      s.sw = s.in ? __ldg(p.sw + at) : 0.0f;
      s.bias = (s.in && p.bias) ? __ldg(p.bias + at) : 0.0f;
      s.corr = (s.in && p.wsum) ? zx * __ldg(p.wsum + at) : 0;
      return s;
    };
    Side next = {};
    if (unit < total) next = fetch(unit);
    int it = 0;
    for (int t = unit; t < total; t += units, ++it) {
      const Side side = next;
      const Tile& tile = side.tile;
      const int as = it & 1;
      float* const sx = s_sx + as * C::kTokens;
      if (et < C::kTokens) sx[et] = side.sx;
      if (CG == 1 && p.split > 1 && leader && et == 0)
        mbar_expect_tx(part_bar, static_cast<uint32_t>((p.split - 1) * tile.rows * WROWS * 4));
      bool arrived = mbar_wait(acc_full_bar(as), (it >> 1) & 1, budget);
      if (CG == 1 && p.split > 1)
        arrived = arrived && (leader ? mbar_wait_cluster(part_bar, it & 1, budget)
                                     : mbar_wait_cluster(free_bar, (it & 1) ^ 1u, budget));
      // also publishes the staged scales; those of the tile before last are no longer read
      if (!epilogue_all(arrived)) {
        report(p.status, ST_EPILOGUE);
        // sums another rank may still be sending land in this CTA's memory: give them the same time again
        if (CG == 1 && p.split > 1 && leader) mbar_wait_cluster(part_bar, it & 1, budget);
        break;
      }
      tc_fence_after();
      if (t + units < total) next = fetch(t + units);
      Lane l;
      l.t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(as * C::kTokens);
      l.m0 = tile.m0;
      l.rows = tile.rows;
      l.n = side.n;
      l.in = side.in;
      l.sw = side.sw;
      l.bias = side.bias;
      l.corr = side.corr;
      l.sx = sx;
      l.first = group * CH;
      l.slot = local;
      l.red = CG == 1 && p.split > 1 ? s_red : nullptr;
      if (CG == 1 && !leader) {
        const uint32_t dst = map_to_cta(red_base, 0) + static_cast<uint32_t>(l.slot) * 4;
        const uint32_t bar = map_to_cta(part_bar, 0);
#pragma unroll 1
        for (int c = l.first; c < l.rows; c += EPI_WARPS / 4 * CH) {
          uint32_t r[CH];
          tc_ld(l.t_row + static_cast<uint32_t>(c), r);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < CH; ++j)
            if (c + j < l.rows) red_add_async(dst + static_cast<uint32_t>((c + j) * WROWS * 4), r[j], bar);
        }
      } else {
        drain<T, ACT>(p, l);
      }
      tc_fence_before();
      if (CG == 1 && p.split > 1 && leader && t + units < total) {  // the cleared buffer may be added to again
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
        __syncwarp();
        if (lane > 0 && lane < p.split) mbar_arrive_release_cluster(map_to_cta(free_bar, lane));
      }
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2)
          mbar_arrive_cluster(map_to_cta(acc_empty_bar(as), 0));
        else
          mbar_arrive(acc_empty_bar(as));
      }
    }
    // rows behind the last group belong to no group: zero
    if (p.offsets) {
      const int64_t width = ACT == LC_ACT_SWIGLU ? p.N / 2 : p.N;
      for (int64_t row = s_off[p.E] + static_cast<int64_t>(blockIdx.x); row < p.R; row += gridDim.x)
        for (int64_t c = et; c < width; c += EPI_THREADS) static_cast<T*>(p.out)[row * p.ldo + c] = narrow<T>(0.0f);
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA frees TMEM or leaves while another may still reach its memory
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                   "r"(static_cast<uint32_t>(TMEM_COLS))
                   : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                   "r"(static_cast<uint32_t>(TMEM_COLS))
                   : "memory");
  }
}

// ---- host side -------------------------------------------------------------------------------
using Kernel = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, Params);

template <int CG, typename T>
static Kernel kernel_for(int act) {
  switch (act) {
    case LC_ACT_RELU: return grouped_linear_kernel<CG, T, LC_ACT_RELU>;
    case LC_ACT_GELU: return grouped_linear_kernel<CG, T, LC_ACT_GELU>;
    case LC_ACT_GELU_TANH: return grouped_linear_kernel<CG, T, LC_ACT_GELU_TANH>;
    case LC_ACT_SILU: return grouped_linear_kernel<CG, T, LC_ACT_SILU>;
    case LC_ACT_SWIGLU: return grouped_linear_kernel<CG, T, LC_ACT_SWIGLU>;
    default: return grouped_linear_kernel<CG, T, LC_ACT_NONE>;
  }
}
template <int CG>
static Kernel kernel_for(int dtype, int act) {
  return dtype == LC_F32    ? kernel_for<CG, float>(act)
         : dtype == LC_BF16 ? kernel_for<CG, __nv_bfloat16>(act)
                            : kernel_for<CG, __half>(act);
}

static void launch_config(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attrs, unsigned grid, int smem, int cluster,
                          cudaStream_t st) {
  *cfg = {};
  cfg->gridDim = dim3(grid);
  cfg->blockDim = dim3(NUM_THREADS);
  cfg->dynamicSmemBytes = smem;
  cfg->stream = st;
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = cluster;
  attrs[0].val.clusterDim.y = 1;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg->attrs = attrs;
  cfg->numAttrs = 2;
}

struct DeviceInfo {
  cudaError_t err;
  int clusters[4];  // resident clusters of 1, 2, 4, 8 CTAs of the split form
};

static int32_t device_info(const DeviceInfo** out) {
  constexpr int kMaxDevices = 64;
  static std::once_flag flags[kMaxDevices];
  static DeviceInfo infos[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return fail(LC_ERR_CUDA, "no current CUDA device");
  std::call_once(flags[dev], [dev]() {
    DeviceInfo& info = infos[dev];
    info.err = cudaSuccess;
    for (int dtype : {LC_F32, LC_BF16, LC_F16})
      for (int act = LC_ACT_NONE; act <= LC_ACT_SWIGLU && info.err == cudaSuccess; ++act) {
        info.err = cudaFuncSetAttribute(kernel_for<1>(dtype, act), cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<1>());
        if (info.err == cudaSuccess)
          info.err = cudaFuncSetAttribute(kernel_for<2>(dtype, act), cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<2>());
      }
    const int sms = sm_count();
    for (int i = 0; i < 4 && info.err == cudaSuccess; ++i) {
      cudaLaunchConfig_t cfg;
      cudaLaunchAttribute attrs[2];
      launch_config(&cfg, attrs, static_cast<unsigned>(sms / (1 << i) << i), smem_bytes<1>(), 1 << i, nullptr);
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kernel_for<1>(LC_F32, LC_ACT_NONE), &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = i == 0 ? sms : 0;
      }
      info.clusters[i] = n;
    }
  });
  if (infos[dev].err != cudaSuccess)
    return fail(LC_ERR_CUDA, "grouped_linear: cannot reserve shared memory: %s", cudaGetErrorString(infos[dev].err));
  *out = &infos[dev];
  return LC_OK;
}

// Row tiles there can be at most: one partly filled one per group that has rows, the rest full.
static int64_t row_tiles(const Params& p, int tokens) {
  const int64_t groups = p.offsets ? (p.E < p.R ? p.E : p.R) : 1;
  return (p.R - groups) / tokens + groups;
}

struct Plan {
  int ctas, tokens, tile_rows, split;  // CTAs of an MMA (1 or 2), rows of q and weight rows per tile, CTAs along K
  int64_t units;                       // tiles in flight
};

// Form and tile sizes, by the clocks that the busiest CTA is expected to take.  A K block costs the larger of its
// MMAs (2 clocks per row of q in a pair, 1 else), of bringing it in (64 bytes a clock, 40 for weights used once) and of
// 300 clocks for a wait, four MMAs and a commit; the epilogue takes 25 clocks per row of q and runs beside the next tile's main loop; a tile
// costs 600 clocks more, and 1500 where K is split.  Tiles come in waves over the CTAs there are; the number of groups
// that have rows is not known on the host, so that half a tile stands for the last wave of a grouped product.
// Measured, product alone, weights from HBM:
//   16 rows,  [28672, 4096] SwiGLU   pair, 112 rows a CTA 22.8 us; pair, 128 24.0; one CTA, 112 23.7, 128 24.8
//   16 rows,  [4096, 14336]          K over 4 CTAs 14.4 us; over 2 18.0; over 8 18.0; over 4 with 112 rows 19.4
//   333 rows, [1232, 1008]           pair, 64 rows of q a tile 5.7 us, 128 6.1 to 6.8, 192 7.1 to 7.9
//   256 rows, [4096, 4096]           pair, 64 rows of q 11.0 us, 128 11.5, 256 15.4; one CTA, 64 12.5
//   64 groups of 84 rows, [2048, 1408]   pair, 128 rows of q 38.5 us, 64 50.2; one CTA, 64 54.2
//   32 groups of 8 rows, [4096, 4096]    pair 80.8 us, one CTA 83.3
static Plan make_plan(const Params& p, const DeviceInfo& info, int64_t sms, int variant) {
  const int num_kb = static_cast<int>((p.K + BK - 1) / BK);
  const int forced = variant > 2 ? 1 << (variant - 3) : 0;
  double groups = 1.0;  // that have rows, were these drawn evenly
  if (p.offsets) {
    const double empty = pow(1.0 - 1.0 / static_cast<double>(p.E), static_cast<double>(p.R));
    groups = static_cast<double>(p.E) * (1.0 - empty);
  }
  const double rows = static_cast<double>(p.R) / groups;
  const int64_t step = p.act == LC_ACT_SWIGLU ? 16 : 8;  // gate and up rows of a unit stay in one tile
  Plan plan = {2, 256, 256, 1, sms / 2};
  double best = 0.0;
  auto consider = [&](int ctas, int split, int64_t units, int tokens) {
    const double row_tiles = groups * ceil(rows / tokens), cols = rows < tokens ? rows : tokens;
    int64_t cta_rows = 128, across = (p.N + ctas * 128 - 1) / (ctas * 128);
    double waves = row_tiles * static_cast<double>(across) / static_cast<double>(units);
    if (p.offsets) {
      waves += 0.5;
    } else {
      waves = ceil(waves);
    }
    if (!p.offsets && rows <= tokens) {  // weights read once: as few rows as the same number of waves allows
      const int64_t room = static_cast<int64_t>(waves * static_cast<double>(units) / row_tiles);
      cta_rows = ((p.N + room * ctas - 1) / (room * ctas) + step - 1) / step * step;
      if (cta_rows < 48) cta_rows = 48;
      if (cta_rows > 128) cta_rows = 128;
    }
    // (weights that only one row tile reads come from HBM, of which a CTA gets less than of the L2)
    const double load = static_cast<double>(cta_rows * BK) / (rows <= tokens ? 40.0 : 64.0) + cols / ctas * BK / 64.0;
    double block = ctas * cols > 300.0 ? ctas * cols : 300.0;
    if (load > block) block = load;
    const double loop = (num_kb + split - 1) / split * block, drain = 25.0 * cols;
    const double cost = waves * ((loop > drain ? loop : drain) + (split > 1 ? 2100.0 : 600.0)) + (loop > drain ? drain : loop);
    if (best == 0.0 || cost < 0.98 * best) {
      best = cost;
      plan = {ctas, tokens, static_cast<int>(ctas * cta_rows), split, units};
    }
  };
  if (variant == 0 || variant == 2)
    for (int tokens : {64, 128, 192, 256}) consider(2, 1, sms / 2, tokens);
  if (variant != 2) {
    const double most = p.offsets ? 2.0 * rows : rows;  // groups differ in size
    const int tokens = most > 48.0 ? 64 : (static_cast<int>(most) + 15) / 16 * 16;
    for (int i = 0; i < 4; ++i) {
      const int split = 1 << i;
      if (info.clusters[i] < 1 || num_kb < (forced ? 1 : 4) * split) break;
      if (forced && split != forced && !(i == 0 && num_kb < forced)) continue;
      consider(1, split, info.clusters[i], tokens < 16 ? 16 : tokens);
    }
  }
  return plan;
}

static int32_t launch(const void* q, int64_t ldq, const int8_t* w, int64_t ldw, int64_t group_stride, int q_unsigned,
                      Params& p, int variant, cudaStream_t st) {
  const DeviceInfo* info = nullptr;
  if (int32_t rc = device_info(&info)) return rc;
  const Plan plan = make_plan(p, *info, sm_count(), variant);
  const bool pair = plan.ctas == 2;
  p.tokens = plan.tokens;
  p.tile_rows = plan.tile_rows;
  p.split = plan.split;
  p.stage_bytes = A_BYTES + plan.tokens / plan.ctas * BK;
  const int fit = (pair ? Cfg<2>::kRing : Cfg<1>::kRing) / p.stage_bytes;
  p.stages = fit < MAX_STAGES ? fit : MAX_STAGES;
  CUtensorMap map_w, map_q, map_q_full;
  if (int32_t rc = encode_tensor_map_3d(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, p.K, p.N, p.E, ldw, group_stride, BK,
                                        plan.tile_rows / plan.ctas, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  if (int32_t rc = encode_tensor_map_2d(&map_q, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, p.K, p.R, ldq, BK,
                                        pair ? Cfg<2>::kBox : Cfg<1>::kBox, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  if (int32_t rc = encode_tensor_map_2d(&map_q_full, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, p.K, p.R, ldq, BK,
                                        plan.tokens / plan.ctas, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  // kind::i8: D s32 (2) in bits [4,6); A (weight, s8 = 1) in [7,10), B (codes, s8 = 1 or u8 = 0) in [10,13); both
  // K-major; N >> 3 in [17,23) is filled in per tile; M >> 4 in [24,29)
  p.idesc = (2u << 4) | (1u << 7) | ((q_unsigned ? 0u : 1u) << 10) |
            (static_cast<uint32_t>((128 * plan.ctas) >> 4) << 24);
  const int64_t tiles = row_tiles(p, plan.tokens) * ((p.N + plan.tile_rows - 1) / plan.tile_rows);
  if (tiles > 0x7fffffffLL) return fail(LC_ERR_UNSUPPORTED, "grouped_linear: too many tiles");
  const int64_t units = plan.units < tiles ? plan.units : tiles;
  const int cluster = plan.ctas * plan.split;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attrs[2];
  launch_config(&cfg, attrs, static_cast<unsigned>(units * cluster), pair ? smem_bytes<2>() : smem_bytes<1>(), cluster, st);
  const cudaError_t err = cudaLaunchKernelEx(&cfg, pair ? kernel_for<2>(p.out_dtype, p.act) : kernel_for<1>(p.out_dtype, p.act),
                                             map_w, map_q, map_q_full, p);
  if (err != cudaSuccess) return fail(LC_ERR_CUDA, "grouped_linear: %s", cudaGetErrorString(err));
  return check_launch("grouped_linear");
}

static int32_t check_and_launch(const char* what, const void* q, int q_unsigned, int64_t ldq, int64_t R,
                                const int32_t* offsets, int64_t E, const int8_t* w, int64_t ldw, int64_t group_stride,
                                int64_t N, int64_t K, const float* sx, int sx_per_row, const float* zx,
                                const int32_t* wsum, const float* sw, const float* bias, int act, const void* residual,
                                int64_t ldr, void* out, int out_dtype, int64_t ldo, int32_t* status, int variant,
                                int early_weights, bool only_check, cudaStream_t st) {
  const int wait_test = (variant & LC_QLINEAR_WAIT_TEST) ? 1 : 0;
  variant &= ~LC_QLINEAR_WAIT_TEST;
  if (wait_test && !status) return fail(LC_ERR_INVALID_ARG, "%s: the wait test needs a status word", what);
  if (variant < 0 || variant > 6) return fail(LC_ERR_INVALID_ARG, "%s: variant must be between 0 and 6", what);
  if (R < 0 || N < 0 || K <= 0 || E < 1) return fail(LC_ERR_INVALID_ARG, "%s: bad shape", what);
  if (act < LC_ACT_NONE || act > LC_ACT_SWIGLU) return fail(LC_ERR_INVALID_ARG, "%s: unknown activation %d", what, act);
  if (act == LC_ACT_SWIGLU && N % 16)
    return fail(LC_ERR_INVALID_ARG, "%s: swiglu needs weight rows in interleaved blocks of 8 gate and 8 up rows", what);
  if (out_dtype != LC_F32 && out_dtype != LC_BF16 && out_dtype != LC_F16)
    return fail(LC_ERR_UNSUPPORTED, "%s: out_dtype %d not supported", what, out_dtype);
  if (!offsets && E != 1) return fail(LC_ERR_INVALID_ARG, "%s: more than one group needs offsets", what);
  if (E > MAX_GROUPS) return fail(LC_ERR_UNSUPPORTED, "%s: at most %d groups", what, MAX_GROUPS);
  if (R == 0 || N == 0) return LC_OK;
  if (!q || !w || !sx || !sw || !out) return fail(LC_ERR_INVALID_ARG, "%s: null pointer", what);
  if ((zx == nullptr) != (wsum == nullptr)) return fail(LC_ERR_INVALID_ARG, "%s: zx and wsum go together", what);
  const int64_t width = act == LC_ACT_SWIGLU ? N / 2 : N;
  if (ldq < K || ldw < K || ldo < width || (residual && ldr < width) || (E > 1 && group_stride < N * ldw - (ldw - K)))
    return fail(LC_ERR_INVALID_ARG, "%s: leading dimension too small", what);
  if (ldq % 16 || ldw % 16 || (E > 1 && group_stride % 16) || !aligned(q, 16) || !aligned(w, 16))
    return fail(LC_ERR_UNSUPPORTED, "%s: operand rows must start on 16-byte boundaries (pad ldq / ldw to 16)", what);
  // |sum| <= K * 255 * 128 must stay inside int32; rows and columns inside the TMA coordinate range
  if (K > 65536) return fail(LC_ERR_UNSUPPORTED, "%s: K above 65536 could overflow int32", what);
  if (R > 0x7fffffffLL - 512 || N > 0x7fffffffLL - 512) return fail(LC_ERR_UNSUPPORTED, "%s: dimension too large", what);
  if (only_check) return LC_OK;
  Params p = {};
  p.R = R;
  p.N = N;
  p.K = K;
  p.E = static_cast<int>(E);
  p.offsets = offsets;
  p.sx = sx;
  p.sx_per_row = sx_per_row;
  p.zx = zx;
  p.wsum = wsum;
  p.sw = sw;
  p.bias = bias;
  p.act = act;
  p.residual = residual;
  p.ldr = ldr;
  p.out = out;
  p.out_dtype = out_dtype;
  p.ldo = ldo;
  p.status = status;
  p.wait_test = wait_test;
  p.early_weights = early_weights;
  return launch(q, ldq, w, ldw, E > 1 ? group_stride : N * ldw, q_unsigned, p, variant, st);
}

}  // namespace grouped
}  // namespace lc

using namespace lc;

extern "C" int32_t lc_grouped_qlinear_i8(const void* q, int32_t q_unsigned, int64_t ldq, int64_t rows,
                                         const int32_t* offsets, int64_t groups, const int8_t* wq, int64_t ldw,
                                         int64_t group_stride, int64_t N, int64_t K, const float* sx,
                                         int32_t sx_per_row, const float* zx, const int32_t* wsum, const float* sw,
                                         const float* bias, int32_t activation, const void* residual, int64_t ldr,
                                         void* out, int32_t out_dtype, int64_t ldo, int32_t* status, int32_t variant,
                                         void* stream) {
  return grouped::check_and_launch("grouped_qlinear_i8", q, q_unsigned, ldq, rows, offsets, groups, wq, ldw,
                                   group_stride, N, K, sx, sx_per_row, zx, wsum, sw, bias, activation, residual, ldr,
                                   out, out_dtype, ldo, status, variant, 0, false, as_stream(stream));
}

// ---- quantization of the activations and the product as one call --------------------------------
static inline int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }
static inline int64_t pad16(int64_t k) { return (k + 15) / 16 * 16; }

extern "C" int64_t lc_expert_linear_workspace_bytes(int64_t rows, int64_t K) {
  if (rows < 0 || K <= 0) return 0;
  return round256(rows * pad16(K)) + round256(rows * 4);  // codes, one scale per row
}

extern "C" int32_t lc_expert_linear(const void* x, int32_t x_dtype, int64_t x_rows, int64_t ldx,
                                    const int32_t* positions, int64_t top_k, const int32_t* offsets, int64_t groups,
                                    int64_t rows, const int8_t* wq, int64_t ldw, int64_t group_stride, int64_t N,
                                    int64_t K, const float* sw, const float* bias, int32_t activation,
                                    const void* residual, int64_t ldr, void* out, int32_t out_dtype, int64_t ldo,
                                    void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  if (rows < 0 || K <= 0 || N < 0) return fail(LC_ERR_INVALID_ARG, "expert_linear: bad shape");
  if (rows == 0 || N == 0) return LC_OK;
  if (positions ? x_rows * top_k != rows : x_rows != rows)
    return fail(LC_ERR_INVALID_ARG, "expert_linear: the input's rows do not match the number of product rows");
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < lc_expert_linear_workspace_bytes(rows, K))
    return fail(LC_ERR_WORKSPACE, "expert_linear: workspace of %lld bytes (256-byte aligned) required",
                (long long)lc_expert_linear_workspace_bytes(rows, K));
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  float* scale = reinterpret_cast<float*>(codes + round256(rows * pad16(K)));
  auto product = [&](bool only_check) {
    return grouped::check_and_launch("expert_linear", codes, 0, pad16(K), rows, offsets, groups, wq, ldw, group_stride, N, K,
                                     scale, 1, nullptr, nullptr, sw, bias, activation, residual, ldr, out, out_dtype, ldo,
                                     status, 0, 1, only_check, as_stream(stream));
  };
  if (int32_t rc = product(true)) return rc;  // refused before anything is launched
  if (int32_t rc = lc_quantize_tokens(x, x_dtype, x_rows, K, ldx, positions, top_k, rows,
                                      offsets && !positions ? offsets + groups : nullptr,
                                      reinterpret_cast<int8_t*>(codes), pad16(K), scale, stream))
    return rc;
  return product(false);
}
