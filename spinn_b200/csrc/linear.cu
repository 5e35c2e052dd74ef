// linear.cu -- y = act(x w^T + bias) + residual in 16-bit types, accumulated in fp32.
//
// Two kernels, by the number of rows m of x and the size of w (see linear_plan):
//
// * linear_rows_kernel, m <= 32 (single tokens, small decoding batches) with a w that its CTAs
//   cover in about one wave: bound by reading w once.
//   No staging: the fragments of mma.sync come straight from global memory, 16 bytes per lane,
//   with k permuted the same way in both operands so that a lane's 16 contiguous bytes are its
//   fragment.  Any alignment up to 16 rows, aligned rows past them.
//
// * linear_tile_kernel: tcgen05 with TMA-fed swizzled stages.  The rows of w are the MMA's rows
//   (TMEM lanes) and the rows of x its columns, i.e. it computes y^T tiles: a warp that drains
//   its 32 lanes then holds 32 consecutive outputs of one row of y, so residual and y are read
//   and written in whole segments at any alignment, without a transposing stage.  Few rows of x
//   only make the MMA narrower, so the same kernel serves decoding batches, where k is split
//   over a cluster whose CTAs add their partial tiles through distributed shared memory.
//   Operands whose rows are not 16-byte aligned are first copied to an aligned pitch.
#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "cache.h"
#include "internal.h"
#include "launch.h"
#include "ptx.cuh"

namespace spinn {
namespace {

constexpr uint64_t kTimeoutNs = 4000000000ull;  // bounded barrier waits
constexpr uint64_t kDrainNs = 1000000000ull;
constexpr int kRowsMax = 32;  // most rows of x that linear_rows_kernel takes

struct LinearParams {
  const void* x;
  const void* w;
  const void* bias;
  const void* res;
  void* y;
  long long ldx, ldw, ldr, ldy;
  int m, n, k;
  int act;
  int num_kb, tiles_m, tiles_n, num_tiles;
  bool vec;    // rows of x and w on 16-byte boundaries
  bool vec_y;  // rows of y and the residual on 16-byte boundaries
  unsigned* err;
};

template <typename T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (std::is_same<T, __half>::value)
    return __half2float(x);
  else
    return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T round_to(float x) {
  if constexpr (std::is_same<T, __half>::value)
    return __float2half_rn(x);
  else
    return __float2bfloat16_rn(x);
}

// The activations of the fp32 accumulators, chosen once per block of values: a switch per value
// cost a third of a whole launch (4096 x 4096 x 8192 with SiLU: 234 us, 207 us without it).  SiLU
// and the tanh form share v / (1 + e^-z): the tanh form is 0.5 v (1 + tanh u) = v / (1 + e^(-2 u)).
// The fast quotient is off by 2 ulp of fp32, the fast exponential by 2 + 1.17 |z| (some 100 where it leaves
// fp32's range, 2^-16): far below the rounding of y.
//
// GELU by erf: v Phi(v) with Phi(-|v|) = erfc(x) / 2, x = |v| / sqrt(2), and erfc(x) = t e^(Q(t) - x^2),
// t = 1 / (1 + 0.6 x).  Q is a degree-8 Chebyshev fit over t in (0, 1] of the logarithm of the scaled
// function, erfc(x) e^(x^2) / t, in powers of two and with the factor 1/2 in its constant: within
// 5e-6 of the value over [-9, 9] and 1e-5 down to -13, where the value leaves fp32's normal range and becomes
// 0, in a third of erff's instructions (777 x 1024 x 2048 10.5 us, 11.5 with erff).
__device__ __forceinline__ float gelu_erf(float v) {
  const float t = __fdividef(1.0f, fmaf(0.42426407f, fabsf(v), 1.0f));  // 0.6 / sqrt(2)
  float q = 0.268522114f;
  q = fmaf(q, t, -1.28184319f);
  q = fmaf(q, t, 2.30145049f);
  q = fmaf(q, t, -1.66434383f);
  q = fmaf(q, t, 0.144887894f);
  q = fmaf(q, t, -0.116924897f);
  q = fmaf(q, t, 0.468497783f);
  q = fmaf(q, t, 1.44246602f);
  q = fmaf(q, t, -2.56271243f);
  q = fmaf(-0.72134752f * v, v, q);  // - x^2 log2(e)
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(q));
  const float h = t * e;
  return v * (v < 0.0f ? h : 1.0f - h);
}
__device__ __forceinline__ float sigmoid_times(float v, float z) { return __fdividef(v, 1.0f + __expf(-z)); }
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
  switch (act) {
    case 1:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];
      break;
    case 3:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = sigmoid_times(v[i], v[i]);
      break;
    case SPINN_CUDA_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = gelu_erf(v[i]);
      break;
    case SPINN_CUDA_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i)  // 2 sqrt(2 / pi) (v + 0.044715 v^3)
        v[i] = sigmoid_times(v[i], 1.5957691216057308f * (v[i] + 0.044715f * v[i] * v[i] * v[i]));
      break;
    default:
      break;
  }
}

// ------------------------------------------------------------------ few rows
template <typename T>
__device__ __forceinline__ void mma_rows(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Elements k .. k + 7 of a row (zeros past `end`; nothing is read where !live).  Operands are read
// by ordinary loads: a kernel that starts while its predecessor still writes them may not take the
// read-only path.
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* row, bool live, int k, int end) {
  uint4 r = make_uint4(0, 0, 0, 0);
  if (!live || k >= end) return r;
  if (VEC && k + 8 <= end) return *reinterpret_cast<const uint4*>(row + k);
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = k + i < end ? row[k + i] : 0;
  r.x = h[0] | h[1] << 16;
  r.y = h[2] | h[3] << 16;
  r.z = h[4] | h[5] << 16;
  r.w = h[6] | h[7] << 16;
  return r;
}

constexpr int kRowWarps = 8;

constexpr int row_ctas(int nt) { return nt == 1 ? 3 : 2; }  // at a time on an SM

// CTA: 16 rows of w, all rows of x (NT blocks of 8); its warps take interleaved chunks of k and are
// summed in order through shared memory.  Asking for the next chunk before this one is used gained
// 13% on 1 x 4096 x 4096 and cost more elsewhere (8 x 4096 x 11008 19.6 -> 21.7 us: fewer CTAs at a time).
template <typename T, int NT, bool VEC>
__global__ void __launch_bounds__(kRowWarps * 32, row_ctas(NT)) linear_rows_kernel(const LinearParams p) {
  __shared__ float part[kRowWarps][NT * 8][16];
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * 16, r = lane >> 2, q = lane & 3;
  const uint16_t* w0 = static_cast<const uint16_t*>(p.w) + (long long)(n0 + r) * p.ldw;
  const uint16_t* w1 = w0 + 8 * p.ldw;
  const bool live0 = n0 + r < p.n, live1 = n0 + r + 8 < p.n;
  float acc[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.0f;
  constexpr int U = NT == 4 ? 2 : 4;  // 32-element steps in flight: what the registers hold
  for (int k0 = warp * 32 * U; k0 < p.k; k0 += kRowWarps * 32 * U) {
    uint4 a[U], b[U], x[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * 32 + q * 8;
      a[u] = load8<VEC>(w0, live0, k, p.k);
      b[u] = load8<VEC>(w1, live1, k, p.k);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        x[u][t] = load8<VEC>(static_cast<const uint16_t*>(p.x) + (t * 8 + r) * p.ldx, t * 8 + r < p.m, k, p.k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        mma_rows<T>(acc[t], a[u].x, b[u].x, a[u].y, b[u].y, x[u][t].x, x[u][t].y);
        mma_rows<T>(acc[t], a[u].z, b[u].z, a[u].w, b[u].w, x[u][t].z, x[u][t].w);
      }
  }
  // accumulator: rows r and r + 8 of w, tokens 2 q and 2 q + 1
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    part[warp][t * 8 + 2 * q][r] = acc[t][0];
    part[warp][t * 8 + 2 * q + 1][r] = acc[t][1];
    part[warp][t * 8 + 2 * q][r + 8] = acc[t][2];
    part[warp][t * 8 + 2 * q + 1][r + 8] = acc[t][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 8 * 16; i += kRowWarps * 32) {
    const int row = i >> 4, n = n0 + (i & 15);
    if (row >= p.m || n >= p.n) continue;
    float v[1] = {0.0f};
#pragma unroll
    for (int s = 0; s < kRowWarps; ++s) v[0] += part[s][row][i & 15];
    if (p.bias) v[0] += to_float(static_cast<const T*>(p.bias)[n]);
    activate(v, p.act);
    if (p.res) v[0] += to_float(static_cast<const T*>(p.res)[row * p.ldr + n]);
    static_cast<T*>(p.y)[row * p.ldy + n] = round_to<T>(v[0]);
  }
}

// ------------------------------------------------------------------ rows to an aligned pitch
// dst[r][0 .. pitch) = src[r][0 .. k), zeros behind.  One launch for both operands.
struct PitchParams {
  const uint16_t* src[2];
  uint16_t* dst[2];
  long long ld[2];
  int rows[2];
  int k, pitch;
};
// A thread makes 16-byte pieces out of the two aligned 16-byte words that hold them: a word is
// read only when it holds an element of the row, so nothing outside the rows' own words is touched.
__global__ void __launch_bounds__(256) pitch_kernel(const PitchParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const int o = blockIdx.y, pieces = p.pitch >> 3, lane = threadIdx.x & 31;
  constexpr int U = 4;
  for (int r = blockIdx.x * 8 + (threadIdx.x >> 5); r < p.rows[o]; r += gridDim.x * 8) {  // a row to a warp
    const uint16_t* src = p.src[o] + r * p.ld[o];
    uint4* dst = reinterpret_cast<uint4*>(p.dst[o] + (long long)r * p.pitch);
    const int shift = (int)(reinterpret_cast<uintptr_t>(src) & 15) >> 1;  // elements; the same for all of the row
    for (int i0 = lane; i0 < pieces; i0 += 32 * U) {
      uint4 lo[U], hi[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * 32;
        lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
        if (i < pieces) {
          const uint4* word = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(src + i * 8) & ~uintptr_t(15));
          lo[u] = *word;
          if (shift + min(8, p.k - i * 8) > 8) hi[u] = word[1];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * 32;
        if (i >= pieces) continue;
        // the 16 bytes at `shift` elements of lo : hi
        const uint32_t w[8] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w, hi[u].x, hi[u].y, hi[u].z, hi[u].w};
        const int whole = shift >> 1;
        uint32_t d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a = 0, b = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q == whole) {
              a = w[j + q];
              b = j + q + 1 < 8 ? w[j + q + 1] : 0;
            }
          d[j] = shift & 1 ? __funnelshift_r(a, b, 16) : a;
          const int left = p.k - i * 8 - 2 * j;  // elements of the row from this word on
          d[j] = left >= 2 ? d[j] : left == 1 ? d[j] & 0xffffu : 0u;
        }
        dst[i] = make_uint4(d[0], d[1], d[2], d[3]);
      }
    }
  }
}

// ------------------------------------------------------------------ tiles on tcgen05
// kind::f16: D fp32 [4,6) = 1, A and B type 0 fp16 / 1 bf16 at [7,10) and [10,13), both K-major.
template <typename T>
__host__ __device__ constexpr uint32_t make_idesc_16(uint32_t M, uint32_t N) {
  constexpr uint32_t f = std::is_same<T, __half>::value ? 0 : 1;
  return (1u << 4) | (f << 7) | (f << 10) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// One lane of a converged warp.  The compiler keeps the operands of what it issues in uniform
// registers; under `lane == 0` an MMA took 64 clocks to issue, longer than it runs with up to 128
// columns (1024 x 1024 x 1024: 7.8 us so, 7.0 with this).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ bool warp_wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, kTimeoutNs));
}
__device__ __forceinline__ bool warp_abort(volatile int* abort) { return __any_sync(0xffffffffu, *abort != 0); }

// Barrier of the four epilogue warps of one group.
__device__ __forceinline__ void group_sync(int group) {
  asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory");
}
// Waits for `bar` in the four warps of one group, which go on together or give up together: by itself
// a warp may see another's abort just before the barrier completes, and leave its neighbours in the
// group_sync that follows.  The vote costs a barrier per tile.
__device__ __forceinline__ bool group_wait(uint64_t* bar, uint32_t parity, volatile int* abort, uint64_t timeout_ns,
                                           int group) {
  const uint32_t mine = __all_sync(0xffffffffu, mbar_wait_backoff(bar, parity, abort, timeout_ns));
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(mine), "r"(group + 1)
      : "memory");
  return all != 0;
}
template <typename T>
union Pack {
  uint4 u;
  T t[8];
  __device__ Pack() {}
};

template <typename T>
union Pair {
  uint32_t u;
  T t[2];
  __device__ Pair() {}
};

template <typename T>
__device__ __forceinline__ uint32_t round_pair(float a, float b) {  // a in the low half
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

constexpr int kTileThreads = 384;  // producer, MMA, TMEM and a spare warp, eight epilogue warps

// BN: rows of x of a tile.  PAIR 2: a CTA pair works on 256 rows of w with one cta_group::2 MMA
// stream, each CTA holding its 128 rows of w and half of the rows of x.  SPL: the CTAs of a
// cluster share one tile and split its k.
//
// A stage holds 128 elements of k, two 128-byte swizzle spans: with one span per stage the
// barrier handoffs showed (4096 x 4096 x 8192 without activation: 207 us, 178 us with two).
template <int BN_, int PAIR_, bool SPL_>
struct LinCfg {
  static constexpr int BN = BN_, PAIR = PAIR_;
  static constexpr bool SPL = SPL_;
  static constexpr int BK = 128, SPAN = 64;  // elements of k per stage and per swizzle span
  static constexpr int A_SPAN = 128 * 128, B_SPAN = BN / PAIR * 128;
  static constexpr int A_STAGE = 2 * A_SPAN, B_STAGE = 2 * B_SPAN, STAGE = A_STAGE + B_STAGE;
  static constexpr int PART = SPL ? BN * 128 * 4 : 0;  // partial sums received from the cluster
  // The epilogue's staging, [16 rows of x][128 rows of w] per group of four warps: y leaves in
  // 16-byte pieces of 256-byte row segments.
  static constexpr int STG_PITCH = 128 + 4, STG = SPL ? 0 : 2 * 16 * STG_PITCH * 4;
  static constexpr int FIT = (222 * 1024 - PART - STG) / STAGE;
  static constexpr int STAGES = FIT > 6 ? 6 : FIT;
  static constexpr int NACC = SPL ? 1 : 2;          // accumulators: the epilogue drains one while the other fills
  static constexpr int COLS = NACC * BN < 32 ? 32 : NACC * BN;
  static constexpr int SMEM = STAGES * STAGE + PART + STG + 512 + 1024;
  static_assert(COLS <= 512, "TMEM");
  static_assert(STAGES >= 2, "pipeline needs two stages");
};

template <typename T, typename C>
__global__ void __launch_bounds__(kTileThreads, 1)
    linear_tile_kernel(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapX,
                       const LinearParams p) {
  constexpr int BN = C::BN, PAIR = C::PAIR, STAGES = C::STAGES, NACC = C::NACC;
  constexpr bool SPL = C::SPL;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * C::A_STAGE;
  float* part = reinterpret_cast<float*>(smem + STAGES * C::STAGE);  // [rank][slot][128 rows of w]
  float* staging = reinterpret_cast<float*>(smem + STAGES * C::STAGE + C::PART);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE + C::PART + C::STG);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + NACC;
  uint64_t* drain = tempty + NACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = PAIR == 2 || SPL ? cluster_ctarank() : 0;
  const uint32_t side = PAIR == 2 ? crank & 1 : 0, leader = crank - side;  // place in the pair, its leader
  const uint32_t rank = SPL ? crank / PAIR : 0;                              // place in the split
  const uint32_t splits = SPL ? cluster_size() / PAIR : 1;
  const int unit0 = SPL ? blockIdx.x / (splits * PAIR) : blockIdx.x / PAIR;
  const int step = SPL ? p.num_tiles : gridDim.x / PAIR;  // a cluster has one tile
  const int kb0 = SPL ? (int)((long long)p.num_kb * rank / splits) : 0;
  const int kb1 = SPL ? (int)((long long)p.num_kb * (rank + 1) / splits) : p.num_kb;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < NACC; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 8 * PAIR);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&mapW);
    prefetch_tmap(&mapX);
  }
  if (warp == 2) {
    if constexpr (PAIR == 2) {
      tmem_alloc_pair(tmem_slot, C::COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, C::COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR == 2) cluster_sync();  // the peer's barriers are initialised before use
  if constexpr (SPL && PAIR == 1) cluster_arrive();  // waited for before the first store to another CTA
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_launch_dependents();
  griddep_wait();

  // Tile order: blocks of eight w tiles walk the x tiles, so that the CTAs working at the same
  // time share both operands in L2.
  auto decode = [&](int tile, int* tm, int* tn) {
    const int per = 8 * p.tiles_m, g = tile / per, r = tile - g * per;
    const int gn = min(8, p.tiles_n - g * 8);
    *tm = r / gn;
    *tn = g * 8 + (r - *tm * gn);
  };

  if (warp == 0) {
    // ---- producer
    int s = 0;
    uint32_t ph = 0, armed = 0, armed_ph = 0;
    for (int t = unit0; t < p.num_tiles && !warp_abort(abort_flag); t += step) {
      int tm, tn;
      decode(t, &tm, &tn);
      const int w_row = (tn * PAIR + side) * 128;
      const int x_row = tm * BN + side * (BN / 2);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!warp_wait_bar(&empty[s], ph ^ 1, abort_flag)) break;
        if (lane == 0) {
          if (side == 0) {
            mbar_arrive_expect_tx(&full[s], C::STAGE * PAIR);
            armed |= 1u << s;
            armed_ph = (armed_ph & ~(1u << s)) | (ph << s);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // the second span may lie wholly past k: it reads as zeros
            uint8_t *a = sA + s * C::A_STAGE + h * C::A_SPAN, *b = sB + s * C::B_STAGE + h * C::B_SPAN;
            const int k = kb * C::BK + h * C::SPAN;
            if constexpr (PAIR == 2) {
              const uint32_t bar = mapa_shared(smem_u32(&full[s]), leader);
              tma_load_2d_pair(&mapW, bar, a, k, w_row);
              tma_load_2d_pair(&mapX, bar, b, k, x_row);
            } else {
              tma_load_2d(&mapW, &full[s], a, k, w_row);
              tma_load_2d(&mapX, &full[s], b, k, x_row);
            }
          }
        }
        __syncwarp();
        if (++s == STAGES) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    if (warp_abort(abort_flag) && lane == 0) {
      // copies in flight land before the shared memory goes away
      volatile int dummy = 0;
      for (int i = 0; i < STAGES; ++i)
        if (armed & (1u << i)) mbar_wait(&full[i], (armed_ph >> i) & 1, &dummy, kDrainNs);
    }
    __syncwarp();
  } else if (warp == 1 && side == 0) {
    // ---- MMA issuer (the pair's leader)
    constexpr uint32_t idesc = make_idesc_16<T>(128 * PAIR, BN);
    const uint64_t adesc = make_smem_desc(smem_u32(sA), 16, 1024, kSw128);
    const uint64_t bdesc = make_smem_desc(smem_u32(sB), 16, 1024, kSw128);
    int s = 0, it = 0;
    uint32_t ph = 0;
    bool issued = false;
    for (int t = unit0; t < p.num_tiles && !warp_abort(abort_flag); t += step, ++it) {
      const int b = it % NACC;
      if (!warp_wait_bar(&tempty[b], ((it / NACC) & 1) ^ 1, abort_flag)) break;
      tc_fence_after();
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!warp_wait_bar(&full[s], ph, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t a = adesc + ((s * C::A_STAGE) >> 4), x = bdesc + ((s * C::B_STAGE) >> 4);
#pragma unroll
          for (int j = 0; j < C::BK / 16; ++j) {
            const uint32_t acc = kb != kb0 || j != 0 ? 1u : 0u;
            const uint64_t aj = a + (j >> 2) * (C::A_SPAN >> 4) + 2 * (j & 3);
            const uint64_t xj = x + (j >> 2) * (C::B_SPAN >> 4) + 2 * (j & 3);
            if constexpr (PAIR == 2)
              umma_f16_pair(tmem + b * BN, aj, xj, idesc, acc);
            else
              umma_f16(tmem + b * BN, aj, xj, idesc, acc);
          }
          if constexpr (PAIR == 2) {
            umma_commit_pair(mapa_shared(smem_u32(&empty[s]), leader));
            umma_commit_pair(mapa_shared(smem_u32(&empty[s]), leader + 1));
          } else {
            umma_commit(&empty[s]);
          }
        }
        __syncwarp();
        issued = true;
        if (++s == STAGES) {
          s = 0;
          ph ^= 1;
        }
      }
      if (!ok) break;
      if (elect_one()) {
        if constexpr (PAIR == 2) {
          umma_commit_pair(mapa_shared(smem_u32(&tfull[b]), leader));
          umma_commit_pair(mapa_shared(smem_u32(&tfull[b]), leader + 1));
        } else {
          umma_commit(&tfull[b]);
        }
      }
      __syncwarp();
    }
    if (warp_abort(abort_flag) && issued && elect_one()) {  // the lane that issued
      volatile int dummy = 0;
      if constexpr (PAIR == 2)
        umma_commit_pair(mapa_shared(smem_u32(drain), leader));
      else
        umma_commit(drain);
      mbar_wait(drain, 0, &dummy, kDrainNs);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ---- epilogue: warp pairs share a TMEM lane quarter and alternate over its column chunks
    constexpr int CW = 16;  // columns (rows of x) per step
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    if constexpr (SPL && PAIR == 1) cluster_wait();  // the cluster's other CTAs run: they may be written to
    int it = 0;
    for (int t = unit0; t < p.num_tiles; t += step, ++it) {
      int tm, tn;
      decode(t, &tm, &tn);
      const int n = (tn * PAIR + side) * 128 + quarter * 32 + lane;
      const int m0 = tm * BN;
      const float bias = !SPL && p.bias && n < p.n ? to_float(static_cast<const T*>(p.bias)[n]) : 0.0f;
      const int b = it % NACC;
      bool ok;
      if constexpr (SPL)  // no barrier of the group follows: a warp that gives up goes to the cluster's like the others
        ok = __all_sync(0xffffffffu, mbar_wait_backoff(&tfull[b], 0, abort_flag, kTimeoutNs));
      else
        ok = group_wait(&tfull[b], (it / NACC) & 1, abort_flag, kTimeoutNs, half);
      if (!ok) break;
      tc_fence_after();
      for (int c = half * CW; c < BN && m0 + c < p.m; c += 2 * CW) {
        uint32_t r[CW];
        tmem_ld_32x32b_x16(tmem + b * BN + c + ((uint32_t)(quarter * 32) << 16), r);
        const int rows = min(CW, p.m - m0 - c);
        if constexpr (SPL) {
          // rows of x in groups of four, group g finished by rank g % splits at slot g / splits
          tmem_ld_wait();
          uint4* own = reinterpret_cast<uint4*>(part) + rank * (BN / 4 / splits) * 128 + quarter * 32 + lane;
          const uint32_t mine = smem_u32(own);
#pragma unroll
          for (int i = 0; i < CW; i += 4) {
            const uint32_t g = (c + i) >> 2, to = g & (splits - 1), slot = g / splits;
            if (i >= rows) continue;
            if (to == rank)  // no way through the cluster (256 x 4096 x 4096: 17.7 -> 17.2 us)
              own[slot * 128] = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
            else
              st_cluster_v4(mapa_shared(mine + slot * 2048, to * PAIR + side), r[i], r[i + 1], r[i + 2], r[i + 3]);
          }
        } else {
          // this thread's part of the output: eight consecutive n of two rows of x
          const int on = (tn * PAIR + side) * 128 + (lane & 15) * 8;
          const int orow = quarter * 4 + (lane >> 4);
          uint4 res[2];
          if (p.res && p.vec_y && on + 8 <= p.n) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (orow + 2 * j < rows)
                res[j] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.res) +
                                                         (long long)(m0 + c + orow + 2 * j) * p.ldr + on);
          }
          // the same for rows off alignment, as they are stored below
          const int n0 = (tn * PAIR + side) * 128, width = min(128, p.n - n0);
          T loose[4][3][2];
          if (p.res && !p.vec_y) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int row = quarter * 4 + q;
              const T* extra = static_cast<const T*>(p.res) + (long long)(m0 + c + row) * p.ldr + n0;
              const int odd = ((uintptr_t)(static_cast<T*>(p.y) + (long long)(m0 + c + row) * p.ldy + n0) >> 1) & 1;
#pragma unroll
              for (int j = 0; j < 3; ++j) {
                const int e = 2 * (lane + 32 * j) - odd;
                const bool live = row < rows && !(j == 2 && e > 127);
                if (live && e >= 0 && e < width) loose[q][j][0] = extra[e];
                if (live && e + 1 >= 0 && e + 1 < width) loose[q][j][1] = extra[e + 1];
              }
            }
          }
          tmem_ld_wait();
          float v[CW];
#pragma unroll
          for (int i = 0; i < CW; ++i) v[i] = __uint_as_float(r[i]) + bias;
          activate(v, p.act);
          float* stage = staging + half * 16 * C::STG_PITCH;
          group_sync(half);  // the previous step's values have been read
#pragma unroll
          for (int i = 0; i < CW; ++i) stage[i * C::STG_PITCH + quarter * 32 + lane] = v[i];
          group_sync(half);
          if (p.vec_y) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int row = orow + 2 * j;
              if (row >= rows || on >= p.n) continue;
              const float4* src = reinterpret_cast<const float4*>(stage + row * C::STG_PITCH + (lane & 15) * 8);
              const float4 lo = src[0], hi = src[1];
              float o[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
              T* dst = static_cast<T*>(p.y) + (long long)(m0 + c + row) * p.ldy + on;
              if (on + 8 <= p.n) {
                Pack<T> x;
                if (p.res) {
                  x.u = res[j];
#pragma unroll
                  for (int i = 0; i < 8; ++i) o[i] += to_float(x.t[i]);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) x.t[i] = round_to<T>(o[i]);
                *reinterpret_cast<uint4*>(dst) = x.u;
              } else {
                const T* extra = static_cast<const T*>(p.res) + (p.res ? (long long)(m0 + c + row) * p.ldr + on : 0);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  if (on + i < p.n) dst[i] = round_to<T>(p.res ? o[i] + to_float(extra[i]) : o[i]);
              }
            }
          } else {
            // rows off alignment: 4-byte words at the row's own parity, its ends in single elements
            for (int q = 0; q < 4; ++q) {
              const int row = quarter * 4 + q;
              if (row >= rows) break;
              T* dst = static_cast<T*>(p.y) + (long long)(m0 + c + row) * p.ldy + n0;
              const float* src = stage + row * C::STG_PITCH;
              const int odd = ((uintptr_t)dst >> 1) & 1;
#pragma unroll
              for (int j = 0; j < 3; ++j) {
                const int e = 2 * (lane + 32 * j) - odd;
                if (e >= width || (j == 2 && e > 127)) continue;
                const bool first = e >= 0, second = e + 1 < width;
                const float o0 = first ? src[e] : 0.0f, o1 = second ? src[e + 1] : 0.0f;
                Pair<T> x;
                x.t[0] = round_to<T>(p.res ? o0 + to_float(loose[q][j][0]) : o0);
                x.t[1] = round_to<T>(p.res ? o1 + to_float(loose[q][j][1]) : o1);
                if (first && second)
                  *reinterpret_cast<uint32_t*>(dst + e) = x.u;
                else if (first)
                  dst[e] = x.t[0];
                else
                  dst[e + 1] = x.t[1];
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR == 2)
          mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[b]), leader));
        else
          mbar_arrive(&tempty[b]);
      }
    }
  }

  if constexpr (SPL) {
    // Every CTA sends its partial sums to the CTAs that finish them, which add them in rank order
    // out of their own shared memory.  A thread finishes two n of every sixth group of four rows;
    // what it needs from global memory is asked for before the barrier.
    int tm, tn;
    decode(unit0, &tm, &tn);
    const int rows = min(BN, p.m - tm * BN), groups = (rows + 3) >> 2;
    const int mine = (groups - (int)rank + (int)splits - 1) / (int)splits;  // groups rank, rank + splits, ...
    const int n = (tn * PAIR + side) * 128 + 2 * (threadIdx.x & 63);
    const bool one = n < p.n, two = n + 1 < p.n;
    const float bias0 = p.bias && one ? to_float(static_cast<const T*>(p.bias)[n]) : 0.0f;
    const float bias1 = p.bias && two ? to_float(static_cast<const T*>(p.bias)[n + 1]) : 0.0f;
    const bool words = two && ((uintptr_t)p.y & 3) == 0 && (p.ldy & 1) == 0;  // n is even
    const bool res_words = two && ((uintptr_t)p.res & 3) == 0 && (p.ldr & 1) == 0;
    const float4* sums = reinterpret_cast<const float4*>(part);
    const int plane = BN / 4 / (int)splits * 128;
    bool joined = false;
    for (int g = threadIdx.x >> 6; g < mine || !joined; g += kTileThreads / 64) {
      const int row = (g * (int)splits + (int)rank) * 4, m = tm * BN + row;
      float res[4][2] = {};
      if (p.res && one && g < mine) {
        const T* src = static_cast<const T*>(p.res) + (long long)m * p.ldr + n;
#pragma unroll
        for (int e = 0; e < 4; ++e, src += p.ldr) {
          if (row + e >= rows) continue;
          if (res_words) {
            Pair<T> x;
            x.u = *reinterpret_cast<const uint32_t*>(src);
            res[e][0] = to_float(x.t[0]);
            res[e][1] = to_float(x.t[1]);
          } else {
            res[e][0] = to_float(src[0]);
            if (two) res[e][1] = to_float(src[1]);
          }
        }
      }
      if (!joined) {
        if (PAIR == 1 && warp < 4) cluster_wait();
        cluster_arrive();
        cluster_wait();
        joined = true;
      }
      if (g >= mine || !one) continue;
      float v[8] = {};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j >= (int)splits) break;
        const float4 a = sums[j * plane + g * 128 + 2 * (threadIdx.x & 63)];
        const float4 b = sums[j * plane + g * 128 + 2 * (threadIdx.x & 63) + 1];
        v[0] += a.x;
        v[1] += b.x;
        v[2] += a.y;
        v[3] += b.y;
        v[4] += a.z;
        v[5] += b.z;
        v[6] += a.w;
        v[7] += b.w;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += e & 1 ? bias1 : bias0;
      activate(v, p.act);
      if (p.res)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += res[e >> 1][e & 1];
      T* dst = static_cast<T*>(p.y) + (long long)m * p.ldy + n;
#pragma unroll
      for (int e = 0; e < 4; ++e, dst += p.ldy) {
        if (row + e >= rows) continue;
        if (words) {
          *reinterpret_cast<uint32_t*>(dst) = round_pair<T>(v[2 * e], v[2 * e + 1]);
        } else {
          dst[0] = round_to<T>(v[2 * e]);
          if (two) dst[1] = round_to<T>(v[2 * e + 1]);
        }
      }
    }
  }
  __syncthreads();
  if constexpr (PAIR == 2) cluster_sync();  // no CTA leaves while its peer may use its memory
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.err, kWaitExpired);
  if (warp == 2) {
    tc_fence_after();
    if constexpr (PAIR == 2)
      tmem_dealloc_pair(tmem, C::COLS);
    else
      tmem_dealloc(tmem, C::COLS);
  }
}

// Four warps of a group wait for a barrier that a fifth completes after `arrive_ns`; the first gives up
// after `limit_ns`, by an abort flag of its own.  Bit w of the result: warp w goes on.
__device__ unsigned g_group_went_on;
__global__ void __launch_bounds__(160) group_wait_selftest_kernel(uint64_t arrive_ns, uint64_t limit_ns) {
  __shared__ uint64_t bar;
  __shared__ int abort_flag[2];
  __shared__ unsigned went_on;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    fence_mbar_init();
    abort_flag[0] = abort_flag[1] = 0;
    went_on = 0;
  }
  __syncthreads();
  if (warp == 4) {
    if (lane == 0) {
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < arrive_ns) __nanosleep(1000);
      mbar_arrive(&bar);
    }
  } else {
    const bool on = group_wait(&bar, 0, &abort_flag[warp != 0], warp ? kTimeoutNs : limit_ns, 0);
    if (on && lane == 0) atomicOr(&went_on, 1u << warp);
  }
  __syncthreads();
  if (threadIdx.x == 0) g_group_went_on = went_on;
}

// ------------------------------------------------------------------ host
struct LinearPlan {
  int bn = 0, pair = 1, split = 1;  // bn 0: linear_rows_kernel
  bool copy_x = false, copy_w = false;
  size_t x_bytes = 0, w_bytes = 0;
};

bool tma_rows(const void* p, long long ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }

LinearPlan linear_plan(const LinearParams& p, int sms) {
  LinearPlan pl;
  const size_t pitch = ((size_t)p.k + 7) / 8 * 8 * 2;
  pl.copy_x = !tma_rows(p.x, p.ldx);
  pl.copy_w = !tma_rows(p.w, p.ldw);
  pl.x_bytes = pl.copy_x ? (pitch * p.m + 255) / 256 * 256 : 0;
  pl.w_bytes = pl.copy_w ? (pitch * p.n + 255) / 256 * 256 : 0;
  // Shape by estimated clocks, fitted to a sweep of every shape over 41 sizes (device time in a
  // captured queue; what it picks takes 0.5% longer than the best, geometric mean).  A stage of 128
  // k takes 600, 650 and 870 clocks on a single CTA of 32, 64 and 128 columns -- the issue of its
  // eight MMAs and the barriers around them, then the operands' way into shared memory -- and 800
  // and 1,200 on pairs (650 split).  Around the stages lie the launch and first loads (2,600; 900
  // more for a cluster), and the last tile's epilogue.  Splitting k pays when there are few tiles:
  // it adds the exchange of the partial sums.
  const int kb = (p.k + 127) / 128;
  double best = 0;
  auto consider = [&](int bn, int pair, int split) {
    const long long tiles = (long long)((p.m + bn - 1) / bn) * ((p.n + 128 * pair - 1) / (128 * pair));
    const long long waves = (tiles * pair * split + sms - 1) / sms;
    if (split > 1 && (waves > 1 || kb < 2 * split)) return;
    // clusters that the GPCs of 148 SMs hold at once
    if (split > 1 && (split * pair == 8 ? tiles > 15 : split * pair == 4 && tiles > 34)) return;
    const double stage = pair == 1 ? (bn == 32 ? 600.0 : bn == 64 ? 650.0 : 870.0)
                                   : bn == 256 ? 1200.0 : split > 1 ? 650.0 : 800.0;
    double clocks = 2600.0 + (pair * split > 1 ? 900.0 : 0.0) + (double)waves * ((kb + split - 1) / split) * stage;
    clocks += bn * 30.0 + 300.0;
    if (split > 1) clocks += 1100.0 + bn * 26.0 / split + (pair == 2 ? 1000.0 : 0.0);
    if (pl.bn == 0 || clocks < best) {
      pl.bn = bn;
      pl.pair = pair;
      pl.split = split;
      best = clocks;
    }
  };
  for (int split = 1; split <= 8; split *= 2)
    for (int bn = 32; bn <= 128; bn *= 2) consider(bn, 1, split);
  for (int split = 1; split <= 4; split *= 2) consider(128, 2, split);
  consider(256, 2, 1);
  if (p.m > (p.vec ? kRowsMax : 16)) return pl;
  // The kernel for few rows, or these tiles?  Tiles read w at HBM's bandwidth at best, after 9,500
  // clocks of start and finish; rows off alignment cost a copy of them first.  The other kernel
  // takes waves of CTAs through k, 1,024 elements at a time: longer the more of them share an SM,
  // and some three times as long off alignment.  Fitted to 1, 8, 16 and 32 rows of 28 sizes (us,
  // few-rows kernel : tiles; 1 x 1024 x 4096 3.0 : 5.6, 8 x 4096 x 1000 4.9 : 5.8, 8 x 4096 x 4096
  // 10.0 : 10.4, 8 x 4096 x 8192 18.7 : 15.3, 16 x 4096 x 4096 10.7 : 10.6, 16 x 11008 x 4096 22.5 :
  // 19.3, 16 x 4096 x 32000 61.1 : 45.1, 32 x 1024 x 1024 3.7 : 5.0, 32 x 2048 x 2048 6.6 : 5.9; off
  // alignment 1 x 1001 x 1000 6.2 : 7.3, 8 x 4095 x 4096 31.1 : 21.9; past 16 rows 10 : 7.5).
  const double hbm = 5.9e-4;  // clocks for an element read, or for a byte copied
  const double tiles = std::max(best, 9500.0 + hbm * p.n * p.k) +
                       (pl.copy_x || pl.copy_w ? 3500.0 + hbm * (double)(pl.x_bytes + pl.w_bytes) : 0.0);
  const int nt = p.m <= 8 ? 1 : p.m <= 16 ? 2 : 4;
  const long long ctas = (p.n + 15) / 16, at_once = (long long)row_ctas(nt) * sms;
  const double waves = (double)((ctas + at_once - 1) / at_once);
  const double share = std::min((double)row_ctas(nt), (double)ctas / sms);
  const double steps = p.k >= 1024 ? p.k / 1024.0 : 0.5 + p.k / 2048.0;
  double step = (nt == 1 ? 1500.0 : nt == 2 ? 2200.0 : 3600.0) + 1100.0 * share;
  if (!p.vec) step *= 3.4;
  if (2600.0 + waves * (1000.0 + steps * step) <= tiles) return LinearPlan();
  return pl;
}

template <typename T, typename C>
int launch_tiles(const LinearParams& p0, const LinearPlan& pl, const void* x, long long ldx, const void* w, long long ldw,
                 int sms, cudaStream_t st) {
  LinearParams p = p0;
  p.num_kb = (p.k + C::BK - 1) / C::BK;
  p.tiles_m = (p.m + C::BN - 1) / C::BN;
  p.tiles_n = (p.n + 128 * C::PAIR - 1) / (128 * C::PAIR);
  const long long tiles = (long long)p.tiles_m * p.tiles_n;
  SPINN_CHECK_ARG(tiles < (1ll << 30), "linear: too many tiles");
  p.num_tiles = (int)tiles;
  CUtensorMap mw, mx;
  const bool half = std::is_same<T, __half>::value;
  int rc = encode_tiled_2d_16(&mw, w, p.k, p.n, (uint64_t)ldw * 2, C::SPAN, 128, half);
  if (rc) return rc;
  rc = encode_tiled_2d_16(&mx, x, p.k, p.m, (uint64_t)ldx * 2, C::SPAN, C::BN / C::PAIR, half);
  if (rc) return rc;
  auto* kernel = linear_tile_kernel<T, C>;
  SPINN_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
  const int cluster = C::SPL ? pl.split * C::PAIR : C::PAIR;
  const int grid = C::SPL ? p.num_tiles * cluster : std::min(p.num_tiles, sms / C::PAIR) * C::PAIR;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  SPINN_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, mw, mx, p));
  return 0;
}

template <typename T>
int linear_launch(const LinearParams& p, const LinearPlan& pl, void* ws, int sms, cudaStream_t st) {
  if (pl.bn == 0) {
    const dim3 grid((p.n + 15) / 16);
    const int threads = kRowWarps * 32;
    if (p.m <= 8)
      return p.vec ? launch_dependent(linear_rows_kernel<T, 1, true>, grid, threads, 0, st, p)
                   : launch_dependent(linear_rows_kernel<T, 1, false>, grid, threads, 0, st, p);
    if (p.m > 16) return launch_dependent(linear_rows_kernel<T, 4, true>, grid, threads, 0, st, p);
    return p.vec ? launch_dependent(linear_rows_kernel<T, 2, true>, grid, threads, 0, st, p)
                 : launch_dependent(linear_rows_kernel<T, 2, false>, grid, threads, 0, st, p);
  }
  const void *x = p.x, *w = p.w;
  long long ldx = p.ldx, ldw = p.ldw;
  if (pl.copy_x || pl.copy_w) {
    PitchParams c = {};
    c.k = p.k;
    c.pitch = (p.k + 7) / 8 * 8;
    if (pl.copy_x) {
      c.src[0] = static_cast<const uint16_t*>(p.x);
      c.dst[0] = static_cast<uint16_t*>(ws);
      c.ld[0] = p.ldx;
      c.rows[0] = p.m;
      x = ws;
      ldx = c.pitch;
    }
    if (pl.copy_w) {
      c.src[1] = static_cast<const uint16_t*>(p.w);
      c.dst[1] = reinterpret_cast<uint16_t*>(static_cast<char*>(ws) + pl.x_bytes);
      c.ld[1] = p.ldw;
      c.rows[1] = p.n;
      w = c.dst[1];
      ldw = c.pitch;
    }
    const int rc = launch_dependent(pitch_kernel, dim3((unsigned)std::min((std::max(c.rows[0], c.rows[1]) + 7) / 8, sms * 8), 2), 256, 0, st, c);
    if (rc) return rc;
  }
  const bool spl = pl.split > 1;
  if (pl.pair == 2 && pl.bn == 256) return launch_tiles<T, LinCfg<256, 2, false>>(p, pl, x, ldx, w, ldw, sms, st);
  if (pl.pair == 2)
    return spl ? launch_tiles<T, LinCfg<128, 2, true>>(p, pl, x, ldx, w, ldw, sms, st)
               : launch_tiles<T, LinCfg<128, 2, false>>(p, pl, x, ldx, w, ldw, sms, st);
#define LINEAR_BN(W)                                                                        \
  if (pl.bn == W)                                                                           \
    return spl ? launch_tiles<T, LinCfg<W, 1, true>>(p, pl, x, ldx, w, ldw, sms, st)        \
               : launch_tiles<T, LinCfg<W, 1, false>>(p, pl, x, ldx, w, ldw, sms, st);
  LINEAR_BN(32)
  LINEAR_BN(64)
  LINEAR_BN(128)
#undef LINEAR_BN
  set_error("linear: no kernel for tile %d", pl.bn);
  return SPINN_CUDA_EUNSUPPORTED;
}

int linear_params(const SpinnCudaLinear* l, LinearParams* p) {
  SPINN_CHECK_ARG(l && l->x && l->w && l->y, "linear: x, w and y are required");
  SPINN_CHECK_ARG(l->dtype == SPINN_CUDA_FP16 || l->dtype == SPINN_CUDA_BF16,
                  "linear: element type %d not supported (fp16 or bf16; spinn_cuda_gemm takes fp32)", l->dtype);
  SPINN_CHECK_ARG(l->m > 0 && l->n > 0 && l->k > 0 && l->m <= kMaxLength && l->n <= kMaxLength && l->k <= kMaxLength,
                  "linear: bad sizes %d x %d x %d", l->m, l->n, l->k);
  SPINN_CHECK_ARG(l->x_stride >= l->k && l->w_stride >= l->k && l->y_stride >= l->n &&
                      (!l->residual || l->residual_stride >= l->n),
                  "linear: a row stride is shorter than its row");
  SPINN_CHECK_ARG(l->act == 0 || l->act == 1 || l->act == 3 || l->act == SPINN_CUDA_ACT_GELU ||
                      l->act == SPINN_CUDA_ACT_GELU_TANH,
                  "linear: activation %d not supported", l->act);
  SPINN_CHECK_ARG((((uintptr_t)l->x | (uintptr_t)l->w | (uintptr_t)l->y | (uintptr_t)l->bias | (uintptr_t)l->residual) & 1) == 0,
                  "linear: misaligned pointer");
  p->x = l->x;
  p->w = l->w;
  p->bias = l->bias;
  p->res = l->residual;
  p->y = l->y;
  p->ldx = l->x_stride;
  p->ldw = l->w_stride;
  p->ldr = l->residual_stride;
  p->ldy = l->y_stride;
  p->m = l->m;
  p->n = l->n;
  p->k = l->k;
  p->act = l->act;
  p->vec = tma_rows(l->x, l->x_stride) && tma_rows(l->w, l->w_stride);
  p->vec_y = tma_rows(l->y, l->y_stride) && (!l->residual || tma_rows(l->residual, l->residual_stride));
  p->err = nullptr;
  return 0;
}

}  // namespace

extern "C" {

__attribute__((visibility("default"))) size_t spinn_cuda_linear_workspace(const SpinnCudaLinear* l) {
  LinearParams p;
  if (linear_params(l, &p)) return 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    dev = -1;
  }
  const LinearPlan pl = linear_plan(p, dev < 0 ? 148 : sm_count(dev));
  return pl.x_bytes + pl.w_bytes;
}

__attribute__((visibility("default"))) int spinn_cuda_selftest_group_wait(uint64_t arrive_ns, uint64_t limit_ns) {
  SPINN_CHECK_ARG(arrive_ns <= 100000000 && limit_ns > 0 && limit_ns <= 1000000000,
                  "selftest_group_wait: at most 100 ms to the arrival and a limit of at most 1 s");
  group_wait_selftest_kernel<<<1, 160>>>(arrive_ns, limit_ns);
  SPINN_CUDA_TRY(cudaGetLastError());
  unsigned went_on = 0;
  SPINN_CUDA_TRY(cudaMemcpyFromSymbol(&went_on, g_group_went_on, sizeof(went_on)));
  return (int)went_on;
}

__attribute__((visibility("default"))) int spinn_cuda_diag_linear_plan(const SpinnCudaLinear* l, int sms, int* out5) {
  LinearParams p;
  const int rc = linear_params(l, &p);
  if (rc) return rc;
  SPINN_CHECK_ARG(sms > 0 && out5, "diag_linear_plan: invalid arguments");
  const LinearPlan pl = linear_plan(p, sms);
  out5[0] = pl.bn;
  out5[1] = pl.pair;
  out5[2] = pl.split;
  out5[3] = pl.copy_x;
  out5[4] = pl.copy_w;
  return 0;
}

__attribute__((visibility("default"))) int spinn_cuda_linear(const SpinnCudaLinear* l, void* workspace,
                                                             size_t workspace_bytes, void* stream) {
  LinearParams p;
  int rc = linear_params(l, &p);
  if (rc) return rc;
  int dev;
  rc = check_stream_device("linear", stream, &dev);
  if (rc) return rc;
  const int sms = sm_count(dev);
  const LinearPlan pl = linear_plan(p, sms);
  const size_t need = pl.x_bytes + pl.w_bytes;
  SPINN_CHECK_ARG(!need || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                  "linear: workspace of %zu bytes (16-byte aligned) needed, %zu given", need, workspace_bytes);
  rc = decode_error_word(dev, &p.err);
  if (rc) return rc;
  const auto rows = [](const void* q, int count, int width, int64_t stride) {
    return Rows{q, 2, width, {count, 1, 1}, {stride, 0, 0}};
  };
  const Rows y = rows(l->y, l->m, l->n, l->y_stride);
  SPINN_CHECK_ARG(rows_apart(y, rows(l->x, l->m, l->k, l->x_stride)) && rows_apart(y, rows(l->w, l->n, l->k, l->w_stride)) &&
                      (!l->bias || rows_apart(y, rows(l->bias, 1, l->n, l->n))),
                  "linear: y overlaps x, w or bias");
  SPINN_CHECK_ARG(!l->residual || (l->residual == l->y && (l->m == 1 || l->residual_stride == l->y_stride)) ||
                      rows_apart(y, rows(l->residual, l->m, l->n, l->residual_stride)),
                  "linear: y must be the residual itself or apart from it");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return l->dtype == SPINN_CUDA_FP16 ? linear_launch<__half>(p, pl, workspace, sms, st)
                                     : linear_launch<__nv_bfloat16>(p, pl, workspace, sms, st);
}

}  // extern "C"
}  // namespace spinn
