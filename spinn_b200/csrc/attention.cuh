// attention.cuh -- attention of one new token per sequence over a paged key-value cache.
//
//   y[s][h] = sum_t p_t v_t,   p = softmax_t(scale * q[s][h] . k_t),   t < lens[s]
//
// The heads of a group share their keys and values, so the cache is read once per group: at a few
// FLOP per byte the kernel is bound by HBM, and everything here serves to keep enough loads in
// flight and the tokens evenly dealt.
//
// Work split.  All tokens of the batch, in order (sequence, head block, tile of TK tokens), are
// dealt to a fixed number of CTAs in equal contiguous shares, whatever the lengths; every CTA
// finds its share from the lengths on the device, so the host needs to know none of them and a
// ragged batch is as balanced as an even one.  A (sequence, head) that lies in one share is
// finished there; one that crosses shares leaves a partial result per share (running maximum,
// sum and unnormalised output), and the second kernel joins them.
//
// Inside a CTA the four warps take a quarter of each tile and run on their own: each has its own
// ring of cp.async stages and its own running softmax, without a barrier in the loop, and the
// four states are joined when a (sequence, head) ends.
#pragma once
#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention.h"
#include "internal.h"
#include "launch.h"
#include "ptx.cuh"

namespace spinn {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kJoinWarps = 8;

// Tile shapes.  GB: heads of one block (8 or 16 with 16-bit types, where they are the columns of
// an MMA; up to 8 with fp32).  DPAD: head_dim padded to the next instantiated size.
template <typename T, int DPAD_, int GB_>
struct Tile {
  static constexpr int DPAD = DPAD_, GB = GB_;
  static constexpr bool k16 = sizeof(T) == 2;
  static constexpr int RW = k16 ? 16 : 8;   // tokens of a warp
  static constexpr int TK = RW * kWarps;    // tokens of a unit
  static constexpr int CH = DPAD * sizeof(T) / 16;
  // Row pitch in 16-byte chunks, against bank conflicts: odd for ldmatrix (eight rows of one
  // chunk); 4 mod 8 for the fp32 reads of two rows by four chunks.
  static constexpr int PITCH = k16 ? CH + 1 : (CH % 8 == 4 ? CH : CH + 4);
  static constexpr int HALF = RW * PITCH * 16;    // bytes of one warp's K (or V) rows
  static constexpr int STAGE = 2 * HALF * kWarps;
  static constexpr int CPL = (CH + 31) / 32;      // fp32: float4 chunks of an output row per lane
  static constexpr int NR = k16 ? GB / 8 * (DPAD / 16) * 4 : GB * CPL * 4;  // output registers
  static constexpr int MLR = k16 ? GB / 8 * 2 : GB;  // heads whose state a lane holds
  static constexpr int DUMP = (NR + 2 * MLR) * 32 * 4;
  static constexpr int EXTRA = 2 * DUMP + (k16 ? 0 : GB * DPAD * 4) + 2 * GB * 4 + 128;
  // Two CTAs per SM where three stages fit in half of the shared memory, else one
  static constexpr int kHalfSm = 113 * 1024, kSm = 226 * 1024;
  static constexpr int FIT2 = (kHalfSm - EXTRA) / STAGE, FIT1 = (kSm - EXTRA) / STAGE;
  static constexpr int CTAS = FIT2 >= 3 ? 2 : 1;
  static constexpr int NS = CTAS == 2 ? (FIT2 > 6 ? 6 : FIT2) : (FIT1 > 6 ? 6 : FIT1);
  static constexpr int SMEM = NS * STAGE + EXTRA;
  static_assert(NS >= 2, "pipeline needs two stages");
};

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 2^(a - b) where b is a maximum that may be -infinity (nothing seen so far).
__device__ __forceinline__ float exp2_from(float a, float b) { return exp2_approx(a - (b == -INFINITY ? 0.0f : b)); }

__device__ __forceinline__ void cp_async_16_zfill(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (std::is_same<T, float>::value)
    return x;
  else if constexpr (std::is_same<T, __half>::value)
    return __float2half_rn(x);
  else
    return __float2bfloat16_rn(x);
}
// (a, b) rounded to T and packed, a in the low half; lo gets what the rounding left, rounded too
template <typename T>
__device__ __forceinline__ uint32_t pack_split(float a, float b, uint32_t* lo) {
  const T ha = from_float<T>(a), hb = from_float<T>(b);
  float fa, fb;
  if constexpr (std::is_same<T, __half>::value) {
    fa = __half2float(ha);
    fb = __half2float(hb);
  } else {
    fa = __bfloat162float(ha);
    fb = __bfloat162float(hb);
  }
  union {
    T t[2];
    uint32_t u;
  } h, l;
  h.t[0] = ha;
  h.t[1] = hb;
  l.t[0] = from_float<T>(a - fa);
  l.t[1] = from_float<T>(b - fb);
  *lo = l.u;
  return h.u;
}

// Length of sequence s for the launch: 0 (and the error raised) when it is out of range.
__device__ __forceinline__ int attn_len(const AttnParams& p, int s) {
  const int n = p.c.lens[s];
  return n < 0 || n > p.capacity ? 0 : n;
}

// Position in the work: tile t of head block hb of sequence s, whose units start at `base`.
struct Walk {
  long long base;
  int s, hb, t, nt, len;
};
template <int TK>
__device__ __forceinline__ void walk_next(const AttnParams& p, Walk& w) {
  if (++w.t < w.nt) return;
  w.t = 0;
  w.base += w.nt;  // base is the head block's first unit
  if (++w.hb < p.hblocks) return;
  w.hb = 0;
  do {
    ++w.s;
    w.len = w.s < p.c.seqs ? attn_len(p, w.s) : 1;
  } while (w.len == 0);
  w.nt = (w.len + TK - 1) / TK;
}

template <typename T, int DPAD, int GB, bool WTS>
__global__ void __launch_bounds__(kThreads, Tile<T, DPAD, GB>::CTAS) attention_kernel(const AttnParams p) {
  using C = Tile<T, DPAD, GB>;
  constexpr int TK = C::TK, RW = C::RW, NS = C::NS, NR = C::NR, MLR = C::MLR;
  extern __shared__ __align__(16) uint8_t smem[];
  float* dump = reinterpret_cast<float*>(smem + NS * C::STAGE);
  float* qs = dump + 2 * (C::DUMP / 4);             // fp32: [GB][DPAD] queries of the segment
  float* fin = qs + (C::k16 ? 0 : GB * DPAD);       // [2][GB] final maximum and 1 / sum (weights)
  long long* sh = reinterpret_cast<long long*>(fin + 2 * GB);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  griddep_launch_dependents();

  // ---- this CTA's share, from the lengths
  const int workers = gridDim.x, me = blockIdx.x;
  long long mine = 0;
  bool bad = false;
  for (int s = tid; s < p.c.seqs; s += kThreads) {
    const int n = p.c.lens[s];
    bad |= n < 0 || n > p.capacity;
    mine += (attn_len(p, s) + TK - 1) / TK;
  }
  if (bad && me == 0) atomicOr(p.c.err, kCacheBadLength);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
  if (lane == 0) sh[warp] = mine;
  // empty sequences have no units: their outputs are zeros
  for (int s = me; s < p.c.seqs; s += workers)
    if (attn_len(p, s) == 0)
      for (int i = tid; i < p.q_heads * p.c.dim; i += kThreads) {
        const int h = i / p.c.dim;
        static_cast<T*>(p.y)[s * p.y_seq + h * p.y_head + (i - h * p.c.dim)] = from_float<T>(0.0f);
      }
  __syncthreads();
  const long long units = (sh[0] + sh[1] + sh[2] + sh[3]) * p.hblocks;
  const long long u0 = units > 0 ? attn_start(units, workers, me) : 0;
  const long long u1 = units > 0 ? attn_start(units, workers, me + 1) : 0;
  if (u0 >= u1) {
    if (tid < 2) p.pieces[me * 2 + tid].s = -1;
    return;
  }
  // ---- the sequence of unit u0: scan of the tile counts, kThreads sequences at a time
  Walk cur;
  {
    long long before = 0;  // tiles of the sequences before this batch of them
    for (int s0 = 0;; s0 += kThreads) {
      const int s = s0 + tid;
      const int nt = s < p.c.seqs ? (attn_len(p, s) + TK - 1) / TK : 0;
      long long incl = nt;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      __syncthreads();
      if (lane == 31) sh[warp] = incl;
      __syncthreads();
      for (int w = 0; w < warp; ++w) incl += sh[w];
      const long long total = sh[0] + sh[1] + sh[2] + sh[3];
      const long long first = (before + incl - nt) * p.hblocks;
      if (nt > 0 && first <= u0 && u0 < first + (long long)nt * p.hblocks) {
        sh[4] = first;
        sh[5] = s;
      }
      before += total;
      if (before * p.hblocks > u0) break;
    }
    __syncthreads();
    cur.s = (int)sh[5];
    cur.len = attn_len(p, cur.s);
    cur.nt = (cur.len + TK - 1) / TK;
    const int r = (int)(u0 - sh[4]);  // < nt * hblocks; a sequence has below 2^31 of them
    cur.hb = r / cur.nt;
    cur.t = r - cur.hb * cur.nt;
    cur.base = u0 - cur.t;
  }

  // ---- loads: this warp's RW rows of a tile into its part of a stage
  const int count = (int)(u1 - u0);
  const uint32_t stage0 = smem_u32(smem) + warp * 2 * C::HALF;
  Walk ahead = cur;
  // Offset of this lane's row (lanes below RW) of tile `w`, or -1 when the row is past the end
  // or its page is bad.
  auto row_offset = [&](const Walk& w) -> long long {
    const int pos = w.t * TK + warp * RW + (lane & (RW - 1));
    if (lane >= RW || pos >= w.len) return -1;
    const long long o = cache_slot(p.c.table + w.s * p.c.table_stride, pos, p.c.page_size, p.c.num_pages,
                                   p.c.page_stride, p.c.token_stride);
    if (o < 0) {
      atomicOr(p.c.err, kCacheBadPage);
      return -1;
    }
    return o + (w.hb / p.gblocks) * p.c.head_stride;
  };
  long long off = row_offset(ahead);
  auto issue = [&](int stage) {
    const uint32_t kdst = stage0 + stage * C::STAGE, vdst = kdst + C::HALF;
    if (p.vec) {
      // 32 lanes cover 32 / CH rows (or a part of one row), chunk by chunk
#pragma unroll
      for (int i = 0; i < RW * C::CH / 32; ++i) {
        const int e = i * 32 + lane, r = e / C::CH, ch = e - r * C::CH;
        const long long o = __shfl_sync(0xffffffffu, off, r);
        const bool ok = o >= 0 && ch * (int)(16 / sizeof(T)) < p.c.dim;
        const long long at = ok ? o + ch * (int)(16 / sizeof(T)) : 0;
        const uint32_t d = (r * C::PITCH + ch) * 16;
        cp_async_16_zfill(kdst + d, static_cast<const T*>(p.c.k) + at, ok);
        cp_async_16_zfill(vdst + d, static_cast<const T*>(p.c.v) + at, ok);
      }
    } else {
      T* ks = reinterpret_cast<T*>(smem + stage * C::STAGE + warp * 2 * C::HALF);
      T* vs = reinterpret_cast<T*>(smem + stage * C::STAGE + warp * 2 * C::HALF + C::HALF);
      constexpr int PE = C::PITCH * 16 / sizeof(T);
      for (int r = 0; r < RW; ++r) {
        const long long o = __shfl_sync(0xffffffffu, off, r);
        for (int e = lane; e < DPAD; e += 32) {
          const bool ok = o >= 0 && e < p.c.dim;
          ks[r * PE + e] = ok ? static_cast<const T*>(p.c.k)[o + e] : from_float<T>(0.0f);
          vs[r * PE + e] = ok ? static_cast<const T*>(p.c.v)[o + e] : from_float<T>(0.0f);
        }
      }
    }
  };
  // the next tile's table entries are read a whole tile before its rows are asked for
  auto advance = [&](int issued) {
    if (issued < count) {
      walk_next<TK>(p, ahead);
      off = row_offset(ahead);
    }
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    if (i < count) {
      issue(i);
      advance(i + 1);
    }
    cp_async_commit();
  }

  // ---- running state of this warp
  float o[NR / 4][4], m[MLR], l[MLR];
  uint32_t qf[C::k16 ? GB / 8 : 1][C::k16 ? DPAD / 16 : 1][2];  // 16-bit: queries as MMA fragments
  auto begin_segment = [&]() {
#pragma unroll
    for (int i = 0; i < NR; ++i) o[i / 4][i & 3] = 0.0f;
#pragma unroll
    for (int i = 0; i < MLR; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
    }
    const int kvh = cur.hb / p.gblocks, g0 = (cur.hb - kvh * p.gblocks) * GB;
    const T* q = static_cast<const T*>(p.q) + cur.s * p.q_seq + (long long)(kvh * p.group + g0) * p.q_head;
    const int heads = min(GB, p.group - g0);
    if constexpr (C::k16) {
#pragma unroll
      for (int n = 0; n < GB / 8; ++n)
#pragma unroll
        for (int k = 0; k < DPAD / 16; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int h = n * 8 + (lane >> 2), d = k * 16 + j * 8 + (lane & 3) * 2;
            union {
              T t[2];
              uint32_t u;
            } x;
            x.u = 0;
            if (h < heads && d < p.c.dim) x.t[0] = q[h * p.q_head + d];
            if (h < heads && d + 1 < p.c.dim) x.t[1] = q[h * p.q_head + d + 1];
            qf[n][k][j] = x.u;
          }
    } else {
      __syncthreads();  // the previous segment's reads are done
      for (int i = tid; i < GB * DPAD; i += kThreads) {
        const int h = i / DPAD, d = i - h * DPAD;
        qs[i] = h < heads && d < p.c.dim ? q[h * p.q_head + d] : 0.0f;
      }
      __syncthreads();
    }
  };

  // ---- one tile: scores, running softmax, output
  auto compute = [&](int stage, long long unit) {
    const int left = cur.len - cur.t * TK - warp * RW;  // valid rows of this warp (may be <= 0)
    if constexpr (C::k16) {
      constexpr int NT = GB / 8, KD = DPAD / 16;
      const uint32_t kb = stage0 + stage * C::STAGE, vb = kb + C::HALF;
      // S^T = K Q^T: tokens are the rows, heads the columns of the MMA
      float sc[NT][2][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][0][i] = sc[n][1][i] = 0.0f;
      const uint32_t ka = kb + ((lane & 15) * C::PITCH + (lane >> 4)) * 16;
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        uint32_t a[4];
        ldmatrix_x4(ka + k * 32, a);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_16816<T>(sc[n][k & 1], a, qf[n][k][0], qf[n][k][1]);
      }
      const int r0 = lane >> 2;
      const bool ok0 = r0 < left, ok1 = r0 + 8 < left;
      uint32_t ph[NT][2], pl[NT][2];
      bool grew = false;
      float s[NT][4], mx[MLR];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][i] = (sc[n][0][i] + sc[n][1][i]) * p.scale_log2;
          if (!(i < 2 ? ok0 : ok1)) s[n][i] = -INFINITY;
        }
        if constexpr (WTS) {
          float* lg = p.logits + ((unit * TK + warp * RW + r0) * GB + n * 8 + (lane & 3) * 2);
          if (ok0) *reinterpret_cast<float2*>(lg) = make_float2(s[n][0], s[n][1]);
          if (ok1) *reinterpret_cast<float2*>(lg + 8 * GB) = make_float2(s[n][2], s[n][3]);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = fmaxf(s[n][c], s[n][2 + c]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          mx[n * 2 + c] = fmaxf(x, m[n * 2 + c]);
          grew |= mx[n * 2 + c] > m[n * 2 + c];
        }
      }
      if (__any_sync(0xffffffffu, grew)) {
        float f[MLR];
#pragma unroll
        for (int i = 0; i < MLR; ++i) {
          f[i] = exp2_from(m[i], mx[i]);
          l[i] *= f[i];
          m[i] = mx[i];
        }
#pragma unroll
        for (int i = 0; i < NR; ++i) o[i / 4][i & 3] *= f[i / (KD * 4) * 2 + (i & 1)];
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = exp2_from(s[n][i], m[n * 2 + (i & 1)]);
        l[n * 2] += e[0] + e[2];
        l[n * 2 + 1] += e[1] + e[3];
        // P^T as the B operand: 8 x 8 blocks transposed in registers.  The probabilities enter
        // the product as a sum of two 16-bit parts, so that y carries one rounding, its own.
        uint32_t lo0, lo1;
        const uint32_t hi0 = pack_split<T>(e[0], e[1], &lo0), hi1 = pack_split<T>(e[2], e[3], &lo1);
        ph[n][0] = movmatrix_trans(hi0);
        ph[n][1] = movmatrix_trans(hi1);
        pl[n][0] = movmatrix_trans(lo0);
        pl[n][1] = movmatrix_trans(lo1);
      }
      // O^T += V^T P^T: output dims are the rows
      const uint32_t va = vb + (((lane & 7) + (lane >> 4) * 8) * C::PITCH + ((lane >> 3) & 1)) * 16;
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        uint32_t a[4];
        ldmatrix_x4_trans(va + k * 32, a);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_16816<T>(o[n * KD + k], a, ph[n][0], ph[n][1]);
          mma_16816<T>(o[n * KD + k], a, pl[n][0], pl[n][1]);
        }
      }
    } else {
      // fp32 on the FMA units: lane = (token of eight, quarter of the row) for the scores, a
      // chunk of four output dims for the products
      const float4* ks = reinterpret_cast<const float4*>(smem + stage * C::STAGE + warp * 2 * C::HALF);
      const float4* vs = ks + C::HALF / 16;
      const float4* q4 = reinterpret_cast<const float4*>(qs);
      const int key = lane >> 2, part = lane & 3;
      float s[GB];
#pragma unroll
      for (int g = 0; g < GB; ++g) s[g] = 0.0f;
#pragma unroll 4
      for (int i = 0; i < C::CH / 4; ++i) {
        const float4 x = ks[key * C::PITCH + part + 4 * i];
#pragma unroll
        for (int g = 0; g < GB; ++g) {
          const float4 y = q4[g * (DPAD / 4) + part + 4 * i];
          s[g] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s[g]))));
        }
      }
      bool grew = false;
      float mx[GB];
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        s[g] += __shfl_xor_sync(0xffffffffu, s[g], 1);
        s[g] += __shfl_xor_sync(0xffffffffu, s[g], 2);
        s[g] = key < left ? s[g] * p.scale_log2 : -INFINITY;
        float x = s[g];
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        mx[g] = fmaxf(x, m[g]);
        grew |= mx[g] > m[g];
        if constexpr (WTS) {
          if (part == 0 && key < left) p.logits[(unit * TK + warp * RW + key) * GB + g] = s[g];
        }
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int g = 0; g < GB; ++g) {
          const float f = exp2_from(m[g], mx[g]);
          l[g] *= f;
          m[g] = mx[g];
#pragma unroll
          for (int i = 0; i < C::CPL * 4; ++i) o[g * C::CPL + i / 4][i & 3] *= f;
        }
      }
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        s[g] = exp2_from(s[g], m[g]);
        l[g] += s[g];
      }
#pragma unroll
      for (int r = 0; r < RW; ++r) {
#pragma unroll
        for (int ci = 0; ci < C::CPL; ++ci) {
          const int ch = lane + 32 * ci;
          const float4 x = ch < C::CH ? vs[r * C::PITCH + ch] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int g = 0; g < GB; ++g) {
            const float w = __shfl_sync(0xffffffffu, s[g], r * 4);
            float(&acc)[4] = o[g * C::CPL + ci];
            acc[0] = fmaf(w, x.x, acc[0]);
            acc[1] = fmaf(w, x.y, acc[1]);
            acc[2] = fmaf(w, x.z, acc[2]);
            acc[3] = fmaf(w, x.w, acc[3]);
          }
        }
      }
    }
  };

  // head (of the block) of state register i
  auto head_of_state = [&](int i) -> int { return C::k16 ? (i >> 1) * 8 + (lane & 3) * 2 + (i & 1) : i; };

  // ---- a segment's end: the four warps' states joined by warp 0, then written out
  auto write_state = [&](float* d) {
#pragma unroll
    for (int i = 0; i < NR; ++i) d[i * 32 + lane] = o[i / 4][i & 3];
#pragma unroll
    for (int i = 0; i < MLR; ++i) {
      d[(NR + i) * 32 + lane] = m[i];
      d[(NR + MLR + i) * 32 + lane] = l[i];
    }
  };
  auto absorb_state = [&](const float* d) {
    float mine[MLR], other[MLR];
#pragma unroll
    for (int i = 0; i < MLR; ++i) {
      const float om = d[(NR + i) * 32 + lane], top = fmaxf(m[i], om);
      mine[i] = exp2_from(m[i], top);
      other[i] = exp2_from(om, top);
      l[i] = l[i] * mine[i] + d[(NR + MLR + i) * 32 + lane] * other[i];
      m[i] = top;
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int st = C::k16 ? i / (DPAD / 16 * 4) * 2 + (i & 1) : i / (C::CPL * 4);
      o[i / 4][i & 3] = o[i / 4][i & 3] * mine[st] + d[i * 32 + lane] * other[st];
    }
  };
  auto end_segment = [&](long long begin, long long end) {
    // every lane's own share of the sum so far (16-bit: its rows; fp32: its token)
#pragma unroll
    for (int i = 0; i < MLR; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 4);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 8);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 16);
    }
    float* da = dump;
    float* db = dump + C::DUMP / 4;
    __syncthreads();  // warp 0 is done with the buffers of the previous segment
    if (warp & 1) write_state(warp == 1 ? da : db);
    __syncthreads();
    if (!(warp & 1)) absorb_state(warp == 0 ? da : db);
    if (warp == 2) write_state(db);
    __syncthreads();
    const bool whole = begin >= u0 && end <= u1;
    if (warp == 0) {
      absorb_state(db);
      const int kvh = cur.hb / p.gblocks, g0 = (cur.hb - kvh * p.gblocks) * GB;
      const int heads = min(GB, p.group - g0);
      if (whole) {
        float inv[MLR];
#pragma unroll
        for (int i = 0; i < MLR; ++i) inv[i] = 1.0f / l[i];
        T* y = static_cast<T*>(p.y) + cur.s * p.y_seq + (long long)(kvh * p.group + g0) * p.y_head;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          int h, d, st;
          if constexpr (C::k16) {
            const int kd = i / 4 % (DPAD / 16);
            st = i / (DPAD / 16 * 4) * 2 + (i & 1);
            h = head_of_state(st);
            d = kd * 16 + (lane >> 2) + ((i >> 1) & 1) * 8;
          } else {
            st = h = i / (C::CPL * 4);
            d = (lane + 32 * (i / 4 % C::CPL)) * 4 + (i & 3);
          }
          if (h < heads && d < p.c.dim) y[h * p.y_head + d] = from_float<T>(o[i / 4][i & 3] * inv[st]);
        }
        if constexpr (WTS) {
#pragma unroll
          for (int i = 0; i < MLR; ++i)
            if (C::k16 ? lane < 4 : lane == 0) {
              fin[head_of_state(i)] = m[i];
              fin[GB + head_of_state(i)] = inv[i];
            }
        }
      } else {
        const int slot = me * 2 + (begin >= u0 ? 1 : 0);
        float* d = p.part + (size_t)slot * NR * 32;
#pragma unroll
        for (int i = 0; i < NR; ++i) d[i * 32 + lane] = o[i / 4][i & 3];
        float* ml = p.ml + (size_t)slot * 2 * GB;
#pragma unroll
        for (int i = 0; i < MLR; ++i)
          if (C::k16 ? lane < 4 : lane == 0) {
            ml[head_of_state(i)] = m[i];
            ml[GB + head_of_state(i)] = l[i];
          }
      }
    }
    if constexpr (WTS) {
      if (whole) {
        __syncthreads();
        const int heads = p.group;  // one head block per key head with weights
        const float* win = p.win ? p.win + cur.s * p.win_seq + cur.hb * p.win_head : nullptr;
        float* wout = p.wout + cur.s * p.wout_seq + cur.hb * p.wout_head;
        for (int i = tid; i < cur.len; i += kThreads) {
          const float* lg = p.logits + (begin * TK + i) * GB;
          float sum = 0.0f;
          for (int g = 0; g < heads; ++g) sum += exp2_from(lg[g], fin[g]) * fin[GB + g];
          wout[i] = (win ? win[i] : 0.0f) + sum;
        }
      }
    }
  };

  if (tid < 2) p.pieces[me * 2 + tid].s = -1;
  __syncthreads();
  bool fresh = true;
  for (int i = 0; i < count; ++i) {
    if (fresh) begin_segment();
    cp_async_wait<NS - 2>();
    __syncwarp();  // this tile has landed, and every lane is done with the one before it
    if (i + NS - 1 < count) {
      issue((i + NS - 1) % NS);
      advance(i + NS);
    }
    cp_async_commit();
    compute(i % NS, u0 + i);
    fresh = cur.t + 1 == cur.nt;
    if (fresh || i + 1 == count) {
      const long long begin = cur.base, end = begin + cur.nt;
      end_segment(begin, end);
      if (tid == 0 && (begin < u0 || end > u1)) {
        Piece& r = p.pieces[me * 2 + (begin >= u0 ? 1 : 0)];
        r.hb = cur.hb;
        r.w0 = attn_owner(units, workers, begin);
        r.w1 = attn_owner(units, workers, end - 1);
        r.begin = begin;
        r.lo = begin >= u0 ? begin : u0;
        r.hi = end <= u1 ? end : u1;
        r.s = cur.s;
      }
    }
    if (i + 1 < count) walk_next<TK>(p, cur);
  }
}

// ------------------------------------------------------------------ join
// Block (w, slice): when worker w is the second one of a segment, the block joins four of the
// output registers of all the segment's workers -- an online softmax over the partials, dealt to
// eight warps.  With weights, the slices above NR / 4 turn the scores of the worker's own tokens
// in split segments into probabilities.
template <typename T, int DPAD, int GB, bool WTS>
__global__ void __launch_bounds__(kJoinWarps * 32) attention_join_kernel(const AttnParams p, int weight_slices) {
  using C = Tile<T, DPAD, GB>;
  constexpr int TK = C::TK, NR = C::NR;
  griddep_wait();
  const int me = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((int)blockIdx.y < NR / 4) {
    const Piece pc = p.pieces[me * 2];
    if (pc.s < 0) return;
    // the first worker after w0 with a share joins; workers between without one have no piece
    for (int w = pc.w0 + 1; w < me; ++w)
      if (p.pieces[w * 2].s >= 0) return;
    __shared__ float sm[kJoinWarps][32][8];
    const int i0 = blockIdx.y * 4;
    int h0, h1, d[4];
    if constexpr (C::k16) {
      const int n = i0 / (DPAD / 16 * 4), kd = i0 / 4 % (DPAD / 16);
      h0 = n * 8 + (lane & 3) * 2;
      h1 = h0 + 1;
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = kd * 16 + (lane >> 2) + (i >> 1) * 8;
    } else {
      h0 = h1 = i0 / (C::CPL * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = (lane + 32 * (i0 / 4 % C::CPL)) * 4 + i;
    }
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int w = pc.w0 + warp; w <= pc.w1; w += kJoinWarps) {
      const int slot = w * 2 + (w == pc.w0 ? 1 : 0);
      if (w != pc.w0 && p.pieces[slot].s < 0) continue;
      const float* ml = p.ml + (size_t)slot * 2 * GB;
      const float* src = p.part + ((size_t)slot * NR + i0) * 32 + lane;
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = src[i * 32];
      const float a0 = ml[h0], a1 = ml[h1], b0 = ml[GB + h0], b1 = ml[GB + h1];
      const float t0 = fmaxf(m0, a0), t1 = fmaxf(m1, a1);
      const float f0 = exp2_from(m0, t0), f1 = exp2_from(m1, t1), e0 = exp2_from(a0, t0), e1 = exp2_from(a1, t1);
      m0 = t0;
      m1 = t1;
      l0 = l0 * f0 + b0 * e0;
      l1 = l1 * f1 + b1 * e1;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = C::k16 && (i & 1) ? o[i] * f1 + x[i] * e1 : o[i] * f0 + x[i] * e0;
    }
    float* mine = sm[warp][lane];
    mine[0] = m0;
    mine[1] = m1;
    mine[2] = l0;
    mine[3] = l1;
#pragma unroll
    for (int i = 0; i < 4; ++i) mine[4 + i] = o[i];
    __syncthreads();
    if (warp != 0) return;
    for (int w = 1; w < kJoinWarps; ++w) {
      const float* x = sm[w][lane];
      const float t0 = fmaxf(m0, x[0]), t1 = fmaxf(m1, x[1]);
      const float f0 = exp2_from(m0, t0), f1 = exp2_from(m1, t1), e0 = exp2_from(x[0], t0), e1 = exp2_from(x[1], t1);
      m0 = t0;
      m1 = t1;
      l0 = l0 * f0 + x[2] * e0;
      l1 = l1 * f1 + x[3] * e1;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = C::k16 && (i & 1) ? o[i] * f1 + x[4 + i] * e1 : o[i] * f0 + x[4 + i] * e0;
    }
    const int kvh = pc.hb / p.gblocks, g0 = (pc.hb - kvh * p.gblocks) * GB;
    const int heads = min(GB, p.group - g0);
    T* y = static_cast<T*>(p.y) + pc.s * p.y_seq + (long long)(kvh * p.group + g0) * p.y_head;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = C::k16 && (i & 1) ? h1 : h0;
      if (h < heads && d[i] < p.c.dim) y[h * p.y_head + d[i]] = from_float<T>(o[i] / (C::k16 && (i & 1) ? l1 : l0));
    }
    return;
  }
  if constexpr (WTS) {
    __shared__ float top[GB], inv[GB];
    const int slice = blockIdx.y - NR / 4;
    for (int kind = 0; kind < 2; ++kind) {
      const Piece pc = p.pieces[me * 2 + kind];
      if (pc.s < 0) continue;
      const int len = p.c.lens[pc.s];
      for (int g = warp; g < p.group; g += kJoinWarps) {
        float m = -INFINITY, l = 0.0f;
        for (int w = pc.w0 + lane; w <= pc.w1; w += 32) {
          const int slot = w * 2 + (w == pc.w0 ? 1 : 0);
          if (w != pc.w0 && p.pieces[slot].s < 0) continue;
          const float a = p.ml[(size_t)slot * 2 * GB + g], b = p.ml[(size_t)slot * 2 * GB + GB + g];
          const float t = fmaxf(m, a);
          l = l * exp2_from(m, t) + b * exp2_from(a, t);
          m = t;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
          const float a = __shfl_xor_sync(0xffffffffu, m, d), b = __shfl_xor_sync(0xffffffffu, l, d);
          const float t = fmaxf(m, a);
          l = l * exp2_from(m, t) + b * exp2_from(a, t);
          m = t;
        }
        if (lane == 0) {
          top[g] = m;
          inv[g] = 1.0f / l;
        }
      }
      __syncthreads();
      const float* win = p.win ? p.win + pc.s * p.win_seq + pc.hb * p.win_head : nullptr;
      float* wout = p.wout + pc.s * p.wout_seq + pc.hb * p.wout_head;
      // this worker's tokens of the segment, dealt to the slices
      const int t0 = (int)(pc.lo - pc.begin) * TK, t1 = min(len, (int)(pc.hi - pc.begin) * TK);
      for (int i = t0 + slice * kJoinWarps * 32 + tid; i < t1; i += weight_slices * kJoinWarps * 32) {
        const float* lg = p.logits + (pc.begin * TK + i) * GB;
        float sum = 0.0f;
        for (int g = 0; g < p.group; ++g) sum += exp2_from(lg[g], top[g]) * inv[g];
        wout[i] = (win ? win[i] : 0.0f) + sum;
      }
      __syncthreads();
    }
  }
}

// Workspace of a launch (bytes of its parts, each rounded to 256).
template <typename T, int DPAD, int GB>
AttnPlan attention_plan_for(const AttnParams& p, int sms, bool weights) {
  using C = Tile<T, DPAD, GB>;
  const long long tiles = ((long long)p.capacity + C::TK - 1) / C::TK;
  const long long units = tiles * p.c.seqs * p.hblocks;  // at most
  AttnPlan pl;
  pl.workers = (int)std::min<long long>(units, (long long)sms * C::CTAS);
  pl.part = up256((size_t)pl.workers * 2 * C::NR * 32 * 4);
  pl.ml = up256((size_t)pl.workers * 2 * 2 * GB * 4);
  pl.pieces = up256((size_t)pl.workers * 2 * sizeof(Piece));
  pl.logits = weights ? up256((size_t)units * C::TK * GB * 4) : 0;
  return pl;
}

template <typename T, int DPAD, int GB, bool WTS>
int attention_launch_for(const AttnParams& p, const AttnPlan& pl, cudaStream_t st) {
  using C = Tile<T, DPAD, GB>;
  auto* kernel = attention_kernel<T, DPAD, GB, WTS>;
  SPINN_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
  kernel<<<pl.workers, kThreads, C::SMEM, st>>>(p);
  SPINN_CUDA_TRY(cudaGetLastError());
  const int slices = WTS ? 4 : 0;
  return launch_dependent(attention_join_kernel<T, DPAD, GB, WTS>, dim3(pl.workers, C::NR / 4 + slices), kJoinWarps * 32,
                          0, st, p, slices);
}

// The instantiation for a head size and group: `go` gets the Tile as a tag.
template <typename T, typename F>
auto attention_dispatch(int dim, int group, F go) {
  constexpr int SMALL = sizeof(T) == 2 ? 8 : 1, LARGE = sizeof(T) == 2 ? 16 : 8;
  if (group <= SMALL) {
    if (dim <= 64) return go(Tile<T, 64, SMALL>());
    if (dim <= 128) return go(Tile<T, 128, SMALL>());
    return go(Tile<T, 256, SMALL>());
  }
  if (dim <= 64) return go(Tile<T, 64, LARGE>());
  if (dim <= 128) return go(Tile<T, 128, LARGE>());
  return go(Tile<T, 256, LARGE>());
}

template <typename T>
AttnPlan attention_plan_t(const AttnParams& p, int sms, bool weights) {
  return attention_dispatch<T>(p.c.dim, p.group, [&](auto t) {
    using C = decltype(t);
    return attention_plan_for<T, C::DPAD, C::GB>(p, sms, weights);
  });
}
template <typename T>
int attention_launch_t(const AttnParams& p, const AttnPlan& pl, cudaStream_t st) {
  return attention_dispatch<T>(p.c.dim, p.group, [&](auto t) {
    using C = decltype(t);
    return p.wout ? attention_launch_for<T, C::DPAD, C::GB, true>(p, pl, st)
                  : attention_launch_for<T, C::DPAD, C::GB, false>(p, pl, st);
  });
}

}  // namespace
}  // namespace spinn
