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
// finished there; one that crosses shares leaves a partial result per share (running
// reference, sum and unnormalised output), and the second kernel joins them.
//
// A batch whose caches are all short (the table holds at most eight tiles, and there is an SM slot
// for every (sequence, head)) is not split: each CTA takes one (sequence, head) and there is
// nothing to join.
//
// Inside a CTA the four warps take a quarter of each tile and run on their own: each has its own
// ring of stages and its own running softmax, without a barrier in the loop, and the four states
// are joined when a (sequence, head) ends.  Where a page holds a whole number of a warp's rows, one
// lane fetches them with TMA boxes (two or so instructions for 4 KB, instead of a row lookup, two
// shuffles and an address for every 512 bytes); otherwise every lane copies 16-byte pieces, or
// single elements where rows are not aligned.
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
constexpr int kJoinWarps = 16;
constexpr int kWholeTiles = 8;  // longest cache, in tiles, that is left to one CTA
constexpr uint64_t kTimeoutNs = 4000000000ull, kDrainNs = 200000000ull;  // bounded barrier waits

// Tile shapes.  GB: heads of one block (8 or 16 with 16-bit types, where they are the columns of
// an MMA; 1, 4 or 8 with fp32).  DPAD: head_dim padded to the next instantiated size.
template <typename T, int DPAD_, int GB_>
struct Tile {
  static constexpr int DPAD = DPAD_, GB = GB_;
  static constexpr bool k16 = sizeof(T) == 2;
  static constexpr bool kScaled = std::is_same<T, __half>::value;  // small probabilities are scaled for the product with V
  // Tokens of a warp.  What a tile costs beside its bytes (fetching, waiting, the softmax's chain) makes
  // 16 the better number wherever two CTAs still fit (64 x 4096 fp32 of 64: 128 us with 8, 98 with 16).
  static constexpr int RW = k16 || DPAD <= 96 ? 16 : 8;
  static constexpr int TK = RW * kWarps;    // tokens of a unit
  static constexpr int CH = DPAD * sizeof(T) / 16;  // 16-byte chunks of a row
  // 16-bit rows lie in sub-tiles of 128 bytes a row, chunk c at c ^ (row % 8): the TMA's 128-byte
  // swizzle, under which ldmatrix is free of bank conflicts.  fp32 rows lie one behind the other.
  static constexpr int SUBS = CH / 8, SUB = RW * 128, HALF = RW * CH * 16;  // HALF: one warp's K (or V) rows
  static constexpr int SPAN = k16 ? 64 : 0;                                 // elements of a sub-tile's row
  static constexpr int STAGE = 2 * HALF * kWarps;
  static constexpr int CPL = (CH + 31) / 32;      // fp32: float4 chunks of an output row per lane
  static constexpr int NR = k16 ? GB / 8 * (DPAD / 16) * 4 : GB * CPL * 4;  // output registers
  static constexpr int MLR = k16 ? GB / 8 * 2 : GB;  // heads whose state a lane holds
  static constexpr int DUMP = (NR + 2 * MLR) * 32 * 4;
  static constexpr int EXTRA = 2 * DUMP + (k16 ? 0 : GB * DPAD * 4) + 2 * GB * 4 + 64 + kWarps * 6 * 8 + 16 + 1024;
  // Two CTAs per SM where three stages fit in half of the shared memory (two stages, for rows of 384
  // bytes: 32 x 8192 16-bit of 192 takes 159 us, 193 padded to 256 with one CTA), else one; three and
  // four CTAs measured no faster.
  static constexpr int kHalfSm = 113 * 1024, kSm = 226 * 1024;
  static constexpr int FIT2 = (kHalfSm - EXTRA) / STAGE, FIT1 = (kSm - EXTRA) / STAGE;
  static constexpr int CTAS = FIT2 >= (CH == 24 ? 2 : 3) ? 2 : 1;
  static constexpr int NS = CTAS == 2 ? (FIT2 > 6 ? 6 : FIT2) : (FIT1 > 6 ? 6 : FIT1);
  static constexpr int SMEM = NS * STAGE + EXTRA;
  static_assert(NS >= 2, "pipeline needs two stages");
};

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 2^(a - b), b a reference that is finite (kNothing while nothing has been seen).
constexpr float kNothing = -3.0e38f;
__device__ __forceinline__ float exp2_from(float a, float b) { return exp2_approx(a - b); }

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
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    *lo = *reinterpret_cast<const uint32_t*>(&l);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(a - __uint_as_float(u << 16), b - __uint_as_float(u & 0xffff0000u));
    *lo = *reinterpret_cast<const uint32_t*>(&l);
    return u;
  }
}

// Length of sequence s for the launch: 0 (and the error raised) when it is out of range.
__device__ __forceinline__ int attn_len(const AttnParams& p, int s) {
  const int n = p.c.lens[s];
  return n < 0 || n > p.capacity ? 0 : n;
}

// Position in the work: tile t of the nt tiles of head block hb of sequence s; `base` is the head
// block's first unit.
struct Walk {
  unsigned base;
  int s, hb, t, nt, len;
};
// Carries t over into the following head blocks and sequences.
template <int TK>
__device__ __forceinline__ void walk_carry(const AttnParams& p, Walk& w) {
  while (w.t >= w.nt) {
    w.t -= w.nt;
    w.base += w.nt;
    if (++w.hb < p.hblocks) continue;
    w.hb = 0;
    do {
      ++w.s;
      w.len = w.s < p.c.seqs ? attn_len(p, w.s) : 0x7fffffff;  // past the last: stay there
    } while (w.len == 0);
    w.nt = w.len == 0x7fffffff ? 0x7fffffff : (w.len + TK - 1) / TK;
  }
}
template <int TK>
__device__ __forceinline__ void walk_next(const AttnParams& p, Walk& w) {
  ++w.t;
  walk_carry<TK>(p, w);
}

template <typename T, int DPAD, int GB, bool WTS>
__global__ void __launch_bounds__(kThreads, Tile<T, DPAD, GB>::CTAS) attention_kernel(const __grid_constant__ AttnParams p) {
  using C = Tile<T, DPAD, GB>;
  constexpr int TK = C::TK, RW = C::RW, NS = C::NS, NR = C::NR, MLR = C::MLR;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* dump = reinterpret_cast<float*>(smem + NS * C::STAGE);
  float* qs = dump + 2 * (C::DUMP / 4);             // fp32: [GB][DPAD] queries of the segment
  float* fin = qs + (C::k16 ? 0 : GB * DPAD);       // [2][GB] final maximum and 1 / sum (weights)
  unsigned* sh = reinterpret_cast<unsigned*>(fin + 2 * GB);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sh + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + kWarps * 6);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint64_t* full = bars + warp * 6;  // this warp's stages
  if (lane == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  if (tid == 0) {
    *abort_flag = 0;
    if (p.mode == kCopyTma) {
      prefetch_tmap(&p.map_k);
      prefetch_tmap(&p.map_v);
    }
  }
  griddep_launch_dependents();
  griddep_wait();
  __syncthreads();

  // ---- this CTA's share, from the lengths
  const int workers = gridDim.x, me = blockIdx.x;
  unsigned units = 0, u0 = 0, u1 = 0;
  Walk cur;
  if (p.whole) {
    // one (sequence, head block) per CTA, its units numbered from me * whole
    cur.s = me / p.hblocks;
    cur.hb = me - cur.s * p.hblocks;
    const int n = p.c.lens[cur.s];
    if ((n < 0 || n > p.capacity) && tid == 0) atomicOr(p.c.err, kCacheBadLength);
    cur.len = n < 0 || n > p.capacity ? 0 : n;
    cur.nt = (cur.len + TK - 1) / TK;
    cur.t = 0;
    cur.base = u0 = (unsigned)me * p.whole;
    u1 = u0 + cur.nt;
    if (cur.len == 0) {
      const int kvh = cur.hb / p.gblocks, g0 = (cur.hb - kvh * p.gblocks) * GB, heads = min(GB, p.group - g0);
      T* y = static_cast<T*>(p.y) + cur.s * p.y_seq + (long long)(kvh * p.group + g0) * p.y_head;
      for (int i = tid; i < heads * p.c.dim; i += kThreads) y[i / p.c.dim * p.y_head + i % p.c.dim] = from_float<T>(0.0f);
      return;
    }
  } else {
    // Tiles of all sequences (kThreads of them at a time), then the sequence of unit u0.  With no
    // more sequences than threads the first scan serves for both.
    const bool once = p.c.seqs <= kThreads;
    unsigned total = 0, incl = 0;
    int len = 0, nt = 0;
    bool bad = false;
    auto scan = [&](int s0) -> unsigned {  // inclusive over this batch, and its total
      const int s = s0 + tid, n = s < p.c.seqs ? p.c.lens[s] : 0;
      bad |= n < 0 || n > p.capacity;
      len = n < 0 || n > p.capacity ? 0 : n;
      nt = (len + TK - 1) / TK;
      incl = nt;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      if (lane == 31) sh[warp] = incl;
      __syncthreads();
      unsigned sum = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) incl += sh[w];
        sum += sh[w];
      }
      return sum;
    };
    for (int s0 = 0; s0 < p.c.seqs; s0 += kThreads) {
      total += scan(s0);
      if (!once) __syncthreads();
    }
    if (bad && me == 0) atomicOr(p.c.err, kCacheBadLength);
    units = total * p.hblocks;
    const AttnShares shares(units, workers);
    u0 = shares.start(me);
    u1 = shares.start(me + 1);
    unsigned before = 0;  // tiles of the sequences before this batch of them
    for (int s0 = 0; u0 < u1; s0 += kThreads) {
      const unsigned sum = once ? total : scan(s0);
      const unsigned first = (before + incl - nt) * p.hblocks;
      if (nt > 0 && first <= u0 && u0 - first < (unsigned)nt * p.hblocks) {
        sh[4] = first;
        sh[5] = s0 + tid;
        sh[6] = len;
      }
      before += sum;
      __syncthreads();
      if (before * p.hblocks > u0) break;
    }
    if (u0 < u1) {
      cur.s = (int)sh[5];
      cur.len = (int)sh[6];
      cur.nt = (cur.len + TK - 1) / TK;
      const unsigned r = u0 - sh[4];
      cur.hb = (int)(r / cur.nt);
      cur.t = (int)(r - (unsigned)cur.hb * cur.nt);
      cur.base = u0 - cur.t;
    }
  }
  // empty sequences have no units: their outputs are zeros
  auto clear_empty = [&]() {
    for (int s = me; s < p.c.seqs; s += workers)
      if (attn_len(p, s) == 0) {
        for (int i = tid; i < p.q_heads * p.c.dim; i += kThreads) {
          const int h = i / p.c.dim;
          static_cast<T*>(p.y)[s * p.y_seq + h * p.y_head + (i - h * p.c.dim)] = from_float<T>(0.0f);
        }
        if (p.by_segment)
          for (int i = tid; i < p.hblocks; i += kThreads) p.segs[s * p.hblocks + i] = {0, -1};
      }
  };
  if (u0 >= u1) {
    if (tid < 2) p.pieces[me * 2 + tid].s = -1;
    clear_empty();
    return;
  }

  // ---- loads: this warp's RW rows of a tile into its part of a stage
  // Boxes start sooner and cost few instructions, copies by the lanes draw a little more bandwidth
  // out of long shares and out of rows that are not whole sub-tiles (bf16, boxes : lanes: 8 x 8192
  // of 128 34.3 : 35.9 us, 48 x 8192 of 128 147 : 145, 64 x 8192 of 64 134 : 140 and of 80 206 : 181).
  int mode = p.mode;
  if (C::k16 && mode == kCopyTma && (u1 - u0) >= 40 && !p.whole &&
      (p.c.dim % 64 || (p.c.dim > 64 && p.c.dim <= 128)))
    mode = kCopyVec;
  const int count = (int)(u1 - u0);
  uint8_t* ring = smem + warp * 2 * C::HALF;
  const uint32_t ring32 = smem_u32(ring);
  // fp32: bytes from row to row, which a box of whole rows lays end to end
  const int pitch = mode == kCopyTma ? p.c.dim * 4 : DPAD * 4;
  auto chunk_at = [&](int row, int ch) -> int {
    return C::k16 ? (ch >> 3) * C::SUB + row * 128 + ((ch ^ row) & 7) * 16 : row * pitch + ch * 16;
  };
  Walk ahead = cur;
  // Lanes copying: offset of this lane's row (lanes below RW) of tile `w`, or -1 when the row is
  // past the end or its page is bad.
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
  // TMA: where the boxes of 32 tiles lie, a tile to a lane, looked up 32 tiles ahead so that no
  // tile waits for its page number.  page -1: nothing to fetch; -2: a bad page.
  struct Boxes {
    int page, tok, head;
  };
  // sub-tiles past head_dim are never fetched: they stay the zeros they are made here
  const int boxes = C::k16 ? (p.c.dim + 63) / 64 : 1;
  const uint32_t fetched = C::k16 ? 2 * boxes * C::SUB : 2 * RW * pitch;  // bytes of a warp's tile
  if (C::k16 && mode == kCopyTma && boxes < C::SUBS) {
    for (int i = 0; i < NS; ++i)
      for (int h = 0; h < 2; ++h)
        for (int j = boxes * (C::SUB / 16) + lane; j < C::HALF / 16; j += 32)
          *reinterpret_cast<uint4*>(ring + i * C::STAGE + h * C::HALF + j * 16) = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  Boxes now = {-1, 0, 0}, next = {-1, 0, 0};
  auto look_up = [&](int first) -> Boxes {  // tiles first .. first + 31 of this share; `ahead` is the first
    Boxes b = {-1, 0, 0};
    Walk w = ahead;
    w.t += lane;
    walk_carry<TK>(p, w);
    const int pos = w.t * TK + warp * RW;
    if (first + lane < count && pos < w.len) {
      const int blk = (int)((unsigned)pos / (unsigned)p.c.page_size);
      b.page = p.c.table[w.s * p.c.table_stride + blk];
      b.tok = pos - blk * p.c.page_size;
      b.head = w.hb / p.gblocks;
      if (b.page < 0 || b.page >= p.c.num_pages) {
        atomicOr(p.c.err, kCacheBadPage);
        b.page = -2;
      }
    }
    ahead.t += 32;
    if (first + 32 < count) walk_carry<TK>(p, ahead);
    return b;
  };
  long long off = -1;
  if (mode == kCopyTma) {
    now = look_up(0);
    if (count > 32) next = look_up(32);
  } else {
    off = row_offset(ahead);
  }
  CopyRing stages;
  auto issue = [&](int i, int stage) {  // tile i of this share
    uint8_t* kdst = ring + stage * C::STAGE;
    uint8_t* vdst = kdst + C::HALF;
    if (mode == kCopyTma) {
      if (i > 0 && (i & 31) == 0) {
        now = next;
        if (i + 32 < count) next = look_up(i + 32);
      }
      const int page = __shfl_sync(0xffffffffu, now.page, i & 31), tok = __shfl_sync(0xffffffffu, now.tok, i & 31);
      const int head = __shfl_sync(0xffffffffu, now.head, i & 31);
      if (page == -1 || !stages.arm(stage)) return;  // all of the rows are past the end: the tile is skipped
      if (page < 0) {
        for (int j = lane; j < 2 * C::HALF / 16; j += 32) reinterpret_cast<uint4*>(kdst)[j] = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[stage]);
        return;
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[stage], fetched);
        const int c1 = p.heads_inner ? head : tok, c2 = p.heads_inner ? tok : head;
#pragma unroll
        for (int j = 0; j < (C::k16 ? C::SUBS : 1); ++j) {
          if (j >= boxes) break;
          tma_load_4d(&p.map_k, &full[stage], kdst + j * C::SUB, j * C::SPAN, c1, c2, page);
          tma_load_4d(&p.map_v, &full[stage], vdst + j * C::SUB, j * C::SPAN, c1, c2, page);
        }
      }
    } else if (mode == kCopyVec) {
      // 32 lanes cover 32 / CH rows (or a part of one row), chunk by chunk
#pragma unroll
      for (int i = 0; i < RW * C::CH / 32; ++i) {
        const int e = i * 32 + lane, r = e / C::CH, ch = e - r * C::CH;
        const long long o = __shfl_sync(0xffffffffu, off, r);
        const bool ok = o >= 0 && ch * (int)(16 / sizeof(T)) < p.c.dim;
        const long long at = ok ? o + ch * (int)(16 / sizeof(T)) : 0;
        const int d = chunk_at(r, ch);
        cp_async_16_zfill(smem_u32(kdst + d), static_cast<const T*>(p.c.k) + at, ok);
        cp_async_16_zfill(smem_u32(vdst + d), static_cast<const T*>(p.c.v) + at, ok);
      }
    } else {
      constexpr int PER = 16 / sizeof(T);
      for (int r = 0; r < RW; ++r) {
        const long long o = __shfl_sync(0xffffffffu, off, r);
        for (int e = lane; e < DPAD; e += 32) {
          const bool ok = o >= 0 && e < p.c.dim;
          const int d = chunk_at(r, e / PER) + e % PER * (int)sizeof(T);
          *reinterpret_cast<T*>(kdst + d) = ok ? static_cast<const T*>(p.c.k)[o + e] : from_float<T>(0.0f);
          *reinterpret_cast<T*>(vdst + d) = ok ? static_cast<const T*>(p.c.v)[o + e] : from_float<T>(0.0f);
        }
      }
    }
  };
  // lanes copying: the next tile's table entries are read a tile before its rows are asked for
  auto advance = [&](int issued) {
    if (mode != kCopyTma && issued < count) {
      walk_next<TK>(p, ahead);
      off = row_offset(ahead);
    }
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    if (i < count) {
      issue(i, i);
      advance(i + 1);
    }
    cp_async_commit();
  }

  // ---- running state of this warp
  uint32_t koff[4], voff[4];  // ldmatrix addresses of the four 16-element steps of a sub-tile
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    koff[k] = (uint32_t)chunk_at(lane & 15, 2 * k + (lane >> 4));
    voff[k] = (uint32_t)chunk_at((lane & 7) + (lane >> 4) * 8, 2 * k + ((lane >> 3) & 1));
  }
  float o[NR / 4][4], m[MLR], l[MLR];
  uint32_t qf[C::k16 ? GB / 8 : 1][C::k16 ? DPAD / 16 : 1][2];  // 16-bit: queries as MMA fragments
  auto begin_segment = [&]() {
#pragma unroll
    for (int i = 0; i < NR; ++i) o[i / 4][i & 3] = 0.0f;
#pragma unroll
    for (int i = 0; i < MLR; ++i) {
      m[i] = kNothing;
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
  auto compute = [&](int stage, unsigned unit) {
    const int left = cur.len - cur.t * TK - warp * RW;  // valid rows of this warp
    if (left <= 0) return;
    uint8_t* tile = ring + stage * C::STAGE;
    if (mode == kCopyTma) {
      const bool landed = mbar_wait(&full[stage], stages.parity_of(stage), abort_flag, kTimeoutNs);
      if (!landed && lane == 0) atomicOr(p.c.err, kWaitExpired);
      stages.waited(stage, landed);
      if (left < RW) {
        // what lies behind the end of the cache may be anything, and 0 * NaN is NaN
        if constexpr (C::k16) {
          for (int i = lane; i < (RW - left) * C::CH; i += 32)
            *reinterpret_cast<uint4*>(tile + C::HALF + chunk_at(left + i / C::CH, i % C::CH)) = make_uint4(0, 0, 0, 0);
        } else {
          for (int i = left * pitch + lane * 16; i < RW * pitch; i += 512)
            *reinterpret_cast<uint4*>(tile + C::HALF + i) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
    }
    if constexpr (C::k16) {
      constexpr int NT = GB / 8, KD = DPAD / 16;
      const uint32_t kb = ring32 + stage * C::STAGE, vb = kb + C::HALF;
      // S^T = K Q^T: tokens are the rows, heads the columns of the MMA
      float sc[NT][2][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][0][i] = sc[n][1][i] = 0.0f;
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        uint32_t a[4];
        ldmatrix_x4(kb + koff[k & 3] + (k >> 2) * C::SUB, a);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_16816<T>(sc[n][k & 1], a, qf[n][k][0], qf[n][k][1]);
      }
      const int r0 = lane >> 2;
      float t[NT][4];  // scores in log2 units, less the running reference
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) t[n][i] = (sc[n][0][i] + sc[n][1][i]) * p.scale_log2;
      if (left < RW) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (r0 + (i < 2 ? 0 : 8) >= left) t[n][i] = -INFINITY;
      }
      if constexpr (WTS) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int h = n * 8 + (lane & 3) * 2;
          float* lg = p.logits + ((long long)unit * TK + warp * RW + r0) * p.lstride + h;
          if (h < p.lstride) {
            if (r0 < left) *reinterpret_cast<float2*>(lg) = make_float2(t[n][0], t[n][1]);
            if (r0 + 8 < left) *reinterpret_cast<float2*>(lg + 8 * p.lstride) = make_float2(t[n][2], t[n][3]);
          }
        }
      }
      // O^T += V^T P^T: output dims are the rows.  P^T is the B operand, 8 x 8 blocks transposed in registers; the
      // probabilities enter the product as a sum of two 16-bit parts, so that y carries one rounding, its
      // own.  SCALED: each head's largest of the sixteen is brought to [2^14, 2^15) first, its sums with
      // it, and these back afterwards: by powers of two, exactly.
      auto add_values = [&](auto tag) {
        constexpr bool SCALED = decltype(tag)::value;
        float e[NT][4], f[SCALED ? MLR : 1], back[SCALED ? MLR : 1];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) e[n][i] = exp2_from(t[n][i], m[n * 2 + (i & 1)]);
          l[n * 2] += e[n][0] + e[n][2];
          l[n * 2 + 1] += e[n][1] + e[n][3];
        }
        if constexpr (SCALED) {
#pragma unroll
          for (int i = 0; i < MLR; ++i) {
            float x = fmaxf(e[i >> 1][i & 1], e[i >> 1][2 + (i & 1)]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            // biased exponents: 268 - that of x, no more than 2^64, by which no sum overflows
            const uint32_t up = min(268u - (__float_as_uint(x) >> 23), 191u);
            f[i] = __uint_as_float(up << 23);
            back[i] = __uint_as_float((254u - up) << 23);
            e[i >> 1][i & 1] *= f[i];
            e[i >> 1][2 + (i & 1)] *= f[i];
          }
#pragma unroll
          for (int i = 0; i < NR; ++i) o[i / 4][i & 3] *= f[i / (KD * 4) * 2 + (i & 1)];
        }
        uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t lo0, lo1;
          const uint32_t hi0 = pack_split<T>(e[n][0], e[n][1], &lo0), hi1 = pack_split<T>(e[n][2], e[n][3], &lo1);
          ph[n][0] = movmatrix_trans(hi0);
          ph[n][1] = movmatrix_trans(hi1);
          pl[n][0] = movmatrix_trans(lo0);
          pl[n][1] = movmatrix_trans(lo1);
        }
#pragma unroll
        for (int k = 0; k < KD; ++k) {
          uint32_t a[4];
          ldmatrix_x4_trans(vb + voff[k & 3] + (k >> 2) * C::SUB, a);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_16816<T>(o[n * KD + k], a, ph[n][0], ph[n][1]);
            mma_16816<T>(o[n * KD + k], a, pl[n][0], pl[n][1]);
          }
        }
        if constexpr (SCALED) {
#pragma unroll
          for (int i = 0; i < NR; ++i) o[i / 4][i & 3] *= back[i / (KD * 4) * 2 + (i & 1)];
        }
      };
      // The reference is raised, and what is summed so far scaled down, only when a score passes it
      // by more than 2^8: it need not be the maximum, only keep the powers in range.
      //
      // fp16 ends at 2^-24, where the tokens behind one that dominates may still add up to all of y.  Its
      // reference therefore lies 2^11 below the maximum and is raised by scores 2^15 above it; and a tile in
      // which a lane's two scores of a head lie 2^8 or more below is looked at again: where a head has no
      // score at its reference, its probabilities are scaled.  One vote asks for both.  (us without any of this
      // and with: 32 x up to 8192 of 128 112.3 and 113.1, 64 x 4096 of 64 102.1 and 103.5, 16 x 4096 of 256 89.5
      // and 92.4; with all tiles looked at again 115.5, 105.8 and 92.9, all of them scaled 117.5, 106.5 and 106.6.)
      constexpr float kBelow = C::kScaled ? 11.0f : 0.0f, kAbove = C::kScaled ? 15.0f : 8.0f;
      bool grew = false, low = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) grew |= t[n][i] - m[n * 2 + (i & 1)] > kAbove;
        if constexpr (C::kScaled) {
#pragma unroll
          for (int c = 0; c < 2; ++c) low |= !(fmaxf(t[n][c], t[n][2 + c]) - m[n * 2 + c] > -8.0f);
        }
      }
      if (__any_sync(0xffffffffu, grew || low)) {
        float f[MLR];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int i = n * 2 + c;
            float x = fmaxf(t[n][c], t[n][2 + c]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            x = fmaxf(x - kBelow, m[i]);
            f[i] = exp2_from(m[i], x);
            l[i] *= f[i];
            m[i] = x;
          }
#pragma unroll
        for (int i = 0; i < NR; ++i) o[i / 4][i & 3] *= f[i / (KD * 4) * 2 + (i & 1)];
        if constexpr (C::kScaled) {
          // does some head have no score at its reference in the tile?  (its lanes are four apart)
          uint32_t all = ~0u;
#pragma unroll
          for (int i = 0; i < MLR; ++i) {
            uint32_t b = __ballot_sync(0xffffffffu, fmaxf(t[i >> 1][i & 1], t[i >> 1][2 + (i & 1)]) >= m[i]);
            b |= b >> 16;
            b |= b >> 8;
            all &= b | b >> 4;
          }
          if ((all & 15) != 15) {
            add_values(std::true_type());
            return;
          }
        }
      }
      add_values(std::false_type());
    } else {
      // fp32 on the FMA units: lane = (token of eight, quarter of the row) for the scores, a
      // chunk of four output dims for the products
      constexpr int RB = RW / 8;  // tokens of a lane
      const float4* q4 = reinterpret_cast<const float4*>(qs);
      const int key = lane >> 2, part = lane & 3;
      float s[RB][GB];
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int g = 0; g < GB; ++g) s[b][g] = 0.0f;
      // Four lanes to a token take every fourth chunk.  Where rows start on the same banks, odd tokens
      // take the chunks of a pair of steps in the other order: all eight groups of banks at once.
      const int chunks = (p.c.dim + 3) >> 2;
      const int flip = pitch % 128 == 0 ? (key & 1) << 2 : 0;
#pragma unroll 4
      for (int i = 0; i < chunks; i += 4) {
        const int ch = i + part < chunks && (i ^ flip) + part < chunks ? (i ^ flip) + part : i + part;
        if (ch >= chunks) continue;
        float4 x[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) x[b] = *reinterpret_cast<const float4*>(tile + chunk_at(key + 8 * b, ch));
#pragma unroll
        for (int g = 0; g < GB; ++g) {
          const float4 y = q4[g * (DPAD / 4) + ch];
#pragma unroll
          for (int b = 0; b < RB; ++b)
            s[b][g] = fmaf(x[b].x, y.x, fmaf(x[b].y, y.y, fmaf(x[b].z, y.z, fmaf(x[b].w, y.w, s[b][g]))));
        }
      }
      bool grew = false;
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int g = 0; g < GB; ++g) {
          float& v = s[b][g];
          v += __shfl_xor_sync(0xffffffffu, v, 1);
          v += __shfl_xor_sync(0xffffffffu, v, 2);
          v = key + 8 * b < left ? v * p.scale_log2 : -INFINITY;
          grew |= v - m[g] > 8.0f;
          if constexpr (WTS) {
            if (part == 0 && key + 8 * b < left && g < p.lstride)
              p.logits[((long long)unit * TK + warp * RW + key + 8 * b) * p.lstride + g] = v;
          }
        }
      if (__any_sync(0xffffffffu, grew)) {  // as above
#pragma unroll
        for (int g = 0; g < GB; ++g) {
          float x = s[0][g];
          if constexpr (RB > 1) x = fmaxf(x, s[RB - 1][g]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          x = fmaxf(x, m[g]);
          const float f = exp2_from(m[g], x);
          l[g] *= f;
          m[g] = x;
#pragma unroll
          for (int i = 0; i < C::CPL * 4; ++i) o[g * C::CPL + i / 4][i & 3] *= f;
        }
      }
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int g = 0; g < GB; ++g) {
          s[b][g] = exp2_from(s[b][g], m[g]);
          l[g] += s[b][g];
        }
#pragma unroll
      for (int r = 0; r < RW; ++r) {
#pragma unroll
        for (int ci = 0; ci < C::CPL; ++ci) {
          const int ch = lane + 32 * ci;
          const float4 x = ch < (p.c.dim + 3) >> 2 ? *reinterpret_cast<const float4*>(tile + C::HALF + chunk_at(r, ch))
                                      : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int g = 0; g < GB; ++g) {
            const float w = __shfl_sync(0xffffffffu, s[r / 8][g], r % 8 * 4);
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
  auto end_segment = [&](unsigned begin, unsigned end) {
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
#pragma unroll 2
        for (int i = tid; i < cur.len; i += kThreads) {
          const float* lg = p.logits + ((long long)begin * TK + i) * p.lstride;
          float sum = 0.0f;
          for (int g = 0; g < heads; ++g) sum += exp2_from(lg[g], fin[g]) * fin[GB + g];
          wout[i] = (win ? win[i] : 0.0f) + sum;
        }
      }
    }
  };

  if (!p.whole) {
    if (tid < 2) p.pieces[me * 2 + tid].s = -1;
    clear_empty();
  }
  __syncthreads();
  bool fresh = true;
  for (int i = 0; i < count; ++i) {
    if (fresh) begin_segment();
    if (mode != kCopyTma) cp_async_wait<NS - 2>();
    __syncwarp();  // every lane is done with the tile before this one (and this one's copies have landed)
    if (i + NS - 1 < count) {
      issue(i + NS - 1, (i + NS - 1) % NS);
      advance(i + NS);
    }
    cp_async_commit();
    compute(i % NS, u0 + i);
    fresh = cur.t + 1 == cur.nt;
    if (fresh || i + 1 == count) {
      const unsigned begin = cur.base, end = begin + cur.nt;
      end_segment(begin, end);
      if (tid == 0 && (begin < u0 || end > u1)) {
        Piece& r = p.pieces[me * 2 + (begin >= u0 ? 1 : 0)];
        r.hb = cur.hb;
        const AttnShares shares(units, workers);
        r.w0 = shares.owner(begin);
        r.w1 = shares.owner(end - 1);
        r.begin = begin;
        r.lo = begin >= u0 ? begin : u0;
        r.hi = end <= u1 ? end : u1;
        r.s = cur.s;
      }
      // its first worker records a split segment for the join, a whole one that there is nothing to
      if (!p.whole && p.by_segment && tid == 0 && begin >= u0)
        p.segs[cur.s * p.hblocks + cur.hb] = {me, end > u1 ? AttnShares(units, workers).owner(end - 1) : -1};
    }
    if (i + 1 < count) walk_next<TK>(p, cur);
  }
  // after an expired wait: copies in flight land before the shared memory goes away
  if (stages.flight) {
    for (int i = 0; i < NS; ++i) {
      volatile int dummy = 0;
      if (stages.flight >> i & 1) mbar_wait(&full[i], stages.parity_of(i), &dummy, kDrainNs);
    }
  }
}

// ------------------------------------------------------------------ join
// Joins the partials of split segments by an online softmax, four output registers (a slice) to a
// warp.  A chain of dependent loads and launches bounds it, so its blocks are laid out for one
// round of loads:
//   by_segment (few segments, of many workers each): a block per (segment, slice), the workers
//     dealt to its sixteen warps, whose states meet in a tree;
//   else: a block per worker, which joins the segment whose second worker it is, its warps dealt
//     to the slices first and to the workers with what is left.
// With weights the first blocks, one per worker, turn the scores of the worker's own tokens in
// split segments into probabilities.
// (8 heads of 32768 tokens, 37 workers each: 40.3 us with the second layout alone, 31.9 with both.)
template <typename T, int DPAD, int GB, bool WTS>
__global__ void __launch_bounds__(kJoinWarps * 32) attention_join_kernel(const __grid_constant__ AttnParams p) {
  using C = Tile<T, DPAD, GB>;
  constexpr int TK = C::TK, NR = C::NR, SLICES = NR / 4;
  constexpr int GROUPS = SLICES >= kJoinWarps ? 1 : kJoinWarps / SLICES;  // warps that share a slice
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int weight_blocks = WTS ? p.workers : 0;
  if ((int)blockIdx.x >= weight_blocks) {
    const int job = blockIdx.x - weight_blocks;
    int s, hb, w0, w1, slice, slice_step, group, groups;
    if (p.by_segment) {
      const int seg = job / SLICES;
      const Segment rec = p.segs[seg];
      if (rec.w1 < 0) return;
      s = seg / p.hblocks;
      hb = seg - s * p.hblocks;
      w0 = rec.w0;
      w1 = rec.w1;
      slice = job - seg * SLICES;
      slice_step = SLICES;
      group = warp;
      groups = kJoinWarps;
    } else {
      const Piece pc = p.pieces[job * 2];
      if (pc.s < 0 || pc.w0 + 1 != job) return;
      s = pc.s;
      hb = pc.hb;
      w0 = pc.w0;
      w1 = pc.w1;
      slice = warp / GROUPS;
      slice_step = kJoinWarps / GROUPS;
      group = warp % GROUPS;
      groups = GROUPS;
    }
    __shared__ float sm[kJoinWarps][32][9];
    for (; slice < SLICES; slice += slice_step) {
      const int i0 = slice * 4;
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
      float m0 = kNothing, m1 = kNothing, l0 = 0.0f, l1 = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      auto add = [&](float a0, float a1, float b0, float b1, const float(&x)[4]) {
        const float t0 = fmaxf(m0, a0), t1 = fmaxf(m1, a1);
        const float f0 = exp2_from(m0, t0), f1 = exp2_from(m1, t1), e0 = exp2_from(a0, t0), e1 = exp2_from(a1, t1);
        m0 = t0;
        m1 = t1;
        l0 = l0 * f0 + b0 * e0;
        l1 = l1 * f1 + b1 * e1;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = C::k16 && (i & 1) ? o[i] * f1 + x[i] * e1 : o[i] * f0 + x[i] * e0;
      };
      constexpr int U = 4;  // partials in flight
      for (int wb = w0 + group; wb <= w1; wb += U * groups) {
        float x[U][4], a0[U], a1[U], b0[U], b1[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int w = wb + u * groups, slot = w * 2 + (w == w0 ? 1 : 0);
          a0[u] = a1[u] = kNothing;
          b0[u] = b1[u] = x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.0f;
          if (w > w1) continue;
          const float* ml = p.ml + (size_t)slot * 2 * GB;
          const float* src = p.part + ((size_t)slot * NR + i0) * 32 + lane;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[u][i] = src[i * 32];
          a0[u] = ml[h0];
          a1[u] = ml[h1];
          b0[u] = ml[GB + h0];
          b1[u] = ml[GB + h1];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) add(a0[u], a1[u], b0[u], b1[u], x[u]);
      }
      // the warps of a slice meet in a tree (blocks whose warps all have their own slice loop instead)
      const int live = min(groups, w1 - w0 + 1);  // the others have nothing
      for (int step = kJoinWarps / 2; step > 0; step >>= 1) {
        if (step >= live) continue;
        if (group >= step && group < 2 * step) {
          float* mine = sm[warp][lane];
          mine[0] = m0;
          mine[1] = m1;
          mine[2] = l0;
          mine[3] = l1;
#pragma unroll
          for (int i = 0; i < 4; ++i) mine[4 + i] = o[i];
        }
        __syncthreads();
        if (group < step && group + step < live) {
          const float* x = sm[warp + step][lane];
          const float xo[4] = {x[4], x[5], x[6], x[7]};
          add(x[0], x[1], x[2], x[3], xo);
        }
      }
      if (group == 0) {
        const int kvh = hb / p.gblocks, g0 = (hb - kvh * p.gblocks) * GB;
        const int heads = min(GB, p.group - g0);
        T* y = static_cast<T*>(p.y) + s * p.y_seq + (long long)(kvh * p.group + g0) * p.y_head;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int h = C::k16 && (i & 1) ? h1 : h0;
          if (h < heads && d[i] < p.c.dim) y[h * p.y_head + d[i]] = from_float<T>(o[i] / (C::k16 && (i & 1) ? l1 : l0));
        }
      }
    }
    return;
  }
  if constexpr (WTS) {
    const int me = blockIdx.x;
    __shared__ float top[GB], inv[GB];
    for (int kind = 0; kind < 2; ++kind) {
      const Piece pc = p.pieces[me * 2 + kind];
      if (pc.s < 0) continue;
      const int len = p.c.lens[pc.s];
      for (int g = warp; g < p.group; g += kJoinWarps) {
        float m = kNothing, l = 0.0f;
        for (int w = pc.w0 + lane; w <= pc.w1; w += 32) {
          const int slot = w * 2 + (w == pc.w0 ? 1 : 0);
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
      // this worker's tokens of the segment
      const int t0 = (int)(pc.lo - pc.begin) * TK, t1 = min(len, (int)(pc.hi - pc.begin) * TK);
      constexpr int U = 4;  // tokens of a thread in flight
      constexpr int step = kJoinWarps * 32;
      for (int i0 = t0 + tid; i0 < t1; i0 += U * step) {
        float w[U], sum[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * step;
          w[u] = win && i < t1 ? win[i] : 0.0f;
          sum[u] = 0.0f;
        }
        const float* lg = p.logits + ((long long)pc.begin * TK + i0) * p.lstride;
        const long long lstep = (long long)step * p.lstride;
        if (C::k16) {  // an even number of scores per token
          for (int g = 0; g < p.lstride; g += 2) {
            float2 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
              x[u] = i0 + u * step < t1 ? *reinterpret_cast<const float2*>(lg + u * lstep + g) : make_float2(0.0f, 0.0f);
#pragma unroll
            for (int u = 0; u < U; ++u) {
              sum[u] += exp2_from(x[u].x, top[g]) * inv[g];
              if (g + 1 < p.group) sum[u] += exp2_from(x[u].y, top[g + 1]) * inv[g + 1];
            }
          }
        } else {
          for (int g = 0; g < p.group; ++g)
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (i0 + u * step < t1) sum[u] += exp2_from(lg[u * lstep + g], top[g]) * inv[g];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i0 + u * step < t1) wout[i0 + u * step] = w[u] + sum[u];
      }
      __syncthreads();
    }
  }
}

// CTAs of a launch and the bytes of the parts of its workspace.
template <typename T, int DPAD, int GB>
AttnPlan attention_plan_for(const AttnParams& p, int sms, bool weights) {
  using C = Tile<T, DPAD, GB>;
  const long long tiles = ((long long)p.capacity + C::TK - 1) / C::TK;
  const long long segments = (long long)p.c.seqs * p.hblocks, units = tiles * segments;  // at most
  AttnPlan pl;
  // Short caches, a CTA each: the join costs more than the few tiles in a row (333 tokens, 4
  // heads of 64: 10.2 us split, 8.7 whole)
  pl.whole = tiles <= kWholeTiles && segments <= (long long)sms * C::CTAS;
  pl.workers = pl.whole ? (int)segments : (int)std::min<long long>(units, (long long)sms * C::CTAS);
  pl.part = pl.whole ? 0 : up256((size_t)pl.workers * 2 * C::NR * 32 * 4);
  pl.ml = pl.whole ? 0 : up256((size_t)pl.workers * 2 * 2 * GB * 4);
  pl.pieces = pl.whole ? 0 : up256((size_t)pl.workers * 2 * sizeof(Piece));
  pl.by_segment = segments * (C::NR / 4) <= 2 * sms;  // a block each in one round
  pl.segs = pl.whole || !pl.by_segment ? 0 : up256((size_t)segments * sizeof(Segment));
  pl.lstride = C::k16 ? (p.group + 1) / 2 * 2 : p.group;
  pl.logits = weights ? up256((size_t)units * C::TK * pl.lstride * 4) : 0;
  return pl;
}

// Tensor maps of the pools for boxes of a warp's rows of one head, when their layout allows: false
// leaves the copies to the lanes.
template <typename C, typename T>
bool attention_maps(AttnParams* p) {
  const CacheView& c = p->c;
  if (!p->vec || c.page_size % C::RW) return false;
  const long long tok = c.token_stride, head = c.head_stride;
  p->heads_inner = head <= tok;
  const long long in = p->heads_inner ? head : tok, out = p->heads_inner ? tok : head;
  if (in <= 0 || out % in || c.page_stride < out || c.page_stride % out) return false;
  const int n_in = p->heads_inner ? c.kv_heads : c.page_size, n_out = p->heads_inner ? c.page_size : c.kv_heads;
  const int b_in = p->heads_inner ? 1 : C::RW, b_out = p->heads_inner ? C::RW : 1;
  const uint64_t dims[4] = {(uint64_t)c.dim, (uint64_t)n_in, (uint64_t)n_out, (uint64_t)c.num_pages};
  const uint64_t strides[3] = {(uint64_t)in * sizeof(T), (uint64_t)out * sizeof(T), (uint64_t)c.page_stride * sizeof(T)};
  const uint32_t box[4] = {C::k16 ? 64u : (uint32_t)c.dim, (uint32_t)b_in, (uint32_t)b_out, 1};
  if (c.dim < 16 / (int)sizeof(T) || strides[2] >= (1ull << 40)) return false;
  return encode_tiled_4d(&p->map_k, c.k, sizeof(T), dims, strides, box) == 0 &&
         encode_tiled_4d(&p->map_v, c.v, sizeof(T), dims, strides, box) == 0;
}

template <typename T, int DPAD, int GB, bool WTS>
int attention_launch_for(AttnParams& p, const AttnPlan& pl, cudaStream_t st) {
  using C = Tile<T, DPAD, GB>;
  p.mode = attention_maps<C, T>(&p) ? kCopyTma : p.vec ? kCopyVec : kCopyElements;
  p.whole = pl.whole ? (p.capacity + C::TK - 1) / C::TK : 0;
  p.lstride = pl.lstride;
  p.workers = pl.workers;
  p.by_segment = !pl.whole && pl.by_segment;
  auto* kernel = attention_kernel<T, DPAD, GB, WTS>;
  SPINN_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
  const int rc = launch_dependent(kernel, dim3(pl.workers), kThreads, C::SMEM, st, p);
  if (rc || pl.whole) return rc;
  const int jobs = p.by_segment ? p.c.seqs * p.hblocks * (C::NR / 4) : pl.workers;
  return launch_dependent(attention_join_kernel<T, DPAD, GB, WTS>, dim3((WTS ? pl.workers : 0) + jobs), kJoinWarps * 32, 0,
                          st, p);
}

// The instantiation for a head size and group: `go` gets the Tile as a tag.
template <typename T, typename F>
auto attention_dispatch(int dim, int group, F go) {
  constexpr int SMALL = sizeof(T) == 2 ? 8 : 1, LARGE = sizeof(T) == 2 ? 16 : 8;
  auto by_dim = [&](auto gb) {
    constexpr int GB = decltype(gb)::value;
    if (dim <= 64) return go(Tile<T, 64, GB>());
    if constexpr (sizeof(T) == 4) {
      if (dim <= 96) return go(Tile<T, 96, GB>());
    }
    if (dim <= 128) return go(Tile<T, 128, GB>());
    if constexpr (sizeof(T) == 2) {
      if (dim <= 192) return go(Tile<T, 192, GB>());
    }
    return go(Tile<T, 256, GB>());
  };
  if (group <= SMALL) return by_dim(std::integral_constant<int, SMALL>());
  if constexpr (sizeof(T) == 4) {
    if (group <= 4) return by_dim(std::integral_constant<int, 4>());
  }
  return by_dim(std::integral_constant<int, LARGE>());
}

template <typename T>
AttnPlan attention_plan_t(const AttnParams& p, int sms, bool weights) {
  return attention_dispatch<T>(p.c.dim, p.group, [&](auto t) {
    using C = decltype(t);
    return attention_plan_for<T, C::DPAD, C::GB>(p, sms, weights);
  });
}
template <typename T>
int attention_launch_t(AttnParams& p, const AttnPlan& pl, cudaStream_t st) {
  return attention_dispatch<T>(p.c.dim, p.group, [&](auto t) {
    using C = decltype(t);
    return p.wout ? attention_launch_for<T, C::DPAD, C::GB, true>(p, pl, st)
                  : attention_launch_for<T, C::DPAD, C::GB, false>(p, pl, st);
  });
}

}  // namespace
}  // namespace spinn
