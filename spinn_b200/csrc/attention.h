// attention.h -- parameters of the paged attention launch (attention.cuh), and the instantiations
// for each cache type, one translation unit each.
#pragma once
#include <cuda.h>

#include "cache.h"

namespace spinn {

// What a worker leaves for the join: its first segment when an earlier worker began it (kind 0),
// and its last one when a later worker ends it (kind 1).  A segment is one (sequence, head
// block); it begins at unit `begin`, w0 / w1 are its first and last worker, and [lo, hi) are this
// worker's own units of it.
struct Piece {
  int s, hb;  // s < 0: none
  int w0, w1;
  unsigned begin, lo, hi;
};

// First and last worker of a segment, for a join by segments; w1 < 0: nothing to join.
struct Segment {
  int w0, w1;
};

// Bookkeeping of a warp's ring of stages that TMA fills.  Once a wait has expired nothing is armed any
// more: a stage whose copy is still in flight may not be armed again, and it is that copy's phase
// that has to end before the shared memory is given up.
struct CopyRing {
  unsigned parity = 0;  // bit s: of the next wait for stage s
  unsigned flight = 0;  // bit s: armed, not yet seen to land
  bool expired = false;
  __host__ __device__ bool arm(int s) {
    if (!expired) flight |= 1u << s;
    return !expired;
  }
  __host__ __device__ unsigned parity_of(int s) const { return parity >> s & 1; }
  __host__ __device__ void waited(int s, bool landed) {
    parity ^= (unsigned)landed << s;
    flight &= ~((unsigned)landed << s);
    expired |= !landed;
  }
};

enum AttnCopy { kCopyElements = 0, kCopyVec = 1, kCopyTma = 2 };

struct AttnParams {
  CUtensorMap map_k, map_v;  // kCopyTma: boxes of a warp's rows of one head
  CacheView c;
  const void* q;
  void* y;
  long long q_seq, q_head, y_seq, y_head;
  int q_heads, group, gblocks, hblocks;  // hblocks = kv_heads * gblocks
  int capacity;                          // longest allowed length
  bool vec;                              // 16-byte rows
  bool heads_inner;                      // the maps' second dimension is the head, not the token
  int mode;                              // AttnCopy
  int whole;                             // tiles to number per CTA when nothing is split, else 0
  int lstride;                           // scores kept per token (weights only)
  float scale_log2;
  const float* win;
  float* wout;
  long long win_seq, win_head, wout_seq, wout_head;
  float* part;    // [worker][2][NR * 32] unnormalised outputs, in register order
  float* ml;      // [worker][2][2][GB] maxima and sums
  Piece* pieces;  // [worker][2]
  Segment* segs;  // [sequence][head block], by_segment only
  int workers;
  bool by_segment;  // layout of the join
  float* logits;  // [unit][TK][lstride], scores in log2 units (weights only)
};

// CTAs of a launch and the bytes of each part of its workspace.
struct AttnPlan {
  bool whole;  // one CTA per (sequence, head block), nothing to join
  int workers, lstride;
  bool by_segment;
  size_t part, ml, pieces, segs, logits;
};

inline size_t up256(size_t b) { return (b + 255) & ~size_t(255); }

// Heads of one block: a wider group is split into blocks that each read the cache.
inline int attention_head_block(int bytes, int group) {
  const int small = bytes == 2 ? 8 : 1, large = bytes == 2 ? 16 : 8;
  return group <= small ? small : large;
}

AttnPlan attention_plan_fp16(const AttnParams& p, int sms, bool weights);
AttnPlan attention_plan_bf16(const AttnParams& p, int sms, bool weights);
AttnPlan attention_plan_fp32(const AttnParams& p, int sms, bool weights);
int attention_launch_fp16(AttnParams& p, const AttnPlan& pl, cudaStream_t st);
int attention_launch_bf16(AttnParams& p, const AttnPlan& pl, cudaStream_t st);
int attention_launch_fp32(AttnParams& p, const AttnPlan& pl, cudaStream_t st);

}  // namespace spinn
