// attention.cu -- entry points of the paged attention (kernels in attention.cuh).
#include <algorithm>

#include "attention.h"
#include "internal.h"

namespace spinn {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

int attention_params(const SpinnCudaCache* cache, const SpinnCudaPageTable* table, const SpinnCudaAttention* a,
                     AttnParams* p) {
  int rc = cache_view("paged_attention", cache, table, &p->c);
  if (rc) return rc;
  SPINN_CHECK_ARG(a && a->q && a->y, "paged_attention: q and y are required");
  SPINN_CHECK_ARG(a->q_heads > 0 && a->q_heads % cache->kv_heads == 0,
                  "paged_attention: %d query heads are no multiple of %d key heads", a->q_heads, cache->kv_heads);
  SPINN_CHECK_ARG(a->q_seq_stride >= 0 && a->q_head_stride >= 0 && a->y_seq_stride >= 0 && a->y_head_stride >= 0,
                  "paged_attention: negative stride");
  const int es = dtype_bytes(cache->dtype);
  SPINN_CHECK_ARG(((uintptr_t)a->q | (uintptr_t)a->y) % es == 0 &&
                      ((uintptr_t)a->weights_in | (uintptr_t)a->weights_out) % 4 == 0,
                  "paged_attention: misaligned pointer");
  p->q = a->q;
  p->y = a->y;
  p->q_seq = a->q_seq_stride;
  p->q_head = a->q_head_stride;
  p->y_seq = a->y_seq_stride;
  p->y_head = a->y_head_stride;
  p->q_heads = a->q_heads;
  p->group = a->q_heads / cache->kv_heads;
  const int gb = attention_head_block(es, p->group);
  p->gblocks = (p->group + gb - 1) / gb;
  SPINN_CHECK_ARG((long long)cache->kv_heads * p->gblocks <= 65535, "paged_attention: too many heads");
  p->hblocks = cache->kv_heads * p->gblocks;
  p->capacity = cache_capacity(table->max_pages, cache->page_size);
  // (a tile holds at least 32 tokens)
  SPINN_CHECK_ARG(((long long)p->capacity + 31) / 32 * table->seqs * p->hblocks <= kMaxUnits,
                  "paged_attention: %d sequences of up to %d tokens in %d head blocks are too much for one call", table->seqs,
                  p->capacity, p->hblocks);
  p->vec = cache_vec16(p->c, es);
  p->scale_log2 = a->scale * kLog2e;
  p->win = a->weights_in;
  p->wout = a->weights_out;
  p->win_seq = a->win_seq_stride;
  p->win_head = a->win_head_stride;
  p->wout_seq = a->wout_seq_stride;
  p->wout_head = a->wout_head_stride;
  SPINN_CHECK_ARG(!a->weights_in || a->weights_out, "paged_attention: weights_in without weights_out");
  if (a->weights_out) {
    SPINN_CHECK_ARG(p->gblocks == 1, "paged_attention: weights need at most %d query heads per key head, not %d", gb,
                    p->group);
    SPINN_CHECK_ARG(a->weights_capacity > 0 && a->win_seq_stride >= 0 && a->win_head_stride >= 0 &&
                        a->wout_seq_stride >= 0 && a->wout_head_stride >= 0,
                    "paged_attention: bad weights geometry");
    SPINN_CHECK_ARG(a->weights_in != a->weights_out ||
                        (a->win_seq_stride == a->wout_seq_stride && a->win_head_stride == a->wout_head_stride),
                    "paged_attention: weights in place need equal strides");
    p->capacity = std::min(p->capacity, a->weights_capacity);
  }
  return 0;
}

AttnPlan attention_plan(const AttnParams& p, int dtype, int sms) {
  const bool w = p.wout != nullptr;
  return dtype == SPINN_CUDA_FP16   ? attention_plan_fp16(p, sms, w)
         : dtype == SPINN_CUDA_BF16 ? attention_plan_bf16(p, sms, w)
                                    : attention_plan_fp32(p, sms, w);
}

}  // namespace

extern "C" {

__attribute__((visibility("default"))) size_t spinn_cuda_paged_attention_workspace(const SpinnCudaCache* cache,
                                                                                   const SpinnCudaPageTable* table,
                                                                                   const SpinnCudaAttention* a) {
  AttnParams p;
  int dev = 0;
  if (attention_params(cache, table, a, &p)) return 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  const AttnPlan pl = attention_plan(p, cache->dtype, sm_count(dev));
  return pl.part + pl.ml + pl.pieces + pl.segs + pl.logits;
}

__attribute__((visibility("default"))) int spinn_cuda_paged_attention(const SpinnCudaCache* cache,
                                                                      const SpinnCudaPageTable* table,
                                                                      const SpinnCudaAttention* a, void* workspace,
                                                                      size_t workspace_bytes, void* stream) {
  AttnParams p;
  int rc = attention_params(cache, table, a, &p);
  if (rc) return rc;
  const int es = dtype_bytes(cache->dtype);
  const Rows q = {a->q, es, cache->head_dim, {table->seqs, a->q_heads, 1}, {a->q_seq_stride, a->q_head_stride, 0}};
  const Rows y = {a->y, es, cache->head_dim, {table->seqs, a->q_heads, 1}, {a->y_seq_stride, a->y_head_stride, 0}};
  SPINN_CHECK_ARG(rows_distinct(y) && rows_apart(y, q), "paged_attention: rows of y overlap one another or q");
  if (a->weights_out) {
    const Rows wout = {a->weights_out, 4, a->weights_capacity, {table->seqs, cache->kv_heads, 1},
                       {a->wout_seq_stride, a->wout_head_stride, 0}};
    const Rows win = {a->weights_in, 4, a->weights_capacity, {table->seqs, cache->kv_heads, 1},
                      {a->win_seq_stride, a->win_head_stride, 0}};
    SPINN_CHECK_ARG(rows_distinct(wout), "paged_attention: rows of weights_out overlap");
    SPINN_CHECK_ARG(rows_apart(wout, q) && rows_apart(wout, y) && (!a->weights_in || rows_apart(win, y)),
                    "paged_attention: weights overlap y, or weights_out q");
    SPINN_CHECK_ARG(!a->weights_in || a->weights_in == a->weights_out || rows_apart(wout, win),
                    "paged_attention: weights_out must be weights_in itself or apart from it");
  }
  int dev;
  rc = check_stream_device("paged_attention", stream, &dev);
  if (rc) return rc;
  rc = decode_error_word(dev, &p.c.err);
  if (rc) return rc;
  const AttnPlan pl = attention_plan(p, cache->dtype, sm_count(dev));
  const size_t need = pl.part + pl.ml + pl.pieces + pl.segs + pl.logits;
  SPINN_CHECK_ARG(!need || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                  "paged_attention: workspace of %zu bytes (16-byte aligned) needed, %zu given", need, workspace_bytes);
  char* ws = static_cast<char*>(workspace);
  p.part = reinterpret_cast<float*>(ws);
  p.ml = reinterpret_cast<float*>(ws + pl.part);
  p.pieces = reinterpret_cast<Piece*>(ws + pl.part + pl.ml);
  p.segs = reinterpret_cast<Segment*>(ws + pl.part + pl.ml + pl.pieces);
  p.logits = reinterpret_cast<float*>(ws + pl.part + pl.ml + pl.pieces + pl.segs);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->dtype == SPINN_CUDA_FP16   ? attention_launch_fp16(p, pl, st)
         : cache->dtype == SPINN_CUDA_BF16 ? attention_launch_bf16(p, pl, st)
                                           : attention_launch_fp32(p, pl, st);
}

__attribute__((visibility("default"))) int spinn_cuda_diag_attention_ring(const int32_t* ops, int count, int32_t* out) {
  SPINN_CHECK_ARG(ops && out && count >= 0, "diag_attention_ring: invalid arguments");
  CopyRing r;
  for (int i = 0; i < count; ++i) {
    const int s = ops[i] & 15;
    SPINN_CHECK_ARG((ops[i] >> 4) >= 0 && (ops[i] >> 4) <= 2, "diag_attention_ring: operation %d", ops[i]);
    const bool armed = ops[i] >> 4 == 0 && r.arm(s);
    if (ops[i] >> 4) r.waited(s, ops[i] >> 4 == 1);
    out[3 * i] = armed;
    out[3 * i + 1] = (int32_t)r.parity;
    out[3 * i + 2] = (int32_t)r.flight;
  }
  return 0;
}

}  // extern "C"
}  // namespace spinn
