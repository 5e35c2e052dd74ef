// cache.cu -- the paged key-value cache: host checks shared by its entry points, appending new
// tokens, and eviction by accumulated attention weight.  Attention itself is in attention.cu.
#include <algorithm>
#include <atomic>

#include "cache.h"
#include "internal.h"
#include "launch.h"
#include "ptx.cuh"

namespace spinn {

constexpr int kMaxDevices = 64;

// One word per device, in the library's own image: no allocation, so that a first call may be a
// captured one.
__device__ unsigned g_decode_err = 0;

int decode_error_word(int device, unsigned** word) {
  static std::atomic<unsigned*> addr[kMaxDevices];
  SPINN_CHECK_ARG(device >= 0 && device < kMaxDevices, "device %d is past the %d supported", device, kMaxDevices);
  *word = addr[device].load();
  if (*word) return 0;
  void* p = nullptr;
  SPINN_CUDA_TRY(cudaGetSymbolAddress(&p, g_decode_err));
  *word = static_cast<unsigned*>(p);
  addr[device].store(*word);
  return 0;
}

int dtype_bytes(int dtype) {
  return dtype == SPINN_CUDA_FP32 ? 4 : (dtype == SPINN_CUDA_FP16 || dtype == SPINN_CUDA_BF16) ? 2 : 0;
}

// Clears what has been reported, and no more: another stream's kernel may raise an error meanwhile.
__global__ void clear_errors_kernel(unsigned* word, unsigned bits) { atomicAnd(word, ~bits); }

int check_stream_device(const char* who, void* stream, int* device) {
  SPINN_CUDA_TRY(cudaGetDevice(device));
  if (stream) {
    // a capturing stream may not be asked; a launch into one of another device fails by itself
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    SPINN_CUDA_TRY(cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &cap));
    if (cap != cudaStreamCaptureStatusNone) return 0;
    int sdev = -1;
    SPINN_CUDA_TRY(cudaStreamGetDevice(static_cast<cudaStream_t>(stream), &sdev));
    SPINN_CHECK_ARG(sdev == *device, "%s: stream belongs to device %d, the current device is %d", who, sdev, *device);
  }
  return 0;
}

int cache_view(const char* who, const SpinnCudaCache* c, const SpinnCudaPageTable* t, CacheView* v) {
  SPINN_CHECK_ARG(c && t, "%s: cache and page table are required", who);
  SPINN_CHECK_ARG(c->k && c->v && t->pages && t->lens, "%s: null pool, page table or lengths", who);
  SPINN_CHECK_ARG(dtype_bytes(c->dtype), "%s: element type %d not supported (fp32, fp16 or bf16)", who, c->dtype);
  SPINN_CHECK_ARG(c->num_pages > 0 && c->page_size > 0 && c->kv_heads > 0 && c->kv_heads <= 65535,
                  "%s: bad pool geometry (%d pages of %d tokens, %d heads)", who, c->num_pages, c->page_size,
                  c->kv_heads);
  SPINN_CHECK_ARG(c->head_dim > 0 && c->head_dim <= 256, "%s: head_dim %d outside [1, 256]", who, c->head_dim);
  SPINN_CHECK_ARG(c->page_stride >= 0 && c->token_stride >= 0 && c->head_stride >= 0, "%s: negative stride", who);
  SPINN_CHECK_ARG(t->seqs > 0 && t->max_pages > 0 && t->row_stride >= 0, "%s: bad page table (%d rows of %d)", who,
                  t->seqs, t->max_pages);
  v->k = c->k;
  v->v = c->v;
  v->page_stride = c->page_stride;
  v->token_stride = c->token_stride;
  v->head_stride = c->head_stride;
  v->num_pages = c->num_pages;
  v->page_size = c->page_size;
  v->kv_heads = c->kv_heads;
  v->dim = c->head_dim;
  v->table = t->pages;
  v->table_stride = t->row_stride;
  v->max_pages = t->max_pages;
  v->seqs = t->seqs;
  v->lens = t->lens;
  const int es = dtype_bytes(c->dtype);
  SPINN_CHECK_ARG(((uintptr_t)v->k | (uintptr_t)v->v) % es == 0 &&
                      ((uintptr_t)v->table | (uintptr_t)v->lens) % 4 == 0,
                  "%s: misaligned pointer", who);
  return 0;
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

bool cache_vec16(const CacheView& v, int bytes) {
  const int per = 16 / bytes;
  return aligned16(v.k) && aligned16(v.v) && v.dim % per == 0 && v.page_stride % per == 0 &&
         v.token_stride % per == 0 && v.head_stride % per == 0;
}

namespace {

// What rows cover in bytes, and whether their dimensions nest.
struct Extent {
  long long all;
  bool nested;
};

Extent extent(const Rows& r) {
  int order[3] = {0, 1, 2};
  std::sort(order, order + 3, [&](int a, int b) { return r.stride[a] < r.stride[b]; });
  Extent e = {r.width * r.bytes, true};
  for (int i : order) {
    if (r.count[i] <= 1) continue;
    const long long stride = r.stride[i] * r.bytes;
    e.nested &= stride >= e.all;
    e.all += (r.count[i] - 1) * stride;
  }
  return e;
}

}  // namespace

// A dimension of two operands: its stride in bytes, the steps of each, and what each covers below it.
struct Level {
  long long stride, na, nb, ea, eb;
};

// Whether b, d bytes behind a, meets no element of it: at each stride only the few relative steps at which
// what lies below may meet are followed.  More than a few (one operand's rows are longer than the
// other's stride) counts as meeting.
bool levels_apart(const Level* l, int levels, long long d, long long wa, long long wb) {
  if (!levels) return d >= wa || -d >= wb;
  const Level& v = l[levels - 1];
  const auto floor_div = [](long long x, long long y) { return x / y - (x % y < 0); };
  const long long lo = std::max(floor_div(-v.eb - d, v.stride) + 1, -(v.na - 1));
  const long long hi = std::min(floor_div(v.ea - 1 - d, v.stride), v.nb - 1);
  if (hi - lo > 3) return false;
  for (long long k = lo; k <= hi; ++k)
    if (!levels_apart(l, levels - 1, d + k * v.stride, wa, wb)) return false;
  return true;
}

bool rows_distinct(const Rows& r) { return extent(r).nested; }

bool rows_apart(const Rows& a, const Rows& b) {
  const Extent x = extent(a), y = extent(b);
  const long long d = (long long)((uintptr_t)b.p - (uintptr_t)a.p);
  if (d >= x.all || -d >= y.all) return true;
  if (!x.nested || !y.nested) return false;
  Level l[6];
  int n = 0;
  const auto add = [&](const Rows& r, bool first) {
    for (int i = 0; i < 3; ++i) {
      if (r.count[i] <= 1) continue;
      const long long s = r.stride[i] * r.bytes;
      int j = 0;
      while (j < n && l[j].stride != s) ++j;
      if (j == n) l[n++] = {s, 1, 1, 0, 0};
      (first ? l[j].na : l[j].nb) = r.count[i];
    }
  };
  add(a, true);
  add(b, false);
  std::sort(l, l + n, [](const Level& p, const Level& q) { return p.stride < q.stride; });
  long long ea = a.width * a.bytes, eb = b.width * b.bytes;
  for (int i = 0; i < n; ++i) {
    l[i].ea = ea;
    l[i].eb = eb;
    ea += (l[i].na - 1) * l[i].stride;
    eb += (l[i].nb - 1) * l[i].stride;
  }
  return levels_apart(l, n, d, a.width * a.bytes, b.width * b.bytes);
}

namespace {

// ------------------------------------------------------------------ append
struct AppendParams {
  CacheView c;
  const void* k;
  const void* v;
  long long k_tok, k_head, v_tok, v_head;
  const int* starts;
  int tokens;
};

constexpr int kAppendTokens = 32;  // most tokens of one CTA

// A CTA copies `per` tokens' key and value rows (every head): its first threads find a token's
// sequence and slot each, then all threads copy, four independent units in flight per thread.
// U is the copied unit, a 16-byte vector where pointers, strides and head_dim allow it, one
// element otherwise.  Few tokens get a CTA each (bound by latency); prompts 32 to a CTA, bound by
// HBM: the chain of lookups (sequence, length, page) is walked once for 128 KB, where a warp to
// a token walked it for every 2 KB and reached 5.2 TB/s.
template <typename U, int ESZ>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p, int per) {
  __shared__ long long slots[kAppendTokens];
  const int t0 = blockIdx.x * per, tokens = min(per, p.tokens - t0);
  griddep_launch_dependents();
  griddep_wait();
  if ((int)threadIdx.x < tokens) {
    const int tok = t0 + threadIdx.x;
    long long slot = -1;
    unsigned err = 0;
    int seq = tok, first = tok;
    if (p.starts) {
      // the last sequence whose first row is at or before tok (empty sequences share their start)
      int lo = 0, hi = p.c.seqs;  // starts[lo] <= tok < starts[hi]
      if (p.starts[0] > tok || p.starts[hi] <= tok) err = kCacheBadLength;
      while (!err && hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.starts[mid] <= tok)
          lo = mid;
        else
          hi = mid;
      }
      seq = lo;
      first = p.starts[lo];
    }
    if (!err) {
      const int past = p.c.lens[seq];
      const long long pos = (long long)past + (tok - first);
      if (past < 0 || tok < first || pos >= cache_capacity(p.c.max_pages, p.c.page_size)) {
        err = kCacheBadLength;
      } else {
        slot = cache_slot(p.c.table + seq * p.c.table_stride, (int)pos, p.c.page_size, p.c.num_pages, p.c.page_stride,
                          p.c.token_stride);
        if (slot < 0) err = kCacheBadPage;
      }
    }
    if (err) atomicOr(p.c.err, err);
    slots[threadIdx.x] = slot;
  }
  __syncthreads();
  constexpr int PER = sizeof(U) / ESZ, Q = 4;
  const int row = p.c.dim / PER, width = row * p.c.kv_heads, total = tokens * width;
  const U* ks = static_cast<const U*>(p.k) + t0 * (p.k_tok / PER);
  const U* vs = static_cast<const U*>(p.v) + t0 * (p.v_tok / PER);
  U* kd = static_cast<U*>(p.c.k);
  U* vd = static_cast<U*>(p.c.v);
  const long long kt = p.k_tok / PER, kh = p.k_head / PER, vt = p.v_tok / PER, vh = p.v_head / PER;
  const long long dh = p.c.head_stride / PER;
  for (int i0 = threadIdx.x; i0 < total; i0 += Q * 256) {
    U a[Q], b[Q];
    long long to[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = i0 + q * 256;
      to[q] = -1;
      if (i < total) {
        const int t = i / width, e = i - t * width, h = e / row, c = e - h * row;
        if (slots[t] >= 0) {
          to[q] = slots[t] / PER + h * dh + c;
          a[q] = ks[t * kt + h * kh + c];
          b[q] = vs[t * vt + h * vh + c];
        }
      }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (to[q] >= 0) {
        kd[to[q]] = a[q];
        vd[to[q]] = b[q];
      }
  }
}

// ------------------------------------------------------------------ eviction
__device__ __forceinline__ uint32_t cluster_nctas() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
struct EvictParams {
  CacheView c;
  const float* win;
  float* wout;
  long long win_seq, win_head, wout_seq, wout_head;
  const int* out_table;
  long long out_stride;
  int out_pages, wcap;
  int* new_lens;
  int* kept;
  int budget, recent;
  bool same_weights, in_place;
};

// Length of sequence s, or -1 (and the error raised) when the table, the weights or the
// destination cannot hold it.
__device__ __forceinline__ int evict_length(const EvictParams& p, int s) {
  const int len = p.c.lens[s];
  const int n = min(len, p.budget);
  if (len < 0 || len > min(cache_capacity(p.c.max_pages, p.c.page_size), p.wcap) ||
      n > cache_capacity(p.out_pages, p.c.page_size)) {
    if (threadIdx.x == 0) atomicOr(p.c.err, kCacheBadLength);
    return -1;
  }
  return len;
}

// Order-preserving bits of a weight: larger weight, larger key; -0 as +0, NaN as -infinity.
__device__ __forceinline__ unsigned weight_key(float w) {
  if (w != w) w = -__int_as_float(0x7f800000);
  const unsigned u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;

// Chooses the kept tokens of one (sequence, head) and compacts its weights.  The n - r largest
// of the first len - r weights are found by radix selection: four passes over 8-bit digits, each
// narrowing the threshold key.  Then every warp takes a contiguous part of the tokens, counts
// the kept ones, and writes their slots in order; ties at the threshold go to the first ones.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
  griddep_launch_dependents();
  __shared__ unsigned hist[8][256];
  __shared__ int warp_gt[kSelWarps], warp_eq[kSelWarps];
  __shared__ unsigned sh_prefix;
  __shared__ int sh_need;
  const int s = blockIdx.x / p.c.kv_heads, h = blockIdx.x - s * p.c.kv_heads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int len = evict_length(p, s);
  int* kept = p.kept + (long long)blockIdx.x * p.budget;
  const float* win = p.win + s * p.win_seq + h * p.win_head;
  float* wout = p.wout + s * p.wout_seq + h * p.wout_head;
  const int n = len < 0 ? 0 : min(len, p.budget);
  if (tid == 0 && h == 0) p.new_lens[s] = n;
  for (int j = n + tid; j < p.budget; j += kSelThreads) kept[j] = -1;
  if (len <= 0) return;
  if (n == len) {  // everything stays
    for (int j = tid; j < n; j += kSelThreads) {
      kept[j] = j;
      if (!p.same_weights) wout[j] = win[j];
    }
    return;
  }
  const int r = min(p.recent, n), old = len - r, need = n - r;
  // threshold: the need-th largest key of [0, old); `ties` of the keys equal to it are kept
  unsigned prefix = 0;
  int ties = need;
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 8 * 256; i += kSelThreads) hist[0][i] = 0;
      __syncthreads();
      for (int i = tid; i < old; i += kSelThreads) {
        const unsigned key = weight_key(win[i]);
        if (shift == 24 || (key >> (shift + 8)) == prefix >> (shift + 8)) atomicAdd(&hist[warp & 7][(key >> shift) & 255], 1u);
      }
      __syncthreads();
      if (warp == 0) {
        // lane l holds the digits 255 - 8 l .. 248 - 8 l, largest first
        int cnt[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          cnt[j] = 0;
#pragma unroll
          for (int c = 0; c < 8; ++c) cnt[j] += hist[c][255 - 8 * lane - j];
          sum += cnt[j];
        }
        int before = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, before, d);
          if (lane >= d) before += o;
        }
        before -= sum;  // keys with a larger digit held by lower lanes
        if (before < ties && before + sum >= ties) {
          int left = ties - before;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (left > 0 && left <= cnt[j]) {
              sh_prefix = prefix | (unsigned)(255 - 8 * lane - j) << shift;
              sh_need = left;
            }
            left -= cnt[j];
          }
        }
      }
      __syncthreads();
      prefix = sh_prefix;
      ties = sh_need;
    }
  }
  // contiguous part of each warp, a multiple of 32 tokens
  const int part = ((len + kSelThreads - 1) / kSelThreads) * 32;
  const int i0 = warp * part, i1 = min(len, i0 + part);
  int gt = 0, eq = 0;
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const unsigned key = i < i1 && i < old ? weight_key(win[i]) : 0;
    const bool more = i < i1 && (i >= old || (need > 0 && key > prefix));
    const bool same = i < i1 && i < old && need > 0 && key == prefix;
    gt += __popc(__ballot_sync(0xffffffffu, more));
    eq += __popc(__ballot_sync(0xffffffffu, same));
  }
  if (lane == 0) {
    warp_gt[warp] = gt;
    warp_eq[warp] = eq;
  }
  __syncthreads();
  int at = 0, seen = 0;  // kept tokens and threshold keys before this warp's part
  for (int w = 0; w < warp; ++w) {
    at += warp_gt[w];
    seen += warp_eq[w];
  }
  at += min(seen, ties);
  const unsigned below = (1u << lane) - 1;
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const unsigned key = i < i1 && i < old ? weight_key(win[i]) : 0;
    const bool same = i < i1 && i < old && need > 0 && key == prefix;
    const unsigned eqs = __ballot_sync(0xffffffffu, same);
    const bool keep = i < i1 && (i >= old || (need > 0 && key > prefix) || (same && seen + __popc(eqs & below) < ties));
    const unsigned ks = __ballot_sync(0xffffffffu, keep);
    if (keep) kept[at + __popc(ks & below)] = i;
    at += __popc(ks);
    seen += __popc(eqs);
  }
  __syncthreads();
  // Weights in order.  In place, a block of them is read before any of it is written: slot j
  // comes from kept[j] >= j, so what a later block reads lies behind what this one writes.
  for (int j0 = 0; j0 < n; j0 += 4 * kSelThreads) {
    float w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = j0 + q * kSelThreads + tid;
      if (j < n) w[q] = win[kept[j]];
    }
    if (p.same_weights) __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = j0 + q * kSelThreads + tid;
      if (j < n) wout[j] = w[q];
    }
  }
  __syncthreads();
  for (int j = n + tid; j < len; j += kSelThreads) wout[j] = 0.0f;
}

// The same choice where the weights of a (sequence, head) fit into the shared memory of a cluster,
// which is nearly always: they are read once, and being copies, in place needs no staging.  The
// digit counts are summed over the cluster through distributed shared memory, and the passes end
// as soon as all of the threshold digit's keys are kept (with distinct weights mostly after
// three).  Digits of 12 bits need one pass less, but their 4096 counts cost more to sum over the
// cluster than a pass (20,000 clocks against 2,000).
//
// Bound by instructions, about two clocks per token on an SM, and by its chain of barriers: 16 x 8
// heads of up to 4096 tokens take 9.7 us, 3 x 8 of up to 131072 33 us, where one CTA per head that
// re-reads the weights takes 12.4 and 147.
constexpr int kClThreads = 512, kClWarps = kClThreads / 32;
constexpr int kClTokens = 26 * 1024;  // of one CTA: 208 KB of keys and weights

__global__ void __launch_bounds__(kClThreads) evict_select_cluster_kernel(const EvictParams p) {
  griddep_launch_dependents();
  // this CTA's keys and then its weights, warp by warp: both, because a key does not give back a
  // NaN's weight, and making keys out of weights in every pass took half of its time
  extern __shared__ unsigned cached[];
  __shared__ unsigned hist[4][256];
  __shared__ unsigned mine[2][256];  // this CTA's digit counts, by parity of the pass
  __shared__ int scan[8], warp_gt[kClWarps], warp_eq[kClWarps], total[2];
  __shared__ unsigned sh_prefix;
  __shared__ int sh_need, sh_count;
  const int ctas = (int)cluster_nctas(), rank = ctas > 1 ? (int)cluster_ctarank() : 0;
  const int pair = blockIdx.x / ctas;
  const int s = pair / p.c.kv_heads, h = pair - s * p.c.kv_heads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int all = ctas * kClThreads, me = rank * kClThreads + tid;
  const int len = evict_length(p, s);
  int* kept = p.kept + (long long)pair * p.budget;
  const float* win = p.win + s * p.win_seq + h * p.win_head;
  float* wout = p.wout + s * p.wout_seq + h * p.wout_head;
  const int n = len < 0 ? 0 : min(len, p.budget);
  if (me == 0 && h == 0) p.new_lens[s] = n;
  for (int j = n + me; j < p.budget; j += all) kept[j] = -1;
  if (len <= 0) return;
  if (n == len) {  // everything stays
    for (int j = me; j < n; j += all) {
      kept[j] = j;
      if (!p.same_weights) wout[j] = win[j];
    }
    return;
  }
  // Kept are the n largest keys, where a recent token's key is above every weight's and that of a
  // slot past the end below.
  const int old = len - min(p.recent, n);
  // contiguous part of each warp, `steps` times 32 tokens
  const int steps = (len + all - 1) / all;
  const int i0 = (rank * kClWarps + warp) * steps * 32;
  unsigned* keys = cached + warp * steps * 32 + lane;
  unsigned* w = keys + kClThreads * steps;
  // all of the weights are asked for at once
  for (int j = 0; j < steps; ++j) {
    const int i = i0 + j * 32 + lane;
    if (i < len) cp_async_4(w + j * 32, win + i);
  }
  cp_async_wait_all();
#pragma unroll 4
  for (int j = 0; j < steps; ++j) {
    const int i = i0 + j * 32 + lane;
    keys[j * 32] = i < old ? weight_key(__uint_as_float(w[j * 32])) : i < len ? 0xffffffffu : 0u;
  }
  // threshold: of the keys whose bits under `mask` equal `prefix`, the first `ties` are kept, and
  // all larger ones
  unsigned prefix = 0, mask = 0;
  int ties = n;
  for (int shift = 24, pass = 0; shift >= 0; shift -= 8, ++pass) {
    for (int q = tid; q < 4 * 256; q += kClThreads) hist[0][q] = 0;
    __syncthreads();
#pragma unroll 4
    for (int j = 0; j < steps; ++j) {
      const unsigned key = keys[j * 32];
      if ((key & mask) == prefix) atomicAdd(&hist[warp & 3][(key >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid < 256) mine[pass & 1][tid] = hist[0][tid] + hist[1][tid] + hist[2][tid] + hist[3][tid];
    if (ctas > 1)
      cluster_sync();
    else
      __syncthreads();
    // thread t < 256 has digit 255 - t: an inclusive scan counts the keys from the largest on
    unsigned count = 0, incl = 0;
    if (tid < 256) {
      if (ctas > 1) {
        const uint32_t at = smem_u32(&mine[pass & 1][255 - tid]);
        unsigned c[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) c[k] = k < ctas ? ld_cluster_u32(mapa_shared(at, k)) : 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) count += c[k];
      } else {
        count = mine[pass & 1][255 - tid];
      }
      incl = count;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      if (lane == 31) scan[warp] = (int)incl;
    }
    __syncthreads();
    if (tid < 256) {
      incl += __reduce_add_sync(0xffffffffu, lane < warp ? scan[lane & 7] : 0);
      if ((int)(incl - count) < ties && (int)incl >= ties) {
        sh_prefix = prefix | (unsigned)(255 - tid) << shift;
        sh_need = ties - (int)(incl - count);
        sh_count = (int)count;
      }
    }
    __syncthreads();
    prefix = sh_prefix;
    ties = sh_need;
    mask |= 255u << shift;
    if (sh_count == ties) break;
  }
  // keys above the threshold and at it, per warp
  int gt = 0, eq = 0;
#pragma unroll 4
  for (int j = 0; j < steps; ++j) {
    const unsigned key = keys[j * 32] & mask;
    gt += key > prefix;
    eq += key == prefix;
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) {
    warp_gt[warp] = gt;
    warp_eq[warp] = eq;
  }
  __syncthreads();
  // larger keys and threshold keys before this warp's part
  const int g = warp_gt[lane & (kClWarps - 1)], e = warp_eq[lane & (kClWarps - 1)];
  int at = __reduce_add_sync(0xffffffffu, lane < warp ? g : 0);
  int seen = __reduce_add_sync(0xffffffffu, lane < warp ? e : 0);
  if (ctas > 1) {
    if (warp == 0) {
      const int a = __reduce_add_sync(0xffffffffu, lane < kClWarps ? g : 0);
      const int b = __reduce_add_sync(0xffffffffu, lane < kClWarps ? e : 0);
      if (lane == 0) {
        total[0] = a;
        total[1] = b;
      }
    }
    cluster_sync();
    int a = 0, b = 0;
    if (lane < rank) {
      a = (int)ld_cluster_u32(mapa_shared(smem_u32(&total[0]), lane));
      b = (int)ld_cluster_u32(mapa_shared(smem_u32(&total[1]), lane));
    }
    at += __reduce_add_sync(0xffffffffu, a);
    seen += __reduce_add_sync(0xffffffffu, b);
    cluster_arrive();  // waited for before leaving: the totals have been read
  }
  at += min(seen, ties);
  // Slots, 32 steps at a time: lane j holds the masks of step j, so that the steps' positions come
  // from one scan instead of a chain over the steps.
  const unsigned below = (1u << lane) - 1;
  for (int j0 = 0; j0 < steps; j0 += 32) {
    const int count = min(32, steps - j0);
    unsigned more = 0, same = 0;
#pragma unroll 4
    for (int j = 0; j < count; ++j) {
      const unsigned key = keys[(j0 + j) * 32] & mask;
      const unsigned m = __ballot_sync(0xffffffffu, key > prefix), t = __ballot_sync(0xffffffffu, key == prefix);
      if (lane == j) {
        more = m;
        same = t;
      }
    }
    int before = __popc(same);
    const int mine_eq = before;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before += o;
    }
    const int eqs = __shfl_sync(0xffffffffu, before, 31);
    // the first `ties` threshold keys in all are kept
    int take = min(mine_eq, max(0, ties - (seen + before - mine_eq)));
    unsigned keep = more;
    for (; take > 0; --take) {
      keep |= same & (0u - same);
      same &= same - 1;
    }
    int base = __popc(keep);
    const int own = base;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, base, d);
      if (lane >= d) base += o;
    }
    const int ks = __shfl_sync(0xffffffffu, base, 31);
    base += at - own;
#pragma unroll 4
    for (int j = 0; j < count; ++j) {
      const unsigned k = __shfl_sync(0xffffffffu, keep, j);
      const int to = __shfl_sync(0xffffffffu, base, j) + __popc(k & below);
      if (k >> lane & 1) {
        kept[to] = i0 + (j0 + j) * 32 + lane;
        wout[to] = __uint_as_float(w[(j0 + j) * 32]);
      }
    }
    at += ks;
    seen += eqs;
  }
  for (int j = n + me; j < len; j += all) wout[j] = 0.0f;
  if (ctas > 1) cluster_wait();
}

// Offsets of a kept row's source and destination; false (error raised) when a page is bad.
__device__ __forceinline__ bool evict_offsets(const EvictParams& p, int s, int h, int j, int from, long long* src,
                                              long long* dst) {
  const int* row = p.c.table + s * p.c.table_stride;
  const int* out = p.out_table + s * p.out_stride;
  const long long a = cache_slot(row, from, p.c.page_size, p.c.num_pages, p.c.page_stride, p.c.token_stride);
  const long long b = cache_slot(out, j, p.c.page_size, p.c.num_pages, p.c.page_stride, p.c.token_stride);
  if (a < 0 || b < 0) {
    atomicOr(p.c.err, kCacheBadPage);
    return false;
  }
  if (!p.in_place && row[j / p.c.page_size] == out[j / p.c.page_size]) {
    atomicOr(p.c.err, kCacheSamePage);
    return false;
  }
  *src = a + h * p.c.head_stride;
  *dst = b + h * p.c.head_stride;
  return true;
}

constexpr int kMoveRows = 64;  // kept rows of one CTA

// Rows to other pages: every CTA moves 64 kept rows of one (sequence, head), keys and values
// together, with eight independent loads per thread.
template <typename U, int ESZ>
__global__ void __launch_bounds__(256) evict_copy_kernel(const EvictParams p) {
  griddep_wait();
  const int s = blockIdx.y / p.c.kv_heads, h = blockIdx.y - s * p.c.kv_heads;
  const int len = evict_length(p, s);
  const int n = len < 0 ? 0 : min(len, p.budget);
  const int j0 = blockIdx.x * kMoveRows;
  if (j0 >= n) return;
  __shared__ long long src[kMoveRows], dst[kMoveRows];
  const int rows = min(kMoveRows, n - j0);
  if (threadIdx.x < rows) {
    const int j = j0 + threadIdx.x;
    if (!evict_offsets(p, s, h, j, p.kept[(long long)blockIdx.y * p.budget + j], &src[threadIdx.x], &dst[threadIdx.x]))
      src[threadIdx.x] = -1;
  }
  __syncthreads();
  constexpr int PER = sizeof(U) / ESZ;
  const int row = p.c.dim / PER, total = rows * row;
  const U* k = static_cast<const U*>(p.c.k);
  const U* v = static_cast<const U*>(p.c.v);
  U* ko = static_cast<U*>(p.c.k);
  U* vo = static_cast<U*>(p.c.v);
  for (int i0 = threadIdx.x; i0 < total; i0 += 4 * 256) {
    U a[4], b[4];
    long long to[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int i = i0 + q * 256;
      to[q] = -1;
      if (i < total) {
        const int j = i / row, e = i - j * row;
        if (src[j] >= 0) {
          const long long from = src[j] / PER + e;
          to[q] = dst[j] / PER + e;
          a[q] = k[from];
          b[q] = v[from];
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (to[q] >= 0) {
        ko[to[q]] = a[q];
        vo[to[q]] = b[q];
      }
  }
}

// Rows within their own pages: slot j comes from kept[j] >= j, so a CTA that walks the rows in
// order, reading a block of them before writing any of it, never overwrites what it has still
// to read.  The next block is read before this one is written, which the same order allows; where
// its rows lie is worked out, a row to a thread, one block earlier, and their slots are read another
// block earlier (24 heads of 16384 rows of 128, bf16: 300 us with every thread waiting for all of it
// in turn, 138 so; 128 heads of 1024 rows: 42 and 31).  The chain of blocks of one head bounds it.
// One CTA takes `slice` units of every row of one pool, so that a (sequence, head) has several.
template <typename U, int ESZ>
__global__ void __launch_bounds__(256) evict_shift_kernel(const EvictParams p, int slice) {
  griddep_wait();
  const int s = blockIdx.y / p.c.kv_heads, h = blockIdx.y - s * p.c.kv_heads;
  const int len = evict_length(p, s);
  if (len <= p.budget) return;
  const int n = p.budget;
  constexpr int PER = sizeof(U) / ESZ, Q = 4, ROWS = 256;
  __shared__ long long src[3][ROWS], dst[3][ROWS];  // of three blocks; src -1: the row stays or has a bad page
  const int row = p.c.dim / PER;
  const int e0 = blockIdx.x * slice, width = min(slice, row - e0);
  U* pool = static_cast<U*>(blockIdx.z ? p.c.v : p.c.k);
  const int* kept = p.kept + (long long)blockIdx.y * p.budget;
  // Rows of one pass over the threads and of a block.  A slice of fewer than Q units leaves threads
  // idle: a block has no more rows than there are places for.
  const int per_pass = min(256 / slice, ROWS / Q), block = Q * per_pass;
  const int tid = threadIdx.x, tr = tid / slice, te = tid - tr * slice;
  const bool live = tr < per_pass && te < width;
  auto slot = [&](int c) -> int {
    const unsigned j = (unsigned)c * block + tid;
    return tid < block && j < (unsigned)n ? kept[j] : -1;
  };
  auto place = [&](int c, int from) {
    const int j = c * block + tid;
    long long a, b;
    const bool move = from >= 0 && from != j && evict_offsets(p, s, h, j, from, &a, &b);
    src[c % 3][tid] = move ? a / PER + e0 : -1;
    dst[c % 3][tid] = move ? b / PER + e0 : -1;
  };
  U now[Q], next[Q];
  long long to[Q], to_next[Q];
  auto fetch = [&](int c, U(&r)[Q], long long(&d)[Q]) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = q * per_pass + tr;
      d[q] = -1;
      if (live && src[c % 3][i] >= 0) {
        r[q] = pool[src[c % 3][i] + te];
        d[q] = dst[c % 3][i] + te;
      }
    }
  };
  const int blocks = (int)(((unsigned)n + block - 1) / block);
  place(0, slot(0));
  place(1, slot(1));
  int ahead = slot(2);
  __syncthreads();
  fetch(0, now, to);
  for (int c = 0; c < blocks; ++c) {
    if (c + 1 < blocks) fetch(c + 1, next, to_next);
    place(c + 2, ahead);
    ahead = slot(c + 3);
    __syncthreads();  // block c has been read by every thread, block c + 2 placed
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (to[q] >= 0) pool[to[q]] = now[q];
      if (c + 1 < blocks) {
        now[q] = next[q];
        to[q] = to_next[q];
      }
    }
  }
}

// Clusters of 1 .. 8 CTAs of the selection kernel, at their largest, that the device holds at once
// (its GPCs do not divide evenly: 15 of eight, 22 of six, 26 of five on 148 SMs).
int select_clusters(int device, int ctas) {
  static std::atomic<int> known[kMaxDevices][9];  // ctas <= 8
  int n = known[device][ctas].load();
  if (!n) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kClThreads);
    cfg.dynamicSmemBytes = kClTokens * 8;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, evict_select_cluster_kernel, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 1;
    }
    known[device][ctas].store(n);
  }
  return n;
}

// As many CTAs per (sequence, head), up to a cluster of eight, as leave each 2048 tokens while all
// clusters run at once; past the 212,992 tokens that eight hold, the kernel that re-reads the
// weights.
int launch_select(const EvictParams& p, int pairs, int device, cudaStream_t st) {
  const int cap = std::min(cache_capacity(p.c.max_pages, p.c.page_size), p.wcap);
  auto tokens = [&](int c) { return ((long long)cap + c * kClThreads - 1) / (c * kClThreads) * kClThreads; };
  SPINN_CUDA_TRY(cudaFuncSetAttribute(evict_select_cluster_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      kClTokens * 8));
  int ctas = std::max(1, std::min(8, cap / 2048));
  while (ctas > 1 && pairs > select_clusters(device, ctas)) --ctas;
  while (ctas < 8 && tokens(ctas) > kClTokens) ++ctas;
  if (tokens(ctas) > kClTokens) {
    evict_select_kernel<<<(unsigned)pairs, kSelThreads, 0, st>>>(p);
    SPINN_CUDA_TRY(cudaGetLastError());
    return 0;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pairs * ctas));
  cfg.blockDim = dim3(kClThreads);
  cfg.dynamicSmemBytes = (size_t)tokens(ctas) * 8;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  SPINN_CUDA_TRY(cudaLaunchKernelEx(&cfg, evict_select_cluster_kernel, p));
  return 0;
}

// Pools that are written: two of them, and no row twice.
bool pools_distinct(const SpinnCudaCache& c, int bytes) {
  const Rows k = {c.k, bytes, c.head_dim, {c.num_pages, c.page_size, c.kv_heads},
                  {c.page_stride, c.token_stride, c.head_stride}};
  Rows v = k;
  v.p = c.v;
  return rows_distinct(k) && rows_apart(k, v);
}

// [rows][width] of 4-byte elements; one row: contiguous.
Rows words(const void* p, long long width, long long rows = 1, long long stride = 0) {
  return {p, 4, width, {rows, 1, 1}, {stride, 0, 0}};
}

}  // namespace

extern "C" {

__attribute__((visibility("default"))) int spinn_cuda_stream_sync(void* stream) {
  int dev;
  int rc = check_stream_device("stream_sync", stream, &dev);
  if (rc) return rc;
  unsigned* word = nullptr;
  rc = decode_error_word(dev, &word);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  SPINN_CUDA_TRY(cudaStreamIsCapturing(st, &cap));
  SPINN_CHECK_ARG(cap == cudaStreamCaptureStatusNone, "stream_sync: the stream is being captured");
  unsigned bits = 0;
  SPINN_CUDA_TRY(cudaMemcpyAsync(&bits, word, sizeof(bits), cudaMemcpyDeviceToHost, st));
  SPINN_CUDA_TRY(cudaStreamSynchronize(st));
  if (!bits) return 0;
  clear_errors_kernel<<<1, 1, 0, st>>>(word, bits);
  SPINN_CUDA_TRY(cudaGetLastError());
  SPINN_CUDA_TRY(cudaStreamSynchronize(st));
  if (bits & kWaitExpired) {
    set_error("a kernel's bounded wait expired");
    return SPINN_CUDA_ETIMEOUT;
  }
  set_error("paged cache:%s%s%s", bits & kCacheBadPage ? " a page number outside the pool;" : "",
            bits & kCacheBadLength ? " a length outside its table, weights or rows;" : "",
            bits & kCacheSamePage ? " an output page that its row also reads (in place takes the same table pointer);" : "");
  return SPINN_CUDA_EINVAL;
}

__attribute__((visibility("default"))) int spinn_cuda_cache_append(const SpinnCudaCache* cache,
                                                                   const SpinnCudaPageTable* table,
                                                                   const SpinnCudaAppend* rows, void* stream) {
  AppendParams p;
  int rc = cache_view("cache_append", cache, table, &p.c);
  if (rc) return rc;
  SPINN_CHECK_ARG(rows && rows->k && rows->v, "cache_append: k and v are required");
  SPINN_CHECK_ARG(rows->tokens >= 0, "cache_append: %d tokens", rows->tokens);
  SPINN_CHECK_ARG(rows->starts || rows->tokens == table->seqs, "cache_append: %d tokens for %d sequences without starts",
                  rows->tokens, table->seqs);
  SPINN_CHECK_ARG(rows->k_token_stride >= 0 && rows->k_head_stride >= 0 && rows->v_token_stride >= 0 &&
                      rows->v_head_stride >= 0,
                  "cache_append: negative stride");
  const int es = dtype_bytes(cache->dtype);
  SPINN_CHECK_ARG(((uintptr_t)rows->k | (uintptr_t)rows->v) % es == 0 && (uintptr_t)rows->starts % 4 == 0,
                  "cache_append: misaligned pointer");
  SPINN_CHECK_ARG(pools_distinct(*cache, es), "cache_append: the pools' rows overlap");
  SPINN_CHECK_ARG(rows->tokens <= kMaxLength, "cache_append: %d tokens", rows->tokens);
  int dev;
  rc = check_stream_device("cache_append", stream, &dev);
  if (rc) return rc;
  if (rows->tokens == 0) return 0;
  rc = decode_error_word(dev, &p.c.err);
  if (rc) return rc;
  p.k = rows->k;
  p.v = rows->v;
  p.k_tok = rows->k_token_stride;
  p.k_head = rows->k_head_stride;
  p.v_tok = rows->v_token_stride;
  p.v_head = rows->v_head_stride;
  p.starts = rows->starts;
  p.tokens = rows->tokens;
  const int per = 16 / es;
  const bool vec = cache_vec16(p.c, es) && aligned16(p.k) && aligned16(p.v) && p.k_tok % per == 0 &&
                   p.k_head % per == 0 && p.v_tok % per == 0 && p.v_head % per == 0;
  // two CTAs or more to an SM before a CTA takes more tokens
  const int each = std::max(1, std::min(kAppendTokens, p.tokens / (4 * sm_count(dev))));
  const dim3 grid((unsigned)((p.tokens + each - 1) / each));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (vec && es == 2) return launch_dependent(append_kernel<uint4, 2>, grid, 256, 0, st, p, each);
  if (vec) return launch_dependent(append_kernel<uint4, 4>, grid, 256, 0, st, p, each);
  if (es == 2) return launch_dependent(append_kernel<uint16_t, 2>, grid, 256, 0, st, p, each);
  return launch_dependent(append_kernel<uint32_t, 4>, grid, 256, 0, st, p, each);
}

__attribute__((visibility("default"))) int spinn_cuda_cache_evict(const SpinnCudaCache* cache,
                                                                  const SpinnCudaPageTable* table,
                                                                  const SpinnCudaEvict* e, void* stream) {
  EvictParams p;
  int rc = cache_view("cache_evict", cache, table, &p.c);
  if (rc) return rc;
  SPINN_CHECK_ARG(e && e->weights_in && e->weights_out && e->out_pages && e->new_lens && e->kept,
                  "cache_evict: weights, out_pages, new_lens and kept are required");
  SPINN_CHECK_ARG(e->budget > 0 && e->budget <= kMaxLength && e->recent >= 0, "cache_evict: budget %d, recent %d",
                  e->budget, e->recent);
  SPINN_CHECK_ARG(e->out_max_pages > 0 && e->out_row_stride >= 0 && e->weights_capacity > 0,
                  "cache_evict: bad output table or weights");
  SPINN_CHECK_ARG(e->win_seq_stride >= 0 && e->win_head_stride >= 0 && e->wout_seq_stride >= 0 &&
                      e->wout_head_stride >= 0,
                  "cache_evict: negative stride");
  SPINN_CHECK_ARG(e->new_lens != table->lens, "cache_evict: new_lens must not be the lengths it is read from");
  SPINN_CHECK_ARG((((uintptr_t)e->weights_in | (uintptr_t)e->weights_out | (uintptr_t)e->out_pages |
                    (uintptr_t)e->new_lens | (uintptr_t)e->kept) & 3) == 0,
                  "cache_evict: misaligned pointer");
  const long long pairs = (long long)table->seqs * cache->kv_heads;
  SPINN_CHECK_ARG(pairs <= 65535, "cache_evict: %lld (sequence, head) pairs, at most 65535", pairs);
  p.in_place = e->out_pages == table->pages;
  SPINN_CHECK_ARG(!p.in_place || table->seqs == 1 || e->out_row_stride == table->row_stride,
                  "cache_evict: in place, the output table's stride must be the table's");
  p.same_weights = e->weights_in == e->weights_out;
  const Rows weights = {e->weights_out, 4, e->weights_capacity, {table->seqs, cache->kv_heads, 1},
                        {e->wout_seq_stride, e->wout_head_stride, 0}};
  const Rows win = {e->weights_in, 4, e->weights_capacity, {table->seqs, cache->kv_heads, 1},
                    {e->win_seq_stride, e->win_head_stride, 0}};
  SPINN_CHECK_ARG(p.same_weights ? e->win_seq_stride == e->wout_seq_stride && e->win_head_stride == e->wout_head_stride
                                 : rows_apart(weights, win),
                  "cache_evict: weights_out must be weights_in itself or apart from it");
  const int es = dtype_bytes(cache->dtype);
  SPINN_CHECK_ARG(pools_distinct(*cache, es), "cache_evict: the pools' rows overlap");
  SPINN_CHECK_ARG(rows_distinct(weights), "cache_evict: rows of weights_out overlap");
  // what is written against what is read and against one another
  const Rows kept = words(e->kept, pairs * e->budget), new_lens = words(e->new_lens, table->seqs);
  const Rows reads[] = {words(table->lens, table->seqs), words(table->pages, table->max_pages, table->seqs, table->row_stride),
                        words(e->out_pages, e->out_max_pages, table->seqs, e->out_row_stride)};
  for (const Rows& r : reads)
    SPINN_CHECK_ARG(rows_apart(kept, r) && rows_apart(new_lens, r) && rows_apart(weights, r),
                    "cache_evict: kept, new_lens or weights_out overlaps the lengths or a table");
  SPINN_CHECK_ARG(rows_apart(kept, new_lens) && rows_apart(kept, weights) && rows_apart(new_lens, weights) &&
                      rows_apart(kept, win) && rows_apart(new_lens, win),
                  "cache_evict: kept, new_lens and the weights overlap one another");
  int dev;
  rc = check_stream_device("cache_evict", stream, &dev);
  if (rc) return rc;
  rc = decode_error_word(dev, &p.c.err);
  if (rc) return rc;
  p.win = e->weights_in;
  p.wout = e->weights_out;
  p.win_seq = e->win_seq_stride;
  p.win_head = e->win_head_stride;
  p.wout_seq = e->wout_seq_stride;
  p.wout_head = e->wout_head_stride;
  p.out_table = e->out_pages;
  p.out_stride = e->out_row_stride;
  p.out_pages = e->out_max_pages;
  p.wcap = std::min(e->weights_capacity, kMaxLength);
  p.new_lens = e->new_lens;
  p.kept = e->kept;
  p.budget = e->budget;
  p.recent = e->recent;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = launch_select(p, (int)pairs, dev, st);
  if (rc) return rc;
  const bool vec = cache_vec16(p.c, es);
  const int units = vec ? p.c.dim * es / 16 : p.c.dim;  // copied units of a row
  if (p.in_place) {
    // 64 bytes of a row per CTA keep DRAM bursts whole
    const int slice = std::min(units, vec ? 4 : 64 / es);
    const dim3 grid((units + slice - 1) / slice, (unsigned)pairs, 2);
    if (vec && es == 2) return launch_dependent(evict_shift_kernel<uint4, 2>, grid, 256, 0, st, p, slice);
    if (vec) return launch_dependent(evict_shift_kernel<uint4, 4>, grid, 256, 0, st, p, slice);
    if (es == 2) return launch_dependent(evict_shift_kernel<uint16_t, 2>, grid, 256, 0, st, p, slice);
    return launch_dependent(evict_shift_kernel<uint32_t, 4>, grid, 256, 0, st, p, slice);
  }
  const int most = std::min(std::min(p.budget, p.wcap), cache_capacity(p.c.max_pages, p.c.page_size));
  const dim3 grid((most + kMoveRows - 1) / kMoveRows, (unsigned)pairs, 1);
  if (vec && es == 2) return launch_dependent(evict_copy_kernel<uint4, 2>, grid, 256, 0, st, p);
  if (vec) return launch_dependent(evict_copy_kernel<uint4, 4>, grid, 256, 0, st, p);
  if (es == 2) return launch_dependent(evict_copy_kernel<uint16_t, 2>, grid, 256, 0, st, p);
  return launch_dependent(evict_copy_kernel<uint32_t, 4>, grid, 256, 0, st, p);
}

__attribute__((visibility("default"))) int64_t spinn_cuda_diag_cache_slot(const int32_t* row, int max_pages, int pos,
                                                                          int page_size, int num_pages,
                                                                          int64_t page_stride, int64_t token_stride) {
  if (!row || max_pages <= 0 || page_size <= 0 || pos < 0 || pos >= cache_capacity(max_pages, page_size)) return -2;
  return cache_slot(row, pos, page_size, num_pages, page_stride, token_stride);
}

__attribute__((visibility("default"))) int spinn_cuda_diag_rows(const int64_t* a, const int64_t* b) {
  SPINN_CHECK_ARG(a && b, "diag_rows: two operands are required");
  const auto rows = [](const int64_t* r) {
    return Rows{(const void*)(uintptr_t)r[0], (int)r[1], r[2], {r[3], r[4], r[5]}, {r[6], r[7], r[8]}};
  };
  return (rows_distinct(rows(a)) ? 1 : 0) | (rows_apart(rows(a), rows(b)) ? 2 : 0);
}

__attribute__((visibility("default"))) int spinn_cuda_diag_attention_share(int64_t units, int workers, int worker,
                                                                           int64_t unit, int64_t* out3) {
  SPINN_CHECK_ARG(out3 && units > 0 && units <= kMaxUnits && workers > 0 && worker >= 0 && worker < workers && unit >= 0 &&
                      unit < units,
                  "spinn_cuda_diag_attention_share: invalid arguments");
  const AttnShares sh((unsigned)units, (unsigned)workers);
  out3[0] = sh.start((unsigned)worker);
  out3[1] = sh.start((unsigned)worker + 1);
  out3[2] = sh.owner((unsigned)unit);
  return 0;
}

}  // extern "C"
}  // namespace spinn
