// cache.h -- the paged key-value cache shared by cache.cu (append, eviction) and attention.cu:
// where a token's row lies, and how one attention launch splits its work.  The arithmetic is
// host code as well, so that the CPU tests run what the kernels run.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/spinn_cuda.h"

namespace spinn {

// Deferred errors of the decoder-serving operators, raised by a kernel that skips the access instead of
// making it (spinn_cuda_stream_sync reports and clears them).
enum DecodeErr : unsigned { kCacheBadPage = 1, kCacheBadLength = 2, kCacheSamePage = 4, kWaitExpired = 8 };

// The pools and their page table as the kernels see them.  Strides are in elements.
struct CacheView {
  void* k;
  void* v;
  long long page_stride, token_stride, head_stride;
  int num_pages, page_size, kv_heads, dim;
  const int* table;
  long long table_stride;
  int max_pages, seqs;
  const int* lens;
  unsigned* err;  // deferred error word of the device
};

// Sizes and lengths end 65536 before 2^31: indices in 32 bits step past their end by a tile.
constexpr int kMaxLength = 0x7fff0000;

// Tokens that a table row can hold.
__host__ __device__ inline int cache_capacity(int max_pages, int page_size) {
  const long long c = (long long)max_pages * page_size;
  return c > kMaxLength ? kMaxLength : (int)c;
}

// Element offset of token `pos` in either pool (head 0) through the table row `row`, or -1 when
// its page lies outside the pool.  pos must be within the row's capacity.  64-bit: a pool of
// more than 2^31 elements is ordinary.
__host__ __device__ inline long long cache_slot(const int* row, int pos, int page_size, int num_pages,
                                                long long page_stride, long long token_stride) {
  const int blk = (int)((unsigned)pos / (unsigned)page_size);
  const int page = row[blk];
  if (page < 0 || page >= num_pages) return -1;
  return (long long)page * page_stride + (long long)(pos - blk * page_size) * token_stride;
}

// Attention's work: `units` tiles of tokens in the order (sequence, head block, tile), dealt to
// `workers` CTAs in contiguous shares of units / workers, the first units % workers of them one
// more.  Worker w has [start(w), start(w + 1)); owner(u) is the worker that has unit u.
struct AttnShares {
  unsigned each, more;
  __host__ __device__ AttnShares(unsigned units, unsigned workers) : each(units / workers), more(units - each * workers) {}
  __host__ __device__ unsigned start(unsigned w) const { return w * each + (w < more ? w : more); }
  __host__ __device__ int owner(unsigned u) const {
    const unsigned big = more * (each + 1);
    return (int)(u < big ? u / (each + 1) : more + (u - big) / each);
  }
};
constexpr long long kMaxUnits = 0x7fffffffLL;

// Host-side checks common to the cache entry points; fills `v`.
int cache_view(const char* who, const SpinnCudaCache* c, const SpinnCudaPageTable* t, CacheView* v);
// The current device when `stream` belongs to it, an error otherwise.
int check_stream_device(const char* who, void* stream, int* device);
// 16-byte vector access possible: `bytes`-sized elements, pointers and strides (elements).
bool cache_vec16(const CacheView& v, int bytes);
int dtype_bytes(int dtype);

// What an operand covers: rows of `width` elements of `bytes` each, count[i] of them at stride[i]
// (elements, >= 0) along up to three dimensions.
struct Rows {
  const void* p;
  int bytes;
  long long width;
  long long count[3], stride[3];
};
// No two rows share an element (a tensor that is written must not: its rows are written by many
// CTAs).  Dimensions nest, in any order.
bool rows_distinct(const Rows& r);
// No element of `a` is one of `b`.  Operands that interleave in one buffer (slices of its rows, keys and
// values of one pool in any order of dimensions) are told apart where their strides agree.
bool rows_apart(const Rows& a, const Rows& b);

// The current device's deferred error word (device memory; DecodeErr bits).
int decode_error_word(int device, unsigned** word);

}  // namespace spinn
