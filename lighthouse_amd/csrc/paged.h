// A key / value cache in pages, as the kernels that fill, read and compact it see it: position t of sequence b lies on
// page table[b][t / size], slot t % size.  A page id outside 0 .. pages - 1 holds nothing: it is never followed.
#pragma once

#include "common.h"

namespace lh {

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, "Division by invariant integers using
// multiplication", 1994): m = floor(2^32 (2^s - d) / d) + 1 with s = ceil(log2 d).
struct FastDiv {
  uint32_t d = 1, m = 1, s = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t divisor) : d(divisor) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)((((1ull << s) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

struct Paged {
  void* k;
  void* v;
  const int32_t* table;
  int64_t table_stride;
  lh_strides3 sk, sv;  // elements: page, head, slot
  int32_t pages, max_pages, size, heads, d;
  float k_scale, v_scale;
  FastDiv by_size;

  // Entry i of the table, through the address space of what no kernel writes while it runs: where i is the same for the wave, the
  // scalar unit loads it.  (As a plain load, which the compiler has to keep in order with the kernel's stores, it went through
  // the vector memory unit, and waiting for it meant waiting for every key and value on the way.)
  __device__ __forceinline__ int entry(int64_t i) const {
    typedef const int32_t __attribute__((address_space(4))) constant_i32;
    return reinterpret_cast<constant_i32*>(reinterpret_cast<uintptr_t>(table))[i];
  }
  // The page of position t < max_pages * size of sequence b, or -1.
  __device__ __forceinline__ int page_of(int b, int t, int* slot) const {
    const int i = (int)by_size.div((uint32_t)t);
    *slot = t - i * size;
    const int p = entry(b * table_stride + i);
    return (uint32_t)p < (uint32_t)pages ? p : -1;
  }
  __host__ __device__ int capacity() const { return max_pages * size; }
};

// Checks what every entry point asks of a cache and fills `out`.
int paged_cache(const lh_paged_cache* c, const char* what, Paged* out);

}  // namespace lh
