// What the kernels of paged caches share: element types of the pages, lengths, 8-bit codes as fp16.
#pragma once

#include "fal_launch.h"
#include "sm100_ptx.cuh"

namespace fal {

struct S8 {
  uint8_t bits;
};
struct E4M3 {
  uint8_t bits;
};

__device__ __forceinline__ int paged_capacity(const PagedCache& c) { return c.pages_per_entry << c.page_shift; }
// Positions of entry b that attention sees.
__device__ __forceinline__ int paged_len(const PagedCache& c, int b) {
  const int length = c.lens[b], capacity = paged_capacity(c);
  if (length < 0) return 0;
  const unsigned n = static_cast<unsigned>(min(length, capacity)) + static_cast<unsigned>(c.appended);
  return static_cast<int>(min(n, static_cast<unsigned>(capacity)));
}
// First position that the first of `rows` query tokens of entry b, which has n positions, does not see.  Where rows were appended
// and may have run over the capacity, n does not tell their positions.
__device__ __forceinline__ int paged_first_limit(const PagedCache& c, int b, int n, int rows) {
  if (c.appended != 0 && n == paged_capacity(c)) return min(c.lens[b], n) + 1;
  return n - rows + 1;
}
__device__ __forceinline__ int paged_len_in_pages(const PagedCache& c, int n) {
  return c.type == kPagedF16 ? n : n >> c.page_shift << c.page_shift;
}

template <class T>
struct Elem {
  static constexpr bool kScaled = true;
  static constexpr int kBytes = 1;
};
template <>
struct Elem<__half> {
  static constexpr bool kScaled = false;
  static constexpr int kBytes = 2;
};
// Four 8-bit codes as two pairs of fp16.
__device__ __forceinline__ void widen(const S8*, uint32_t w, uint32_t& lo, uint32_t& hi) {
  // 1024 + u, u = code + 128, as fp16 is 0x6400 + u
  const uint32_t u = w ^ 0x80808080u;
  lo = __byte_perm(u, 0x64646464u, 0x4140);
  hi = __byte_perm(u, 0x64646464u, 0x4342);
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(0x64806480u));
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(0x64806480u));
}
__device__ __forceinline__ void widen(const E4M3*, uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t"
      ".reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t"
      "}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

}  // namespace fal
