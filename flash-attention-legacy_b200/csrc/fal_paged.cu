// Paged key/value caches: append of new rows with the position rotation on the way, attention over the pages (fp16, or
// 8 bits with a scale for each page and head), and the pages' rows in order for the forward kernel.
//
// The reference has no paged cache; its hook attends eagerly over dense ones (flash_attn_legacy/integrations.py:77-98).
//
// 8-bit pages.  A value is rounded to 8 bits once, when its page is full: a = max |x| over the page's rows of a head,
// scale = a / m and code = round(x m / a), m = 127 (int8, nearest whole number) or 448 (e4m3, nearest such number).  Until
// then the row waits as fp16 in the entry's tail, so that the cache does not depend on how the rows came in, token by
// token or as chunks, and no page is rounded again when a larger value arrives.  x m is exact in 32 bits (11 + 7 bits) and
// its quotient by a, rounded once, is on the same side of every rounding border as the exact one: the border is a multiple
// of 2^-5 of the code's leading bit at least 2^-16 away relative to it, or the quotient is exactly the border.
#include <type_traits>

#include "fal_combine.cuh"
#include "fal_common.h"
#include "fal_launch.h"
#include "sm100_ptx.cuh"

namespace fal {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct S8 {
  uint8_t bits;
};
struct E4M3 {
  uint8_t bits;
};

__device__ __forceinline__ int paged_capacity(const PagedCache& c) { return c.pages_per_entry << c.page_shift; }
__device__ __forceinline__ int paged_len(const PagedCache& c, int b) { return min(max(c.lens[b], 0), paged_capacity(c)); }

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
// Bound by HBM on prompts, by latency for single tokens.  A thread takes 16 columns of a head: the two 8-column pieces
// whose columns are rotated with each other, or two neighbouring ones.
constexpr int kAppendThreads = 256;

struct Piece {
  int first, second;  // columns of the two pieces
  bool rotated;
};
__device__ __forceinline__ Piece append_piece(const PagedAppendParams& p, int c) {
  Piece x;
  x.rotated = c * 16 < p.rotary_dim;
  const bool apart = x.rotated && !p.interleaved;
  x.first = apart ? c * 8 : c * 16;
  x.second = x.first + (apart ? p.rotary_dim / 2 : 8);
  return x;
}

__device__ __forceinline__ void load_angles(const void* table, int half_tables, int64_t at, float (&x)[8]) {
  if (half_tables) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(table) + at));
    const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
    const float4* t = reinterpret_cast<const float4*>(static_cast<const float*>(table) + at);
    const float4 a = __ldg(t), b = __ldg(t + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
}

// (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin) in 32 bits, rounded once to the cache's fp16.
__device__ __forceinline__ void turn(float& x1, float& x2, float c, float s) {
  const float y1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
  const float y2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
  x1 = y1;
  x2 = y2;
}

// The two pieces of a row of q or k (v: not rotated) at position pos, rotated.
__device__ __forceinline__ void append_load(const PagedAppendParams& p, const __half* row, int c, bool turned, int pos,
                                            uint4& a, uint4& b, Piece& at) {
  at = append_piece(p, c);
  if (!turned) at = Piece{c * 16, c * 16 + 8, false};
  a = *reinterpret_cast<const uint4*>(row + at.first);
  b = *reinterpret_cast<const uint4*>(row + at.second);
  if (!at.rotated) return;
  __half2* ha = reinterpret_cast<__half2*>(&a);
  __half2* hb = reinterpret_cast<__half2*>(&b);
  float cs[8], sn[8];
  const int64_t angle = static_cast<int64_t>(pos) * (p.rotary_dim / 2) + c * 8;
  load_angles(p.cos, p.half_tables, angle, cs);
  load_angles(p.sin, p.half_tables, angle, sn);
  if (p.interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 x = __half22float2(ha[i]), y = __half22float2(hb[i]);
      turn(x.x, x.y, cs[i], sn[i]);
      turn(y.x, y.y, cs[4 + i], sn[4 + i]);
      ha[i] = __floats2half2_rn(x.x, x.y);
      hb[i] = __floats2half2_rn(y.x, y.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 x = __half22float2(ha[i]), y = __half22float2(hb[i]);
      turn(x.x, y.x, cs[2 * i], sn[2 * i]);
      turn(x.y, y.y, cs[2 * i + 1], sn[2 * i + 1]);
      ha[i] = __floats2half2_rn(x.x, x.y);
      hb[i] = __floats2half2_rn(y.x, y.y);
    }
  }
}

__device__ __forceinline__ const __half* new_row(const void* base, const RowStrides& s, int b, int h, int r) {
  return static_cast<const __half*>(base) + b * s.batch + h * s.head + r * s.row;
}

// Page of position pos of entry b, or -1 (and the status word says so).
__device__ __forceinline__ int append_page(const PagedAppendParams& p, int b, int pos) {
  int page = -1;
  if (pos < paged_capacity(p.c)) page = p.c.table[b * p.c.table_stride + (pos >> p.c.page_shift)];
  if (page < 0 || page >= p.c.num_pages) {
    if (p.status) atomicCAS(p.status, 0, kDevAppendOverflow);
    page = -1;
  }
  return page;
}

// Grid: (token, piece of its q, k and v heads).  Rows of 8-bit caches that finish a page are the next kernel's business,
// and so are those behind such a page: their places in the tail are read there first.
__global__ void __launch_bounds__(kAppendThreads) fal_paged_append_kernel(const PagedAppendParams p) {
  grid_dependency_wait();
  grid_dependency_launch();
  const int b = blockIdx.x / p.rows;
  const int i = blockIdx.x % p.rows;
  const int start = p.c.lens[b];
  const int capacity = paged_capacity(p.c);
  if (i == 0 && blockIdx.y == 0 && threadIdx.x == 0)
    p.new_lens[b] = start < 0 ? start : static_cast<int>(min(static_cast<int64_t>(start) + p.rows, static_cast<int64_t>(capacity)));
  const int pieces = p.c.head_dim / 16;
  const int task = blockIdx.y * kAppendThreads + threadIdx.x;
  int h = task / pieces;
  const int c = task % pieces;
  if (h >= p.heads_q + 2 * p.c.heads_kv) return;
  const int64_t pos64 = static_cast<int64_t>(start) + i;
  const bool placed = start >= 0 && pos64 < capacity;  // (start < 0: an unused entry of a padded batch)
  const int pos = placed ? static_cast<int>(pos64) : 0;
  uint4 a, z;
  Piece at;
  if (h < p.heads_q) {
    append_load(p, new_row(p.q, p.q_strides, b, h, i), c, true, pos, a, z, at);
    if (!placed) a = z = make_uint4(0, 0, 0, 0);
    __half* out = static_cast<__half*>(p.q_out) + (static_cast<int64_t>(blockIdx.x) * p.heads_q + h) * p.c.head_dim;
    *reinterpret_cast<uint4*>(out + at.first) = a;
    *reinterpret_cast<uint4*>(out + at.second) = z;
    return;
  }
  h -= p.heads_q;
  const bool is_v = h >= p.c.heads_kv;
  if (is_v) h -= p.c.heads_kv;
  if (!placed) {
    if (start >= 0 && p.status) atomicCAS(p.status, 0, kDevAppendOverflow);
    return;
  }
  __half* dst;
  const int shift = p.c.page_shift;
  const int in_page = pos & ((1 << shift) - 1);
  if (p.c.type == kPagedF16) {
    const int page = append_page(p, b, pos);
    if (page < 0) return;
    const RowStrides& s = is_v ? p.c.v_strides : p.c.k_strides;
    dst = static_cast<__half*>(is_v ? p.c.v_pages : p.c.k_pages) + page * s.batch + h * s.head + in_page * s.row;
  } else {
    const int64_t end = min(static_cast<int64_t>(start) + p.rows, static_cast<int64_t>(capacity));
    if ((end >> shift) != (start >> shift)) return;
    const RowStrides& s = is_v ? p.c.v_tail_strides : p.c.k_tail_strides;
    dst = static_cast<__half*>(is_v ? p.c.v_tail : p.c.k_tail) + b * s.batch + h * s.head + in_page * s.row;
  }
  const __half* src = is_v ? new_row(p.v, p.v_new_strides, b, h, i) : new_row(p.k, p.k_new_strides, b, h, i);
  append_load(p, src, c, !is_v, pos, a, z, at);
  *reinterpret_cast<uint4*>(dst + at.first) = a;
  *reinterpret_cast<uint4*>(dst + at.second) = z;
}

// The codes of two fp16 values as two bytes; most: the page's largest magnitude, not 0.
__device__ __forceinline__ uint32_t codes_of(const S8*, float2 x, float most) {
  const int lo = __float2int_rn(__fdiv_rn(x.x * 127.f, most)), hi = __float2int_rn(__fdiv_rn(x.y * 127.f, most));
  return (lo & 0xff) | ((hi & 0xff) << 8);
}
__device__ __forceinline__ uint32_t codes_of(const E4M3*, float2 x, float most) {
  uint16_t out;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
      : "=h"(out)
      : "f"(__fdiv_rn(x.y * 448.f, most)), "f"(__fdiv_rn(x.x * 448.f, most)));
  return out;
}
__device__ __forceinline__ float code_max(const S8*) { return 127.f; }
__device__ __forceinline__ float code_max(const E4M3*) { return 448.f; }

// Full pages of 8-bit caches.  Grid: (page counted from the one of the first new row, KV head of K then of V, entry).
// The rows of a page are put together in shared memory -- the first page's earlier rows from the tail, the others from
// the call, rotated --, their largest magnitude is found, and the codes leave in 16-byte stores.  The first page's block
// also writes the rows behind the last full page to the tail, once it has read it.
template <class T>
__global__ void __launch_bounds__(kAppendThreads) fal_paged_seal_kernel(const PagedAppendParams p) {
  extern __shared__ __align__(16) __half seal_rows[];
  __shared__ uint32_t warp_most[kAppendThreads / 32];
  grid_dependency_wait();
  grid_dependency_launch();
  const int b = blockIdx.z;
  const int start = p.c.lens[b];
  const int capacity = paged_capacity(p.c);
  const int shift = p.c.page_shift;
  if (start < 0 || start >= capacity) return;
  const int end = static_cast<int>(min(static_cast<int64_t>(start) + p.rows, static_cast<int64_t>(capacity)));
  const int index = (start >> shift) + blockIdx.x;  // page of the entry
  if (index >= (end >> shift)) return;              // not full
  const bool is_v = blockIdx.y >= static_cast<unsigned>(p.c.heads_kv);
  const int h = is_v ? blockIdx.y - p.c.heads_kv : blockIdx.y;
  const int d = p.c.head_dim, pieces = d / 16, page_rows = 1 << shift;
  const RowStrides& ts = is_v ? p.c.v_tail_strides : p.c.k_tail_strides;
  __half* tail = static_cast<__half*>(is_v ? p.c.v_tail : p.c.k_tail) + b * ts.batch + h * ts.head;
  const void* src = is_v ? p.v : p.k;
  const RowStrides& ss = is_v ? p.v_new_strides : p.k_new_strides;

  uint32_t most = 0;  // of the magnitudes' bits: infinities and NaN are larger than any number
  for (int task = threadIdx.x; task < page_rows * pieces; task += kAppendThreads) {
    const int r = task / pieces, c = task % pieces;
    const int pos = (index << shift) + r;
    uint4 a, z;
    Piece at;
    if (pos < start) {
      at = Piece{c * 16, c * 16 + 8, false};
      a = *reinterpret_cast<const uint4*>(tail + r * ts.row + at.first);
      z = *reinterpret_cast<const uint4*>(tail + r * ts.row + at.second);
    } else {
      append_load(p, new_row(src, ss, b, h, pos - start), c, !is_v, pos, a, z, at);
    }
    *reinterpret_cast<uint4*>(seal_rows + r * d + at.first) = a;
    *reinterpret_cast<uint4*>(seal_rows + r * d + at.second) = z;
    for (const uint32_t w : {a.x, a.y, a.z, a.w, z.x, z.y, z.z, z.w}) most = __vmaxu2(most, w & 0x7fff7fffu);
  }
  most = max(most & 0xffffu, most >> 16);
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) warp_most[threadIdx.x >> 5] = most;
  __syncthreads();
  most = warp_most[0];
#pragma unroll
  for (int w = 1; w < kAppendThreads / 32; ++w) most = max(most, warp_most[w]);
  const float a = __half2float(__ushort_as_half(static_cast<unsigned short>(most)));
  const bool finite = most < 0x7c00u;
  const bool some = finite && most != 0;

  const int page = threadIdx.x == 0 ? append_page(p, b, index << shift) : p.c.table[b * p.c.table_stride + index];
  if (page >= 0 && page < p.c.num_pages) {
    const RowStrides& s = is_v ? p.c.v_strides : p.c.k_strides;
    uint8_t* out = static_cast<uint8_t*>(is_v ? p.c.v_pages : p.c.k_pages) + page * s.batch + h * s.head;
    for (int task = threadIdx.x; task < page_rows * pieces; task += kAppendThreads) {
      const int r = task / pieces, c = task % pieces;
      const __half2* x = reinterpret_cast<const __half2*>(seal_rows + r * d + c * 16);
      uint32_t w[4] = {0, 0, 0, 0};
      if (some) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = codes_of(static_cast<const T*>(nullptr), __half22float2(x[2 * k]), a) |
                 (codes_of(static_cast<const T*>(nullptr), __half22float2(x[2 * k + 1]), a) << 16);
      }
      *reinterpret_cast<uint4*>(out + r * s.row + c * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (threadIdx.x == 0) {
      float* scales = is_v ? p.c.v_scales : p.c.k_scales;
      // a page with an infinity or a NaN has none that stands for it: what sees the page becomes NaN
      scales[static_cast<int64_t>(page) * p.c.heads_kv + h] =
          finite ? __fdiv_rn(a, code_max(static_cast<const T*>(nullptr))) : __int_as_float(0x7fffffff);
    }
  }
  if (blockIdx.x != 0) return;
  const int left = end & (page_rows - 1);  // rows behind the last full page (the tail was read before the barrier above)
  const int first = end - left;
  for (int task = threadIdx.x; task < left * pieces; task += kAppendThreads) {
    const int r = task / pieces, c = task % pieces;
    uint4 x, z;
    Piece at;
    append_load(p, new_row(src, ss, b, h, first + r - start), c, !is_v, first + r, x, z, at);
    *reinterpret_cast<uint4*>(tail + r * ts.row + at.first) = x;
    *reinterpret_cast<uint4*>(tail + r * ts.row + at.second) = z;
  }
}

template <class T>
cudaError_t launch_seal(const PagedAppendParams& p, cudaStream_t stream) {
  auto kern = fal_paged_seal_kernel<T>;
  static DeviceOnce configured;
  cudaError_t e = configured.run([&] {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPagedMostRows * 256 * 2);
  });
  if (e != cudaSuccess) return e;
  const int64_t page_rows = 1 << p.c.page_shift;
  const unsigned pages = static_cast<unsigned>((p.rows + page_rows - 1) >> p.c.page_shift);  // that one entry can finish
  return launch_dependent(kern, dim3(pages, 2 * p.c.heads_kv, p.c.batch), dim3(kAppendThreads),
                          static_cast<size_t>(p.c.head_dim) * page_rows * 2, stream, p);
}

// ---------------------------------------------------------------------------
// Attention over the pages, few query rows per KV head
// ---------------------------------------------------------------------------
// Bound by HBM: every K and V row is read once for all query rows of its KV head.  The products are mma.sync m16n8k16 with
// 16 keys (scores) or 16 columns of V (output) as the M rows and 8 query rows as N: S^T = K Q^T, O^T = V^T P^T.  Query rows
// are (token, head of the group) pairs, 8 NT to a CTA.  K and V fragments are read from shared memory as the lanes' own 16
// bytes, without ldmatrix: a contraction may take its columns in any order, so lane t of four takes the columns 16 t' ...
// of a key row that are next to each other, and Q is laid out to match; lane g of eight takes D / 8 neighbouring columns of V.
// 8-bit codes become fp16 in registers (exact), the scales enter in 32 bits: K's with the softmax scale, V's where the
// product of a 16-key slice is added to the output.  P^T of the scores' layout becomes the second product's operand by
// movmatrix.
constexpr int kPagedWarps = 4;
constexpr int kPagedThreads = kPagedWarps * 32;
constexpr int kPagedSlice = 16;

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
  const uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(l), "r"(0x64806480u));
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(h), "r"(0x64806480u));
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

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void cp_async_4_zfill(uint32_t dst, const void* src, bool valid) {
  const uint32_t n = valid ? 4u : 0u;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

__device__ __forceinline__ void lds16(uint32_t addr, uint32_t (&w)[4]) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "r"(addr));
}
__device__ __forceinline__ void lds8(uint32_t addr, uint32_t (&w)[2]) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
}

// Rows of D elements in shared memory, 16-byte chunks permuted so that eight lanes of a 16-byte load hit different
// banks: for K they are two rows of four chunks, for V four rows (2 t) of one or two lanes' columns.
template <int D, class T>
struct PagedTile {
  static constexpr int kRowBytes = D * Elem<T>::kBytes;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kSliceBytes = kPagedSlice * kRowBytes;  // K or V
  static constexpr int kLaneBytes = kRowBytes / 8;             // of a V row
  static __device__ __forceinline__ int k_chunk(int row, int ch) { return kChunks >= 8 ? ch ^ ((row & 1) << 2) : ch; }
  static __device__ __forceinline__ int v_chunk(int row, int ch) {
    const int t = (row >> 1) & 3;
    if (kLaneBytes == 8 || kLaneBytes == 64) return ch ^ t;
    if (kLaneBytes == 16) return ch ^ (t << 1);
    return ch ^ ((t & 1) | ((t & 2) << 1));
  }
};

template <int D, class T>
struct PagedSmem {
  static constexpr int kStages = Elem<T>::kScaled ? 4 : 3;
  static constexpr int kRingBytes = kStages * 2 * PagedTile<D, T>::kSliceBytes;  // per warp
  static constexpr int kScaleBytes = kStages * 8;
  static constexpr int kTailStages = kRingBytes / (2 * PagedTile<D, __half>::kSliceBytes);
  static_assert(kTailStages >= 1, "a slice of the tail fits");
  static constexpr int kScaleOffset = kPagedWarps * kRingBytes;
  static constexpr int kPipeBytes = kScaleOffset + kPagedWarps * kScaleBytes;
  static constexpr int merge_bytes(int rows) { return kPagedWarps * rows * (D + 2) * 4; }
  static constexpr int bytes(int rows) { return kPipeBytes > merge_bytes(rows) ? kPipeBytes : merge_bytes(rows); }
};

// log2 of the positions per split of an entry with `len` positions in pages.
__device__ __forceinline__ int paged_split_shift(const PagedAttnParams& p, int len) {
  int shift = kDecodeFinestShift;
  while (shift < p.split_shift && ((len - 1) >> shift) + 1 > p.fine_splits) ++shift;
  return shift;
}
// Positions of an entry of n that are in pages.
__device__ __forceinline__ int paged_len_in_pages(const PagedCache& c, int n) {
  return c.type == kPagedF16 ? n : n >> c.page_shift << c.page_shift;
}

template <int D, int NT>
struct PagedState {
  uint32_t q[D / 16][2][NT];
  float o[NT][D / 16][4];
  float m[NT][2];  // running maximum, log2 domain
  float l[NT][2];  // this lane's part of the sum
};

// Where a warp finds its keys: pages through the table (T as stored), or the tail (fp16).
template <class T>
struct PagedSource {
  const uint8_t* k;  // of the KV head
  const uint8_t* v;
  int64_t k_page, v_page, k_row, v_row;  // bytes
  const int32_t* table;  // of the entry; null for the tail
  int page_shift, num_pages;
  const float* k_scales;  // of the KV head
  const float* v_scales;
  int heads_kv;
  int* status;
};

// Keys pos0 ... pos_end - 1 for the query rows of a CTA, one 16-key slice of every kPagedWarps to a warp.
template <int D, class T, int NT, int STAGES>
__device__ __forceinline__ void paged_stream(const PagedSource<T>& src, uint32_t ring, uint32_t ring_scales, int pos0,
                                             int pos_end, int real_chunks, float c2, const int (&limit)[NT][2], int min_limit,
                                             PagedState<D, NT>& st) {
  using Tile = PagedTile<D, T>;
  constexpr bool kScaled = Elem<T>::kScaled;
  constexpr int kLoads = kPagedSlice * Tile::kChunks / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int slices = (pos_end - pos0 + kPagedSlice - 1) / kPagedSlice;
  const int mine = (slices - warp + kPagedWarps - 1) / kPagedWarps;
  const int page_mask = (1 << src.page_shift) - 1;

  auto page_of = [&](int i) {
    const int slice = i * kPagedWarps + warp;
    return src.table != nullptr && slice < slices ? __ldg(src.table + ((pos0 + slice * kPagedSlice) >> src.page_shift)) : 0;
  };
  int next_page = page_of(0);
  auto issue = [&](int i) {
    const int slice = i * kPagedWarps + warp;
    const int page = next_page;
    next_page = page_of(i + 1);
    if (slice < slices) {
      const int key0 = pos0 + slice * kPagedSlice;
      const uint32_t sb = ring + (i % STAGES) * 2 * Tile::kSliceBytes;
      const bool there = page >= 0 && page < src.num_pages;  // (else its rows are zeros)
      if (!there && lane == 0 && src.status) atomicCAS(src.status, 0, kDevNoPage);
      const int64_t id = there ? page : 0;
      const int row0 = src.table != nullptr ? key0 & page_mask : key0;
      const uint8_t* kp = src.k + id * src.k_page + row0 * src.k_row;
      const uint8_t* vp = src.v + id * src.v_page + row0 * src.v_row;
#pragma unroll
      for (int it = 0; it < kLoads; ++it) {
        const int idx = it * 32 + lane;
        const int row = idx / Tile::kChunks, ch = idx % Tile::kChunks;
        const bool ok = there && key0 + row < pos_end && ch < real_chunks;
        const int64_t r = ok ? row : 0;
        const int sc = ok ? ch : 0;
        cp_async_16_zfill(sb + row * Tile::kRowBytes + Tile::k_chunk(row, ch) * 16, kp + r * src.k_row + sc * 16, ok);
        cp_async_16_zfill(sb + Tile::kSliceBytes + row * Tile::kRowBytes + Tile::v_chunk(row, ch) * 16,
                          vp + r * src.v_row + sc * 16, ok);
      }
      if (kScaled && lane < 2)
        cp_async_4_zfill(ring_scales + (i % STAGES) * 8 + lane * 4, (lane == 0 ? src.k_scales : src.v_scales) + id * src.heads_kv,
                         there);
    }
    cp_async_commit();  // (always, so that the groups count the same)
  };

#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(i);
  for (int i = 0; i < mine; ++i) {
    issue(i + STAGES - 1);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const uint32_t sb = ring + (i % STAGES) * 2 * Tile::kSliceBytes;
    const int key0 = pos0 + (i * kPagedWarps + warp) * kPagedSlice;
    float k_scale = 1.f, v_scale = 1.f;
    if constexpr (kScaled)
      asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(k_scale), "=f"(v_scale) : "r"(ring_scales + (i % STAGES) * 8));

    // ---- S^T = K Q^T: 16 keys x 8 NT query rows ----
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
#pragma unroll
    for (int seg = 0; seg < Tile::kRowBytes / 64; ++seg) {
      uint32_t r0[4], r1[4];
      lds16(sb + g * Tile::kRowBytes + Tile::k_chunk(g, seg * 4 + t) * 16, r0);
      lds16(sb + (g + 8) * Tile::kRowBytes + Tile::k_chunk(g + 8, seg * 4 + t) * 16, r1);
      if constexpr (kScaled) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t a[4];
          widen(static_cast<const T*>(nullptr), r0[k], a[0], a[2]);
          widen(static_cast<const T*>(nullptr), r1[k], a[1], a[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816(s[nt], a, st.q[seg * 4 + k][0][nt], st.q[seg * 4 + k][1][nt]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t a[4] = {r0[2 * k], r1[2 * k], r0[2 * k + 1], r1[2 * k + 1]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816(s[nt], a, st.q[seg * 2 + k][0][nt], st.q[seg * 2 + k][1][nt]);
        }
      }
    }

    // ---- softmax over the keys: this lane has keys g and g + 8 of query rows 2 t and 2 t + 1 of every eight ----
    const float f = c2 * k_scale;
    const bool masked = key0 + kPagedSlice > min_limit;
    uint32_t pb[NT][2];
    float mx[NT][2];
    bool grows = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[nt][e] *= f;
        if (masked && key0 + g + (e >> 1) * 8 >= limit[nt][e & 1]) s[nt][e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = fmaxf(s[nt][e], s[nt][2 + e]);
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        mx[nt][e] = x;
        grows = grows || x > st.m[nt][e];
      }
    }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float m_new = fmaxf(st.m[nt][e], mx[nt][e]);
          alpha[e] = fast_exp2(st.m[nt][e] - (m_new == -INFINITY ? 0.f : m_new));
          st.l[nt][e] *= alpha[e];
          st.m[nt][e] = m_new;
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          st.o[nt][j][0] *= alpha[0];
          st.o[nt][j][1] *= alpha[1];
          st.o[nt][j][2] *= alpha[0];
          st.o[nt][j][3] *= alpha[1];
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float m_use = st.m[nt][e] == -INFINITY ? 0.f : st.m[nt][e];
        s[nt][e] = fast_exp2(s[nt][e] - m_use);
        s[nt][2 + e] = fast_exp2(s[nt][2 + e] - m_use);
        st.l[nt][e] += s[nt][e] + s[nt][2 + e];
      }
      pb[nt][0] = movmatrix(pack_half2(s[nt][0], s[nt][1]));
      pb[nt][1] = movmatrix(pack_half2(s[nt][2], s[nt][3]));
    }

    // ---- O^T += V^T P^T ----
    const uint32_t vb = sb + Tile::kSliceBytes;
    auto product = [&](int j, const uint32_t (&a)[4]) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if constexpr (kScaled) {
          float x[4] = {0.f, 0.f, 0.f, 0.f};
          mma_16816(x, a, pb[nt][0], pb[nt][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) st.o[nt][j][e] += v_scale * x[e];
        } else {
          mma_16816(st.o[nt][j], a, pb[nt][0], pb[nt][1]);
        }
      }
    };
    constexpr int kPiece = Tile::kLaneBytes < 16 ? Tile::kLaneBytes : 16;
#pragma unroll
    for (int piece = 0; piece < Tile::kLaneBytes / kPiece; ++piece) {
      uint32_t w[4][4];  // rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 2 * t + (r & 1) + (r >> 1) * 8;
        const int byte = g * Tile::kLaneBytes + piece * 16;
        const uint32_t addr = vb + row * Tile::kRowBytes + Tile::v_chunk(row, byte >> 4) * 16 + (byte & 15);
        if constexpr (kPiece == 16) {
          lds16(addr, w[r]);
        } else {
          uint32_t half_row[2];
          lds8(addr, half_row);
          w[r][0] = half_row[0];
          w[r][1] = half_row[1];
        }
      }
#pragma unroll
      for (int k = 0; k < kPiece / 4; ++k) {
        if constexpr (kScaled) {
          const int j = piece * 8 + 2 * k;  // two output tiles of two columns a lane
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t a[4];
            widen(static_cast<const T*>(nullptr), __byte_perm(w[0][k], w[1][k], u == 0 ? 0x5140 : 0x7362), a[0], a[1]);
            widen(static_cast<const T*>(nullptr), __byte_perm(w[2][k], w[3][k], u == 0 ? 0x5140 : 0x7362), a[2], a[3]);
            product(j + u, a);
          }
        } else {
          const uint32_t a[4] = {__byte_perm(w[0][k], w[1][k], 0x5410), __byte_perm(w[0][k], w[1][k], 0x7632),
                                 __byte_perm(w[2][k], w[3][k], 0x5410), __byte_perm(w[2][k], w[3][k], 0x7632)};
          product(piece * 4 + k, a);
        }
      }
    }
    __syncwarp();  // all lanes are done with this stage before it is refilled
  }
  cp_async_wait<0>();
}

// Grid: (KV head x chunk of 8 NT query rows, split -- the last one of 8-bit caches is the tail --, entry).
template <int D, class T, int NT>
__global__ void __launch_bounds__(kPagedThreads) fal_paged_splitk_kernel(const PagedAttnParams p) {
  using L = PagedSmem<D, T>;
  constexpr int kRows = 8 * NT;
  extern __shared__ __align__(128) uint8_t paged_smem[];
  grid_dependency_wait();    // the append of this step's rows may still run up to here
  grid_dependency_launch();
  const PagedCache& c = p.c;
  const int group = p.heads_q / c.heads_kv;
  const int chunks = (p.rows * group + kRows - 1) / kRows;
  const int kv_head = blockIdx.x / chunks;
  const int row0 = blockIdx.x % chunks * kRows;  // of the KV head's rows * group query rows
  const int rows_valid = min(kRows, p.rows * group - row0);
  const int b = blockIdx.z;
  const int n = paged_len(c, b);
  const int in_pages = paged_len_in_pages(c, n);
  const int shift = paged_split_shift(p, in_pages);
  const bool is_tail = Elem<T>::kScaled && blockIdx.y == static_cast<unsigned>(p.grid_splits);
  const int split = is_tail ? ((in_pages - 1) >> shift) + 1 : blockIdx.y;  // of the partial results
  const int pos0 = is_tail ? in_pages : split << shift;
  const int pos_end = is_tail ? n : min(pos0 + (1 << shift), in_pages);
  if (pos0 >= pos_end) return;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  PagedState<D, NT> st;
  int limit[NT][2];  // first key that a query row does not see
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      limit[nt][e] = min(pos_end, n - p.rows + (row0 + nt * 8 + 2 * t + e) / group + 1);
      st.m[nt][e] = -INFINITY;
      st.l[nt][e] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[nt][j][e] = 0.f;
  }
  const int min_limit = min(pos_end, n - p.rows + row0 / group + 1);
  const float c2 = p.scale * kLog2e;
  const uint32_t ring = smem_u32(paged_smem) + warp * L::kRingBytes;
  const uint32_t ring_scales = smem_u32(paged_smem) + L::kScaleOffset + warp * L::kScaleBytes;

  // Q as the first product's second operand: of every group of four columns that a lane's key fragment holds, two each.
  auto load_q = [&](auto elem) {
    constexpr int kE = 16 / Elem<decltype(elem)>::kBytes;  // columns of a lane's 16 bytes
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = nt * 8 + g;
      const __half* q = nullptr;
      if (row < rows_valid)
        q = static_cast<const __half*>(p.q) + b * p.q_strides.batch + (row0 + row) / group * p.q_strides.row +
            (kv_head * group + (row0 + row) % group) * p.q_strides.head;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int col = (ks / (kE / 4)) * 4 * kE + t * kE + (ks % (kE / 4)) * 4;
        uint2 x = make_uint2(0u, 0u);
        if (row < rows_valid && col < c.head_dim) x = *reinterpret_cast<const uint2*>(q + col);
        st.q[ks][0][nt] = x.x;
        st.q[ks][1][nt] = x.y;
      }
    }
  };
  const int real_bytes = c.head_dim;  // x the element's bytes
  if (is_tail) {
    if constexpr (Elem<T>::kScaled) {
      load_q(__half{});
      PagedSource<__half> src{};
      src.k_row = c.k_tail_strides.row * 2;
      src.v_row = c.v_tail_strides.row * 2;
      src.k = static_cast<const uint8_t*>(c.k_tail) + (b * c.k_tail_strides.batch + kv_head * c.k_tail_strides.head) * 2 -
              in_pages * src.k_row;
      src.v = static_cast<const uint8_t*>(c.v_tail) + (b * c.v_tail_strides.batch + kv_head * c.v_tail_strides.head) * 2 -
              in_pages * src.v_row;
      src.num_pages = 1;
      paged_stream<D, __half, NT, L::kTailStages>(src, ring, ring_scales, pos0, pos_end, real_bytes / 8, c2, limit, min_limit, st);
    }
  } else {
    load_q(T{});
    constexpr int kB = Elem<T>::kBytes;
    PagedSource<T> src{};
    src.k = static_cast<const uint8_t*>(c.k_pages) + kv_head * c.k_strides.head * kB;
    src.v = static_cast<const uint8_t*>(c.v_pages) + kv_head * c.v_strides.head * kB;
    src.k_page = c.k_strides.batch * kB;
    src.v_page = c.v_strides.batch * kB;
    src.k_row = c.k_strides.row * kB;
    src.v_row = c.v_strides.row * kB;
    src.table = c.table + b * c.table_stride;
    src.page_shift = c.page_shift;
    src.num_pages = c.num_pages;
    src.k_scales = c.k_scales + (Elem<T>::kScaled ? kv_head : 0);
    src.v_scales = c.v_scales + (Elem<T>::kScaled ? kv_head : 0);
    src.heads_kv = c.heads_kv;
    src.status = p.status;
    paged_stream<D, T, NT, L::kStages>(src, ring, ring_scales, pos0, pos_end, real_bytes * kB / 16, c2, limit, min_limit, st);
  }
  __syncthreads();  // the ring becomes the place of the warps' results

  float* mo = reinterpret_cast<float*>(paged_smem);  // [warp][row][D]
  float* mml = mo + kPagedWarps * kRows * D;         // [warp][row][2]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = warp * kRows + nt * 8 + 2 * t + e;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
        *reinterpret_cast<float2*>(mo + row * D + g * (D / 8) + 2 * j) = make_float2(st.o[nt][j][e], st.o[nt][j][2 + e]);
      float l = st.l[nt][e];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      if (g == 0) *reinterpret_cast<float2*>(mml + row * 2) = make_float2(st.m[nt][e], l);
    }
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < rows_valid * D; idx += kPagedThreads) {
    const int r = idx / D, col = idx % D;
    float most = -INFINITY;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) most = fmaxf(most, mml[(w * kRows + r) * 2]);
    const float use = most == -INFINITY ? 0.f : most;
    float o = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) {
      const float x = fast_exp2(mml[(w * kRows + r) * 2] - use);
      o += x * mo[(w * kRows + r) * D + col];
      l += x * mml[(w * kRows + r) * 2 + 1];
    }
    const int64_t head = kv_head * group + (row0 + r) % group;
    const int64_t at = ((static_cast<int64_t>(b) * p.rows + (row0 + r) / group) * p.heads_q + head) * p.splits + split;
    p.part_o[at * D + col] = o;
    if (col == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(most, l);
  }
}

template <int D, int WARPS>
__global__ void __launch_bounds__(kCombineThreads) fal_paged_combine_kernel(const PagedAttnParams p) {
  constexpr int kRows = kCombineThreads / (32 * WARPS);
  const int tid = threadIdx.x % (32 * WARPS);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / (32 * WARPS);
  const bool row_ok = row < static_cast<int64_t>(p.c.batch) * p.rows * p.heads_q;
  int n = 0;
  if (row_ok) {
    const int len = paged_len(p.c, static_cast<int>(row / (static_cast<int64_t>(p.rows) * p.heads_q)));
    const int in_pages = paged_len_in_pages(p.c, len);
    n = ((in_pages - 1) >> paged_split_shift(p, in_pages)) + 1 + (len > in_pages ? 1 : 0);
  }
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + row * p.splits;
  const float4* po = reinterpret_cast<const float4*>(p.part_o) + row * p.splits * (D / 4);
  combine_row<D, WARPS>(tid, row_ok, n, ml, po, static_cast<__half*>(p.o) + row * p.c.head_dim, p.c.head_dim, nullptr);
}

template <int D, class T, int NT>
cudaError_t launch_splitk_t(const PagedAttnParams& p, cudaStream_t stream) {
  auto kern = fal_paged_splitk_kernel<D, T, NT>;
  constexpr int kBytes = PagedSmem<D, T>::bytes(8 * NT);
  static DeviceOnce configured;
  cudaError_t e = configured.run([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes); });
  if (e != cudaSuccess) return e;
  const int group = p.heads_q / p.c.heads_kv;
  const dim3 grid(p.c.heads_kv * ((p.rows * group + 8 * NT - 1) / (8 * NT)), p.splits, p.c.batch);
  e = launch_dependent(kern, grid, dim3(kPagedThreads), kBytes, stream, p);
  if (e != cudaSuccess) return e;
  const int64_t rows = static_cast<int64_t>(p.c.batch) * p.rows * p.heads_q;
  if (p.splits * p.kernel_dim * 4 <= (rows >= 256 ? 4096 : 2048))
    return launch_dependent(fal_paged_combine_kernel<D, 1>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(kCombineThreads), 0, stream, p);
  return launch_dependent(fal_paged_combine_kernel<D, 4>, dim3(static_cast<unsigned>(rows)), dim3(kCombineThreads), 0, stream, p);
}

template <int D, class T>
cudaError_t launch_splitk_d(const PagedAttnParams& p, cudaStream_t stream) {
  if constexpr (D < 256) {
    if (paged_rows_per_cta(p.rows * (p.heads_q / p.c.heads_kv), D) == 16) return launch_splitk_t<D, T, 2>(p, stream);
  }
  return launch_splitk_t<D, T, 1>(p, stream);
}

template <class T>
cudaError_t launch_splitk(const PagedAttnParams& p, cudaStream_t stream) {
  if (p.kernel_dim == 64) return launch_splitk_d<64, T>(p, stream);
  if (p.kernel_dim == 128) return launch_splitk_d<128, T>(p, stream);
  return launch_splitk_d<256, T>(p, stream);
}

// ---------------------------------------------------------------------------
// Rows in order, for the forward kernel
// ---------------------------------------------------------------------------
// Bound by HBM.  A thread takes 16 columns of a row; code x scale is rounded to fp16, which the forward kernel's operands are.
template <class T>
__global__ void __launch_bounds__(256) fal_paged_gather_kernel(const PagedGatherParams p) {
  const PagedCache& c = p.c;
  const int pieces = c.head_dim / 16;
  const int e = blockIdx.z;
  const int b = p.b0 + e;
  const bool is_v = blockIdx.y >= static_cast<unsigned>(p.heads);
  const int hh = is_v ? blockIdx.y - p.heads : blockIdx.y;
  const int h = p.h0 + hh;
  const int n = paged_len(c, b), in_pages = paged_len_in_pages(c, n);
  const int64_t task = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t pos = task / pieces;
  const int col = static_cast<int>(task % pieces) * 16;
  if (pos >= n) return;
  uint4 out[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (pos >= in_pages) {
    const RowStrides& s = is_v ? c.v_tail_strides : c.k_tail_strides;
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __half*>(is_v ? c.v_tail : c.k_tail) + b * s.batch +
                                                      h * s.head + (pos - in_pages) * s.row + col);
    out[0] = src[0];
    out[1] = src[1];
  } else {
    const int page = c.table[b * c.table_stride + (pos >> c.page_shift)];
    if (page >= 0 && page < c.num_pages) {
      const RowStrides& s = is_v ? c.v_strides : c.k_strides;
      const int64_t at = page * s.batch + h * s.head + (pos & ((1 << c.page_shift) - 1)) * s.row + col;
      if constexpr (Elem<T>::kScaled) {
        const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(is_v ? c.v_pages : c.k_pages) + at);
        const float scale = (is_v ? c.v_scales : c.k_scales)[static_cast<int64_t>(page) * c.heads_kv + h];
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t lo, hi;
          widen(static_cast<const T*>(nullptr), w[i], lo, hi);
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo));
          const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          y[2 * i] = pack_half2(x.x * scale, x.y * scale);
          y[2 * i + 1] = pack_half2(z.x * scale, z.y * scale);
        }
        out[0] = make_uint4(y[0], y[1], y[2], y[3]);
        out[1] = make_uint4(y[4], y[5], y[6], y[7]);
      } else {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __half*>(is_v ? c.v_pages : c.k_pages) + at);
        out[0] = src[0];
        out[1] = src[1];
      }
    } else if (col == 0 && p.status) {
      atomicCAS(p.status, 0, kDevNoPage);
    }
  }
  const int64_t capacity = paged_capacity(c);
  __half* dst = static_cast<__half*>(is_v ? p.v_out : p.k_out) + ((static_cast<int64_t>(e) * p.heads + hh) * capacity + pos) * c.head_dim + col;
  reinterpret_cast<uint4*>(dst)[0] = out[0];
  reinterpret_cast<uint4*>(dst)[1] = out[1];
}

}  // namespace

int paged_rows_per_cta(int rows, int kernel_dim) { return rows > 8 && kernel_dim < 256 ? 16 : 8; }

cudaError_t launch_paged_append(const PagedAppendParams& p, cudaStream_t stream) {
  const int tasks = (p.heads_q + 2 * p.c.heads_kv) * (p.c.head_dim / 16);
  const int64_t tokens = static_cast<int64_t>(p.c.batch) * p.rows;
  const int groups = (tasks + kAppendThreads - 1) / kAppendThreads;
  if (tokens > 0x7fffffff || groups > 65535) return cudaErrorInvalidValue;
  cudaError_t e = launch_dependent(fal_paged_append_kernel, dim3(static_cast<unsigned>(tokens), groups), dim3(kAppendThreads), 0, stream, p);
  if (e != cudaSuccess || p.c.type == kPagedF16) return e;
  return p.c.type == kPagedS8 ? launch_seal<S8>(p, stream) : launch_seal<E4M3>(p, stream);
}

cudaError_t launch_paged_attn(const PagedAttnParams& p, cudaStream_t stream) {
  if (p.c.type == kPagedF16) return launch_splitk<__half>(p, stream);
  if (p.c.type == kPagedS8) return launch_splitk<S8>(p, stream);
  return launch_splitk<E4M3>(p, stream);
}

cudaError_t launch_paged_gather(const PagedGatherParams& p, cudaStream_t stream) {
  const int64_t tasks = (static_cast<int64_t>(p.c.pages_per_entry) << p.c.page_shift) * (p.c.head_dim / 16);
  const int64_t blocks = (tasks + 255) / 256;
  if (blocks > 0x7fffffff || 2 * p.heads > 65535 || p.entries > 65535) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks), 2 * p.heads, p.entries);
  if (p.c.type == kPagedF16) fal_paged_gather_kernel<__half><<<grid, 256, 0, stream>>>(p);
  else if (p.c.type == kPagedS8) fal_paged_gather_kernel<S8><<<grid, 256, 0, stream>>>(p);
  else fal_paged_gather_kernel<E4M3><<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace fal
