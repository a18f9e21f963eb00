// Append of new rows to a paged key/value cache, with the position rotation on the way.
//
// The reference has no paged cache; its hook attends eagerly over dense ones (flash_attn_legacy/integrations.py:77-98).
//
// 8-bit pages.  A value is rounded to 8 bits once, when its page is full: a = max |x| over the page's rows of a head,
// scale = a / m and code = round(x m / a), m = 127 (int8, nearest whole number) or 448 (e4m3, nearest such number).  Until
// then the row waits as fp16 in the entry's tail, so that the cache does not depend on how the rows came in, token by
// token or as chunks, and no page is rounded again when a larger value arrives.  The codes are those of the exact quotients: one
// is on a rounding border or at least 2^-19 of itself away, because a border is a number of 8 bits at most, a one of 11, and
// the difference of x m and border x a a whole number in the units of both.
#include <algorithm>
#include <type_traits>

#include "fal_paged.cuh"

namespace fal {

namespace {

// Prompts are bound by HBM with fp16 pages (0.90 of a copy's rate), by the integer and floating pipes with 8-bit ones (4 x 1 024
// tokens of 32 + 8 + 8 heads of 128, int8, 22.9 us, 4.2 TB/s); single tokens by latency.  A thread takes 16 columns of a head:
// the two 8-column pieces whose columns are rotated with each other, or two neighbouring ones.
constexpr int kAppendThreads = 256;
// Blocks per SM: 48 registers a thread, at which the kernels of 8-bit pages store 192 bytes a thread and load 124 that four blocks
// would leave in registers (fp16 pages: 8).  us with 4 / 5 / 6 blocks on 4 x 2 987 tokens of 40 + 8 + 8 heads of 128, fp16: 63.3 / 59.9
// (5.8 TB/s) / 60.1; with 3 / 4 / 5 on the same in int8, 81.2 / 70.2 / 69.6, on 13 x 1 027 of 24 + 8 + 8, 73.1 / 63.4 / 61.4.
constexpr int kAppendBlocks = 5;

// How a launch is laid out: a grid row per entry, first its page blocks, then its token blocks.
struct AppendGrid {
  unsigned page_blocks;   // of an entry
  unsigned head_groups;   // page blocks of a page
  int head_threads_log2;  // of a page block, to a head
  unsigned per_piece;     // 65 536 / pieces of a row, rounded up
};
// x / pieces of a row, for x < 65 536 / 6: a multiplication, because divisions were a third of the instructions of a kernel that
// the integer pipe bounded (13 x 1 027 tokens of 24 / 8 heads of 128, int8, 69.7 us, without them 63.4).
__device__ __forceinline__ int over_pieces(const AppendGrid& g, int x) { return static_cast<int>(x * g.per_piece >> 16); }

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

// cos and sin of the eight column pairs of piece c at position pos.
struct Angles {
  float cs[8], sn[8];
};
__device__ __forceinline__ Angles append_angles(const PagedAppendParams& p, int c, int pos) {
  Angles x;
  const int64_t at = static_cast<int64_t>(pos) * (p.rotary_dim / 2) + c * 8;
  load_angles(p.cos, p.half_tables, at, x.cs);
  load_angles(p.sin, p.half_tables, at, x.sn);
  return x;
}
__device__ __forceinline__ void append_turn(const PagedAppendParams& p, const Angles& x, uint4& a, uint4& b) {
  __half2* ha = reinterpret_cast<__half2*>(&a);
  __half2* hb = reinterpret_cast<__half2*>(&b);
  if (p.interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 u = __half22float2(ha[i]), v = __half22float2(hb[i]);
      turn(u.x, u.y, x.cs[i], x.sn[i]);
      turn(v.x, v.y, x.cs[4 + i], x.sn[4 + i]);
      ha[i] = __floats2half2_rn(u.x, u.y);
      hb[i] = __floats2half2_rn(v.x, v.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 u = __half22float2(ha[i]), v = __half22float2(hb[i]);
      turn(u.x, v.x, x.cs[2 * i], x.sn[2 * i]);
      turn(u.y, v.y, x.cs[2 * i + 1], x.sn[2 * i + 1]);
      ha[i] = __floats2half2_rn(u.x, u.y);
      hb[i] = __floats2half2_rn(v.x, v.y);
    }
  }
}

// The two pieces of a row of k (v: not rotated) at position pos, rotated.
__device__ __forceinline__ void append_load(const PagedAppendParams& p, const __half* row, int c, bool turned, int pos,
                                            uint4& a, uint4& b, Piece& at) {
  at = append_piece(p, c);
  if (!turned) at = Piece{c * 16, c * 16 + 8, false};
  a = *reinterpret_cast<const uint4*>(row + at.first);
  b = *reinterpret_cast<const uint4*>(row + at.second);
  if (at.rotated) append_turn(p, append_angles(p, c, pos), a, b);
}

__device__ __forceinline__ const __half* new_row(const void* base, const RowStrides& s, int b, int h, int r) {
  return static_cast<const __half*>(base) + b * s.batch + h * s.head + r * s.row;
}

// Half a token block: one token.  A thread takes one piece of every few heads, so that it fetches its angles once (a thread for
// every piece of a token's heads, angles and all, took 36 us where this took 26: 4 x 1 024 tokens of 48 heads of 128, int8).
// Rows of 8-bit caches that finish a page are the page blocks' business, and so are those behind such a page: their places in
// the tail are read there first.
constexpr int kTokenThreads = kAppendThreads / 2;
__device__ __forceinline__ void append_token(const PagedAppendParams& p, const AppendGrid& grid, int b, int i, int thread) {
  const int start = p.c.lens[b];
  const int capacity = paged_capacity(p.c);
  const int pieces = p.c.head_dim / 16;
  const int lanes = over_pieces(grid, kTokenThreads), lane = over_pieces(grid, thread), c = thread - lane * pieces;
  const int64_t pos64 = static_cast<int64_t>(start) + i;
  const bool placed = start >= 0 && pos64 < capacity;  // (start < 0: an unused entry of a padded batch)
  const int pos = placed ? static_cast<int>(pos64) : 0;
  if (thread == 0) {
    if (i == 0)
      p.new_lens[b] =
          start < 0 ? start : static_cast<int>(min(static_cast<int64_t>(start) + p.rows, static_cast<int64_t>(capacity)));
    if (start >= 0 && !placed && p.status) atomicCAS(p.status, 0, kDevAppendOverflow);
  }
  if (lane >= lanes) return;  // (head_dim 96)
  const int shift = p.c.page_shift;
  const int in_page = pos & ((1 << shift) - 1);
  // where head 0 of the token's K and V rows goes, or nowhere
  __half *k_to = nullptr, *v_to = nullptr;
  int64_t k_head = 0, v_head = 0;
  if (p.c.type == kPagedF16) {
    int page = -1;
    if (placed) {
      page = p.c.table[b * p.c.table_stride + (pos >> shift)];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.c.num_pages)) {
        page = -1;
        if (thread == 0 && p.status) atomicCAS(p.status, 0, kDevAppendOverflow);
      }
    }
    if (page >= 0) {
      k_to = static_cast<__half*>(p.c.k_pages) + page * p.c.k_strides.batch + in_page * p.c.k_strides.row;
      v_to = static_cast<__half*>(p.c.v_pages) + page * p.c.v_strides.batch + in_page * p.c.v_strides.row;
    }
    k_head = p.c.k_strides.head;
    v_head = p.c.v_strides.head;
  } else {
    const int64_t end = min(static_cast<int64_t>(start) + p.rows, static_cast<int64_t>(capacity));
    if (placed && (end >> shift) == (start >> shift)) {
      k_to = static_cast<__half*>(p.c.k_tail) + b * p.c.k_tail_strides.batch + in_page * p.c.k_tail_strides.row;
      v_to = static_cast<__half*>(p.c.v_tail) + b * p.c.v_tail_strides.batch + in_page * p.c.v_tail_strides.row;
    }
    k_head = p.c.k_tail_strides.head;
    v_head = p.c.v_tail_strides.head;
  }
  const Piece turned = append_piece(p, c), plain{c * 16, c * 16 + 8, false};
  Angles angles;
  if (turned.rotated) angles = append_angles(p, c, pos);
  const int heads = p.heads_q + (k_to != nullptr ? 2 * p.c.heads_kv : 0);
  for (int h = lane; h < heads; h += lanes) {
    const int hk = h - p.heads_q, hv = hk - p.c.heads_kv;
    const __half* src = hk < 0 ? new_row(p.q, p.q_strides, b, h, i) : hv < 0 ? new_row(p.k, p.k_new_strides, b, hk, i)
                                                                            : new_row(p.v, p.v_new_strides, b, hv, i);
    const Piece& at = hv < 0 ? turned : plain;
    uint4 a = *reinterpret_cast<const uint4*>(src + at.first), z = *reinterpret_cast<const uint4*>(src + at.second);
    if (at.rotated) append_turn(p, angles, a, z);
    __half* dst = hk < 0 ? static_cast<__half*>(p.q_out) + ((static_cast<int64_t>(b) * p.rows + i) * p.heads_q + h) * p.c.head_dim
                         : hv < 0 ? k_to + hk * k_head : v_to + hv * v_head;
    if (!placed) a = z = make_uint4(0, 0, 0, 0);  // (a query without a position)
    *reinterpret_cast<uint4*>(dst + at.first) = a;
    *reinterpret_cast<uint4*>(dst + at.second) = z;
  }
}

// x m / a, near enough for its rounding to a code: x's product with c = m / a is within 2^-22.9 of itself of the quotient.
// Rounded to 21 bits it is a border of the codes where the quotient is one, and on the quotient's side of every border
// elsewhere, 2^-20.5 against 2^-19.  (A zero keeps its sign.)
__device__ __forceinline__ float quotient(float x, float c) {
  return __uint_as_float((__float_as_uint(__fmul_rn(x, c)) + 4u) & ~7u);
}
// The codes of four fp16 values as four bytes.  A sum with 1.5 x 2^23 is rounded to a whole number, in the lowest bits.
__device__ __forceinline__ uint32_t codes_of(const S8*, float2 x, float2 z, float c) {
  auto whole = [&](float y) { return __float_as_uint(__fadd_rn(quotient(y, c), 12582912.f)); };
  return __byte_perm(__byte_perm(whole(x.x), whole(x.y), 0x0040), __byte_perm(whole(z.x), whole(z.y), 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t codes_of(const E4M3*, float2 x, float2 z, float c) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(quotient(x.y, c)), "f"(quotient(x.x, c)));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(quotient(z.y, c)), "f"(quotient(z.x, c)));
  return lo | static_cast<uint32_t>(hi) << 16;
}
__device__ __forceinline__ float code_max(const S8*) { return 127.f; }
__device__ __forceinline__ float code_max(const E4M3*) { return 448.f; }

// A page block: the index-th page from the one of entry b's first new row, for a few KV heads of K or of V, `threads` to a head.
// A thread keeps the first kSealKept pieces that it reads (the rows before the new ones from the tail, the others from the
// call, rotated) and reads further ones, of pages of more than 8 192 values a head, again: once for the largest magnitude, once
// for the codes.  The first page's block also writes the rows behind the last full page to the tail, once it has read it.
// (256 threads to a head took 104 us where this took 80: 4 x 2 987 tokens, pages of 16 x 128.)
constexpr int kSealKept = 2;
template <class T>
__device__ __forceinline__ void append_page_codes(const PagedAppendParams& p, const AppendGrid& grid, int b, int first_head,
                                                  int index_from) {
  const int threads = 1 << grid.head_threads_log2;
  __shared__ uint32_t warp_most[kAppendThreads / 32];
  const int start = p.c.lens[b];
  const int capacity = paged_capacity(p.c);
  const int shift = p.c.page_shift;
  if (start < 0 || start >= capacity) return;
  const int end = static_cast<int>(min(static_cast<int64_t>(start) + p.rows, static_cast<int64_t>(capacity)));
  const int index = (start >> shift) + index_from;  // page of the entry
  if (index >= (end >> shift)) return;              // not full
  const int wanted = first_head + static_cast<int>(threadIdx.x >> grid.head_threads_log2);
  const int head = min(wanted, 2 * p.c.heads_kv - 1);
  const bool active = wanted == head;
  const int thread = threadIdx.x & (threads - 1);
  const int page = p.c.table[b * p.c.table_stride + index];
  const bool is_v = head >= p.c.heads_kv;
  const int h = is_v ? head - p.c.heads_kv : head;
  const int pieces = p.c.head_dim / 16, page_rows = 1 << shift, tasks = active ? page_rows * pieces : 0;
  const RowStrides& ts = is_v ? p.c.v_tail_strides : p.c.k_tail_strides;
  __half* tail = static_cast<__half*>(is_v ? p.c.v_tail : p.c.k_tail) + b * ts.batch + h * ts.head;
  const void* src = is_v ? p.v : p.k;
  const RowStrides& ss = is_v ? p.v_new_strides : p.k_new_strides;
  auto load = [&](int task, uint4& a, uint4& z, Piece& at) {
    const int r = over_pieces(grid, task), c = task - r * pieces;
    const int pos = (index << shift) + r;
    if (pos < start) {
      // (in the pieces that the rotation of a new row takes together, so that one place holds one piece)
      at = append_piece(p, c);
      if (is_v) at = Piece{c * 16, c * 16 + 8, false};
      a = *reinterpret_cast<const uint4*>(tail + r * ts.row + at.first);
      z = *reinterpret_cast<const uint4*>(tail + r * ts.row + at.second);
    } else {
      append_load(p, new_row(src, ss, b, h, pos - start), c, !is_v, pos, a, z, at);
    }
  };
  uint32_t most = 0;  // of the magnitudes' bits: infinities and NaN are larger than any number
  auto look = [&](const uint4& x) {
    for (const uint32_t w : {x.x, x.y, x.z, x.w}) most = __vmaxu2(most, w & 0x7fff7fffu);
  };
  uint4 kept[kSealKept][2];
  Piece at;
#pragma unroll
  for (int k = 0; k < kSealKept; ++k) {
    kept[k][0] = kept[k][1] = make_uint4(0, 0, 0, 0);
    const int task = thread + k * threads;
    if (task < tasks) load(task, kept[k][0], kept[k][1], at);
    look(kept[k][0]);
    look(kept[k][1]);
  }
  for (int task = thread + kSealKept * threads; task < tasks; task += threads) {
    uint4 a, z;
    load(task, a, z, at);
    look(a);
    look(z);
  }
  most = max(most & 0xffffu, most >> 16);
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) warp_most[threadIdx.x >> 5] = most;
  __syncthreads();
  const int first_warp = (threadIdx.x - thread) / 32;
  for (int w = 0; w < threads / 32; ++w) most = max(most, warp_most[first_warp + w]);
  const float largest = __half2float(__ushort_as_half(static_cast<unsigned short>(most)));
  const bool finite = most < 0x7c00u;
  const bool some = finite && most != 0;
  const float per_value = some ? __fdiv_rn(code_max(static_cast<const T*>(nullptr)), largest) : 0.f;

  if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.c.num_pages)) {
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, kDevAppendOverflow);
  } else {
    const RowStrides& s = is_v ? p.c.v_strides : p.c.k_strides;
    uint8_t* out = static_cast<uint8_t*>(is_v ? p.c.v_pages : p.c.k_pages) + page * s.batch + h * s.head;
    auto codes = [&](const uint4& x) {
      uint2 w = make_uint2(0u, 0u);
      if (some) {
        const __half2* y = reinterpret_cast<const __half2*>(&x);
        const T* type = nullptr;
        w.x = codes_of(type, __half22float2(y[0]), __half22float2(y[1]), per_value);
        w.y = codes_of(type, __half22float2(y[2]), __half22float2(y[3]), per_value);
      }
      return w;
    };
    auto store = [&](int task, const uint4& a, const uint4& z) {
      const int r = over_pieces(grid, task), c = task - r * pieces;
      Piece to = append_piece(p, c);
      if (is_v) to = Piece{c * 16, c * 16 + 8, false};
      *reinterpret_cast<uint2*>(out + r * s.row + to.first) = codes(a);
      *reinterpret_cast<uint2*>(out + r * s.row + to.second) = codes(z);
    };
#pragma unroll
    for (int k = 0; k < kSealKept; ++k) {
      const int task = thread + k * threads;
      if (task < tasks) store(task, kept[k][0], kept[k][1]);
    }
    for (int task = thread + kSealKept * threads; task < tasks; task += threads) {
      uint4 a, z;
      load(task, a, z, at);
      store(task, a, z);
    }
    if (active && thread == 0) {
      float* scales = is_v ? p.c.v_scales : p.c.k_scales;
      // a page with an infinity or a NaN has none that stands for it: what sees the page becomes NaN
      scales[static_cast<int64_t>(page) * p.c.heads_kv + h] =
          finite ? __fdiv_rn(largest, code_max(static_cast<const T*>(nullptr))) : __int_as_float(0x7fffffff);
    }
  }
  if (index_from != 0) return;
  __syncthreads();  // the tail's rows of this page have been read
  const int left = active ? end & (page_rows - 1) : 0;  // rows behind the last full page
  const int first = end & ~(page_rows - 1);
  for (int task = thread; task < left * pieces; task += threads) {
    const int r = over_pieces(grid, task), c = task - r * pieces;
    uint4 x, z;
    append_load(p, new_row(src, ss, b, h, first + r - start), c, !is_v, first + r, x, z, at);
    *reinterpret_cast<uint4*>(tail + r * ts.row + at.first) = x;
    *reinterpret_cast<uint4*>(tail + r * ts.row + at.second) = z;
  }
}

template <class T>
__global__ void __launch_bounds__(kAppendThreads, kAppendBlocks)
fal_paged_append_kernel(const PagedAppendParams p, const AppendGrid grid) {
  grid_dependency_wait();
  grid_dependency_launch();
  const int b = blockIdx.y;
  if constexpr (!std::is_same<T, __half>::value) {
    if (blockIdx.x < grid.page_blocks) {  // (page, then heads of K and of V)
      const unsigned page = blockIdx.x / grid.head_groups, heads = blockIdx.x - page * grid.head_groups;
      append_page_codes<T>(p, grid, b, static_cast<int>(heads * (kAppendThreads >> grid.head_threads_log2)), static_cast<int>(page));
      return;
    }
  }
  const unsigned i = (blockIdx.x - grid.page_blocks) * 2 + threadIdx.x / kTokenThreads;
  if (i < static_cast<unsigned>(p.rows)) append_token(p, grid, b, static_cast<int>(i), threadIdx.x % kTokenThreads);
}

template <class T>
cudaError_t append_t(const PagedAppendParams& p, cudaStream_t stream) {
  // pages that one entry can finish
  const int64_t pages = std::is_same<T, __half>::value ? 0 : (p.rows + (int64_t{1} << p.c.page_shift) - 1) >> p.c.page_shift;
  const int pieces = p.c.head_dim / 16;
  AppendGrid grid{};
  // threads to a head: kSealKept pieces each where that fills warps
  grid.head_threads_log2 = 5;
  while (1 << grid.head_threads_log2 < kAppendThreads && kSealKept << grid.head_threads_log2 < pieces << p.c.page_shift)
    ++grid.head_threads_log2;
  const int64_t at_once = kAppendThreads >> grid.head_threads_log2;
  grid.head_groups = static_cast<unsigned>((2 * p.c.heads_kv + at_once - 1) / at_once);
  grid.per_piece = (65536 + pieces - 1) / pieces;
  const int64_t page_blocks = pages * grid.head_groups;
  const int64_t blocks = page_blocks + (static_cast<int64_t>(p.rows) + 1) / 2;
  if (blocks > 0x7fffffff || p.c.batch > 65535) return cudaErrorInvalidValue;
  grid.page_blocks = static_cast<unsigned>(page_blocks);
  return launch_dependent(fal_paged_append_kernel<T>, dim3(static_cast<unsigned>(blocks), p.c.batch), dim3(kAppendThreads), 0,
                          stream, p, grid);
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendParams& p, cudaStream_t stream) {
  if (p.c.type == kPagedF16) return append_t<__half>(p, stream);
  return p.c.type == kPagedS8 ? append_t<S8>(p, stream) : append_t<E4M3>(p, stream);
}

}  // namespace fal
