// Attention over the pages of a key/value cache, in fp16 or in 8 bits with a scale for each page and head; and the pages' rows
// in order for the forward kernel, which takes the calls with many query tokens.
//
// The reference has no paged cache; its hook attends eagerly over dense ones (flash_attn_legacy/integrations.py:77-98).
#include <algorithm>
#include <type_traits>

#include "fal_combine.cuh"
#include "fal_paged.cuh"

namespace fal {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------------------
// Attention over the pages, few query rows per KV head
// ---------------------------------------------------------------------------
// Bound by HBM: every K and V row is read once for all query rows of its KV head.  The products are mma.sync m16n8k16 with
// 16 keys (scores) or 16 columns of V (output) as the M rows and 8 query rows as N: S^T = K Q^T, O^T = V^T P^T.  Query rows
// are (token, head of the group) pairs, 8 NT to a CTA.  A warp fetches 16-key slices of K and V by TMA (boxes of 16 rows of a
// page) into a ring of its own.  Fragments are read from shared memory as the lanes' own 16 bytes, without ldmatrix: a
// contraction may take its terms in any order, so lane t of four takes 16 bytes of a key row that are next to each other,
// and Q is laid out to match; lane g of eight takes 16 neighbouring bytes of a V row.
// 8-bit codes become fp16 in registers (exact).  The scales enter in 32 bits: K's multiplies the scores, V's is part of the
// weights, P = 2^(s + log2 v - m) with m near the largest such exponent, so that P keeps its bits however the scales differ; the
// softmax sum adds P / v, in 32 bits.  P is rounded to fp16 for the second product (2^-11 of each weight; P in two fp16 parts would
// be twice the products), which adds 1.9e-4 to the 2.1e-4 of rounding the output.  P^T of the scores' layout becomes the second product's operand by movmatrix.
//
// An (entry, KV head, chunk of 8 NT query rows) is a unit; its keys count in steps, one 16-key slice for each of four warps, or
// two.  Entries are cut into parts of one length that the GPU works out from all lengths, so that all units together
// make a few CTAs for every place on the GPU, whatever the lengths are; the units of one part are CTAs next to each other,
// because their rows are next to each other in memory where a page holds all heads of a position.  Parts of a cut entry go
// to the workspace and a second kernel merges them; a CTA that has all keys of its unit writes the result itself.
constexpr int kPagedWarps = 4;
constexpr int kPagedThreads = kPagedWarps * 32;
constexpr int kPagedSlice = 16;

// Slices that a warp takes at a time, of one page or of two.
template <int D, class T, int NT>
constexpr int kPagedSlices = Elem<T>::kScaled && NT == 1 && D <= 128 ? 2 : 1;
template <int D, class T, int NT>
constexpr int kPagedStep = kPagedWarps * kPagedSlice * kPagedSlices<D, T, NT>;  // keys of a step of a CTA

// Where the queries are: in registers, or in shared memory where registers hold many rows of the output.
template <int D, int NT>
constexpr bool kPagedQueriesShared = NT * D > 256;

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// D = A * B + C (fp16 16 x 16 and 16 x 8, fp32)
__device__ __forceinline__ void mma_16816_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                               const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma_16816_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_16816_from(d, a, b0, b1, d);
}
__device__ __forceinline__ void lds16(uint32_t addr, uint32_t* w) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
}
__device__ __forceinline__ void lds8(uint32_t addr, uint32_t* w) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
}

// A slice of 16 rows of a page in shared memory as TMA leaves it: blocks of 16 rows x 128 bytes (64-byte rows: one of 64),
// the 16-byte chunks of a row exclusive-or'ed with the row's number (64-byte rows: half of it).  The eight lanes that a
// 16-byte load serves at a time hit different banks if they are, for K, rows 4 apart, and for V, rows 0 ... 3 and chunks 4
// apart (64-byte rows: rows of both parities).  So row i of the first product's operand is key key_of(i), and lane g takes
// chunk chunk_of(g) of the V rows.
template <int D, class T>
struct PagedTile {
  static constexpr int kRowBytes = D * Elem<T>::kBytes;
  static constexpr int kBlockRow = kRowBytes < 128 ? kRowBytes : 128;
  static constexpr int kBlocks = kRowBytes / kBlockRow;
  static constexpr int kBlockBytes = kPagedSlice * kBlockRow;
  static constexpr int kSliceBytes = kPagedSlice * kRowBytes;  // K or V
  static constexpr int kLaneCols = kBlockRow / 8 / Elem<T>::kBytes;  // of a block's V row that a lane takes
  static constexpr bool kNarrow = kBlockRow == 64;
  static __device__ __forceinline__ int key_of(int i) {  // i: 0 ... 7; 8 ... 15 are 8 further
    return kNarrow ? i ^ ((i >> 1) & 1) : ((i & 1) << 2) | (i >> 1);
  }
  static __device__ __forceinline__ int chunk_of(int g) { return ((g & 1) << 2) | (g >> 1); }
  // Shared address in the K slice of row key_of(g), chunk t; in the V slice of row key_of(2 t), the lane's columns.
  static __device__ __forceinline__ uint32_t k_read(int g, int t) {
    const int row = key_of(g);
    return row * kBlockRow + (t ^ (kNarrow ? row >> 1 : row)) * 16;
  }
  static __device__ __forceinline__ uint32_t v_read(int g, int t) {
    const int row = key_of(2 * t);
    if (kNarrow) return row * kBlockRow + ((g >> 1) ^ (row >> 1)) * 16 + (g & 1) * 8;
    return row * kBlockRow + (chunk_of(g) ^ row) * 16;
  }
  // From there to row key_of(2 t + 1).
  static __device__ __forceinline__ uint32_t v_next(uint32_t at) { return kNarrow ? at ^ 64u : (at ^ 64u) + 4 * kBlockRow; }
  // First of the two columns that a lane has of output tile j.
  static __device__ __forceinline__ int column(int g, int j) {
    const int block = j / (kLaneCols / 2);
    return block * 8 * kLaneCols + (kNarrow ? g : chunk_of(g)) * kLaneCols + j % (kLaneCols / 2) * 2;
  }
};

// A slice of an 8-bit cache's tail: 16 fp16 rows, copied by the lanes (rows behind the end are zeros), chunks permuted for K
// as above with two chunks a lane.  Lanes take the columns that they take of the pages.
template <int D, class T>
struct PagedTailTile {
  static constexpr int kRowBytes = D * 2;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kLoads = kPagedSlice * kChunks / 32;
  static constexpr int kCopyRows = 32 / kChunks;
  static_assert(kCopyRows >= 1, "a row is at most 512 bytes");
  static __device__ __forceinline__ uint32_t place(int row, int ch) { return row * kRowBytes + (ch ^ (row & 7)) * 16; }
};

template <int D, class T, int NT>
struct PagedSmem {
  static constexpr int kStages = D == 64 && kPagedSlices<D, T, NT> == 1 ? 4 : kPagedSlices<D, T, NT> == 1 || D == 64 ? 3 : 2;
  static constexpr int kTensorBytes = kPagedSlices<D, T, NT> * PagedTile<D, T>::kSliceBytes;
  static constexpr int kStageBytes = 2 * kTensorBytes;      // K, then V; or K or V of a slice of the tail
  static constexpr int kRingBytes = kStages * kStageBytes;  // per warp
  static constexpr int kPipeBytes = kPagedWarps * kRingBytes;
  static constexpr int kPitch = D + 4;  // floats of a row of a warp's result
  static constexpr int kMergeBytes = kPagedWarps * 8 * NT * (kPitch + 2) * 4;
  static constexpr int kAlign = 1024;   // of TMA's permuted blocks
  static constexpr int kQueryOffset = kPipeBytes > kMergeBytes ? kPipeBytes : kMergeBytes;
  static constexpr int kBytes = kQueryOffset + (kPagedQueriesShared<D, NT> ? D / 16 * NT * 256 : 0) + kAlign;
};

// ---- the deal ----
// Steps of one unit of an entry with n positions: those of its pages, then those of its tail.
template <int STEP>
__device__ __forceinline__ int paged_steps(const PagedCache& c, int n) {
  const int in_pages = paged_len_in_pages(c, n);
  return (in_pages + STEP - 1) / STEP + (n - in_pages + STEP - 1) / STEP;
}

// Sums over the block's threads up to this one, and over all of them.
struct PagedSums {
  uint64_t warp_sum[kPagedWarps];
};
__device__ __forceinline__ uint64_t paged_block_sum(PagedSums& sums, uint64_t mine, uint64_t& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint64_t x = __shfl_up_sync(0xffffffffu, mine, off);
    if (lane >= off) mine += x;
  }
  __syncthreads();  // (the last sums have been read)
  if (lane == 31) sums.warp_sum[warp] = mine;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < kPagedWarps; ++w) {
    if (w < warp) mine += sums.warp_sum[w];
    all += sums.warp_sum[w];
  }
  return mine;
}

constexpr float kNoKey = -1e30f;  // further below any score than an exponential notices

// A part is as long as makes kPagedWaves CTAs of all units for every place on the GPU (SMs get unequal shares of the memory's
// bandwidth), but no shorter than kPagedGoodSteps, which a CTA's set-up is small beside, as long as there is a CTA for every
// place, nor than kPagedMinKeys.  (A length that makes the CTAs fill the places a whole number of times is no better.)
// us with 1 / 2 / 4 CTAs for every place: 64 entries of 16 000 int8 positions, 8 heads of 128, 421 / 366 / 339, fp16 623 / 604 /
// 605, 16 fp16 - / 167 / 159.  Parts of 8 / 16 / 32 steps: 16 entries of 32 000 int8, 4 heads of 64, 60 / 56 / 53, 16 of 6 000
// with 5 tokens, 8 heads of 64, 57 / 49 / 53; 16 of 16 000 int8, 8 heads of 128, 99 / 104 / -, 20 of 5 000 48 / 59 / - (128 keys
// to a step); with 16 heads to a KV head 57 / 52 / -, 12 of 2 000 fp16 with 5 tokens 39 / 31 / -, one of 30 000 int8
// 38 / 29 / -; 16 of 5 000 e4m3, 16 heads of 256, 119 / 119 / 110.
constexpr int kPagedMinKeys = 256;
constexpr int kPagedWaves = 4;
template <int D, int STEP>
constexpr int kPagedGoodSteps = D == 256 ? 32 : D == 128 && STEP > 64 ? 8 : 16;

// Where that length would give every place one CTA, a few more CTAs than places, from parts that are not of full length, would
// take the GPU twice: then the parts are a quarter to a half longer, if those fit.  us without / with that: 8 entries of 6 000
// int8, 5 tokens, 8 heads of 128, 48.4 / 37.4, of 2 000 28.7 / 23.7; 16 of 3 000, one token, 32.7 / 27.6; 6 of 100 ... 5 000
// e4m3, 16 heads of 256, 36.1 / 30.5; where it does not help, 8 of 500 ... 12 000 38.5 / 39.2, 4 of 8 000 19.9 / 20.6.
constexpr int kPagedChooseEntries = 4096;  // (their parts are counted in 16 bits)

// How an entry is cut.
struct PagedCut {
  int entry;
  int n;          // positions
  int steps;      // of a unit
  int parts;
  int64_t group;  // parts of the entries before it
  int64_t slot;   // the same, of those that are cut (their results go to the workspace)
};
// Finds the entry that has part `group` of all entries' parts.  False: there is none.  Called by all threads of a block, each
// of which looks at batch / kPagedThreads entries in a row.  STEP: keys of a step; heads: units of an entry.
template <int D, int STEP>
__device__ __forceinline__ bool paged_find(PagedSums& sums, PagedCut& found, const PagedAttnParams& p, unsigned heads,
                                           int64_t group) {
  const PagedCache& c = p.c;
  const int per = (c.batch + kPagedThreads - 1) / kPagedThreads;
  const int first = threadIdx.x * per, last = min(first + per, c.batch);
  if (threadIdx.x == 0) found.entry = -1;  // (seen by all behind the sums' barriers)
  const int n_first = first < last ? paged_len(c, first) : 0;
  auto len_of = [&](int e) { return e == first ? n_first : paged_len(c, e); };
  uint64_t total = 0, all;
  for (int e = first; e < last; ++e) total += paged_steps<STEP>(c, len_of(e));
  paged_block_sum(sums, total, all);
  const uint64_t once = (all * heads + p.resident - 1) / p.resident;
  constexpr uint64_t kGood = kPagedGoodSteps<D, STEP>, kLeast = kPagedMinKeys / STEP;
  const uint64_t wanted = max(max((once + kPagedWaves - 1) / kPagedWaves, min(once, kGood)), kLeast);
  uint32_t length = static_cast<uint32_t>(min(wanted, uint64_t{1} << 30));  // (no entry has more steps)
  // Parts, and parts of cut entries: in halves of 32 bits; with a second length to choose from, in quarters.
  const bool choose = once > kLeast && once <= kGood && c.batch <= kPagedChooseEntries;
  const uint32_t even = (static_cast<uint32_t>(all) + p.even_parts - 1) / p.even_parts;  // (to choose, `all` is small)
  const uint32_t longer = max(length + (length + 3) / 4, min(even, length + (length + 1) / 2));
  auto parts_of = [&](int steps, uint32_t len) -> uint64_t { return (static_cast<uint32_t>(steps) + len - 1) / len; };
  uint64_t mine = 0;
  for (int e = first; e < last; ++e) {
    const int steps = paged_steps<STEP>(c, len_of(e));
    const uint64_t parts = parts_of(steps, length);
    if (choose) {
      const uint64_t fewer = parts_of(steps, longer);
      mine += parts | (parts > 1 ? parts << 16 : 0) | fewer << 32 | (fewer > 1 ? fewer << 48 : 0);
    } else {
      mine += parts | (parts > 1 ? parts << 32 : 0);
    }
  }
  uint64_t from = paged_block_sum(sums, mine, all) - mine;
  if (choose) {
    if ((all & 0xffff) * heads > p.resident && (all >> 32 & 0xffff) * heads <= p.resident) {
      length = longer;
      from >>= 32;
      mine >>= 32;
    }
    from = (from & 0xffff) | (from & 0xffff0000u) << 16;
    mine = (mine & 0xffff) | (mine & 0xffff0000u) << 16;
  }
  const int64_t low = static_cast<int64_t>(from & 0xffffffffu), high = low + static_cast<int64_t>(mine & 0xffffffffu);
  if (group >= low && group < high) {
    for (int e = first; e < last; ++e) {
      const int n = len_of(e), steps = paged_steps<STEP>(c, n);
      const int64_t before = static_cast<int64_t>(from & 0xffffffffu), count = static_cast<int64_t>(parts_of(steps, length));
      if (group >= before && group < before + count)
        found = PagedCut{e, n, steps, static_cast<int>(count), before, static_cast<int64_t>(from >> 32)};
      from += count | (count > 1 ? count << 32 : 0);
    }
  }
  __syncthreads();
  return found.entry >= 0;
}

// ---- one piece of a unit ----
template <int D, int NT, int H>
struct PagedState {
  // the first product's second operand, or where it is: [step][n tile][lane], two words each
  uint32_t q[kPagedQueriesShared<D, NT> ? 1 : D / 16][2][kPagedQueriesShared<D, NT> ? 1 : NT];
  uint32_t q_shared;
  uint32_t p[H][NT][2];  // the weights of the slices in hand, as the second product's operand
  float o[NT][D / 16][4];
  float m[NT][2];     // reference of the exponents, log2 domain: at most 8 below the largest score so far; kNoKey before the first
  float l[NT][2];     // this lane's keys' share of the softmax sums
  float c2;
  int min_limit;     // first key that some query row does not see
};

// What follows the first product: scores s of this lane's keys key and key + 8 of H slices, from key0 on, for query rows 2 t and
// 2 t + 1 of every eight become weights.  end: of the keys that the slices are to have; first_limit: first key that the
// entry's first token does not see; a token whose own would be beyond the capacity has no place and sees none.
template <int H, int D, int NT, int HS>
__device__ __forceinline__ void paged_weights(PagedState<D, NT, HS>& st, float (&s)[H][NT][4], int key0, int key, int end,
                                              const float (&k_scale)[H], const float (&v_log)[H], int first_limit, int capacity,
                                              int row0, int group) {
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const float f = st.c2 * k_scale[h];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const uint64_t y = ffma2(pack_f32x2(s[h][nt][e], s[h][nt][e + 1]), pack_f32x2(f, f), pack_f32x2(v_log[h], v_log[h]));
        unpack_f32x2(y, s[h][nt][e], s[h][nt][e + 1]);
      }
  }
  if (key0 + H * kPagedSlice > min(st.min_limit, end)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int sees = first_limit + (row0 + nt * 8 + 2 * static_cast<int>(threadIdx.x & 3) + x) / group;
        const int limit = sees > capacity ? 0 : min(end, sees);
#pragma unroll
        for (int h = 0; h < H; ++h) {
          if (key + h * kPagedSlice >= limit) s[h][nt][x] = -INFINITY;
          if (key + h * kPagedSlice + 8 >= limit) s[h][nt][2 + x] = -INFINITY;
        }
      }
  }
  float most[NT][2];
  bool grows = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      most[nt][e] = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
      if (H == 2) most[nt][e] = fmaxf(most[nt][e], fmaxf(s[H - 1][nt][e], s[H - 1][nt][2 + e]));
      grows = grows || most[nt][e] - st.m[nt][e] > 8.f;
    }
  // The reference follows the largest score only when a weight would exceed 2^8: the output is rescaled a few times per
  // part, and the largest is looked for across the lanes only then.
  if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float alpha[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = most[nt][e];
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        const float m_new = fmaxf(st.m[nt][e], x);
        alpha[e] = fast_exp2(st.m[nt][e] - m_new);
        st.m[nt][e] = m_new;
        st.l[nt][e] *= alpha[e];
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
  for (int h = 0; h < H; ++h) {
    const float inv = fast_exp2(fmaxf(-v_log[h], -126.f));  // 1 / v (of a NaN: any number)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint64_t m = pack_f32x2(-st.m[nt][0], -st.m[nt][1]);
      const uint64_t p0 = exp2_pair(fadd2(pack_f32x2(s[h][nt][0], s[h][nt][1]), m));
      const uint64_t p1 = exp2_pair(fadd2(pack_f32x2(s[h][nt][2], s[h][nt][3]), m));
      unpack_f32x2(p0, s[h][nt][0], s[h][nt][1]);
      unpack_f32x2(p1, s[h][nt][2], s[h][nt][3]);
      st.p[h][nt][0] = movmatrix(pack_half2(s[h][nt][0], s[h][nt][1]));
      st.p[h][nt][1] = movmatrix(pack_half2(s[h][nt][2], s[h][nt][3]));
      const uint64_t l = ffma2(fadd2(p0, p1), pack_f32x2(inv, inv), pack_f32x2(st.l[nt][0], st.l[nt][1]));
      unpack_f32x2(l, st.l[nt][0], st.l[nt][1]);
    }
  }
}

// s (+)= the product of 16 keys' columns of one step and Q's.
template <int D, int NT, int H>
__device__ __forceinline__ void paged_score_step(PagedState<D, NT, H>& st, float (&s)[NT][4], const uint32_t (&a)[4], int ks) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    uint32_t q[2];
    if constexpr (kPagedQueriesShared<D, NT>) {
      lds8(st.q_shared + (ks * NT + nt) * 256, q);
    } else {
      q[0] = st.q[ks][0][nt];
      q[1] = st.q[ks][1][nt];
    }
    if (ks == 0) {
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
      mma_16816_from(s[nt], a, q[0], q[1], zero);
    } else {
      mma_16816_add(s[nt], a, q[0], q[1]);
    }
  }
}

// Scores of a slice of a page; kb: its shared address + k_read.
template <class T, int D, int NT, int H>
__device__ __forceinline__ void paged_scores(PagedState<D, NT, H>& st, float (&s)[NT][4], uint32_t kb) {
  using Tile = PagedTile<D, T>;
  constexpr int kSteps = Elem<T>::kScaled ? 4 : 2;  // of 16 columns in four lanes' 16 bytes
#pragma unroll
  for (int seg = 0; seg < Tile::kRowBytes / 64; ++seg) {
    uint32_t r0[4], r1[4];
    const uint32_t at = (kb ^ (seg & 1) * 64) + (seg >> 1) * Tile::kBlockBytes;
    lds16(at, r0);
    lds16(at + 8 * Tile::kBlockRow, r1);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      uint32_t a[4];
      if constexpr (Elem<T>::kScaled) {
        widen(static_cast<const T*>(nullptr), r0[k], a[0], a[2]);
        widen(static_cast<const T*>(nullptr), r1[k], a[1], a[3]);
      } else {
        a[0] = r0[2 * k];
        a[1] = r1[2 * k];
        a[2] = r0[2 * k + 1];
        a[3] = r1[2 * k + 1];
      }
      paged_score_step(st, s, a, seg * kSteps + k);
    }
  }
}

// O^T += V^T P^T of the h-th slice, of a page; vb: its shared address + v_read.
template <class T, int D, int NT, int H>
__device__ __forceinline__ void paged_output(PagedState<D, NT, H>& st, int h, uint32_t vb) {
  using Tile = PagedTile<D, T>;
  auto product = [&](int j, const uint32_t (&a)[4]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mma_16816_add(st.o[nt][j], a, st.p[h][nt][0], st.p[h][nt][1]);
  };
#pragma unroll
  for (int block = 0; block < Tile::kBlocks; ++block) {
    uint32_t w[4][4];  // rows key_of(2 t), key_of(2 t + 1), and 8 further
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t at = ((r & 1) != 0 ? Tile::v_next(vb) : vb) + (r >> 1) * 8 * Tile::kBlockRow + block * Tile::kBlockBytes;
      if constexpr (Tile::kNarrow) lds8(at, w[r]);
      else lds16(at, w[r]);
    }
#pragma unroll
    for (int k = 0; k < Tile::kBlockRow / 32; ++k) {
      if constexpr (Elem<T>::kScaled) {
        const int j = block * 8 + 2 * k;  // two output tiles of two columns a lane
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
        product(block * 4 + k, a);
      }
    }
  }
}

// The same of a slice of the tail at shared address base; K and V are there one after the other.
template <class T, int D, int NT, int H>
__device__ __forceinline__ void paged_tail_scores(PagedState<D, NT, H>& st, uint32_t base, int key0, int end, int first_limit,
                                                  int capacity, int row0, int group) {
  using Tail = PagedTailTile<D, T>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float s[1][NT][4];
#pragma unroll
  for (int seg = 0; seg < D / 64; ++seg) {
    uint32_t r0[8], r1[8];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      lds16(base + Tail::place(g, (seg * 4 + t) * 2 + x), r0 + 4 * x);
      lds16(base + Tail::place(g + 8, (seg * 4 + t) * 2 + x), r1 + 4 * x);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t a[4] = {r0[2 * k], r1[2 * k], r0[2 * k + 1], r1[2 * k + 1]};
      paged_score_step(st, s[0], a, seg * 4 + k);
    }
  }
  const float k_scale[1] = {1.f}, v_log[1] = {0.f};
  paged_weights<1>(st, s, key0, key0 + g, end, k_scale, v_log, first_limit, capacity, row0, group);
}
template <class T, int D, int NT, int H>
__device__ __forceinline__ void paged_tail_output(PagedState<D, NT, H>& st, uint32_t base) {
  using Tile = PagedTile<D, T>;
  using Tail = PagedTailTile<D, T>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int j = 0; j < D / 16; j += 4) {  // eight columns
    uint32_t w[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r) lds16(base + Tail::place(2 * t + (r & 1) + (r >> 1) * 8, Tile::column(g, j) / 8), w[r]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t a[4] = {__byte_perm(w[0][k], w[1][k], 0x5410), __byte_perm(w[0][k], w[1][k], 0x7632),
                             __byte_perm(w[2][k], w[3][k], 0x5410), __byte_perm(w[2][k], w[3][k], 0x7632)};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_16816_add(st.o[nt][j + k], a, st.p[0][nt][0], st.p[0][nt][1]);
    }
  }
}

// A warp's ring: its shared address, a barrier per stage, and their phases (a bit each).
struct PagedRing {
  uint32_t base;
  uint32_t barriers;
  uint32_t phases;
  WaitCtx wait;
};
constexpr int kPagedBarrierId = 60;
constexpr int kNoSlice = -1;  // in place of a page: beyond the part

// Steps step0 ... step1 - 1 of the unit (entry b of n positions, KV head, query rows row0 ...), this warp's slices of them.
template <int D, class T, int NT>
__device__ __forceinline__ void paged_piece(const PagedAttnParams& p, const CUtensorMap* k_map, const CUtensorMap* v_map,
                                            PagedRing& ring, uint32_t queries, int b, int n, int kv_head, int row0, int rows_valid,
                                            int first_limit, int step0, int step1,
                                            PagedState<D, NT, kPagedSlices<D, T, NT>>& st) {
  using L = PagedSmem<D, T, NT>;
  using Tile = PagedTile<D, T>;
  constexpr bool kScaled = Elem<T>::kScaled;
  constexpr int kH = kPagedSlices<D, T, NT>;
  constexpr int kKeys = kH * kPagedSlice;  // of a warp's turn
  constexpr int kStep = kPagedStep<D, T, NT>;
  constexpr int kQ = 16 / Elem<T>::kBytes;  // neighbouring columns of a lane in Q's layout
  constexpr int kAhead = L::kStages - 1;
  const PagedCache& c = p.c;
  const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = p.heads_q / c.heads_kv;
  const int in_pages = paged_len_in_pages(c, n);
  const int page_steps = (in_pages + kStep - 1) / kStep;

  // this warp's turns: keys first + i * kStep ... + kKeys - 1
  const int first = step0 * kStep + warp * kKeys;
  const int page_end = min(step1 * kStep, in_pages);
  const int turns = page_end > first ? (page_end - first + kStep - 1) / kStep : 0;
  // and its slices of the tail: rows tail_first + i * 64 ... + 15
  const int tail_first = (max(step0, page_steps) - page_steps) * kStep + warp * kPagedSlice;
  const int tail_end = kScaled ? min((step1 - page_steps) * kStep, n - in_pages) : 0;
  constexpr int kTailStep = kPagedWarps * kPagedSlice;
  const int tail_slices = tail_end > tail_first ? (tail_end - tail_first + kTailStep - 1) / kTailStep : 0;

  // Pages and scales of 32 slices at a time, one to a lane: of the slices whose loads are being issued, of the 32 before them
  // (some of which are still to be worked on), and of the 32 behind them.
  constexpr int kBatch = 32 / kH;  // turns
  const int32_t* table = c.table + b * c.table_stride;
  auto pages_of = [&](int i) {
    const int key = first + (i + lane / kH) * kStep + lane % kH * kPagedSlice;
    return key < page_end ? __ldg(table + (key >> c.page_shift)) : kNoSlice;
  };
  auto there = [&](int page) { return static_cast<uint32_t>(page) < static_cast<uint32_t>(c.num_pages); };
  auto scale_of = [&](const float* scales, int page) {
    // (an ordinary load: the append before may still be writing scales while this grid's blocks take their places)
    return kScaled && there(page) ? scales[static_cast<int64_t>(page) * c.heads_kv + kv_head] : 1.f;
  };
  // log2 of V's scale; of 0, which a page of zeros has, of a number small enough for its values to be no more than 0 in fp16, but no
  // smaller: its keys' weights in the softmax sum are those of the exponents v log down from the others', which 2^-126 ends.
  // (At 2^-100 keys with 2^-20 of the weight of one whose V values are the largest of fp16 were lost.)
  auto v_log_of = [&](int page) {
    const float scale = scale_of(c.v_scales, page);
    return kScaled ? __log2f(scale < 0x1p-60f ? 0x1p-60f : scale) : 0.f;  // (a NaN stays one)
  };
  int pages = pages_of(0), next_pages = 0;
  float k_scales = 0.f, v_logs = 0.f, next_k = 0.f, next_v = 0.f, last_k = 0.f, last_v = 0.f;
  uint32_t fill = 0;  // stage that the next loads go to
  auto issue = [&](int i) {
    if (i < turns) {
      const int in_batch = i & (kBatch - 1);
      if (in_batch == 0 && i > 0) {
        pages = next_pages;
        last_k = k_scales;
        last_v = v_logs;
        k_scales = next_k;
        v_logs = next_v;
      }
      if (in_batch == kBatch / 8) next_pages = pages_of((i & ~(kBatch - 1)) + kBatch);
      if (kScaled && in_batch == kBatch * 5 / 8) {
        next_k = scale_of(c.k_scales, next_pages);
        next_v = v_log_of(next_pages);
      }
      int page[kH];
#pragma unroll
      for (int h = 0; h < kH; ++h) page[h] = __shfl_sync(0xffffffffu, pages, in_batch * kH + h);
      const int key0 = first + i * kStep;
      if (elect_one()) {
        const uint32_t bar = ring.barriers + fill * 8;
        const uint32_t stage = ring.base + fill * L::kStageBytes;
        mbar_arrive_expect_tx(bar, L::kStageBytes);
#pragma unroll
        for (int h = 0; h < kH; ++h) {
          const int row = (key0 + h * kPagedSlice) & ((1 << c.page_shift) - 1);
          if (!there(page[h])) {  // (TMA fills a box outside of the tensor with zeros)
            if (key0 + h * kPagedSlice < page_end && p.status) atomicCAS(p.status, 0, kDevNoPage);
            page[h] = c.num_pages;
          }
#pragma unroll
          for (int x = 0; x < Tile::kBlocks; ++x) {
            const int column = x * Tile::kBlockRow / Elem<T>::kBytes;
            const uint32_t at = stage + h * Tile::kSliceBytes + x * Tile::kBlockBytes;
            tma_load_4d(at, k_map, bar, column, row, kv_head, page[h]);
            tma_load_4d(at + L::kTensorBytes, v_map, bar, column, row, kv_head, page[h]);
          }
        }
      }
    } else if (kScaled && i < turns + 2 * tail_slices) {  // K, then V of a slice of the tail
      using Tail = PagedTailTile<D, T>;
      const int j = i - turns;
      const bool is_v = (j & 1) != 0;
      const RowStrides& s = is_v ? c.v_tail_strides : c.k_tail_strides;
      const int row = tail_first + (j >> 1) * kTailStep;
      const __half* src = static_cast<const __half*>(is_v ? c.v_tail : c.k_tail) + b * s.batch + kv_head * s.head + row * s.row;
      const int ch = lane % Tail::kChunks;
#pragma unroll
      for (int it = 0; it < Tail::kLoads; ++it) {
        const int r = it * Tail::kCopyRows + lane / Tail::kChunks;
        const bool ok = row + r < tail_end && ch * 8 < c.head_dim;
        cp_async_16_zfill(ring.base + fill * L::kStageBytes + Tail::place(r, ch), ok ? src + r * s.row + ch * 8 : src, ok);
      }
      cp_async_commit();
    }
    fill = fill + 1 < L::kStages ? fill + 1 : 0;
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) issue(i);
  k_scales = scale_of(c.k_scales, pages);
  v_logs = v_log_of(pages);

  // ---- queries and their limits, under the first loads ----
  auto query = [&](int nt, int ks) {
    const int row = nt * 8 + g;
    const int r = row0 + row;
    const int col = (ks / (kQ / 4)) * 4 * kQ + t * kQ + (ks % (kQ / 4)) * 4;
    if (row >= rows_valid || col >= c.head_dim) return make_uint2(0u, 0u);
    return *reinterpret_cast<const uint2*>(static_cast<const __half*>(p.q) + b * p.q_strides.batch + r / group * p.q_strides.row +
                                           (kv_head * group + r % group) * p.q_strides.head + col);
  };
  if constexpr (kPagedQueriesShared<D, NT>) {
    st.q_shared = queries + lane * 8;
    for (int x = warp; x < D / 16 * NT; x += kPagedWarps) {
      const uint2 q = query(x % NT, x / NT);
      asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(st.q_shared + x * 256), "r"(q.x), "r"(q.y) : "memory");
    }
    __syncthreads();
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if constexpr (!kPagedQueriesShared<D, NT>) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const uint2 q = query(nt, ks);
        st.q[ks][0][nt] = q.x;
        st.q[ks][1][nt] = q.y;
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      st.m[nt][e] = kNoKey;
      st.l[nt][e] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[nt][j][e] = 0.f;
  }
  const int capacity = paged_capacity(c);
  st.min_limit = first_limit + (row0 + rows_valid - 1) / group > capacity ? 0 : first_limit + row0 / group;
  st.c2 = p.scale * kLog2e;

  const uint32_t k_read = Tile::k_read(g, t), v_read = L::kTensorBytes + Tile::v_read(g, t);
  uint32_t drain = 0;
  for (int i = 0; i < turns; ++i) {
    issue(i + kAhead);
    const uint32_t stage = ring.base + drain * L::kStageBytes;
    const int key0 = first + i * kStep;
    float k_scale[kH], v_log[kH];
    const bool before = (min(i + kAhead, turns - 1) ^ i) >= kBatch;
#pragma unroll
    for (int h = 0; h < kH; ++h) {
      k_scale[h] = 1.f;
      v_log[h] = 0.f;
      if constexpr (kScaled) {
        k_scale[h] = __shfl_sync(0xffffffffu, before ? last_k : k_scales, i * kH + h);
        v_log[h] = __shfl_sync(0xffffffffu, before ? last_v : v_logs, i * kH + h);
      }
    }
    mbar_wait(ring.barriers + drain * 8, (ring.phases >> drain) & 1u, ring.wait, kPagedBarrierId);
    ring.phases ^= 1u << drain;
    if (!kScaled && key0 + kPagedSlice > page_end) {
      // whatever the page holds behind the entry's length: as V rows with weights of 0 its NaN would still reach the output
      const int rows = page_end - key0;
      for (int x = rows * (Tile::kBlockRow / 16) + lane; x < kPagedSlice * (Tile::kBlockRow / 16); x += 32)
#pragma unroll
        for (int block = 0; block < Tile::kBlocks; ++block)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};"
                       ::"r"(stage + L::kTensorBytes + block * Tile::kBlockBytes + x * 16),
                       "r"(0)
                       : "memory");
      __syncwarp();
    }
    float s[kH][NT][4];
#pragma unroll
    for (int h = 0; h < kH; ++h) paged_scores<T>(st, s[h], stage + k_read + h * Tile::kSliceBytes);
    paged_weights<kH>(st, s, key0, key0 + Tile::key_of(g), page_end, k_scale, v_log, first_limit, capacity, row0, group);
#pragma unroll
    for (int h = 0; h < kH; ++h) paged_output<T>(st, h, stage + v_read + h * Tile::kSliceBytes);
    drain = drain + 1 < L::kStages ? drain + 1 : 0;
    __syncwarp();  // all lanes are done with this stage before it is refilled
  }
  if constexpr (kScaled) {
    for (int j = 0; j < 2 * tail_slices; ++j) {
      issue(turns + j + kAhead);
      cp_async_wait<0>();
      __syncwarp();
      const uint32_t stage = ring.base + drain * L::kStageBytes;
      if ((j & 1) == 0)
        paged_tail_scores<T>(st, stage, in_pages + tail_first + (j >> 1) * kTailStep, n, first_limit, capacity, row0, group);
      else
        paged_tail_output<T>(st, stage);
      drain = drain + 1 < L::kStages ? drain + 1 : 0;
      __syncwarp();
    }
  }
  // the lanes' shares of the sums
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) st.l[nt][e] += __shfl_xor_sync(0xffffffffu, st.l[nt][e], off);
}

// What a pair of columns is exclusive-or'ed with where the warps' results lie: a number of its lane, below the pairs of a lane.
template <int D, class T>
__device__ __forceinline__ int paged_merge_mix(int pair) {
  constexpr int kPairs = PagedTile<D, T>::kLaneCols / 2;
  return (pair / kPairs >> 1) & (kPairs - 1) & 3;
}

// CTAs per SM: what shared memory holds, as far as the registers of a result of 8 NT rows allow.
template <int D, class T, int NT>
constexpr int paged_ctas_per_sm() {
  const int by_memory = (227 << 10) / (PagedSmem<D, T, NT>::kBytes + (2 << 10));
  constexpr int kOutput = NT * D;  // floats of a lane's share of the output, times four
  const int by_registers = kOutput <= 64                                        ? 5
                           : kOutput <= 128 && kPagedSlices<D, T, NT> == 1      ? 4
                           : kOutput == 384 || (kOutput <= 256 && NT < 4)       ? 3
                                                                                : 2;
  return by_memory < by_registers ? by_memory : by_registers;
}

template <int D, class T, int NT>
__global__ void __launch_bounds__(kPagedThreads, paged_ctas_per_sm<D, T, NT>())
fal_paged_splitk_kernel(const PagedAttnParams p, const __grid_constant__ CUtensorMap k_map,
                        const __grid_constant__ CUtensorMap v_map) {
  using L = PagedSmem<D, T, NT>;
  using Tile = PagedTile<D, T>;
  constexpr int kRows = 8 * NT;
  extern __shared__ __align__(128) uint8_t paged_smem_raw[];
  __shared__ PagedSums sums;
  __shared__ PagedCut cut;
  __shared__ __align__(8) uint64_t barriers[kPagedWarps][L::kStages];
  __shared__ int abort_flag;
  uint8_t* paged_smem = paged_smem_raw + (L::kAlign - smem_u32(paged_smem_raw) % L::kAlign) % L::kAlign;
  if (threadIdx.x < kPagedWarps * L::kStages) mbar_init(smem_u32(&barriers[0][0] + threadIdx.x), 1);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
  }
  fence_mbar_init();
  grid_dependency_wait();    // the append of this step's rows may still run up to here
  grid_dependency_launch();
  const PagedCache& c = p.c;
  const int group = p.heads_q / c.heads_kv;
  const int chunks = (p.rows * group + kRows - 1) / kRows;
  const unsigned heads = c.heads_kv * chunks;  // units of an entry
  const int unit = blockIdx.x % heads;
  if (!paged_find<D, kPagedStep<D, T, NT>>(sums, cut, p, heads, blockIdx.x / heads)) return;
  const int b = cut.entry;
  const unsigned part = blockIdx.x / heads - static_cast<unsigned>(cut.group);
  if (unit == 0 && part == 0 && threadIdx.x == 0) {  // for the merge
    p.cuts[2 * b] = cut.parts;
    p.cuts[2 * b + 1] = cut.slot;
  }
  const unsigned parts = cut.parts, steps = cut.steps, longer = steps % parts;  // the first ones have a step more
  const int step0 = part * (steps / parts) + min(static_cast<unsigned>(part), longer);
  const int step1 = step0 + steps / parts + (part < longer ? 1 : 0);
  const int kv_head = unit / chunks;
  const int row0 = unit % chunks * kRows;  // of the KV head's rows * group query rows
  const int rows_valid = min(kRows, p.rows * group - row0);
  const int first_limit = paged_first_limit(c, b, cut.n, p.rows);
  const int warp = warp_index(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  PagedRing ring{smem_u32(paged_smem) + warp * L::kRingBytes, smem_u32(&barriers[warp][0]), 0u, WaitCtx{&abort_flag, p.status}};
  PagedState<D, NT, kPagedSlices<D, T, NT>> st;
  paged_piece<D, T, NT>(p, &k_map, &v_map, ring, smem_u32(paged_smem) + L::kQueryOffset, b, cut.n, kv_head, row0, rows_valid,
                        first_limit, step0, step1, st);
  __syncthreads();  // the ring becomes the place of the warps' results

  // (column pair c of a row is at c ^ (its lane / 2): eight lanes and four rows of a store hit different banks)
  float* mo = reinterpret_cast<float*>(paged_smem);          // [warp][row][kPitch]
  float* mml = mo + kPagedWarps * kRows * L::kPitch;         // [warp][row][2]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = warp * kRows + nt * 8 + 2 * t + x;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const int pair = Tile::column(g, j) / 2;
        *reinterpret_cast<float2*>(mo + row * L::kPitch + (pair ^ paged_merge_mix<D, T>(pair)) * 2) =
            make_float2(st.o[nt][j][x], st.o[nt][j][2 + x]);
      }
      if (g == 0)
        *reinterpret_cast<float2*>(mml + row * 2) = make_float2(st.m[nt][x], st.l[nt][x]);
    }
  }
  __syncthreads();
  // rows of this chunk whose tokens have a place
  const int placed = min(max(min(paged_capacity(c) + 1 - first_limit, p.rows) * group - row0, 0), rows_valid);
  const int64_t slot = ((cut.slot + part) * heads + unit) * kRows;
  for (int idx = threadIdx.x; idx < rows_valid * (D / 2); idx += kPagedThreads) {
    const int r = idx / (D / 2), pair = idx % (D / 2);
    float most = kNoKey;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) most = fmaxf(most, mml[(w * kRows + r) * 2]);
    float o0 = 0.f, o1 = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) {
      const float x = fast_exp2(mml[(w * kRows + r) * 2] - most);
      const float2 y =
          *reinterpret_cast<const float2*>(mo + (w * kRows + r) * L::kPitch + (pair ^ paged_merge_mix<D, T>(pair)) * 2);
      o0 += x * y.x;
      o1 += x * y.y;
      l += x * mml[(w * kRows + r) * 2 + 1];
    }
    if (r >= placed) o0 = o1 = 0.f;  // (weights of 0 throughout, which an infinity among the values would show through)
    if (cut.parts == 1) {
      const float inv = l != 0.f ? 1.f / l : 0.f;  // (0: the row sees no key)
      const int head = kv_head * group + (row0 + r) % group;
      __half* out =
          static_cast<__half*>(p.o) + ((static_cast<int64_t>(b) * p.rows + (row0 + r) / group) * p.heads_q + head) * c.head_dim;
      if (2 * pair < c.head_dim) *reinterpret_cast<uint32_t*>(out + 2 * pair) = pack_half2(o0 * inv, o1 * inv);
    } else {
      *reinterpret_cast<float2*>(p.part_o + (slot + r) * D + 2 * pair) = make_float2(o0, o1);
      if (pair == 0) *reinterpret_cast<float2*>(p.part_ml + (slot + r) * 2) = make_float2(most, l);
    }
  }
}

// Merges the parts of the entries that were cut, and writes the zeros of entries without positions.
template <int D, int NT>
__global__ void __launch_bounds__(kCombineThreads) fal_paged_combine_kernel(const PagedAttnParams p) {
  constexpr int kRows = 8 * NT;
  const PagedCache& c = p.c;
  const int group = p.heads_q / c.heads_kv;
  const int chunks = (p.rows * group + kRows - 1) / kRows;
  const int heads = c.heads_kv * chunks;
  const int row = blockIdx.x;
  const int head = row % p.heads_q, token = row / p.heads_q % p.rows, b = row / p.heads_q / p.rows;
  grid_dependency_wait();
  const longlong2 cut = *reinterpret_cast<const longlong2*>(p.cuts + 2 * b);
  const int parts = paged_len(c, b) > 0 ? static_cast<int>(cut.x) : 0;
  if (parts == 1) return;
  const int in_head = token * group + head % group;  // query row of the KV head
  const int64_t first = (cut.y * heads + head / group * chunks + in_head / kRows) * kRows + in_head % kRows;
  auto at = [&](int i) { return first + static_cast<int64_t>(i) * heads * kRows; };
  combine_row<D, kCombineThreads / 32>(threadIdx.x, true, parts, reinterpret_cast<const float2*>(p.part_ml),
                                       reinterpret_cast<const float4*>(p.part_o), at,
                                       static_cast<__half*>(p.o) + static_cast<int64_t>(row) * c.head_dim, c.head_dim, nullptr);
}

// CTAs of the split-K kernel that the GPU holds at once.
template <int D, class T, int NT>
cudaError_t resident_ctas(int* ctas) {
  auto kern = fal_paged_splitk_kernel<D, T, NT>;
  constexpr int kBytes = PagedSmem<D, T, NT>::kBytes;
  static DeviceOnce configured;
  static int per_device[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  e = configured.run([&] {
    cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    int per_sm = 0, sms = 0;
    if (err == cudaSuccess) err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, kPagedThreads, kBytes);
    if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    per_device[dev] = per_sm * sms;
    return err == cudaSuccess && per_device[dev] <= 0 ? cudaErrorLaunchOutOfResources : err;
  });
  if (e == cudaSuccess) *ctas = per_device[dev];
  return e;
}

template <int D, class T, int NT>
cudaError_t splitk_t(PagedAttnParams& p, const CUtensorMap* maps, cudaStream_t stream) {
  cudaError_t e = resident_ctas<D, T, NT>(&p.resident);
  if (e != cudaSuccess) return e;
  const int64_t chunks = (static_cast<int64_t>(p.rows) * (p.heads_q / p.c.heads_kv) + 8 * NT - 1) / (8 * NT);
  const int64_t heads = p.c.heads_kv * chunks;
  p.even_parts = static_cast<int>(p.c.batch * std::max<int64_t>(1, p.resident / (p.c.batch * heads)));
  // Parts of all entries: one each, and as many more as there are CTAs to make; and no more than kPagedMinKeys make of full
  // entries.
  constexpr int kStep = kPagedStep<D, T, NT>, kMinSteps = kPagedMinKeys / kStep;
  const int64_t steps = ((static_cast<int64_t>(p.c.pages_per_entry) << p.c.page_shift) + kStep - 1) / kStep + 1;
  const int64_t parts = static_cast<int64_t>(kPagedWaves) * p.resident;
  const int64_t groups = std::min<int64_t>(p.c.batch + parts / heads, p.c.batch * ((steps + kMinSteps - 1) / kMinSteps));
  // (a cut entry is longer than one part: its parts are at most twice its steps in parts)
  p.slots = std::min<int64_t>(groups, 2 * (parts / heads) + 2) * heads;
  if (groups * heads > 0x7fffffff) return cudaErrorInvalidValue;
  if (maps == nullptr) return e;
  p.part_ml = p.part_o + p.slots * 8 * NT * D;
  e = launch_dependent(fal_paged_splitk_kernel<D, T, NT>, dim3(static_cast<unsigned>(groups * heads)), dim3(kPagedThreads),
                       PagedSmem<D, T, NT>::kBytes, stream, p, maps[0], maps[1]);
  if (e != cudaSuccess) return e;
  const unsigned rows = static_cast<unsigned>(p.c.batch) * p.rows * p.heads_q;
  return launch_dependent(fal_paged_combine_kernel<D, NT>, dim3(rows), dim3(kCombineThreads), 0, stream, p);
}

template <int D, class T>
cudaError_t splitk_d(PagedAttnParams& p, const CUtensorMap* maps, cudaStream_t stream) {
  const int tiles = paged_rows_per_cta(p.rows * (p.heads_q / p.c.heads_kv), D) / 8;
  if constexpr (D < 256) {
    if (tiles == 4) return splitk_t<D, T, 4>(p, maps, stream);
    if (tiles == 3) return splitk_t<D, T, 3>(p, maps, stream);
  }
  if (tiles == 2) return splitk_t<D, T, 2>(p, maps, stream);
  return splitk_t<D, T, 1>(p, maps, stream);
}

template <class T>
cudaError_t splitk(PagedAttnParams& p, const CUtensorMap* maps, cudaStream_t stream) {
  if (p.kernel_dim == 64) return splitk_d<64, T>(p, maps, stream);
  if (p.kernel_dim == 128) return splitk_d<128, T>(p, maps, stream);
  return splitk_d<256, T>(p, maps, stream);
}

cudaError_t splitk(PagedAttnParams& p, const CUtensorMap* maps, cudaStream_t stream) {
  if (p.c.type == kPagedF16) return splitk<__half>(p, maps, stream);
  if (p.c.type == kPagedS8) return splitk<S8>(p, maps, stream);
  return splitk<E4M3>(p, maps, stream);
}

// ---------------------------------------------------------------------------
// Rows in order, for the forward kernel
// ---------------------------------------------------------------------------
// Bound by HBM.  A thread takes 16 columns of a row.  Codes stay codes (exact in fp16), a thread for every 16 keys hands their
// scales to the forward kernel.  (With the values rounded to fp16 the output was 1.5 times as far from 64 bits as the split-K
// pass's.)  Where a scale is 0, NaN or beyond what fp16 rows give, the values are written, and their scale is 1.
__device__ __forceinline__ bool paged_scale_apart(float scale) { return scale >= 0x1p-40f && scale <= 0x1p40f; }
// What the first block of an (entry, head) adds where rows were appended: the forward kernel gets a length that tells the positions of
// those that did not run over the table, and zeros behind it that only the rows without a place see.
// (In all blocks, each with its share, the pass took 42 us where this takes 38: 4 x 512 tokens behind 7 000 int8 positions; asked of
// calls that append nothing too, 64 tokens on 32 x 32 768 of 2 heads took 725 us where they take 722.)
template <class T>
__device__ __forceinline__ void paged_gather_over(const PagedGatherParams& p, int e, int hh, bool is_v, int n) {
  const PagedCache& c = p.c;
  const int end = n > 0 ? paged_first_limit(c, p.b0 + e, n, c.appended) - 1 + c.appended : 0;
  if (blockIdx.y == 0 && threadIdx.x == 0) p.lens_out[e] = end;
  const int64_t head = static_cast<int64_t>(e) * p.heads + hh;
  uint4* rows = reinterpret_cast<uint4*>(static_cast<__half*>(is_v ? p.v_out : p.k_out) + (head * p.capacity + n) * c.head_dim);
  for (int64_t i = threadIdx.x; i < static_cast<int64_t>(end - n) * (c.head_dim / 8); i += 256) rows[i] = make_uint4(0, 0, 0, 0);
  if (Elem<T>::kScaled && !is_v && end > n) {
    const int blocks = (end + 127) / 128 * (128 / kPagedBoxRows);  // (n is a whole number of pages)
    for (int i = n / kPagedBoxRows + threadIdx.x; i < blocks; i += 256)
      p.scales_out[head * p.key_blocks + i] = make_float4(p.scale_log2, 0.f, 1.f, 0.f);
  }
}
template <class T, bool APPENDED>
__global__ void __launch_bounds__(256) fal_paged_gather_kernel(const PagedGatherParams p) {
  const PagedCache& c = p.c;
  const int pieces = c.head_dim / 16;
  const int e = blockIdx.z;
  const int b = p.b0 + e;
  const bool is_v = blockIdx.y >= static_cast<unsigned>(p.heads);
  const int hh = is_v ? blockIdx.y - p.heads : blockIdx.y;
  const int h = p.h0 + hh;
  const int n = paged_len(c, b), in_pages = paged_len_in_pages(c, n);
  if constexpr (APPENDED) {
    if (blockIdx.x == 0) paged_gather_over<T>(p, e, hh, is_v, n);
  }
  const int64_t task = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t pos = task / pieces;
  const int col = static_cast<int>(task % pieces) * 16;
  if (pos >= n) return;
  uint4 out[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  float k_scale = 1.f, v_scale = 1.f;  // that the forward kernel applies
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
        const float scales[2] = {__ldg(c.k_scales + static_cast<int64_t>(page) * c.heads_kv + h),
                                 __ldg(c.v_scales + static_cast<int64_t>(page) * c.heads_kv + h)};
        if (paged_scale_apart(scales[0])) k_scale = scales[0];
        if (paged_scale_apart(scales[1])) v_scale = scales[1];
        const float scale = paged_scale_apart(scales[is_v]) ? 1.f : scales[is_v];
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
  if (Elem<T>::kScaled && !is_v && col == 0 && (pos & (kPagedBoxRows - 1)) == 0) {
    float4* to = p.scales_out + (static_cast<int64_t>(e) * p.heads + hh) * p.key_blocks + pos / kPagedBoxRows;
    // (a product of extremes stays a number that neither infinities nor zeros turn into a NaN)
    to[0] = make_float4(fminf(fmaxf(k_scale * p.scale_log2, 0x1p-126f), 0x1p100f), log2f(v_scale), 1.f / v_scale, 0.f);
    if (pos + kPagedBoxRows >= n)  // the rest of the last tile's 128 keys
      for (int64_t i = 1; ((pos / kPagedBoxRows + i) & 7) != 0; ++i) to[i] = make_float4(p.scale_log2, 0.f, 1.f, 0.f);
  }
  __half* dst =
      static_cast<__half*>(is_v ? p.v_out : p.k_out) + ((static_cast<int64_t>(e) * p.heads + hh) * p.capacity + pos) * c.head_dim + col;
  reinterpret_cast<uint4*>(dst)[0] = out[0];
  reinterpret_cast<uint4*>(dst)[1] = out[1];
}

template <class T>
cudaError_t gather_t(const cudaLaunchConfig_t& cfg, const PagedGatherParams& p) {
  return p.c.appended != 0 ? cudaLaunchKernelEx(&cfg, fal_paged_gather_kernel<T, true>, p)
                           : cudaLaunchKernelEx(&cfg, fal_paged_gather_kernel<T, false>, p);
}

// Zeros for the tokens of entry blockIdx.x that have no place.  (Rows that the forward kernel left out itself
// took 1 to 4 % of its other calls: 2 x 200 queries, 16 heads of 256, 44.1 us / 45.2 to 45.7.)
__global__ void __launch_bounds__(256) fal_paged_zero_kernel(const PagedAttnParams p) {
  grid_dependency_wait();
  const int b = blockIdx.x, length = p.c.lens[b], capacity = paged_capacity(p.c);
  if (length < 0 || length <= capacity - p.rows) return;  // (unused: zeros already)
  const int64_t token = static_cast<int64_t>(p.heads_q) * p.c.head_dim / 8;  // pieces of 16 bytes
  uint4* o = static_cast<uint4*>(p.o) + b * p.rows * token;
  for (int64_t i = (capacity - min(length, capacity)) * token + threadIdx.x; i < p.rows * token; i += 256)
    o[i] = make_uint4(0, 0, 0, 0);
}

}  // namespace

int paged_rows_per_cta(int rows, int kernel_dim) {
  const int tiles = (rows + 7) / 8, most = kernel_dim < 256 ? 4 : 2;
  const int passes = (tiles + most - 1) / most;
  return 8 * ((tiles + passes - 1) / passes);
}

cudaError_t paged_attn_plan(PagedAttnParams& p) { return splitk(p, nullptr, nullptr); }

cudaError_t launch_paged_attn(PagedAttnParams& p, const CUtensorMap* maps, cudaStream_t stream) { return splitk(p, maps, stream); }

cudaError_t launch_paged_gather(const PagedGatherParams& p, cudaStream_t stream) {
  const int64_t tasks = (static_cast<int64_t>(p.c.pages_per_entry) << p.c.page_shift) * (p.c.head_dim / 16);
  const int64_t blocks = (tasks + 255) / 256;
  if (blocks > 0x7fffffff || 2 * p.heads > 65535 || p.entries > 65535) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};  // (a launch that returns its own error, and none of another's)
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 2 * p.heads, p.entries);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  if (p.c.type == kPagedF16) return gather_t<__half>(cfg, p);
  return p.c.type == kPagedS8 ? gather_t<S8>(cfg, p) : gather_t<E4M3>(cfg, p);
}

cudaError_t launch_paged_zero(const PagedAttnParams& p, cudaStream_t stream) {
  return launch_dependent(fal_paged_zero_kernel, dim3(p.c.batch), dim3(256), 0, stream, p);
}

}  // namespace fal
