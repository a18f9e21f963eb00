// Merge of the partial results that the splits of a (batch entry, head) row wrote: fp32 rows, each relative to its
// split's maximum, with that maximum (log2 domain) and the sum of the weights.
#pragma once

#include "sm100_ptx.cuh"

namespace fal {

constexpr int kCombineThreads = 128;

// (m, l) <- the merge with another running maximum and sum (log2 domain).
__device__ __forceinline__ void merge_stats(float& m, float& l, float m2, float l2) {
  const float m_new = fmaxf(m, m2);
  const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
  l = l * fast_exp2(m - m_use) + l2 * fast_exp2(m2 - m_use);
  m = m_new;
}

// Called by all threads of a block of kCombineThreads, WARPS warps to a row; tid: the thread's index among its row's.
// Waits for the grids before this one, then merges n partials into head_dim_real columns at out_row: the i-th has its
// statistics at ml[index(i)] and its row at po[index(i) * D / 4].
template <int D, int WARPS, class Index>
__device__ __forceinline__ void combine_row(int tid, bool row_ok, int n, const float2* ml, const float4* po, Index index,
                                            __half* out_row, int head_dim_real, float* lse) {
  static_assert(WARPS == 1 || WARPS * 32 == kCombineThreads, "a row per warp or per block");
  constexpr int kThreads = 32 * WARPS;                       // threads per row
  constexpr int kLanes = D / 4 < kThreads ? D / 4 : kThreads;  // threads per partial row
  constexpr int kVecs = D / (4 * kLanes);                    // 16-byte pieces of it per thread
  constexpr int kGroups = kThreads / kLanes;                 // partial rows in flight
  __shared__ float2 warp_ml[WARPS];
  __shared__ float4 part[kGroups][kLanes];
  // (The lengths were not written by the split-K grid, and whatever wrote them ended before that grid let this one start.)
  grid_dependency_wait();
  if (!row_ok) return;  // (whole warps; a block of one row has that row)

  // The first partial rows of this thread are fetched with the statistics, not behind them: one round trip to L2 for three.
  constexpr int kAhead = 4;
  const int lane = tid % kLanes;
  const int grp = tid / kLanes;
  float mx[kAhead];
  float4 px[kAhead][kVecs];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const int i = grp + k * kGroups;
    mx[k] = -INFINITY;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) px[k][v] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < n) {
      const int64_t at = index(i);
      mx[k] = ml[at].x;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) px[k][v] = po[at * (D / 4) + v * kLanes + lane];
    }
  }
  float m = -INFINITY, l = 0.f;
  for (int i = tid; i < n; i += kThreads) {
    const float2 x = ml[index(i)];
    merge_stats(m, l, x.x, x.y);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, off);
    const float l2 = __shfl_xor_sync(0xffffffffu, l, off);
    merge_stats(m, l, m2, l2);
  }
  if constexpr (WARPS > 1) {
    if ((tid & 31) == 0) warp_ml[tid >> 5] = make_float2(m, l);
    __syncthreads();
    m = warp_ml[0].x;
    l = warp_ml[0].y;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) merge_stats(m, l, warp_ml[w].x, warp_ml[w].y);
  }
  const float muse = (m == -INFINITY) ? 0.f : m;
  const float inv = l > 0.f ? 1.f / l : 0.f;

  float4 o[kVecs];
#pragma unroll
  for (int v = 0; v < kVecs; ++v) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add_weighted = [&](float4& a, float w, const float4& x) {
    a.x += w * x.x;
    a.y += w * x.y;
    a.z += w * x.z;
    a.w += w * x.w;
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    if (grp + k * kGroups < n) {
      const float w = fast_exp2(mx[k] - muse);
#pragma unroll
      for (int v = 0; v < kVecs; ++v) add_weighted(o[v], w, px[k][v]);
    }
  }
#pragma unroll 4
  for (int i = grp + kAhead * kGroups; i < n; i += kGroups) {
    const int64_t at = index(i);
    const float w = fast_exp2(ml[at].x - muse);
#pragma unroll
    for (int v = 0; v < kVecs; ++v) add_weighted(o[v], w, po[at * (D / 4) + v * kLanes + lane]);
  }
  auto add = [&](float4& a, const float4& x) {
    a.x += x.x;
    a.y += x.y;
    a.z += x.z;
    a.w += x.w;
  };
  if constexpr (WARPS > 1) {
    static_assert(kVecs == 1, "one piece per thread");
    part[grp][lane] = o[0];
    __syncthreads();
    if (grp == 0) {
#pragma unroll
      for (int g = 1; g < kGroups; ++g) add(o[0], part[g][lane]);
    }
  } else {
#pragma unroll
    for (int off = kLanes; off < 32; off <<= 1) {  // (one piece per thread then)
      const float4 x = make_float4(__shfl_xor_sync(0xffffffffu, o[0].x, off), __shfl_xor_sync(0xffffffffu, o[0].y, off),
                                   __shfl_xor_sync(0xffffffffu, o[0].z, off), __shfl_xor_sync(0xffffffffu, o[0].w, off));
      add(o[0], x);
    }
  }
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const int col = (v * kLanes + lane) * 4;
    if (grp == 0 && col < head_dim_real) {
      uint2 out;
      out.x = pack_half2(o[v].x * inv, o[v].y * inv);
      out.y = pack_half2(o[v].z * inv, o[v].w * inv);
      *reinterpret_cast<uint2*>(out_row + col) = out;
    }
  }
  if (lse != nullptr && tid == 0) *lse = (l > 0.f) ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace fal
