// Per-beam states after a beam step: beam j of request r goes on with the state of beam parents[r, j].
//
//   state[.., r K + j, ..] <- state[.., r K + parents[r, j], ..]      in place, any number of tensors per launch
//
// In place because most of the traffic then is what cannot be avoided: a beam that keeps its own state is neither read
// (unless another one takes it) nor written, and nothing is copied back.  It needs no buffer and no order between
// threads: a thread owns one column (up to 16 bytes at one offset of all K beams of a request), reads it for every beam
// that changes, and only then writes.  Positions at or behind a request's length are neither read nor written.
//
// Bound by HBM: keys and values of 64 x 8 x 2048 x 64 bf16 for eight requests of four beams, half of the positions live: 376 us
// a call over three draws of parents and lengths, whose reads and writes (2.27 GB) take 352 us at the rate of a plain copy.
// Small states cost a launch, 2.3 us.
#pragma once

#include "fmms_common.cuh"

namespace fmms {

constexpr int kReorderThreads = 256;
constexpr int kReorderMaxStates = 64;     // tensors per launch
constexpr int kReorderMaxRequests = 1024;  // requests per launch
constexpr int kReorderMaxBeams = 64;

struct ReorderState {
  uint8_t* data;
  long long beam_stride;      // bytes from beam to beam
  long long outer_stride[2];  // bytes; the two outer dimensions around the beams
  int outer[2];
  long long seg_bytes;        // contiguous bytes of a beam at one outer index
  long long step_bytes;       // bytes of one position, 0: the state has no positions
};

struct ReorderParams {
  ReorderState st[kReorderMaxStates];
  const void* parents;        // [R, K] int64 or int32
  const int* lengths;         // [R] or null
  int parents_wide;
  int R, K;
};

template <int VEC>
struct ReorderVec;
template <>
struct ReorderVec<16> { using type = uint4; };
template <>
struct ReorderVec<8> { using type = uint2; };
template <>
struct ReorderVec<4> { using type = uint32_t; };
template <>
struct ReorderVec<2> { using type = uint16_t; };
template <>
struct ReorderVec<1> { using type = uint8_t; };

__device__ __forceinline__ int reorder_parent(const ReorderParams& p, int r, int j) {
  const size_t at = (size_t)r * p.K + j;
  const long long v = p.parents_wide ? reinterpret_cast<const long long*>(p.parents)[at]
                                     : (long long)reinterpret_cast<const int*>(p.parents)[at];
  return (v < 0 || v >= p.K) ? j : (int)v;  // not a beam of the request: keep the own state
}

// Columns that a thread handles at a time when a request has up to KM beams (a power of two).  Narrow ones twice as many, or
// too little is in flight (five beams of 5 x 777 x 123 odd bf16 with half of the positions live: 21 us -> 11 us, together with
// a kernel of its own for every width, whose registers then are its own: 64 instead of 108).
__host__ __device__ constexpr int reorder_columns_each(int KM, int vec) {
  const int few = KM <= 4 ? 4 : KM <= 8 ? 2 : 1;
  return vec <= 4 && KM <= 8 ? 2 * few : few;
}

// The columns of one tensor.  KM: beams rounded up.
template <int KM, int VEC>
__device__ __forceinline__ void reorder_columns(const ReorderParams& p, const ReorderState& s, const int* prefix) {
  using V = typename ReorderVec<VEC>::type;
  constexpr int U = reorder_columns_each(KM, VEC), kUnit = kReorderThreads * U;
  const int tid = threadIdx.x;
  const long long cols = s.seg_bytes / VEC;
  const long long outers = (long long)s.outer[0] * s.outer[1];

  if (cols >= kUnit / 2) {
    // Long segments: a unit is kUnit columns of one (outer index, request), so that the parents are read once per unit.
    // prefix[r]: live units of the requests below r.
    const int per_outer = prefix[p.R];
    const long long units = outers * per_outer;
#pragma unroll 1
    for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
      const long long o = unit / per_outer;
      const int i = (int)(unit - o * per_outer);
      int lo = 0, hi = p.R - 1;  // the last r with prefix[r] <= i
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= i) lo = mid; else hi = mid - 1;
      }
      const int r = lo;
      long long live = cols;
      if (p.lengths && s.step_bytes) live = min(cols, max(0, p.lengths[r]) * (s.step_bytes / VEC));
      const long long o0 = o / s.outer[1], o1 = o - o0 * s.outer[1];
      const long long col = (long long)(i - prefix[r]) * kUnit + tid;
      uint8_t* at = s.data + o0 * s.outer_stride[0] + o1 * s.outer_stride[1] + (long long)r * p.K * s.beam_stride + col * VEC;
      int par[KM];
#pragma unroll
      for (int j = 0; j < KM; ++j) par[j] = j < p.K ? reorder_parent(p, r, j) : j;
      V v[U][KM];
#pragma unroll
      for (int j = 0; j < KM; ++j)
        if (par[j] != j) {
          const uint8_t* src = at + par[j] * s.beam_stride;
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (col + u * kReorderThreads < live) v[u][j] = *reinterpret_cast<const V*>(src + u * kReorderThreads * VEC);
        }
#pragma unroll
      for (int j = 0; j < KM; ++j)
        if (par[j] != j) {
          uint8_t* dst = at + j * s.beam_stride;
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (col + u * kReorderThreads < live) *reinterpret_cast<V*>(dst + u * kReorderThreads * VEC) = v[u][j];
        }
    }
    return;
  }
  // Short segments: the columns of all (outer index, request) one after the other.
  const long long total = outers * p.R * cols;
#pragma unroll 1
  for (long long x = (long long)blockIdx.x * kReorderThreads + tid; x < total; x += (long long)gridDim.x * kReorderThreads) {
    const long long seg = x / cols, col = x - seg * cols;
    const long long o = seg / p.R;
    const int r = (int)(seg - o * p.R);
    if (p.lengths && s.step_bytes && col >= max(0, p.lengths[r]) * (s.step_bytes / VEC)) continue;
    const long long o0 = o / s.outer[1], o1 = o - o0 * s.outer[1];
    uint8_t* at = s.data + o0 * s.outer_stride[0] + o1 * s.outer_stride[1] + (long long)r * p.K * s.beam_stride + col * VEC;
    int par[KM];
#pragma unroll
    for (int j = 0; j < KM; ++j) par[j] = j < p.K ? reorder_parent(p, r, j) : j;
    V v[KM];
#pragma unroll
    for (int j = 0; j < KM; ++j)
      if (par[j] != j) v[j] = *reinterpret_cast<const V*>(at + par[j] * s.beam_stride);
#pragma unroll
    for (int j = 0; j < KM; ++j)
      if (par[j] != j) *reinterpret_cast<V*>(at + j * s.beam_stride) = v[j];
  }
}

// grid (CTAs per tensor, tensors); VEC: bytes of a column in all of them
template <int KM, int VEC>
__global__ void __launch_bounds__(kReorderThreads) reorder_kernel(const __grid_constant__ ReorderParams p) {
  __shared__ int prefix[kReorderMaxRequests + 1];
  const ReorderState& s = p.st[blockIdx.y];
  constexpr int kUnit = kReorderThreads * reorder_columns_each(KM, VEC);
  if (s.seg_bytes / VEC >= kUnit / 2) {
    for (int r = threadIdx.x; r < p.R; r += kReorderThreads) {
      long long live = s.seg_bytes;
      if (p.lengths && s.step_bytes) live = min(live, max(0, p.lengths[r]) * s.step_bytes);
      prefix[r + 1] = (int)((live / VEC + kUnit - 1) / kUnit);
    }
    __syncthreads();
    if (threadIdx.x < 32) {  // inclusive sums, 32 at a time
      int carry = 0;
      for (int b = 0; b < p.R; b += 32) {
        const int r = b + threadIdx.x;
        int v = r < p.R ? prefix[r + 1] : 0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, v, off);
          if ((int)threadIdx.x >= off) v += o;
        }
        v += carry;
        if (r < p.R) prefix[r + 1] = v;
        carry = __shfl_sync(0xffffffffu, v, 31);
      }
      if (threadIdx.x == 0) prefix[0] = 0;
    }
    __syncthreads();
  }
  reorder_columns<KM, VEC>(p, s, prefix);
}

}  // namespace fmms
