// One step of a beam search: of all continuations (beam k, token v) of a request the N with the largest
//   total[k, v] = score[k] + x[k, v] - ln sum_v exp x[k, v],
// equal totals in the order of (k, v).
//
// Two kernels.  beam_part_kernel reads the logits once: a CTA holds a slice of one row in registers, takes its maximum,
// its sum of exponentials and its N largest logits (within a row the order of the totals is the order of the logits).
// beam_merge_kernel, one CTA per request, joins the slices' sums and picks the N best of what they kept.
//
// The N largest of a set are found through a bound: split the set into G >= N groups; the N-th largest of the groups'
// maxima cannot exceed the N-th largest element.  What reaches the bound is N elements and, with random order, few more
// (G = 32: 9.2 of 8, 22 of 16); they are counted against each other for their ranks.  Where more reach it than the
// list holds (many equal logits), the N largest are taken one after the other.
//
// Two beams' candidates may lie arbitrarily close, and their order is an integer output, so sums and totals are formed
// to more than 32 bits: exponentials carry the rounding of their argument along, slices join in fp64, and totals are
// fp64 (the sum comes out within some 1e-8 relative).
#pragma once

#include <cuda_fp16.h>

#include "fmms_common.cuh"

namespace fmms {

constexpr int kBeamThreads = 256;
constexpr int kBeamVecs = 4;         // 16-byte loads of a thread: the slice of a CTA is 16 KiB
constexpr int kBeamMaxN = 64;        // candidates
constexpr int kBeamMaxK = 64;        // beams
constexpr int kBeamListCap = 512;    // elements of a slice that reach the bound
constexpr int kBeamMergeCap = 1024;  // the same over a request

struct BeamParams {
  const void* logits;          // row (r, k) at r * stride_r + k * stride_k elements
  long long stride_r, stride_k;
  const float* scores;         // [R, K]
  const uint8_t* finished;     // [R, K] or null
  int R, K, V, N, splits;
  long long pad_token;
  unsigned long long* keys;    // [R * K][splits][N] (value, index), descending; 0: none
  double* sums;                // [R * K][splits] sum of exp(x - max)
  float* maxima;               // [R * K][splits]
  float* out_scores;           // [R, N]
  long long* out_tokens;
  long long* out_parents;
};

template <typename T>
__device__ __forceinline__ float2 beam_pair(uint32_t w);
template <>
__device__ __forceinline__ float2 beam_pair<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 beam_pair<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// the elements of a 16-byte vector as fp32
template <typename T>
__device__ __forceinline__ void beam_unpack(const uint4& u, float (&v)[16 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(w[i]);
    } else {
      const float2 f = beam_pair<T>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

template <typename T>
__host__ __device__ constexpr int beam_tile() {
  return kBeamThreads * kBeamVecs * (int)(16 / sizeof(T));
}

__device__ __forceinline__ bool beam_live(const BeamParams& p, int row) {
  const float s = p.scores[row];
  return s - s == 0.f;  // neither infinite nor NaN
}

template <typename T>
__global__ void __launch_bounds__(kBeamThreads) beam_part_kernel(const BeamParams p) {
  constexpr int VE = 16 / sizeof(T);
  __shared__ __align__(16) float gmax[128];
  __shared__ float sh_pivot;
  __shared__ int sh_count;
  __shared__ unsigned long long list[kBeamListCap];
  __shared__ double wsum[kBeamThreads / 32];
  __shared__ unsigned long long wbest[kBeamThreads / 32];
  griddep_launch_dependents();
  const int row = blockIdx.y, split = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((p.finished && p.finished[row]) || !beam_live(p, row)) return;  // the merge does not look at such rows either
  const T* x = reinterpret_cast<const T*>(p.logits) + (row / p.K) * p.stride_r + (row % p.K) * p.stride_k;
  const int lead = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));  // elements back to a 16-byte boundary
  const int first = split * beam_tile<T>() + tid * VE - lead;  // index of the thread's first element (may be < 0)

  uint4 u[kBeamVecs];
#pragma unroll
  for (int j = 0; j < kBeamVecs; ++j) {
    const int i = first + j * kBeamThreads * VE;
    if (i >= 0 && i + VE <= p.V) {
      u[j] = __ldg(reinterpret_cast<const uint4*>(x + i));
    } else {
      alignas(16) T e[VE];
#pragma unroll
      for (int q = 0; q < VE; ++q) e[q] = (i + q >= 0 && i + q < p.V) ? x[i + q] : (T)(-INFINITY);
      u[j] = *reinterpret_cast<const uint4*>(e);
    }
  }
  float m = -INFINITY;  // fmaxf drops NaN
#pragma unroll
  for (int j = 0; j < kBeamVecs; ++j) {
    float v[VE];
    beam_unpack<T>(u[j], v);
#pragma unroll
    for (int q = 0; q < VE; ++q) m = fmaxf(m, v[q]);
  }
  // groups of 8 lanes (32 groups) or of 2 lanes (128 groups)
  const int wide = p.N <= 16;
  float gm = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  if (wide) {
    gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 2));
    gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 4));
  }
  const int G = wide ? 32 : 128, per = kBeamThreads / G;
  if (tid % per == 0) gmax[tid / per] = gm;
  if (tid == 0) sh_count = 0;
  __syncthreads();
  float top = -INFINITY;
  for (int i = lane; i < G; i += 32) top = fmaxf(top, gmax[i]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (tid < G) {
    const float v = gmax[tid];
    int rank = 0;
    for (int i = 0; i < G; i += 4) {
      const float4 o = *reinterpret_cast<const float4*>(&gmax[i]);
      rank += (o.x > v || (o.x == v && i < tid)) + (o.y > v || (o.y == v && i + 1 < tid)) +
              (o.z > v || (o.z == v && i + 2 < tid)) + (o.w > v || (o.w == v && i + 3 < tid));
    }
    if (rank == p.N - 1) sh_pivot = v;
  }
  // sum of exp(x - top): 2^(hi + lo) with hi + lo = (x - top) log2(e) to twice the precision, 2^lo = 1 + lo ln 2.
  // The bound of -200 gives 0 and also stands in for -inf, and for NaN, which fmaxf drops.
  constexpr float kL = kLog2e, kL2 = 1.9259629911266175e-8f;  // log2(e) = kL + kL2
  float s = 0.f, c = 0.f;
#pragma unroll
  for (int j = 0; j < kBeamVecs; ++j) {
    float v[VE];
    beam_unpack<T>(u[j], v);
#pragma unroll
    for (int q = 0; q < VE; ++q) {
      const float d = fmaxf(v[q] - top, -200.f);
      const float hi = d * kL;
      const float lo = fmaf(d, kL2, fmaf(d, kL, -hi));
      const float e = ex2_approx(hi);
      s += e;
      c = fmaf(e, lo, c);
    }
  }
  double sum = (double)s + (double)c * 0.6931471805599453;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane == 0) wsum[warp] = sum;
  __syncthreads();
  const float pivot = sh_pivot;
  if (m >= pivot && m > -INFINITY) {
#pragma unroll
    for (int j = 0; j < kBeamVecs; ++j) {
      float v[VE];
      beam_unpack<T>(u[j], v);
#pragma unroll
      for (int q = 0; q < VE; ++q)
        if (v[q] >= pivot && v[q] > -INFINITY) {
          const int pos = atomicAdd(&sh_count, 1);
          // + 0.f: -0 counts as 0
          if (pos < kBeamListCap) list[pos] = cand_key(v[q] + 0.f, first + j * kBeamThreads * VE + q);
        }
    }
  }
  __syncthreads();
  const int n = sh_count;
  const size_t part = (size_t)row * p.splits + split;
  unsigned long long* out = p.keys + part * p.N;
  if (tid == 0) {
    double total = 0.;
    for (int w = 0; w < kBeamThreads / 32; ++w) total += wsum[w];
    p.sums[part] = total;
    p.maxima[part] = top;
  }
  if (n <= kBeamListCap) {
    for (int i = tid; i < n; i += kBeamThreads) {
      const unsigned long long key = list[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += list[j] > key;
      if (rank < p.N) out[rank] = key;
    }
    for (int i = n + tid; i < p.N; i += kBeamThreads) out[i] = 0ull;
    return;
  }
  // many elements at the bound: one maximum after the other (keys differ, each is below the last)
  unsigned long long last = ~0ull;
  for (int r = 0; r < p.N; ++r) {
    unsigned long long best = 0ull;
#pragma unroll
    for (int j = 0; j < kBeamVecs; ++j) {
      float v[VE];
      beam_unpack<T>(u[j], v);
#pragma unroll
      for (int q = 0; q < VE; ++q)
        if (v[q] > -INFINITY) {
          const unsigned long long key = cand_key(v[q] + 0.f, first + j * kBeamThreads * VE + q);
          if (key < last && key > best) best = key;
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, off));
    __syncthreads();
    if (lane == 0) wbest[warp] = best;
    __syncthreads();
    for (int w = 0; w < kBeamThreads / 32; ++w) best = max(best, wbest[w]);
    if (tid == 0) out[r] = best;
    last = best;
  }
}

struct BeamCand {
  double total;
  unsigned int at;  // k * V + v
};
__device__ __forceinline__ bool beam_before(double t1, unsigned int a1, double t2, unsigned int a2) {
  return t1 > t2 || (t1 == t2 && a1 < a2);
}

__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(const BeamParams p) {
  __shared__ double lse[kBeamMaxK], base[kBeamMaxK];
  __shared__ int kind[kBeamMaxK];  // 0: no candidates, 1: its list, 2: finished (one candidate)
  __shared__ double tmax[kBeamThreads];
  __shared__ double sh_pivot;
  __shared__ int sh_count;
  __shared__ double list_t[kBeamMergeCap];
  __shared__ unsigned int list_a[kBeamMergeCap];
  griddep_wait();  // launched behind beam_part_kernel with programmatic stream serialisation
  const int r = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    sh_count = 0;
    sh_pivot = -INFINITY;
  }
  for (int k = warp; k < p.K; k += kBeamThreads / 32) {
    const int row = r * p.K + k;
    const bool live = beam_live(p, row), done = p.finished && p.finished[row];
    double S = 0.;
    float mx = -INFINITY;
    if (live && !done) {
      for (int i = lane; i < p.splits; i += 32) mx = fmaxf(mx, p.maxima[(size_t)row * p.splits + i]);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      if (mx - mx == 0.f) {
        for (int i = lane; i < p.splits; i += 32) {
          const float mi = p.maxima[(size_t)row * p.splits + i];
          if (mi > -INFINITY) S += p.sums[(size_t)row * p.splits + i] * exp((double)mi - (double)mx);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) S += __shfl_xor_sync(0xffffffffu, S, off);
      }
    }
    if (lane == 0) {
      base[k] = (double)p.scores[row];
      kind[k] = !live ? 0 : done ? 2 : (mx - mx == 0.f) ? 1 : 0;
      lse[k] = kind[k] == 1 ? (double)mx + log(S) : 0.;
    }
  }
  __syncthreads();
  const int per_row = p.splits * p.N, E = p.K * per_row;
  // entry e of the request; false: none
  auto entry = [&](int e, double& t, unsigned int& a) {
    const int k = e / per_row;
    if (kind[k] == 1) {
      const unsigned long long key = p.keys[((size_t)r * p.K) * per_row + e];
      if (key == 0ull) return false;
      float v;
      int idx;
      cand_key_decode(key, v, idx);
      t = base[k] + ((double)v - lse[k]);
      a = (unsigned int)k * (unsigned int)p.V + (unsigned int)idx;
      return true;
    }
    if (kind[k] == 2 && e == k * per_row) {
      t = base[k];
      a = (unsigned int)k * (unsigned int)p.V + (unsigned int)p.pad_token;
      return true;
    }
    return false;
  };
  double m = -INFINITY;
  for (int e = tid; e < E; e += kBeamThreads) {
    double t;
    unsigned int a;
    if (entry(e, t, a)) m = fmax(m, t);
  }
  tmax[tid] = m;
  __syncthreads();
  const int G = p.N <= 16 ? 32 : kBeamThreads;  // groups: equal lanes of the warps, or single threads
  if (G == 32 && tid < 32) {
    for (int w = 1; w < kBeamThreads / 32; ++w) m = fmax(m, tmax[w * 32 + tid]);
    __syncwarp();
    tmax[tid] = m;
    __syncwarp();
  }
  if (tid < G) {
    int rank = 0;
    for (int i = 0; i < G; ++i) rank += tmax[i] > m || (tmax[i] == m && i < tid);
    if (rank == p.N - 1) sh_pivot = m;
  }
  __syncthreads();
  const double pivot = sh_pivot;
  for (int e = tid; e < E; e += kBeamThreads) {
    double t;
    unsigned int a;
    if (entry(e, t, a) && t >= pivot) {
      const int pos = atomicAdd(&sh_count, 1);
      if (pos < kBeamMergeCap) {
        list_t[pos] = t;
        list_a[pos] = a;
      }
    }
  }
  __syncthreads();
  const int n = sh_count;
  const size_t o = (size_t)r * p.N;
  auto put = [&](int rank, double t, unsigned int a) {
    p.out_scores[o + rank] = (float)t;
    p.out_tokens[o + rank] = (long long)(a % (unsigned int)p.V);
    p.out_parents[o + rank] = (long long)(a / (unsigned int)p.V);
  };
  int found = min(n, p.N);
  if (n <= kBeamMergeCap) {
    for (int i = tid; i < n; i += kBeamThreads) {
      const double t = list_t[i];
      const unsigned int a = list_a[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += beam_before(list_t[j], list_a[j], t, a);
      if (rank < p.N) put(rank, t, a);
    }
  } else {
    // one after the other: the best entry behind the last one taken
    double lt = INFINITY;
    unsigned int la = 0u;
    for (int i = 0; i < p.N; ++i) {
      double bt = -INFINITY;
      unsigned int ba = 0xffffffffu;
      for (int e = tid; e < E; e += kBeamThreads) {
        double t;
        unsigned int a;
        if (entry(e, t, a) && (i == 0 || beam_before(lt, la, t, a)) && beam_before(t, a, bt, ba)) {
          bt = t;
          ba = a;
        }
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) {
        const double t2 = __shfl_xor_sync(0xffffffffu, bt, off);
        const unsigned int a2 = __shfl_xor_sync(0xffffffffu, ba, off);
        if (beam_before(t2, a2, bt, ba)) {
          bt = t2;
          ba = a2;
        }
      }
      __syncthreads();
      if (lane == 0) {
        list_t[warp] = bt;
        list_a[warp] = ba;
      }
      __syncthreads();
      for (int w = 0; w < kBeamThreads / 32; ++w)
        if (beam_before(list_t[w], list_a[w], bt, ba)) {
          bt = list_t[w];
          ba = list_a[w];
        }
      if (tid == 0) put(i, bt, ba);  // n > N entries exist: every round finds one
      lt = bt;
      la = ba;
    }
  }
  for (int i = found + tid; i < p.N; i += kBeamThreads) {
    p.out_scores[o + i] = -INFINITY;
    p.out_tokens[o + i] = -1;
    p.out_parents[o + i] = min(i, p.K - 1);
  }
}

}  // namespace fmms
