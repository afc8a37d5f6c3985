// One step of a beam search: of all continuations (beam k, token v) of a request the N with the largest
//   total[k, v] = score[k] + x[k, v] - ln sum_v exp x[k, v],
// equal totals in the order of (k, v).
//
// Two kernels.  beam_part_kernel reads the logits once: a CTA streams a slice of one row through a ring of asynchronous
// copies (each warp, for aligned rows each thread, reads back only what it copied itself, so the loop has no barrier) and keeps the slice's maximum, its
// sum of exponentials and its N largest logits - within a row the order of the totals is the order of the logits.
// beam_merge_kernel, one CTA per request, joins the slices' sums and picks the N best of what they kept.
//
// The N largest of a set are found through a bound: split the set into G >= N groups; the N-th largest of the groups'
// maxima cannot exceed the N-th largest element.  What reaches the bound is N elements and, with random order, few more
// (G = 32: 9.2 of 8, 22 of 16).  A slice takes its bound from its first vectors and keeps the vectors with an element that
// reaches it (from a quarter of the slice: four times as many); their elements are counted against each other for their
// ranks.  Where that is more than the lists hold (tokens masked in the first vectors, logits that rise), the slice is looked
// at again with a bound from all of it, and where even that leaves too many (equal logits), the N largest are taken one
// after the other.
//
// Two beams' candidates may lie arbitrarily close, and their order is an integer output, so more than fp32 goes into the
// totals.  Exponentials are fp32 numbers of the special-function unit (2^-22 relative) whose arguments' rounding is carried
// along; what is not is the rounding of x - max (2^-24 |x - max|, of which the mean over the softmax is at most ln V).  A
// thread adds up to 64 of them in fp32, at most 11 additions deep; from there on, sums, logarithms and totals are fp64.  A
// log-sum-exp is within (15 + ln V) 2^-24, below 2e-6 for 2^18 tokens; measured over rows of all kinds (random, peaked, flat, of
// few values): 1.4e-7 at most.  (In 64 bits throughout, the exponentials of 64 x 8 x 128256 logits alone would be some 15 fp64
// operations each, 50 us at 64 per clock and SM, as much as the whole step takes.)
#pragma once

#include <cuda_fp16.h>

#include <cfloat>
#include <type_traits>

#include "fmms_common.cuh"

namespace fmms {

constexpr int kBeamThreads = 256;
constexpr int kBeamMaxN = 64;       // candidates
constexpr int kBeamMaxK = 64;       // beams
constexpr int kBeamRing = 3;        // pairs of 16-byte vectors a thread has in flight or in hand
constexpr int kBeamFirst = 4;       // vectors of a thread that the bound is taken from
constexpr int kBeamMaxIters = 16;   // vectors of a thread in a slice (even)
constexpr int kBeamVecCap = 448;    // vectors of a slice with an element that reaches the bound
constexpr int kBeamListCap = 512;   // elements of a slice that reach the bound
constexpr int kBeamItems = 1024;    // entries that the merge holds at a time
constexpr int kBeamMergeCap = kBeamItems + kBeamMaxN;

struct BeamParams {
  const void* logits;          // row (r, k) at r * stride_r + k * stride_k elements
  long long stride_r, stride_k;
  const float* scores;         // [R, K]
  const uint8_t* finished;     // [R, K] or null
  int R, K, V, N, splits, iters;  // iters: vectors of a thread in a slice
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

// pair i of the elements of a 16-byte vector, as fp32
template <typename T>
__device__ __forceinline__ float2 beam_get(const uint4& u, int i) {
  if constexpr (sizeof(T) == 4)
    return i == 0 ? make_float2(__uint_as_float(u.x), __uint_as_float(u.y)) : make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  else
    return beam_pair<T>(i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w);
}

// the largest element of a vector; NaN never is (nor does it turn up when all are NaN: the result is then -inf)
template <typename T>
__device__ __forceinline__ float beam_vec_max(const uint4& u) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w))), -INFINITY);
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* h = reinterpret_cast<const T2*>(&u);
    const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    const float2 f = beam_pair<T>(*reinterpret_cast<const uint32_t*>(&m));
    return fmaxf(fmaxf(f.x, f.y), -INFINITY);
  }
}

__device__ __forceinline__ bool beam_live(const BeamParams& p, int row) {
  const float s = p.scores[row];
  return s - s == 0.f;  // neither infinite nor NaN
}

// e^x for x <= 0 to some 1e-12 relative: 2^k times the Taylor polynomial of the rest (|rest| <= ln 2 / 2, rest^11 / 11! <
// 3e-13).  Small where a library call is some hundred instructions, which a kernel of a few microseconds first has to fetch.
__device__ __forceinline__ double beam_exp(double x) {
  if (!(x > -700.)) return 0.;
  const double k = rint(x * 1.4426950408889634), r = fma(k, -0.6931471805599453, x);
  double y = 1. / 3628800.;
  y = fma(y, r, 1. / 362880.);
  y = fma(y, r, 1. / 40320.);
  y = fma(y, r, 1. / 5040.);
  y = fma(y, r, 1. / 720.);
  y = fma(y, r, 1. / 120.);
  y = fma(y, r, 1. / 24.);
  y = fma(y, r, 1. / 6.);
  y = fma(y, r, 0.5);
  y = fma(y, r, 1.);
  y = fma(y, r, 1.);
  return y * __hiloint2double(((int)k + 1023) << 20, 0);
}

// ln x for x >= 1: the fp32 logarithm and one Newton step, y + (x e^-y - 1), whose error is the square of fp32's
__device__ __forceinline__ double beam_log(double x) {
  const double y = (double)logf((float)x);
  return y + fma(x, beam_exp(-y), -1.);
}

// The n-th largest of 32 values, one per lane: sorted by a bitonic network, descending over the lanes.
__device__ __forceinline__ float warp_nth(float v, int n) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int j = size >> 1; j > 0; j >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, j);
      v = ((lane & j) == 0) == ((lane & size) == 0) ? fmaxf(v, o) : fminf(v, o);
    }
  return __shfl_sync(0xffffffffu, v, n - 1);
}

// The same of 128 values, four per lane.
__device__ __noinline__ float warp_nth4(float4 v4, int n) {
  const int lane = threadIdx.x & 31;
  float v[4] = {v4.x, v4.y, v4.z, v4.w};  // value 32 r + lane
#pragma unroll
  for (int size = 2; size <= 128; size <<= 1)
#pragma unroll
    for (int j = size >> 1; j > 0; j >>= 1) {
      float o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = j < 32 ? __shfl_xor_sync(0xffffffffu, v[r], j) : v[r ^ (j >> 5)];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int e = 32 * r + lane;
        v[r] = ((e & j) == 0) == ((e & size) == 0) ? fmaxf(v[r], o[r]) : fminf(v[r], o[r]);
      }
    }
  const int r = (n - 1) >> 5;
  return __shfl_sync(0xffffffffu, r == 0 ? v[0] : r == 1 ? v[1] : r == 2 ? v[2] : v[3], (n - 1) & 31);
}

__device__ __forceinline__ void copy_vector(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// The 16 bytes that begin `offset` bytes (below 16, a multiple of T's size) behind a 16-byte boundary in shared memory.
template <typename T>
__device__ __forceinline__ uint4 load_between(const uint4* at, int offset) {
  const uint2* w = reinterpret_cast<const uint2*>(at) + (offset >> 3);
  const uint2 a = w[0], b = w[1], c = w[2];
  const bool odd = offset & 4;
  const uint4 u = make_uint4(odd ? a.y : a.x, odd ? b.x : a.y, odd ? b.y : b.x, odd ? c.x : b.y);
  if constexpr (sizeof(T) == 4) return u;
  const uint32_t next = odd ? c.y : c.x;
  const int bits = (offset & 2) * 8;
  return make_uint4(__funnelshift_r(u.x, u.y, bits), __funnelshift_r(u.y, u.z, bits), __funnelshift_r(u.z, u.w, bits),
                    __funnelshift_r(u.w, next, bits));
}

// EVEN: every row begins on a 16-byte boundary.
template <typename T, bool EVEN>
__global__ void __launch_bounds__(kBeamThreads, 5) beam_part_kernel(const BeamParams p) {
  constexpr int VE = 16 / sizeof(T);
  constexpr int kWarpVecs = EVEN ? 32 : 33;  // copies of a warp for its 32 vectors
  __shared__ __align__(16) uint4 ring[kBeamRing][2][kBeamThreads / 32 * kWarpVecs];
  __shared__ __align__(16) float gmax[128];
  __shared__ float sh_pivot;
  __shared__ int sh_vecs, sh_count;
  __shared__ __align__(16) uint4 vec_data[kBeamVecCap];
  __shared__ int vec_list[kBeamVecCap];
  __shared__ unsigned long long list[kBeamListCap];
  __shared__ double wsum[kBeamThreads / 32], wsum_up[kBeamThreads / 32];
  __shared__ float wmax[kBeamThreads / 32];
  __shared__ unsigned long long wbest[kBeamThreads / 32];
  griddep_launch_dependents();
  const int row = blockIdx.y, split = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((p.finished && p.finished[row]) || !beam_live(p, row)) return;  // the merge does not look at such rows either
  const T* x = reinterpret_cast<const T*>(p.logits) + (row / p.K) * p.stride_r + (row % p.K) * p.stride_k;
  // A row is cut into vectors from its first element on, wherever it lies, so that rows with the same values have the
  // same sums to the last bit: equal totals of two beams are told apart by (beam, token) alone.  Copies are the 16 bytes on
  // boundaries.  Where a row begins `shift` elements behind one, vector v is the end of copy v and the beginning of copy v + 1,
  // the next lane's, and two lanes of a warp fetch what follows its last vectors.  (64 x 8 x 128257 bf16, 16 candidates: 59 us
  // instead of the 50 us of 128256.)  The last VE to 2 VE - 1 elements, so that no copy ends behind the row, are the last
  // slice's singles.
  const int shift = EVEN ? 0 : (int)(reinterpret_cast<uintptr_t>(x) & 15) / (int)sizeof(T);
  const int vecs = max(p.V / VE - 1, 0), tail = vecs * VE;
  const int v_begin = min(split * p.iters * kBeamThreads, vecs), v_end = min(v_begin + p.iters * kBeamThreads, vecs);
  const int singles = split == p.splits - 1 ? p.V - tail : 0;
  const int copy_end = !EVEN && v_end > v_begin ? v_end + 1 : v_end, place = warp * kWarpVecs + lane;
  const T* boundary = x - shift;

  auto fetch = [&](int v, int slot) {  // vectors v and v + 256 of the row, for this thread
#pragma unroll
    for (int h = 0; h < 2; ++h)
      // (copy 0 begins before the row unless that begins on a boundary)
      if (v + h * kBeamThreads < copy_end && (EVEN || h > 0 || v > 0 || shift == 0))
        copy_vector(&ring[slot][h][place], boundary + (size_t)(v + h * kBeamThreads) * VE);
    if constexpr (!EVEN) {
      const int h = 31 - lane, next = v + h * (kBeamThreads + 1);  // lane 31: its own vector's sequel; lane 30: lane 31's other one's
      if (h < 2 && next < v_end) copy_vector(&ring[slot][h][warp * kWarpVecs + 32], boundary + (size_t)(next + 1) * VE);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (!EVEN && shift && v_begin == 0 && v_end > 0 && tid < VE - shift) reinterpret_cast<T*>(ring[0][0])[shift + tid] = x[tid];
  auto take = [&](int slot, int h) {  // this thread's vector, once the warp's copies are there
    if constexpr (EVEN)
      return ring[slot][h][place];
    else
      return load_between<T>(&ring[slot][h][place], shift * (int)sizeof(T));
  };
#pragma unroll
  for (int i = 0; i < kBeamRing - 1; ++i) fetch(v_begin + 2 * i * kBeamThreads + tid, i);
  float single = -INFINITY;
  int single_at = 0;
  if (tid < singles) {  // at most 2 VE - 1 threads
    single_at = tail + tid;
    single = fmaxf((float)x[single_at], -INFINITY);
  }
  if (tid == 0) sh_vecs = sh_count = 0;

  // bound and first reference of the exponentials from the first vectors (fmaxf drops NaN)
  asm volatile("cp.async.wait_group %0;" ::"n"(kBeamRing - 1 - kBeamFirst / 2) : "memory");
  if constexpr (!EVEN) __syncwarp();
  float m = single;
#pragma unroll
  for (int i = 0; i < kBeamFirst; ++i)
    if (v_begin + i * kBeamThreads + tid < v_end) m = fmaxf(m, beam_vec_max<T>(take(i / 2, i % 2)));
  // The N-th largest of 32 groups' maxima (8 lanes each; up to 32 candidates), or of 128 (2 lanes): into sh_pivot; the
  // largest: returned.
  // Few vectors leave groups of 8 lanes empty, and the bound would be -inf (64 x 12 x 1500 bf16, 24
  // candidates: 26 us, and 15 us with groups of 2).
  const bool wide = p.N <= 32 && v_end - v_begin >= kBeamThreads;
  auto bound = [&](float m) {
    float gm = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    if (wide) {
      gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 2));
      gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 4));
    }
    const int shift = wide ? 3 : 1;
    if ((tid & ((1 << shift) - 1)) == 0) gmax[tid >> shift] = gm;
    __syncthreads();
    float top = gmax[lane];
    if (wide) {
      if (warp == 0) {
        const float v = warp_nth(top, p.N);
        if (lane == 0) sh_pivot = v;
      }
    } else {
      const float4 v4 = make_float4(top, gmax[lane + 32], gmax[lane + 64], gmax[lane + 96]);
      top = fmaxf(fmaxf(v4.x, v4.y), fmaxf(v4.z, v4.w));
      if (warp == 0) {
        const float v = warp_nth4(v4, p.N);
        if (lane == 0) sh_pivot = v;
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    __syncthreads();
    return top;
  };
  const float ref0 = bound(m);
  float pivot = sh_pivot;

  // sum of exp(x - ref): 2^(hi + lo) with hi + lo = (x - ref) log2(e) to twice the precision, 2^lo = 1 + lo ln 2.
  // The bound of -200 gives 0 and also stands in for -inf, and for NaN, which fmaxf drops.
  constexpr float kRest = 1.92596299e-8f;  // log2(e) = kLog2e + kRest
  const float2 kL = make_float2(kLog2e, kLog2e), kNegL = make_float2(-kLog2e, -kLog2e), kNegRest = make_float2(-kRest, -kRest);
  float ref = ref0;
  float2 s = make_float2(0.f, 0.f), c = make_float2(0.f, 0.f);  // sums of e, and of e times minus lo
  auto term = [&](float2 v) {
    float2 d = __fadd2_rn(v, make_float2(-ref, -ref));
    d.x = fmaxf(d.x, -200.f);
    d.y = fmaxf(d.y, -200.f);
    const float2 hi = __fmul2_rn(d, kL);
    const float2 lo = __ffma2_rn(d, kNegRest, __ffma2_rn(d, kNegL, hi));
    const float2 e = make_float2(ex2_approx(hi.x), ex2_approx(hi.y));
    c = __ffma2_rn(e, lo, c);
    return e;
  };
  auto four = [&](float2 a, float2 b, float2 c, float2 d) {
    const float2 ab = __fadd2_rn(term(a), term(b));
    return __fadd2_rn(ab, __fadd2_rn(term(c), term(d)));
  };
  double before = 0.;  // the sum from before the last rise of the reference, in its units
  auto sum_now = [&] { return before + ((double)s.x + (double)s.y) - ((double)c.x + (double)c.y) * 0.6931471805599453; };
  auto raise = [&](float to) {
    const double sum = sum_now();
    before = sum == 0. ? 0. : sum * beam_exp((double)ref - (double)to);
    s = make_float2(0.f, 0.f);
    c = make_float2(0.f, 0.f);
    ref = to;
  };
  if (tid < singles) {
    s = term(make_float2(single, -INFINITY));  // not above ref
  }
  // below this a vector neither raises the reference (which the bound never exceeds) nor is noted; nothing is at -inf
  const float quiet = fmaxf(pivot, -FLT_MAX);
  auto note = [&](int v, const uint4& u) {
    const int pos = atomicAdd(&sh_vecs, 1);
    if (pos < kBeamVecCap) {
      vec_list[pos] = v;
      vec_data[pos] = u;
    }
  };
  const uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;  // -inf
#pragma unroll 1
  for (int i = 0, v = v_begin + tid; i < p.iters / 2; ++i, v += 2 * kBeamThreads) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kBeamRing - 2) : "memory");
    // other lanes' copies are there; and every lane has read the slot before this one, which is filled next
    if constexpr (!EVEN) __syncwarp();
    const int slot = i % kBeamRing;
    uint4 u0 = make_uint4(kNone, kNone, kNone, kNone), u1 = u0;
    if (v < v_end) u0 = take(slot, 0);
    if (v + kBeamThreads < v_end) u1 = take(slot, 1);
    fetch(v + 2 * (kBeamRing - 1) * kBeamThreads, (i + kBeamRing - 1) % kBeamRing);
    const float vm0 = beam_vec_max<T>(u0), vm1 = beam_vec_max<T>(u1), vm = fmaxf(vm0, vm1);
    m = fmaxf(m, vm);
    // rare, and left together: the exponentials below are the warp's again
    if (vm >= quiet) {
      if (vm > ref) raise(vm);
      if (vm0 >= quiet) note(v, u0);
      if (vm1 >= quiet) note(v + kBeamThreads, u1);
    }
    __syncwarp();
    // the two vectors in pairs, pairs of pairs, ..: 3 (fp32: 2) additions deep, and one more for the iteration
    if constexpr (VE == 8) {
      const float2 s0 = four(beam_get<T>(u0, 0), beam_get<T>(u0, 1), beam_get<T>(u0, 2), beam_get<T>(u0, 3));
      const float2 s1 = four(beam_get<T>(u1, 0), beam_get<T>(u1, 1), beam_get<T>(u1, 2), beam_get<T>(u1, 3));
      s = __fadd2_rn(s, __fadd2_rn(s0, s1));
    } else {
      s = __fadd2_rn(s, four(beam_get<T>(u0, 0), beam_get<T>(u0, 1), beam_get<T>(u1, 0), beam_get<T>(u1, 1)));
    }
  }
  const double mine = sum_now();
  float top = m;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (lane == 0) wmax[warp] = top;
  __syncthreads();  // also: the noted vectors are complete
#pragma unroll
  for (int w = 0; w < kBeamThreads / 32; ++w) top = fmaxf(top, wmax[w]);
  // threads whose reference is still the first one add up in its units, the others in those of the slice's maximum
  double sum = ref == ref0 ? mine : 0., sum_up = 0.;
  if (ref != ref0 && mine > 0.) sum_up = mine * beam_exp((double)ref - (double)top);
  const bool any_up = __any_sync(0xffffffffu, sum_up > 0.);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (any_up)
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum_up += __shfl_xor_sync(0xffffffffu, sum_up, off);
  if (lane == 0) {
    wsum[warp] = sum;
    wsum_up[warp] = sum_up;
  }
  // the elements that reach the bound
  auto offer = [&](float v, int at) {
    if (v >= pivot && v > -INFINITY) {
      const int pos = atomicAdd(&sh_count, 1);
      if (pos < kBeamListCap) list[pos] = cand_key(v + 0.f, at);  // + 0.f: -0 counts as 0
    }
  };
  const int vecs_noted = sh_vecs;
  if (vecs_noted <= kBeamVecCap) {
#pragma unroll 1
    for (int i = tid; i < vecs_noted * VE; i += kBeamThreads)
      offer((float)reinterpret_cast<const T*>(vec_data)[i], vec_list[i / VE] * VE + i % VE);
    if (tid < singles) offer(single, single_at);
  }
  __syncthreads();
  int n = sh_count;
  const int from = v_begin * VE, to = split == p.splits - 1 ? p.V : v_end * VE;
  const size_t part = (size_t)row * p.splits + split;
  unsigned long long* out = p.keys + part * p.N;
  if (tid == kBeamThreads - 1) {  // the last warp: the first ones rank the list
    double all = 0., up = 0.;
    for (int w = 0; w < kBeamThreads / 32; ++w) {
      all += wsum[w];
      up += wsum_up[w];
    }
    p.sums[part] = (ref0 == top || all == 0. ? all : all * beam_exp((double)ref0 - (double)top)) + up;
    p.maxima[part] = top;
  }
  if (vecs_noted > kBeamVecCap || n > kBeamListCap) {
    bound(m);  // of the whole slice now
    pivot = sh_pivot;
    if (tid == 0) sh_count = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = from + tid; i < to; i += kBeamThreads) offer((float)x[i], i);
    __syncthreads();
    n = sh_count;
  }
  if (n <= kBeamListCap) {
    if (n > 64 && n <= 256 && p.N <= 32) {
      // The first warp alone: a bound from 32 groups of the list, what reaches it moved to the front, and if that is one
      // element per lane at most, sorted.
      if (warp != 0) return;
      float v = -INFINITY;
      for (int i = lane; i < n; i += 32) v = fmaxf(v, float_key_decode((uint32_t)(list[i] >> 32)));
      const float least = warp_nth(v, p.N);
      int kept = 0;
      for (int i0 = 0; i0 < n; i0 += 32) {
        const unsigned long long key = i0 + lane < n ? list[i0 + lane] : 0ull;
        const bool in = key != 0ull && float_key_decode((uint32_t)(key >> 32)) >= least;
        const unsigned b = __ballot_sync(0xffffffffu, in);
        if (in) list[kept + __popc(b & ((1u << lane) - 1u))] = key;  // at or before where it was read
        kept += __popc(b);
        __syncwarp();
      }
      unsigned long long key = lane < kept ? list[lane] : 0ull;
      if (kept <= 32) {
#pragma unroll
        for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
          for (int j = size >> 1; j > 0; j >>= 1) {
            const unsigned long long o = __shfl_xor_sync(0xffffffffu, key, j);
            key = ((lane & j) == 0) == ((lane & size) == 0) ? max(key, o) : min(key, o);
          }
        if (lane < p.N) out[lane] = key;
        return;
      }
      n = kept;
      for (int i = lane; i < n; i += 32) {
        key = list[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += list[j] > key;
        if (rank < p.N) out[rank] = key;
      }
      return;  // n > 32 >= N: every place is taken
    }
    for (int i = tid; i < n; i += kBeamThreads) {
      const unsigned long long key = list[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += list[j] > key;
      if (rank < p.N) out[rank] = key;
    }
    for (int i = n + tid; i < p.N; i += kBeamThreads) out[i] = 0ull;
    return;
  }
  // many elements at the bound: one maximum after the other (keys differ, each is below the last), read again
  unsigned long long last = ~0ull;
  for (int r = 0; r < p.N; ++r) {
    unsigned long long best = 0ull;
#pragma unroll 1
    for (int i = from + tid; i < to; i += kBeamThreads) {
      const float v = (float)x[i];
      if (v > -INFINITY) {
        const unsigned long long key = cand_key(v + 0.f, i);
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

__device__ __forceinline__ bool beam_before(double t1, unsigned int a1, double t2, unsigned int a2) {
  return t1 > t2 || (t1 == t2 && a1 < a2);
}

// One CTA per request.  What the slices kept is a set of lists, K * splits of them with N entries each in descending order.
// Many lists: the N-th largest of 32 (128) groups' maxima of the lists' first entries is a bound, and every list is read
// as far as it reaches that (1 x 12 x 262208 fp32, 24 candidates: 12384 entries, of which some 50 do; 64 us without, 20 us
// with it).  Otherwise, or when more reach it than there is room for: up to 1024 entries at a time, joined with the best N of
// the ones before, shrink to what reaches their bound (again and again while they are many) and are counted against each
// other.
__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(const BeamParams p) {
  __shared__ double lse[kBeamMaxK], base[kBeamMaxK];
  __shared__ int kind[kBeamMaxK];  // 0: no candidates, 1: its lists, 2: finished (one candidate)
  __shared__ double list_t[2][kBeamMergeCap];
  __shared__ unsigned int list_a[2][kBeamMergeCap];
  __shared__ float gmax[kBeamThreads];
  __shared__ int sh_count[2];
  griddep_wait();  // launched behind beam_part_kernel with programmatic stream serialisation
  const int r = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per_row = p.splits * p.N, items = p.K * per_row;
  const unsigned long long* keys = p.keys + (size_t)r * items;
  const size_t o = (size_t)r * p.N;

  // the first entries (of rows without lists: whatever is there, not looked at) come while the sums do
  const unsigned long long early0 = tid < items ? __ldcg(keys + tid) : 0ull;
  const unsigned long long early1 = tid + kBeamThreads < items ? __ldcg(keys + tid + kBeamThreads) : 0ull;

  // the beams' log-sum-exps: a warp per beam
#pragma unroll 1
  for (int k = warp; k < p.K; k += kBeamThreads / 32) {
    const int at = r * p.K + k;
    const float score = p.scores[at];
    const bool live = score - score == 0.f, done = p.finished && p.finished[at];
    double S = 0.;
    float mx = -INFINITY;
    if (live && !done) {
#pragma unroll 1
      for (int i0 = 0; i0 < p.splits; i0 += 32) {
        const int i = i0 + lane;
        float mi = -INFINITY;
        double si = 0.;
        if (i < p.splits) {
          mi = p.maxima[(size_t)at * p.splits + i];
          si = p.sums[(size_t)at * p.splits + i];
        }
        float all = fmaxf(mi, mx);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, off));
        double term = mi > -INFINITY ? si * beam_exp((double)mi - (double)all) : 0.;
        if (i0 > 0 && lane == 0 && mx > -INFINITY) term += S * beam_exp((double)mx - (double)all);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) term += __shfl_xor_sync(0xffffffffu, term, off);
        S = term;
        mx = all;
      }
    }
    if (lane == 0) {
      base[k] = (double)score;
      kind[k] = !live ? 0 : done ? 2 : (mx - mx == 0.f) ? 1 : 0;
      lse[k] = kind[k] == 1 ? (double)mx + beam_log(S) : 0.;
    }
  }
  int cur = 0, have = 0;  // the list in use; the best candidates so far, at its front
  // the N-th largest of the maxima of 32 (or 128) groups of the threads' m, for everybody
  auto bound = [&](float m) {
    gmax[tid] = m;
    __syncthreads();
    if (p.N <= 32) {
#pragma unroll
      for (int w = 0; w < kBeamThreads / 32; ++w) m = fmaxf(m, gmax[w * 32 + lane]);
      return warp_nth(m, p.N);
    }
    float4 v4;
    v4.x = fmaxf(gmax[lane], gmax[lane + 128]);
    v4.y = fmaxf(gmax[lane + 32], gmax[lane + 160]);
    v4.z = fmaxf(gmax[lane + 64], gmax[lane + 192]);
    v4.w = fmaxf(gmax[lane + 96], gmax[lane + 224]);
    return warp_nth4(v4, p.N);
  };
  bool collected = false;
  const int lists = p.K * p.splits;
  if (items > kBeamItems && lists >= 2 * p.N) {  // of fewer lists the first entries hardly bound anything
    if (tid == 0) sh_count[0] = 0;
    __syncthreads();
    // entry j of list l: its total, and where it comes from; false: there is none
    auto entry = [&](int l, int j, double& t, unsigned int& a) {
      const int k = l / p.splits;
      if (kind[k] == 1) {
        const unsigned long long key = __ldcg(keys + (size_t)l * p.N + j);
        if (key == 0ull) return false;
        float v;
        int idx;
        cand_key_decode(key, v, idx);
        t = base[k] + ((double)v - lse[k]);
        a = (unsigned int)k * (unsigned int)p.V + (unsigned int)idx;
        return true;
      }
      t = base[k];
      a = (unsigned int)k * (unsigned int)p.V + (unsigned int)p.pad_token;
      return kind[k] == 2 && l == k * p.splits && j == 0;
    };
    float m = -INFINITY;
    double t;
    unsigned int a;
    for (int l = tid; l < lists; l += kBeamThreads)
      if (entry(l, 0, t, a)) m = fmaxf(m, __double2float_rd(t));
    const float pivot = bound(m);
    for (int l = tid; l < lists; l += kBeamThreads)
      for (int j = 0; j < p.N; ++j) {
        if (!entry(l, j, t, a) || !(__double2float_rd(t) >= pivot)) break;
        const int pos = atomicAdd(&sh_count[0], 1);
        if (pos >= kBeamMergeCap) break;
        list_t[0][pos] = t;
        list_a[0][pos] = a;
      }
    __syncthreads();
    collected = sh_count[0] <= kBeamMergeCap;
    __syncthreads();  // the count is set anew below
  }
#pragma unroll 1
  for (int first = collected ? items - 1 : 0; first < items; first += kBeamItems) {
    if (!collected && tid == 0) sh_count[cur] = have;
    __syncthreads();
    const int last = collected ? first : min(items, first + kBeamItems);  // collected: nothing more to read
#pragma unroll 1
    for (int j = 0, i = first + tid; i < last; ++j, i += kBeamThreads) {
      const int k = i / per_row;
      const unsigned long long key = first == 0 && j < 2 ? (j == 0 ? early0 : early1) : __ldcg(keys + i);
      double t;
      unsigned int a;
      if (kind[k] == 1) {
        if (key == 0ull) continue;
        float v;
        int idx;
        cand_key_decode(key, v, idx);
        t = base[k] + ((double)v - lse[k]);
        a = (unsigned int)k * (unsigned int)p.V + (unsigned int)idx;
      } else if (kind[k] == 2 && i == k * per_row) {
        t = base[k];
        a = (unsigned int)k * (unsigned int)p.V + (unsigned int)p.pad_token;
      } else {
        continue;
      }
      const int pos = atomicAdd(&sh_count[cur], 1);
      list_t[cur][pos] = t;
      list_a[cur][pos] = a;
    }
    __syncthreads();
    int n = sh_count[cur];
    // Keep what reaches the N-th largest of the maxima of 32 (or 128) groups, item i in group i mod 32 (128).  Rounded
    // down to fp32 the totals keep their order, and a bound need not tell apart what rounding makes equal.
#pragma unroll 1
    while (n > 2 * p.N + 16) {
      float m = -INFINITY;
#pragma unroll 1
      for (int i = tid; i < n; i += kBeamThreads) m = fmaxf(m, __double2float_rd(list_t[cur][i]));
      if (tid == 0) sh_count[cur ^ 1] = 0;
      const float pivot = bound(m);
#pragma unroll 1
      for (int i = tid; i < n; i += kBeamThreads) {
        const double t = list_t[cur][i];
        if (__double2float_rd(t) >= pivot) {
          const int pos = atomicAdd(&sh_count[cur ^ 1], 1);
          list_t[cur ^ 1][pos] = t;
          list_a[cur ^ 1][pos] = list_a[cur][i];
        }
      }
      __syncthreads();
      cur ^= 1;
      if (sh_count[cur] * 4 > n * 3) {  // not much less: many equal totals
        n = sh_count[cur];
        break;
      }
      n = sh_count[cur];
    }
    // ranks; those that make it go out, or to the front of the other list
    const bool end = collected || last == items;
#pragma unroll 1
    for (int i = tid; i < n; i += kBeamThreads) {
      const double t = list_t[cur][i];
      const unsigned int a = list_a[cur][i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += beam_before(list_t[cur][j], list_a[cur][j], t, a);
      if (rank >= p.N) continue;
      if (end) {
        p.out_scores[o + rank] = (float)t;
        p.out_tokens[o + rank] = (long long)(a % (unsigned int)p.V);
        p.out_parents[o + rank] = (long long)(a / (unsigned int)p.V);
      } else {
        list_t[cur ^ 1][rank] = t;
        list_a[cur ^ 1][rank] = a;
      }
    }
    have = min(n, p.N);
    cur ^= 1;
  }
  for (int i = have + tid; i < p.N; i += kBeamThreads) {
    p.out_scores[o + i] = -INFINITY;
    p.out_tokens[o + i] = -1;
    p.out_parents[o + i] = min(i, p.K - 1);
  }
}

}  // namespace fmms
