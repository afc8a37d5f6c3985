// Products with 4-bit weights for more than eight rows of x: the same stored weights, scales and arithmetic as in
// fmms_int4.cuh, on the fifth-generation tensor cores.
//
// mma.sync takes eight cycles for a 16 x 16 x 8 product here, so that beyond eight rows the products and not the weight's
// stream set its pace (151936 x 4096: 55 us for one row, 60 us for 8, 83 us for 16, 216 us for 32, where this kernel takes
// 88 us and 103 us; 128256 x 8192 at 16 rows: 200 us and 143 us).  tcgen05.mma takes 128 weight
// rows against all rows of x at once, and it reads one operand from tensor memory: the weights go from registers there,
// in the very layout the stored order is made for (tcgen05.st .16x128b places what a lane holds of a 16 x 16 operand), and
// never through shared memory as fp16.
//
// A CTA per SM has a contiguous range of tiles and takes eight of them (128 rows) at a time:
//   warps 0-15   stream the weights through rings of asynchronous copies of their own (warp w: every second step, the
//                tiles of tensor-memory lanes 32 (w mod 4).., half of the columns), move the nibbles to bits 4 to 7 of fp16
//                subnormals and store them
//   warps 16-23  read the sums of every group back, a weight row and half of the rows of x per thread: out[n] += s sum[n] in
//                fp32
//   warp 24      issues the products, a group of columns to an accumulator
//   warp 25      fetches x, a bulk copy per step
// The zero points are products as well: behind the columns of a group come 16 more, of which three hold z on the one side
// and minus the sum of x over the group, cut into three fp16 parts, on the other (the z of all groups of a step, up to four,
// lie in one such operand, at columns 4 g.., and the sums of group g meet only those).  That halves what the reading back
// costs (a multiply-add per row of x and group instead of two and a load).
// int4_stage_x writes x beforehand, as fp16 in the swizzled layout of the products with those columns behind every step.
// Its power of two per row puts the row's largest element into [2^7, 2^8), so that a group's sum fits fp16 as well; what lies
// below 2^-24 of that element (2^-21 for fp16 rows) is rounded to 2^-32 of it, far below the rounding of the fp32 sums.
#pragma once

#include <cuda_fp16.h>

#include "fmms_common.cuh"
#include "fmms_int4.cuh"
#include "fmms_tcgen05.cuh"

namespace fmms {

constexpr int kInt4MmaWeightWarps = 16, kInt4MmaSumWarps = 8;
constexpr int kInt4MmaThreads = (kInt4MmaWeightWarps + kInt4MmaSumWarps + 2) * 32;
constexpr int kInt4MmaPass = 64;       // rows of x in a pass, at most
constexpr int kInt4MmaRing = 4;        // steps in a warp's ring (every second one is its own)
constexpr int kInt4MmaMaxX = 6;        // steps of x in shared memory
constexpr int kInt4MmaScaleRing = 8;   // steps of scales
constexpr int kInt4MmaAlign = 1024;    // of the shared memory of a CTA, whose dynamic part has as many bytes more
// A step is what changes hands at a time: 256 columns, for barriers, not arithmetic, set the pace of a shorter one; 128 where
// tensor memory (of a slot: operands at 64 columns a unit, zero points 8, accumulators at a column per row of x and group)
// does not hold two of them.
__host__ __device__ constexpr int int4_step_units(int group, int n) { return group < kInt4Unit || n > 48 ? 1 : 2; }
__host__ __device__ constexpr int int4_step_groups(int group, int n) { return int4_step_units(group, n) * int4_unit_groups(group); }
// Steps in tensor memory.  Three let a weight warp fill while the products of the step before still run; with two it waits for
// them (128256 x 8192 at 16 rows: 147 us, with three 143 us).
__host__ __device__ constexpr int int4_slots(int group, int n) {
  const int fit = kTmemCols / (int4_step_units(group, n) * 64 + 8 + int4_step_groups(group, n) * n);
  return fit < 3 ? fit : 3;
}
__host__ __device__ constexpr int int4_mma_max_n(int group) { return group == 32 ? 32 : kInt4MmaPass; }
__host__ __device__ constexpr int int4_x_bytes(int n, int group) { return (int4_step_units(group, n) * 2 + 1) * n * 128; }  // of a step

struct Int4MmaParams {
  Int4Params base;        // x: for int4_stage_x only
  const uint8_t* staged;  // [passes][steps of a row][int4_x_bytes]
  const int* exponents;   // [passes][64]
  int n, row_steps;       // rows of x in a pass, a multiple of 16
  int x_stages, ring_off, scale_off;
  uint32_t idesc;
  int* status_dev;
  unsigned long long wait_ns;  // how long a wait may take
  int x_limit;                 // steps of x that a CTA fetches, at most: fewer than there are makes the waits for them run out
};

// One CTA per row of x.
template <int GR>
__global__ void __launch_bounds__(256) int4_stage_x_kernel(const Int4MmaParams p, uint8_t* staged, int* exponents) {
  const int step_units = int4_step_units(GR, p.n);
  __shared__ uint32_t wmax[8];
  griddep_launch_dependents();
  const Int4Params& q = p.base;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pass = b / p.n, row = b - pass * p.n;
  const uint16_t* src = reinterpret_cast<const uint16_t*>(q.x) + (size_t)b * q.x_stride;
  auto load = [&](int k, float (&v)[8]) {  // eight columns; zero behind the end
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w = 0u;
      if (k < q.D)
        w = q.x_pairs ? *reinterpret_cast<const uint32_t*>(src + k + 2 * i) : (uint32_t)src[k + 2 * i] | ((uint32_t)src[k + 2 * i + 1] << 16);
      v[2 * i] = half_bits_to_float(w & 0xffffu, q.x_bf16);
      v[2 * i + 1] = half_bits_to_float(w >> 16, q.x_bf16);
    }
  };
  uint32_t m = 0u;
#pragma unroll 2
  for (int k = tid * 8; k < q.D; k += 256 * 8) {
    float v[8];
    load(k, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) wmax[warp] = m;
  __syncthreads();
  m = 0u;
#pragma unroll
  for (int w = 0; w < 8; ++w) m = max(m, wmax[w]);
  const int exponent = m == 0u ? 0 : min(7 - ((int)(m >> 23) - 127), 120);
  if (tid == 0) exponents[pass * kInt4MmaPass + row] = exponent;
  const float up = __uint_as_float((uint32_t)(exponent + 127) << 23);
  const int cols = q.all_units * kInt4Unit;
  uint8_t* out = staged + (size_t)pass * p.row_steps * int4_x_bytes(p.n, GR);
  auto place = [&](int tile, int c16) {  // of the 16 bytes c16 of this row in a tile of n rows of 128 bytes
    return tile * (p.n * 128) + row * 128 + ((c16 ^ (row & 7)) * 16);
  };
  // all threads run the same number of rounds: the sums are shuffled
#pragma unroll 1
  for (int k0 = 0; k0 < cols; k0 += 256 * 8) {
    const int k = k0 + tid * 8;
    float v[8], s = 0.f;
    load(k, v);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = __floats2half2_rn(v[2 * j] * up, v[2 * j + 1] * up);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
      const float2 f = __half22float2(h);
      s += f.x + f.y;
    }
#pragma unroll
    for (int off = 1; off < GR / 8; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (k >= cols) continue;
    const int step = k / (step_units * kInt4Unit), in_step = k - step * (step_units * kInt4Unit);
    uint8_t* dst = out + (size_t)step * int4_x_bytes(p.n, GR);
    *reinterpret_cast<uint4*>(dst + place(in_step / 64, in_step % 64 / 8)) = make_uint4(w[0], w[1], w[2], w[3]);
    if (in_step % GR == 0) {
      // minus the sum, in three parts
      const __half h0 = __float2half_rn(-s), h1 = __float2half_rn(-s - __half2float(h0));
      const __half h2 = __float2half_rn(-s - __half2float(h0) - __half2float(h1));
      const int gi = in_step / GR;
      const uint32_t w0 = (uint32_t)__half_as_ushort(h0) | ((uint32_t)__half_as_ushort(h1) << 16), w1 = (uint32_t)__half_as_ushort(h2);
      const uint4 parts = gi & 1 ? make_uint4(0u, 0u, w0, w1) : make_uint4(w0, w1, 0u, 0u), none = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(dst + place(step_units * 2, gi * 2)) = gi < 2 ? parts : none;
      *reinterpret_cast<uint4*>(dst + place(step_units * 2, gi * 2 + 1)) = gi < 2 ? none : parts;
    }
  }
}

// Four words of codes (64 columns of 16 rows, over the warp) as fp16 subnormals: per word the operands of a 16 x 16 product.
// Masked inside the statement, so that the results are made where the store wants them.
__device__ __forceinline__ void tmem_store_codes(uint32_t taddr, uint4 w) {
  asm volatile(
      "{\n\t"
      ".reg .b32 a<16>;\n\t"
      "shl.b32 a0, %1, 4;\n\t"
      "shr.u32 a2, %1, 4;\n\t"
      "shr.u32 a3, %1, 8;\n\t"
      "shl.b32 a4, %2, 4;\n\t"
      "shr.u32 a6, %2, 4;\n\t"
      "shr.u32 a7, %2, 8;\n\t"
      "shl.b32 a8, %3, 4;\n\t"
      "shr.u32 a10, %3, 4;\n\t"
      "shr.u32 a11, %3, 8;\n\t"
      "shl.b32 a12, %4, 4;\n\t"
      "shr.u32 a14, %4, 4;\n\t"
      "shr.u32 a15, %4, 8;\n\t"
      "and.b32 a0, a0, 0x00f000f0;\n\t"
      "and.b32 a1, %1, 0x00f000f0;\n\t"
      "and.b32 a2, a2, 0x00f000f0;\n\t"
      "and.b32 a3, a3, 0x00f000f0;\n\t"
      "and.b32 a4, a4, 0x00f000f0;\n\t"
      "and.b32 a5, %2, 0x00f000f0;\n\t"
      "and.b32 a6, a6, 0x00f000f0;\n\t"
      "and.b32 a7, a7, 0x00f000f0;\n\t"
      "and.b32 a8, a8, 0x00f000f0;\n\t"
      "and.b32 a9, %3, 0x00f000f0;\n\t"
      "and.b32 a10, a10, 0x00f000f0;\n\t"
      "and.b32 a11, a11, 0x00f000f0;\n\t"
      "and.b32 a12, a12, 0x00f000f0;\n\t"
      "and.b32 a13, %4, 0x00f000f0;\n\t"
      "and.b32 a14, a14, 0x00f000f0;\n\t"
      "and.b32 a15, a15, 0x00f000f0;\n\t"
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {a0, a1, a2, a3, a4, a5, a6, a7, a8, a9, a10, a11, a12, a13, a14, a15};\n\t"
      "}" ::"r"(taddr),
      "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
      : "memory");
}

__device__ __forceinline__ void tmem_load8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_store_zero_points(uint32_t taddr, const uint32_t (&a)[4]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]) : "memory");
}

// A in tensor memory, B in shared memory
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(yes));
  return yes != 0;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// NC: rows of x in a pass (16, 32, 48 or 64).
template <int NC, int GR, bool ZP>
__global__ void __launch_bounds__(kInt4MmaThreads, 1) int4_mma_kernel(const Int4MmaParams p) {
  extern __shared__ uint8_t smem_raw[];
  // swizzled operands begin on 1 KiB boundaries
  uint8_t* const smem = smem_raw + ((kInt4MmaAlign - (smem_u32(smem_raw) & (kInt4MmaAlign - 1))) & (kInt4MmaAlign - 1));
  constexpr int kGroups = int4_unit_groups(GR), kSteps = GR / 16;
  constexpr int kStepU = int4_step_units(GR, NC), kStepG = int4_step_groups(GR, NC);
  constexpr int kXBytes = int4_x_bytes(NC, GR);
  // tensor memory: operands of all slots, zero points (of each slot, or one for all), accumulators of all slots
  constexpr int kSlots = int4_slots(GR, NC), kZeroCols = ZP ? 8 : 0;
  constexpr int kZeroAt = kSlots * kStepU * 64, kSumAt = kZeroAt + (ZP ? kSlots * kZeroCols : 8);
  static_assert(kSlots >= 2 && kStepG <= 4 && kSumAt + kSlots * kStepG * NC <= kTmemCols, "tensor memory");
  constexpr int kScaleBytes = kStepG * 64;  // of a step, for the two tiles of a warp
  constexpr int kScaleCopy = kStepG == 4 ? 8 : 4, kScaleLanes = kStepG * 32 / kScaleCopy;
  __shared__ uint64_t a_full[kSlots], done[kSlots], d_empty[kSlots];
  __shared__ uint64_t x_full[kInt4MmaMaxX], x_empty[kInt4MmaMaxX];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const Int4Params& q = p.base;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = warp & 3;
  const int pass = blockIdx.y;

  // this CTA's tiles, eight to a block; tile s of a block lies in lanes 32 (s mod 4) + 16 (s / 4)..
  const int t_each = q.tiles / (int)gridDim.x, t_rest = q.tiles - t_each * (int)gridDim.x;
  const int t_begin = t_each * (int)blockIdx.x + min((int)blockIdx.x, t_rest), t_count = t_each + ((int)blockIdx.x < t_rest);
  const int blocks = (t_count + 7) / 8, row_steps = p.row_steps, steps = blocks * row_steps;

  if (tid == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&a_full[i], kInt4MmaWeightWarps / 2);
      mbar_init(&done[i], 1);  // the products: operands free, sums there
      mbar_init(&d_empty[i], kInt4MmaSumWarps);
    }
    for (int i = 0; i < p.x_stages; ++i) {
      mbar_init(&x_full[i], 1);
      mbar_init(&x_empty[i], 1);
    }
    abort_word = 0;
    fence_mbar_init();
  }
  if (warp == kInt4MmaWeightWarps + kInt4MmaSumWarps) {
    tmem_alloc(&tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  if (warp < kInt4MmaWeightWarps) {
    // ------------------------------ weights ------------------------------
    const int half = (warp >> 2) & 1, a = warp >> 3;  // chunk of every unit; steps a, a + 2, ..
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    constexpr int kSlot = kStepU * 1024 + (ZP ? 128 : 0);  // bytes of a step: two tiles, one chunk of each unit; zeros
    uint8_t* ring = smem + p.ring_off + warp * (kInt4MmaRing * kSlot);
    const uint32_t ring_at = smem_u32(ring);
    // zeros: the warps of the first half have those of all groups of the step, 16 bytes for each of the two tiles
    const bool zeros_too = ZP && half == 0;
    const int z_tile = lane >> 2 & 1, z_group = lane >> 3;  // lanes below 8 kStepG copy 4 bytes of these
    const long long four = (long long)q.chunks * (4 * 512);  // four tiles on
    int f_block = 0, f_step = a - 2, f_slot = 0;
    const uint8_t *f_q = nullptr, *f_z = nullptr;
    auto next = [&](int& block, int& step) {
      step += 2;
      while (step >= row_steps) {
        step -= row_steps;
        ++block;
      }
    };
    auto fetch = [&] {
      const int old = f_block;
      const bool first = f_step < 0;
      next(f_block, f_step);
      if (f_block < blocks) {
        const int unit = f_step * kStepU;
        if (f_block != old || first) {
          const long long tile = t_begin + f_block * 8 + quad;  // the first of this warp's two
          f_q = q.q + (tile * q.chunks + unit * 2 + half) * 512 + lane * 16;
          if constexpr (ZP) f_z = q.zeros + (tile + z_tile * 4) * q.groups * 16 + (lane & 3) * 4;
        }
        const int left = t_count - f_block * 8 - quad;
        const uint32_t dst = ring_at + f_slot * kSlot;
#pragma unroll
        for (int i = 0; i < kStepU; ++i) {
          const bool in = (unit + i) * 2 + half < q.chunks;  // a row may end within its last step, or its last unit
          if (in && left > 0) copy_async<16>(dst + i * 1024 + lane * 16, f_q + i * 1024);
          if (in && left > 4) copy_async<16>(dst + i * 1024 + 512 + lane * 16, f_q + four + i * 1024);
        }
        if constexpr (ZP) {
          // groups of more than one unit repeat
          const int gr = GR == kInt4Unit ? (q.group_units == 1 ? unit + z_group : (unit + z_group) / q.group_units) : unit * kGroups + z_group;
          if (zeros_too && z_group < kStepG && left > z_tile * 4 && gr < q.groups)
            copy_async<4>(dst + kStepU * 1024 + lane * 4, f_z + gr * 16);
        }
        f_q += 2 * kStepU * 1024;
        if (++f_slot == kInt4MmaRing) f_slot = 0;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < kInt4MmaRing - 1; ++i) fetch();
    // z 2^-20 of group g at columns 4 g, 4 g + 1 and 4 g + 2 of a row: what lane (row, t) holds of the operand for rows `row`
    // and 8 + row is that of group t / 2, and 8 columns on of group 2 + t / 2.  Above 127 that is no subnormal: the number's
    // step doubles at 2^-13.
    const uint32_t z_mask = lane & 1 ? 0x0000ffffu : 0xffffffffu;
    const int z_mine = lane >> 1 & 1;
    auto zero_point = [&](uint32_t z) { return min(z << 4, (z << 3) + 1024u) * 0x00010001u & z_mask; };
    if constexpr (!ZP)
      if (warp < 4) {  // before this warp's first step, and read from step 0 on, which is its own
        const uint32_t eight = zero_point(8), all[4] = {eight, eight, eight, eight};
        tmem_store_zero_points(tmem + lanes + kZeroAt, all);
        tmem_store_zero_points(tmem + lanes + (16u << 16) + kZeroAt, all);
      }
    int slot = 0, at_slot = a, round = 0, block = 0, step = a - 2;  // at_slot, round: where the step goes, for the how manieth time
#pragma unroll 1
    for (;;) {
      next(block, step);
      if (block >= blocks) break;
      const int mine = t_count - block * 8 - quad;  // > 0: the first tile is there, > 4: the second too
      asm volatile("cp.async.wait_group %0;" ::"n"(kInt4MmaRing - 2) : "memory");
      if constexpr (ZP) __syncwarp();  // zeros were copied by other lanes
      const uint8_t* src = ring + slot * kSlot;
      if (round > 0) mbar_wait(&done[at_slot], (uint32_t)(round - 1) & 1u, abort_flag, p.status_dev, p.wait_ns);
      tc_fence_after();
      const uint32_t at = tmem + lanes + at_slot * (kStepU * 64) + half * 32;
#pragma unroll
      for (int i = 0; i < kStepU; ++i)
#pragma unroll
        for (int m = 0; m < 2; ++m)
          if (mine > m * 4) tmem_store_codes(at + ((uint32_t)(m * 16) << 16) + i * 64, *reinterpret_cast<const uint4*>(src + i * 1024 + m * 512 + lane * 16));
      if (zeros_too) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          uint32_t z[4] = {0u, 0u, 0u, 0u};
#pragma unroll
          for (int j = 0; j < kStepG; j += 2) {
            // (a step of one group has no second one: what is read in its place meets zeros of x)
            const uint32_t pair = *reinterpret_cast<const uint16_t*>(src + kStepU * 1024 + ((j + z_mine) * 2 + m) * 16 + (lane >> 2) * 2);
            z[j] = zero_point(pair & 0xffu);
            z[j + 1] = zero_point(pair >> 8);
          }
          tmem_store_zero_points(tmem + lanes + ((uint32_t)(m * 16) << 16) + kZeroAt + at_slot * kZeroCols, z);
        }
        __syncwarp();  // everybody has read the slot's zeros
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&a_full[at_slot]);
      fetch();
      if (++slot == kInt4MmaRing) slot = 0;
      at_slot += 2;
      if (at_slot >= kSlots) {
        at_slot -= kSlots;
        ++round;
      }
    }
  } else if (warp < kInt4MmaWeightWarps + kInt4MmaSumWarps) {
    // ------------------------------ sums ------------------------------
    // two warps to a quarter of the lanes, each with half of the columns
    constexpr int kCols = NC / 2;
    const int first_col = (warp - kInt4MmaWeightWarps) / 4 * kCols;
    uint8_t* ring = smem + p.scale_off + (warp - kInt4MmaWeightWarps) * (kInt4MmaScaleRing * kScaleBytes);
    const uint32_t ring_at = smem_u32(ring);
    int f_block = 0, f_unit = 0, f_slot = 0;
    const int sm = lane / kScaleLanes;                                 // which of the two tiles this lane copies for
    const int sg = (lane % kScaleLanes) * kScaleCopy / 32;             // which group of the step
    const uint8_t* f_s = nullptr;
    auto start = [&] {
      const long long tile = t_begin + f_block * 8 + quad;
      f_s = reinterpret_cast<const uint8_t*>(q.scales) + (tile + sm * 4) * q.groups * 32 + (lane % kScaleLanes) * kScaleCopy % 32;
    };
    auto fetch = [&] {
      if (f_block < blocks) {
        // groups of more than one unit repeat
        const int gr = GR == kInt4Unit ? (q.group_units == 1 ? f_unit + sg : (f_unit + sg) / q.group_units) : f_unit * kGroups + sg;
        if (lane < 2 * kScaleLanes && t_count - f_block * 8 - quad > sm * 4 && gr < q.groups)
          copy_async<kScaleCopy>(ring_at + f_slot * kScaleBytes + lane * kScaleCopy, f_s + gr * 32);
        if (++f_slot == kInt4MmaScaleRing) f_slot = 0;
        f_unit += kStepU;
        if (f_unit >= q.all_units) {
          f_unit = 0;
          ++f_block;
          start();
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    start();
#pragma unroll 1
    for (int i = 0; i < kInt4MmaScaleRing - 1; ++i) fetch();
    griddep_wait();  // the exponents come from the kernel before
    const int r16 = lane & 15, tile_of = lane >> 4;  // row within its tile; first or second tile
    const int place = (r16 & 7) * 2 + (r16 >> 3);    // within the 16 scales of a group
    const int nb = min(NC, q.B - pass * p.n);
    // what brings column first_col + lane back to its row of x, in two halves: no step of it lies beyond both ends
    int e = 0;
    if (lane < kCols && first_col + lane < nb) e = 20 - p.exponents[pass * kInt4MmaPass + first_col + lane];
    const float down0 = __uint_as_float((uint32_t)(127 + (e >> 1)) << 23), down1 = __uint_as_float((uint32_t)(127 + e - (e >> 1)) << 23);
    int slot = 0, d = 0, dround = 0;
#pragma unroll 1
    for (int block = 0; block < blocks; ++block) {
      float2 tot[kCols / 2];
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) tot[i] = make_float2(0.f, 0.f);
#pragma unroll 1
      for (int unit = 0; unit < q.all_units; unit += kStepU) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kInt4MmaScaleRing - 2) : "memory");
        __syncwarp();
        fetch();
        float s[kStepG];
#pragma unroll
        for (int gi = 0; gi < kStepG; ++gi)
          s[gi] = half_bits_to_float(reinterpret_cast<const uint16_t*>(ring + slot * kScaleBytes)[tile_of * (kStepG * 16) + gi * 16 + place], q.s_bf16);
        if (++slot == kInt4MmaScaleRing) slot = 0;
        mbar_wait(&done[d], (uint32_t)dround & 1u, abort_flag, p.status_dev, p.wait_ns);
        __syncwarp();
        tc_fence_after();
        const int groups = GR == kInt4Unit ? min(kStepU, q.all_units - unit) : min(kStepG, q.groups - unit * kGroups);
        const uint32_t at = tmem + ((uint32_t)(quad * 32) << 16) + kSumAt + d * (kStepG * NC) + first_col;
#pragma unroll
        for (int gi = 0; gi < kStepG; ++gi) {
          if (gi >= groups) break;  // the row has ended: no products either
          const float2 s2 = make_float2(s[gi], s[gi]);
#pragma unroll
          for (int i = 0; i < kCols / 8; ++i) {
            uint32_t acc[8];
            tmem_load8(at + gi * NC + i * 8, acc);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              tot[i * 4 + j] = __ffma2_rn(s2, make_float2(__uint_as_float(acc[2 * j]), __uint_as_float(acc[2 * j + 1])), tot[i * 4 + j]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&d_empty[d]);
        if (++d == kSlots) {
          d = 0;
          ++dround;
        }
      }
      // (after a wait that ran out, here or elsewhere, what has been added up need not be sums)
      const bool there = t_count - block * 8 - quad > tile_of * 4 && !*abort_flag;
      const int v = (t_begin + block * 8 + quad + tile_of * 4) * kInt4Tile + r16;
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        const float y = ((i & 1) ? tot[i / 2].y : tot[i / 2].x) * __shfl_sync(0xffffffffu, down0, i) * __shfl_sync(0xffffffffu, down1, i);
        if (there && v < q.V && first_col + i < nb) int4_store(q, pass * p.n + first_col + i, v, y);
      }
      if (__any_sync(0xffffffffu, *abort_flag)) break;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kInt4MmaWeightWarps + kInt4MmaSumWarps) {
    // ------------------------------ products ------------------------------
    // The whole warp runs the loop, so that addresses stay in uniform registers; one elected lane issues.
    int a = 0, around = 0, x = 0, xround = 0, unit = 0, issued = 0;
#pragma unroll 1
    for (; issued < steps; ++issued) {
      // three conditions at once: lanes 0 mod 3 wait for x, 1 for the accumulators, 2 for the weights
      const int what = lane % 3;
      bool ok = true;
      if (what != 1 || around > 0)
        ok = mbar_wait(what == 0 ? &x_full[x] : what == 1 ? &d_empty[a] : &a_full[a],
                       (uint32_t)(what == 0 ? xround : what == 1 ? around - 1 : around) & 1u, abort_flag, p.status_dev, p.wait_ns);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const int groups = GR == kInt4Unit ? min(kStepU, q.all_units - unit) : min(kStepG, q.groups - unit * kGroups);
      const uint64_t desc = umma_smem_desc(smem_u32(smem) + x * kXBytes);
      const uint32_t ta = tmem + a * (kStepU * 64), tz = tmem + kZeroAt + a * kZeroCols, td = tmem + kSumAt + a * (kStepG * NC);
      if (elect_one()) {
#pragma unroll
        for (int gi = 0; gi < kStepG; ++gi) {
          if (gi >= groups) break;
          const uint64_t dz = desc + (uint64_t)(kStepU * 2 * (NC * 128 / 16) + gi * 2);
          umma_f16_ts(td + gi * NC, tz, dz, p.idesc, 0u);
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            const int k = gi * kSteps + j;  // 16 columns: eight of tensor memory, 32 bytes of each row of x
            umma_f16_ts(td + gi * NC, ta + k * 8, desc + (uint64_t)((k >> 2) * (NC * 128 / 16) + (k & 3) * 2), p.idesc, 1u);
          }
        }
        umma_commit(&done[a]);
        umma_commit(&x_empty[x]);
      }
      __syncwarp();
      if (++a == kSlots) {
        a = 0;
        ++around;
      }
      if (++x == p.x_stages) {
        x = 0;
        ++xround;
      }
      unit += kStepU;
      if (unit >= q.all_units) unit = 0;
    }
    // the products that were issued have to end, and the last commit to arrive, while the CTA and its tensor memory are there
    if (issued > 0 && !mbar_wait_plain(&x_empty[(issued - 1) % p.x_stages], (uint32_t)((issued - 1) / p.x_stages) & 1u, kWaitLimitNs) && p.status_dev)
      atomicExch(p.status_dev, kErrTimeout);
  } else if (lane == 0) {
    // ------------------------------ x ------------------------------
    griddep_wait();
    const uint8_t* src = p.staged + (size_t)pass * row_steps * kXBytes;
    int x = 0, round = 0, at = 0, issued = 0;
#pragma unroll 1
    for (int step = 0; step < min(steps, p.x_limit); ++step) {
      if (round > 0 && !mbar_wait(&x_empty[x], (uint32_t)(round - 1) & 1u, abort_flag, p.status_dev, p.wait_ns)) break;
      mbar_arrive_expect_tx(&x_full[x], (uint32_t)kXBytes);
      bulk_load(smem + x * kXBytes, src + (size_t)at * kXBytes, (uint32_t)kXBytes, &x_full[x]);
      ++issued;
      if (++at == row_steps) at = 0;
      if (++x == p.x_stages) {
        x = 0;
        ++round;
      }
    }
    // copies land before the CTA's memory is reused, also when a wait ran out and no product asks for them
    for (int i = 0; i < min(issued, p.x_stages); ++i) {
      const int last = ((issued - 1 - i) / p.x_stages) * p.x_stages + i;
      mbar_wait_plain(&x_full[i], (uint32_t)(last / p.x_stages) & 1u, kWaitLimitNs);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kInt4MmaWeightWarps + kInt4MmaSumWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace fmms
