// Products with 4-bit weights for up to eight rows of x: out[b, v] = sum_k x[b, k] (q[v, k] - z[v, g(k)]) s[v, g(k)], g(k) = k / group.
//
// For a few rows of x the work is the stream of the weight: half a byte and 2 B flops per element.  The arithmetic per
// streamed byte is therefore kept small instead of the arithmetic per product:
//
//   Integers enter the tensor cores as they are stored.  A nibble in bits 4 to 7 of an fp16 number is the subnormal
//   q 2^-20, exact, so eight weights cost four ANDs and three shifts, with no conversion and no subtraction.  (Bits 0 to 3,
//   for one shift, would be exact too, but the tensor cores line products up by their exponent fields, which hide a
//   subnormal's leading zeros: rows with their codes there came out to 1e-6, against 1e-7 in bits 4 to 7.  Subtracting the
//   zero point first costs four fp16 operations more: 151936 x 4096 at one row took 68 us instead of 55.)  The stored order
//   puts the two nibbles of a byte into two different rows of the 16 x 16 operand.
//   The zero point leaves the product: sum_k x (q - z) = sum_k x q - z sum_k x.  The accumulators of a group start at
//   -z sum_k x (the sum over the group is formed once per CTA, in fp32, from the rounded x that the products use, so the
//   two parts cancel exactly), the scale is applied once per group in fp32, and groups add up in fp32.
//   x becomes fp16 after a power-of-two scaling per row that puts its largest element near 2^14: bf16 values down to 2^-28
//   of the row's maximum keep all their bits, smaller ones are rounded to 2^-39 of that maximum, which is below the
//   rounding of the fp32 sums.  fp16 goes in as it is.
//
// Work split.  Tiles of 16 rows are dealt to the CTAs, one per SM, in contiguous ranges; the warps of a CTA share its
// range in equal parts that begin and end anywhere in a pair of tiles (two at a time share the operand loads of x).  A
// warp's part is contiguous in memory and it streams it through a ring of asynchronous copies of its own: between the
// load of x and the end of the stream no warp waits for another.  A pair that several warps have a part of is joined at
// the end in the order of the columns: the first keeps its sums in registers, the others leave theirs in shared memory.
// (Bulk copies cost here: about 75 cycles of issue each from one producer warp, and with 32 to 1024 bytes to a copy
// there are four to six per 2 KiB; per-lane copies of 16 bytes need one instruction per 512.)
// x lies in shared memory in operand order.  Where it does not fit, the columns are taken in phases, and finished sums
// of a phase wait in global memory for the thread that wrote them.
// No atomics, one order of additions: results do not depend on timing, nor a row on the rest of its batch.
#pragma once

#include <cuda_fp16.h>

#include "fmms_common.cuh"

namespace fmms {

constexpr int kInt4Tile = 16;    // weight rows of a tile
constexpr int kInt4Chunk = 64;   // columns of a chunk: 512 bytes of a tile
constexpr int kInt4Rows = 8;     // rows of x, at most (more: fmms_int4_mma.cuh)
constexpr int kInt4Warps = 16;
constexpr int kInt4Stages = 3;   // units in a warp's ring (4 measured worse)
constexpr int kInt4Unit = 128;   // columns a warp fetches at a time; larger groups apply their scale to several units
__host__ __device__ constexpr int int4_unit_groups(int group) { return group < kInt4Unit ? kInt4Unit / group : 1; }
__host__ __device__ constexpr int int4_stage_bytes(int group) { return 2 * (2 * 512 + int4_unit_groups(group) * 48); }

struct Int4Params {
  const void* x;
  long long x_stride;          // elements between rows of x
  const uint8_t* q;            // [tiles][chunks][512]
  const uint16_t* scales;      // [tiles][groups][8][2] bf16 or fp16
  const uint8_t* zeros;        // [tiles][groups][8][2], or null: 8
  void* out;
  long long out_stride;        // elements between rows of out
  float* partial;              // [tiles][128], several phases only
  int V, D, B;
  int tiles, chunks, groups;
  int x_bf16, s_bf16, out_kind;  // out_kind: 0 bf16, 1 fp16, 2 fp32
  int x_pairs;                 // rows of x start on 4-byte boundaries
  int log_rows;                // rows of x in a pass, rounded up to a power of two
  int group_units;             // units of a group (1 for groups of up to 128 columns)
  int phases, units, all_units;  // units of a phase (the last one may have fewer) and of a row
  int xs_off, xs32_off, ring_off, piece_off;  // shared memory
};

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}

// c = A B + c0 for a 16 x 16 A and a 16 x 8 B
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// two fp32 additions, and two multiplications by s with additions, in one instruction each
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
  const float2 r = __fadd2_rn(make_float2(x, y), make_float2(a, b));
  x = r.x;
  y = r.y;
}
__device__ __forceinline__ void fma2(float& x, float& y, float s, float a, float b) {
  const float2 r = __ffma2_rn(make_float2(s, s), make_float2(a, b), make_float2(x, y));
  x = r.x;
  y = r.y;
}

__device__ __forceinline__ float half_bits_to_float(uint32_t bits16, bool bf16) {
  return bf16 ? __uint_as_float(bits16 << 16) : __half2float(__ushort_as_half((unsigned short)bits16));
}

// Columns k, k + 1 and the three pairs 8, 16 and 24 columns on, of a row of x (k is even).
__device__ __forceinline__ uint4 int4_load_x(const Int4Params& p, int b, int k) {
  const uint16_t* src = reinterpret_cast<const uint16_t*>(p.x) + (size_t)b * p.x_stride + k;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = p.x_pairs ? *reinterpret_cast<const uint32_t*>(src + 8 * i) : (uint32_t)src[8 * i] | ((uint32_t)src[8 * i + 1] << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void int4_store(const Int4Params& p, int b, int v, float y) {
  const size_t at = (size_t)b * p.out_stride + v;
  if (p.out_kind == 0)
    reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
  else if (p.out_kind == 1)
    reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(y);
  else
    reinterpret_cast<float*>(p.out)[at] = y;
}

// GR: columns of a group, at most 128; ZP: zero points given.
template <int GR, bool ZP>
__global__ void __launch_bounds__(kInt4Warps * 32, 1) int4_linear_kernel(const Int4Params p) {
  extern __shared__ __align__(128) uint8_t smem_parts[];
  constexpr int kChunks = kInt4Unit / kInt4Chunk, kGroups = int4_unit_groups(GR);  // of a unit
  constexpr int kStage = int4_stage_bytes(GR), S = kInt4Stages;
  constexpr int kScaleOff = 2 * kChunks * 512, kZeroOff = kScaleOff + 2 * kGroups * 32;
  constexpr int kScaleCopy = kGroups == 4 ? 8 : 4;                    // bytes a lane copies of the scales
  constexpr int kScaleLanes = kGroups * 32 / kScaleCopy;              // lanes of one tile
  constexpr int kZeroLanes = kGroups * 4;
  __shared__ unsigned int warp_max[kInt4Warps * kInt4Rows];
  __shared__ int row_exp[kInt4Rows];  // x went in times two to this
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int nb = p.B;

  uint4* xfrag = reinterpret_cast<uint4*>(smem_parts);
  float* xs = reinterpret_cast<float*>(smem_parts + p.xs_off);      // [groups of a phase][kInt4Rows]
  float* xs32 = reinterpret_cast<float*>(smem_parts + p.xs32_off);  // the same for 32 columns each (groups of 32: xs)
  float* pieces = reinterpret_cast<float*>(smem_parts + p.piece_off);  // [warps][8][32]
  const uint8_t* ring = smem_parts + p.ring_off + warp * (S * kStage);
  const uint32_t ring_at = smem_u32(ring);

  // x: a thread has one row and one t, and 8 of every 32 columns: the 16 bytes of one lane's operands.  The first loads go
  // out before anything else, the ring's behind them.
  const int stride = (kInt4Warps * 8) >> p.log_rows, first_block = (tid >> 2) >> p.log_rows;
  const int row = (tid >> 2) & ((1 << p.log_rows) - 1);
  constexpr int kAhead = 4;  // loads in flight
  uint4 raw[kAhead];
  auto load_blocks = [&](int k_begin, int blocks, int from) {  // blocks of 32 columns; zero from p.D on
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int blk = from + i * stride;
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row < nb && blk < blocks && k_begin + blk * 32 < p.D) raw[i] = int4_load_x(p, row, k_begin + blk * 32 + t * 2);
    }
  };
  load_blocks(0, p.units * (kInt4Unit / 32), first_block);

  // this CTA's tiles in pairs, and the warps' parts of them; position = pair * units + unit
  const int t_each = p.tiles / (int)gridDim.x, t_rest = p.tiles - t_each * (int)gridDim.x;
  const int t_begin = t_each * (int)blockIdx.x + min((int)blockIdx.x, t_rest), t_end = t_begin + t_each + ((int)blockIdx.x < t_rest);
  const int span = (t_end - t_begin + 1) / 2 * p.units, s_each = span / kInt4Warps, s_rest = span - s_each * kInt4Warps;
  auto part = [&](int w) { return s_each * w + min(w, s_rest); };
  const int begin = part(warp), end = part(warp + 1);
  const int p_first = begin / p.units, p_last = (end - 1) / p.units;
  // the units of pair `pr` in `phase` that belong to this warp: from lo to before hi
  auto unit_range = [&](int phase, int pr, int& lo, int& hi) {
    lo = max(begin - pr * p.units, 0);
    hi = min(min(end - pr * p.units, p.units), p.all_units - phase * p.units);
  };

  // the ring: one unit of both tiles of a pair at a time, one group of copies each (an empty one behind the end)
  int f_phase = 0, f_pr = p_first, f_unit = 0, f_left = 0, f_slot = 0, f_in_group = 0;
  const uint8_t *f_q = p.q, *f_s = nullptr, *f_z = nullptr;
  long long f_pitch = 0;
  auto seek = [&] {  // (f_phase, f_pr) or the next pair behind it that this warp has units of
    for (; f_phase < p.phases; ++f_phase, f_pr = p_first)
      for (; f_pr <= p_last; ++f_pr) {
        int lo, hi;
        unit_range(f_phase, f_pr, lo, hi);
        if (lo >= hi) continue;
        f_left = hi - lo;
        f_unit = f_phase * p.units + lo;
        const int tile = t_begin + f_pr * 2;
        const int two = tile + 1 < t_end ? 1 : 0;  // the range may end with a single tile: it is fetched twice
        f_pitch = two ? (long long)p.chunks * 512 : 0;
        f_q = p.q + ((long long)tile * p.chunks + f_unit * kChunks) * 512 + lane * 16;
        const int sm = lane / kScaleLanes, zm = lane / kZeroLanes;
        const int gr = GR < kInt4Unit ? f_unit * kGroups : f_unit / p.group_units;
        if (GR == kInt4Unit) f_in_group = f_unit - gr * p.group_units;
        f_s = reinterpret_cast<const uint8_t*>(p.scales) + ((long long)(tile + (sm & two)) * p.groups + gr) * 32 +
              (lane % kScaleLanes) * kScaleCopy;
        if constexpr (ZP)
          f_z = p.zeros + ((long long)(tile + (zm & two)) * p.groups + gr) * 16 + (lane % kZeroLanes) * 4;
        return;
      }
  };
  auto fetch = [&] {
    if (f_left > 0) {
      const uint32_t dst = ring_at + f_slot * kStage;
      // a row may end within its last unit: chunks and groups that are not there are not read
      const int chunks = GR < kInt4Unit ? p.chunks - f_unit * kChunks : kChunks;
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          if (c < chunks) copy_async<16>(dst + (m * kChunks + c) * 512 + lane * 16, f_q + (m ? f_pitch : 0) + c * 512);
      const int left = GR < kInt4Unit ? p.groups - f_unit * kGroups : kGroups;
      if (lane < 2 * kScaleLanes && (GR == kInt4Unit || (lane % kScaleLanes) * kScaleCopy < left * 32))
        copy_async<kScaleCopy>(dst + kScaleOff + lane * kScaleCopy, f_s);
      if constexpr (ZP)
        if (lane < 2 * kZeroLanes && (GR == kInt4Unit || (lane % kZeroLanes) * 4 < left * 16)) copy_async<4>(dst + kZeroOff + lane * 4, f_z);
      f_q += kChunks * 512;
      if (GR < kInt4Unit || ++f_in_group == p.group_units) {
        f_in_group = 0;
        f_s += kGroups * 32;
        if constexpr (ZP) f_z += kGroups * 16;
      }
      ++f_unit;
      if (++f_slot == S) f_slot = 0;
      if (--f_left == 0) {
        ++f_pr;
        seek();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (begin < end) seek();
#pragma unroll
  for (int i = 0; i < S - 1; ++i) fetch();

  auto pow2 = [](int e) { return __uint_as_float((uint32_t)(e + 127) << 23); };
  float tot[2][4];
  auto clear = [&] {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) tot[m][j] = 0.f;
  };
  auto write_out = [&](int pr) {
    const int tile = t_begin + pr * 2;
#pragma unroll
    for (int m = 0; m < 2; ++m)
      if (tile + m < t_end)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = t * 2 + (j & 1), v = (tile + m) * kInt4Tile + g + ((j & 2) ? 8 : 0);
          if (n < nb && v < p.V) int4_store(p, n, v, tot[m][j]);
        }
  };
  int slot = 0;

  for (int phase = 0; phase < p.phases; ++phase) {
    // x as it is into the places of its operands, with the maximum of each row on the way; then, each thread what it
    // wrote itself, in fp16, and the sums over the groups
    const int k_begin = phase * p.units * kInt4Unit, blocks = min(p.units, p.all_units - phase * p.units) * (kInt4Unit / 32);
    uint4* const mine = xfrag + row * 4 + t;
    if (phase > 0) {
      load_blocks(k_begin, blocks, first_block);
      __syncthreads();  // the phase before has been read
    }
    uint32_t m = 0u;  // magnitudes of bf16 compare like integers
#pragma unroll 1
    for (int from = first_block; from < blocks; from += kAhead * stride) {
      if (from != first_block) load_blocks(k_begin, blocks, from);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int blk = from + i * stride;
        if (row < nb && blk < blocks) mine[blk * 32] = raw[i];
        m = __vmaxu2(m, __vmaxu2(__vmaxu2(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu), __vmaxu2(raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu)));
      }
    }
    // the power of two that puts the row's maximum into [2^14, 2^15), clamped to what fp32 can hold; fp16 goes in as it is
    int exponent = 0;
    if (p.x_bf16) {
      m = max(m & 0xffffu, m >> 16);
#pragma unroll
      for (int off = 1; off < 32; off <<= 1)  // lanes of the same row
        if (off < 4 || off >= (4 << p.log_rows)) m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
      if (lane < (4 << p.log_rows) && t == 0) warp_max[warp * kInt4Rows + row] = m;
      __syncthreads();
      m = 0u;
#pragma unroll 4
      for (int w = 0; w < kInt4Warps; ++w) m = max(m, warp_max[w * kInt4Rows + row]);
      if (m != 0u) exponent = min(14 - ((int)(m >> 7) - 127), 120);
    }
    if (first_block == 0 && t == 0 && row < nb) row_exp[row] = exponent;
    const float up = pow2(exponent);
    constexpr int kConvert = 4;
#pragma unroll 1
    for (int from = first_block; from < blocks; from += kConvert * stride) {
      uint4 x4[kConvert];
      float s[kConvert];
#pragma unroll
      for (int i = 0; i < kConvert; ++i) {
        x4[i] = make_uint4(0u, 0u, 0u, 0u);
        if (row < nb && from + i * stride < blocks) x4[i] = mine[(from + i * stride) * 32];
      }
#pragma unroll
      for (int i = 0; i < kConvert; ++i) {
        uint32_t w[4] = {x4[i].x, x4[i].y, x4[i].z, x4[i].w};
        s[i] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (p.x_bf16) {
            const __half2 h = __floats2half2_rn(__uint_as_float(w[j] << 16) * up, __uint_as_float(w[j] & 0xffff0000u) * up);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
          }
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          s[i] += f.x + f.y;
        }
        x4[i] = make_uint4(w[0], w[1], w[2], w[3]);
        s[i] += __shfl_xor_sync(0xfu << (lane & 28), s[i], 1);  // the four lanes of a row and block run together
        s[i] += __shfl_xor_sync(0xfu << (lane & 28), s[i], 2);
      }
#pragma unroll
      for (int i = 0; i < kConvert; ++i) {
        const int blk = from + i * stride;
        if (row >= nb || blk >= blocks) continue;
        if (p.x_bf16) mine[blk * 32] = x4[i];
        // in units of the operands; without zero points times 8
        if (t == 0) (GR == 32 ? xs : xs32)[blk * kInt4Rows + row] = s[i] * (ZP ? -0x1p-20f : -0x1p-17f);
      }
    }
    __syncthreads();
    if constexpr (GR > 32) {
      for (int i = tid; i < blocks / (GR / 32) * kInt4Rows; i += kInt4Warps * 32) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < GR / 32; ++j) s += xs32[(i / kInt4Rows * (GR / 32) + j) * kInt4Rows + i % kInt4Rows];
        xs[i] = s;
      }
      __syncthreads();
    }

    clear();
    for (int pr = p_first; pr <= p_last && begin < end; ++pr) {
      int u, hi;
      unit_range(phase, pr, u, hi);
      if (u >= hi) continue;
      const uint4* xp = xfrag + u * (kChunks * 2 * 32) + lane;
      const float* xsp = xs + u * (kGroups * kInt4Rows) + t * 2;
      for (; u < hi; ++u) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        __syncwarp();  // scales and zeros were copied by other lanes; and everybody is done with the slot before this one
        fetch();
        const uint8_t* src = ring + slot * kStage;
        const uint4* qsrc = reinterpret_cast<const uint4*>(src) + lane;
        const uint32_t* ssrc = reinterpret_cast<const uint32_t*>(src + kScaleOff) + g;
        const uint16_t* zsrc = reinterpret_cast<const uint16_t*>(src + kZeroOff) + g;
        float acc[2][4];
#pragma unroll
        for (int cc = 0; cc < kChunks; ++cc) {
          uint32_t qw[2][4];
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const uint4 qv = qsrc[(m * kChunks + cc) * 32];
            qw[m][0] = qv.x;
            qw[m][1] = qv.y;
            qw[m][2] = qv.z;
            qw[m][3] = qv.w;
          }
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {  // 32 columns: two products
            constexpr int kPairs = GR / 32;  // of a group
            const int gi = (cc * 2 + jj) / kPairs;  // group within the unit
            const bool first = (cc * 2 + jj) % kPairs == 0, last = (cc * 2 + jj) % kPairs == kPairs - 1;
            const uint4 xv = xp[(cc * 2 + jj) * 32];
            // Two products to a chain, chains joined by rounded additions: the tensor cores cut sums off.  All first
            // products, then all second ones.
            float c[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int m = 0; m < 2; ++m) {
                const uint32_t w = qw[m][jj * 2 + h];
                const uint32_t a0 = (w << 4) & 0x00f000f0u, a1 = w & 0x00f000f0u, a2 = (w >> 4) & 0x00f000f0u, a3 = (w >> 8) & 0x00f000f0u;
                if (h == 0)
                  mma_16816(c[m], a0, a1, a2, a3, xv.x, xv.y, 0.f, 0.f, 0.f, 0.f);
                else
                  mma_16816(c[m], a0, a1, a2, a3, xv.z, xv.w, c[m][0], c[m][1], c[m][2], c[m][3]);
              }
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              if (first) {
                float z0 = 1.f, z1 = 1.f;
                if constexpr (ZP) {
                  const uint32_t z = zsrc[(m * kGroups + gi) * 8];
                  z0 = (float)(z & 0xffu);
                  z1 = (float)(z >> 8);
                }
                const float2 xsum = *reinterpret_cast<const float2*>(xsp + gi * kInt4Rows);
                acc[m][0] = c[m][0];
                acc[m][1] = c[m][1];
                acc[m][2] = c[m][2];
                acc[m][3] = c[m][3];
                fma2(acc[m][0], acc[m][1], z0, xsum.x, xsum.y);
                fma2(acc[m][2], acc[m][3], z1, xsum.x, xsum.y);
              } else {
                add2(acc[m][0], acc[m][1], c[m][0], c[m][1]);
                add2(acc[m][2], acc[m][3], c[m][2], c[m][3]);
              }
              if (last && (GR == kInt4Unit || (phase * p.units + u) * kGroups + gi < p.groups)) {
                const uint32_t s2 = ssrc[(m * kGroups + gi) * 8];
                const float s0 = half_bits_to_float(s2 & 0xffffu, p.s_bf16);
                const float s1 = half_bits_to_float(s2 >> 16, p.s_bf16);
                fma2(tot[m][0], tot[m][1], s0, acc[m][0], acc[m][1]);
                fma2(tot[m][2], tot[m][3], s1, acc[m][2], acc[m][3]);
              }
            }
          }
        }
        xp += kChunks * 2 * 32;
        xsp += kGroups * kInt4Rows;
        if (++slot == S) slot = 0;
      }
      // the warp's part of this pair in this phase is complete
      const bool has_start = begin <= pr * p.units, has_end = end >= (pr + 1) * p.units;
      // From the units of the sums to the result, by 2^(20 - exponent) in two halves: no step of it lies beyond both ends.
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e = t * 2 + i < nb ? 20 - row_exp[t * 2 + i] : 0;
        const float down0 = pow2(e >> 1), down1 = pow2(e - (e >> 1));
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          tot[m][i] = tot[m][i] * down0 * down1;
          tot[m][2 + i] = tot[m][2 + i] * down0 * down1;
        }
      }
      if (!has_start) {
        float* mine = pieces + warp * (2 * 128) + lane;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = tot[i / 4][i % 4];
          mine[i * 32] = phase ? mine[i * 32] + y : y;
        }
        clear();
        continue;
      }
      if (p.phases > 1) {  // what the phases before left
        float* mine = p.partial + ((size_t)t_begin + pr * 2) * 128 + lane;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (t_begin + pr * 2 + i / 4 >= t_end) continue;
          float& y = tot[i / 4][i % 4];
          if (phase) y += mine[i * 32];
          if (phase + 1 < p.phases) mine[i * 32] = y;
        }
      }
      // a pair that the next warps go on with is the part's last: at the end its sums stay where they are
      if (has_end && phase + 1 == p.phases) write_out(pr);
      if (has_end || phase + 1 < p.phases) clear();
    }
  }
  __syncthreads();
  if (begin < end) {
    const int pr = p_last, stop = (pr + 1) * p.units;
    if (begin <= pr * p.units && end < stop) {
#pragma unroll 4
      for (int w = warp + 1; w < kInt4Warps && part(w) < stop; ++w) {
        if (part(w) == part(w + 1)) continue;
        const float* other = pieces + w * (2 * 128) + lane;
#pragma unroll
        for (int i = 0; i < 8; ++i) tot[i / 4][i % 4] += other[i * 32];
      }
      write_out(pr);
    }
  }
}

}  // namespace fmms
