// Products with 4-bit weights: out[b, v] = sum_k x[b, k] (q[v, k] - z[v, g(k)]) s[v, g(k)], g(k) = k / group.
//
// For a few rows of x the work is the stream of the weight: half a byte and 2 B flops per element.  The arithmetic per
// streamed byte is therefore kept small instead of the arithmetic per product:
//
//   Integers enter the tensor cores as they are stored.  Masking a 32-bit word with 0x000f000f leaves two fp16
//   subnormals q 2^-24, masking it with 0x00f000f0 two subnormals q 2^-20: both exact, so eight weights cost four
//   ANDs and one shift, with no conversion and no subtraction.  The stored order puts the two nibbles of a byte into
//   two different rows of the 16 x 16 operand, so that the factor 2^4 between the masks belongs to a whole row and
//   joins that row's scale.
//   The zero point leaves the product: sum_k x (q - z) = sum_k x q - z sum_k x.  The accumulators of a group start at
//   -z sum_k x (the sum over the group is formed once per CTA, in fp32, from the rounded x that the products use, so the
//   two parts cancel exactly), the scale is applied once per group in fp32, and groups add up in fp32.
//   x becomes fp16 after a power-of-two scaling per row that puts its largest element near 2^14: bf16 and fp16 values
//   down to 2^-28 of the row's maximum keep all their bits, smaller ones are rounded to 2^-39 of that maximum, which is
//   below the rounding of the fp32 sums.
//
// Work split.  A tile is 16 weight rows over all columns, contiguous in memory.  A persistent CTA (or, for long rows
// and few tiles, a cluster of them) takes one tile at a time; its warps split the columns, so that the hidden states a
// warp multiplies with stay at fixed places of shared memory, laid out in operand order.  Every warp streams its own
// part of the tile through a private ring of bulk copies (one lane issues, the warp waits on the mbarrier; no other warp
// is involved until the tile's sums are joined through shared memory).  Clusters join their sums in the first CTA's
// shared memory.  No atomics, one order of additions: results do not depend on timing, nor a row on its batch.
#pragma once

#include <cuda_fp16.h>

#include "fmms_common.cuh"

namespace fmms {

constexpr int kInt4Tile = 16;        // weight rows of a tile
constexpr int kInt4Chunk = 64;       // columns of a chunk: 512 bytes of a tile
constexpr int kInt4StepChunks = 4;   // chunks a warp fetches at a time
constexpr int kInt4MaxWarps = 16;
constexpr int kInt4MaxStages = 8;

struct Int4Params {
  const void* x;
  long long x_stride;          // elements between rows of x
  const uint8_t* q;            // [tiles][chunks][512]
  const uint16_t* scales;      // [tiles][groups][8][2] bf16 or fp16
  const uint8_t* zeros;        // [tiles][groups][8][2], or null: 8
  void* out;
  long long out_stride;        // elements between rows of out
  int V, D, B;
  int tiles, chunks, groups;
  int x_bf16, s_bf16, out_kind;  // out_kind: 0 bf16, 1 fp16, 2 fp32
  int x_vec;                   // rows of x start on 16-byte boundaries
  int split;                   // CTAs of a cluster, each with its share of the columns
  int stages, stage_bytes;
  int xs_off, ring_off, red_off, join_off, bar_off;  // shared memory
  int* status_dev;
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t pol) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(pol)
      : "memory");
}

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float half_bits_to_float(uint32_t bits16, bool bf16) {
  return bf16 ? __uint_as_float(bits16 << 16) : __half2float(__ushort_as_half((unsigned short)bits16));
}

// Eight consecutive elements of a row of x as fp32 (k is a multiple of 8, the row length a multiple of 32).
__device__ __forceinline__ void int4_load_x8(const Int4Params& p, int b, int k, float (&v)[8]) {
  const uint16_t* src = reinterpret_cast<const uint16_t*>(p.x) + (size_t)b * p.x_stride + k;
  uint32_t w[4];
  if (p.x_vec) {
    const uint4 u = *reinterpret_cast<const uint4*>(src);
    w[0] = u.x;
    w[1] = u.y;
    w[2] = u.z;
    w[3] = u.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)src[2 * i] | ((uint32_t)src[2 * i + 1] << 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = half_bits_to_float(w[i] & 0xffffu, p.x_bf16);
    v[2 * i + 1] = half_bits_to_float(w[i] >> 16, p.x_bf16);
  }
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

// NT: blocks of eight rows of x; GR: columns of a group; ZP: zero points given.
template <int NT, int GR, bool ZP>
__global__ void __launch_bounds__(kInt4MaxWarps * 32, 1) int4_linear_kernel(const Int4Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kGran = GR > kInt4Chunk ? GR / kInt4Chunk : 1;   // chunks of a group
  constexpr int kSteps = GR / 16;                                // products of a group
  constexpr int kPerChunk = GR < kInt4Chunk ? kInt4Chunk / GR : 1;  // groups of a chunk
  constexpr int kOut = NT * 128;                                 // values of a tile
  __shared__ unsigned int row_max[NT * 8];
  __shared__ int abort_word;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, W = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int rank = (int)blockIdx.x % p.split, first_tile = (int)blockIdx.x / p.split, tile_step = (int)gridDim.x / p.split;
  const int b0 = blockIdx.y * NT * 8, nb = min(NT * 8, p.B - b0);

  uint4* xfrag = reinterpret_cast<uint4*>(smem);
  float* xs = reinterpret_cast<float*>(smem + p.xs_off);
  uint8_t* ring = smem + p.ring_off + (size_t)warp * p.stages * p.stage_bytes;
  float* red = reinterpret_cast<float*>(smem + p.red_off);
  float* join = reinterpret_cast<float*>(smem + p.join_off);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + p.bar_off) + warp * p.stages;
  volatile int* abort_flag = &abort_word;

  // columns of this CTA and of this warp, in units of whole groups (whole chunks for groups below 64)
  const int units = p.chunks / kGran;
  const int u_cta = (int)((long long)units * rank / p.split), u_end = (int)((long long)units * (rank + 1) / p.split);
  const int c_cta = u_cta * kGran, cta_units = u_end - u_cta;
  const int c_begin = (u_cta + cta_units * warp / W) * kGran, c_end = (u_cta + cta_units * (warp + 1) / W) * kGran;
  const int nsteps = (c_end - c_begin + kInt4StepChunks - 1) / kInt4StepChunks;

  if (lane == 0)
    for (int i = 0; i < p.stages; ++i) mbar_init(&full[i], 1);
  if (tid == 0) abort_word = 0;
  for (int i = tid; i < NT * 8; i += blockDim.x) row_max[i] = 0u;
  fence_mbar_init();
  __syncthreads();
  if (p.split > 1) {  // every CTA of the cluster runs before one of them writes into the first one's shared memory
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }

  // the ring: the warp's steps of all its tiles, one after the other
  int issue_tile = first_tile, issue_step = 0, issued = 0;
  const uint64_t pol = policy_evict_first();
  auto issue = [&](int slot) {
    if (issue_tile >= p.tiles || nsteps == 0) return;
    const int c = c_begin + issue_step * kInt4StepChunks, n = min(kInt4StepChunks, c_end - c);
    const int gr = c * kPerChunk / kGran;
    const int ng = min(max(n / kGran, 1) * kPerChunk, p.groups - gr);
    uint8_t* dst = ring + (size_t)slot * p.stage_bytes;
    const uint32_t qb = n * 512, sb = ng * 32, zb = ZP ? ng * 16 : 0;
    mbar_arrive_expect_tx(&full[slot], qb + sb + zb);
    bulk_load(dst, p.q + ((size_t)issue_tile * p.chunks + c) * 512, qb, &full[slot], pol);
    constexpr int kMaxGroups = kInt4StepChunks * kPerChunk / kGran;
    bulk_load(dst + kInt4StepChunks * 512, p.scales + ((size_t)issue_tile * p.groups + gr) * 16, sb, &full[slot], pol);
    if constexpr (ZP)
      bulk_load(dst + kInt4StepChunks * 512 + kMaxGroups * 32, p.zeros + ((size_t)issue_tile * p.groups + gr) * 16, zb,
                &full[slot], pol);
    ++issued;
    if (++issue_step == nsteps) {
      issue_step = 0;
      issue_tile += tile_step;
    }
  };
  if (lane == 0)
    for (int i = 0; i < p.stages; ++i) issue(i);

  // x: maximum of each row, then fp16 operands in the order the products read them, and the sums over the groups
  const int k_begin = c_cta * kInt4Chunk, k_end = min(p.D, (u_end * kGran) * kInt4Chunk);
  const int segs = (k_end - k_begin + 255) / 256;
  for (int u = warp; u < nb * segs; u += W) {
    const int b = u / segs, k = k_begin + (u - b * segs) * 256 + lane * 8;
    unsigned int m = 0u;
    if (k < k_end) {
      float v[8];
      int4_load_x8(p, b0 + b, k, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) atomicMax(&row_max[b], m);
  }
  __syncthreads();
  // exponent of the power of two that puts the row's maximum into [2^14, 2^15); clamped to what fp32 can hold
  auto row_exponent = [&](int b) {
    const int e = (int)(row_max[b] >> 23) - 127;
    return row_max[b] == 0u ? 0 : min(14 - e, 120);
  };
  auto pow2 = [](int e) { return __uint_as_float((uint32_t)(e + 127) << 23); };
  for (int u = warp; u < nb * segs; u += W) {
    const int b = u / segs, k = k_begin + (u - b * segs) * 256 + lane * 8;
    float s = 0.f;
    if (k < k_end) {
      const float up = pow2(row_exponent(b));
      float v[8];
      int4_load_x8(p, b0 + b, k, v);
      const int c = (k - k_begin) / kInt4Chunk, step = (k & 63) >> 4, half = (k & 15) >> 3;
      uint32_t* dst = reinterpret_cast<uint32_t*>(xfrag + ((c * 2 + (step >> 1)) * NT + (b >> 3)) * 32 + (b & 7) * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i] * up, v[2 * i + 1] * up);
        dst[i * 4 + (step & 1) * 2 + half] = *reinterpret_cast<const uint32_t*>(&h);
        s += __low2float(h) + __high2float(h);
      }
    }
#pragma unroll
    for (int off = 1; off < GR / 8; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (k < k_end && (lane & (GR / 8 - 1)) == 0)
      xs[((k - k_begin) / GR) * (NT * 8) + b] = s * (ZP ? -0x1p-24f : -0x1p-21f);  // in units of the operands; times 8
  }
  __syncthreads();

  const int gr_cta = c_cta * kPerChunk / kGran;  // first group of the CTA
  int slot = 0, parity = 0, buf = 0, consumed = 0;
  int joined_tile = -1;  // clusters: the tile whose sums are on their way to the first CTA

  auto finish_join = [&](int tile, int jbuf) {  // first CTA of a cluster: add the shares in rank order, write the tile
    for (int j = tid; j < kOut; j += blockDim.x) {
      float y = 0.f;
      for (int r = 0; r < p.split; ++r) y += join[(jbuf * p.split + r) * kOut + j];
      const int i = j >> 5, l = j & 31;
      const int n = (i >> 2) * 8 + (l & 3) * 2 + (i & 1), v = tile * kInt4Tile + (l >> 2) + ((i & 2) ? 8 : 0);
      if (n < nb && v < p.V) int4_store(p, b0 + n, v, y);
    }
  };

  for (int tile = first_tile; tile < p.tiles; tile += tile_step) {
    float tot[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) tot[i][j] = 0.f;
    for (int st = 0; st < nsteps; ++st) {
      mbar_wait(&full[slot], (uint32_t)parity, abort_flag, p.status_dev);
      const int c = c_begin + st * kInt4StepChunks, n = min(kInt4StepChunks, c_end - c);
      const uint8_t* src = ring + (size_t)slot * p.stage_bytes;
      const uint4* qsrc = reinterpret_cast<const uint4*>(src) + lane;
      const uint32_t* ssrc = reinterpret_cast<const uint32_t*>(src + kInt4StepChunks * 512) + g;
      const uint16_t* zsrc = reinterpret_cast<const uint16_t*>(src + kInt4StepChunks * 512 + kInt4StepChunks * kPerChunk / kGran * 32) + g;
      const int gr0 = c * kPerChunk / kGran;
      for (int cu = 0; cu < n; cu += kGran) {
        float acc[NT][4];
#pragma unroll
        for (int cc = 0; cc < kGran; ++cc) {
          const uint4 qv = qsrc[(cu + cc) * 32];
          const uint32_t qw[4] = {qv.x, qv.y, qv.z, qv.w};
          uint4 xv[NT];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int step = cc * 4 + j;               // product within the unit
            const int gi = cu * kPerChunk / kGran + step / kSteps;  // group within the fetched step
            if (step % kSteps == 0) {
              float z0 = 1.f, z1 = 16.f;
              if constexpr (ZP) {
                const uint32_t z = zsrc[gi * 8];
                z0 = (float)(z & 0xffu);
                z1 = (float)(z >> 8) * 16.f;
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const float2 xsum = *reinterpret_cast<const float2*>(xs + (gr0 + gi - gr_cta) * (NT * 8) + nt * 8 + t * 2);
                acc[nt][0] = z0 * xsum.x;
                acc[nt][1] = z0 * xsum.y;
                acc[nt][2] = z1 * xsum.x;
                acc[nt][3] = z1 * xsum.y;
              }
            }
            const uint32_t w = qw[j], w8 = w >> 8;
            const uint32_t a0 = w & 0x000f000fu, a1 = w & 0x00f000f0u, a2 = w8 & 0x000f000fu, a3 = w8 & 0x00f000f0u;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if ((j & 1) == 0) xv[nt] = xfrag[(((c - c_cta + cu + cc) * 2 + (j >> 1)) * NT + nt) * 32 + lane];
              if ((j & 1) == 0)
                mma_16816(acc[nt], a0, a1, a2, a3, xv[nt].x, xv[nt].y);
              else
                mma_16816(acc[nt], a0, a1, a2, a3, xv[nt].z, xv[nt].w);
            }
            if ((step + 1) % kSteps == 0 && (GR > 32 || gr0 + gi < p.groups)) {
              const uint32_t s2 = ssrc[gi * 8];
              const float s0 = half_bits_to_float(s2 & 0xffffu, p.s_bf16), s1 = half_bits_to_float(s2 >> 16, p.s_bf16) * 0.0625f;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                tot[nt][0] = fmaf(s0, acc[nt][0], tot[nt][0]);
                tot[nt][1] = fmaf(s0, acc[nt][1], tot[nt][1]);
                tot[nt][2] = fmaf(s1, acc[nt][2], tot[nt][2]);
                tot[nt][3] = fmaf(s1, acc[nt][3], tot[nt][3]);
              }
            }
          }
        }
      }
      __syncwarp();
      ++consumed;
      if (lane == 0) issue(slot);
      if (++slot == p.stages) {
        slot = 0;
        parity ^= 1;
      }
    }
    // the warps' sums of the tile; two buffers, so that one barrier per tile is enough
    float* mine = red + (size_t)buf * W * kOut + warp * kOut;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) mine[(nt * 4 + j) * 32 + lane] = tot[nt][j];
    __syncthreads();
    if (p.split > 1 && joined_tile >= 0) {
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      if (rank == 0) finish_join(joined_tile, buf ^ 1);
    }
    for (int j = tid; j < kOut; j += blockDim.x) {
      float y = 0.f;
      for (int w = 0; w < W; ++w) y += red[(size_t)(buf * W + w) * kOut + j];
      const int i = j >> 5, l = j & 31;
      const int n = (i >> 2) * 8 + (l & 3) * 2 + (i & 1), v = tile * kInt4Tile + (l >> 2) + ((i & 2) ? 8 : 0);
      if (n < nb) y = (y * 0x1p24f) * pow2(-row_exponent(n));
      if (p.split == 1) {
        if (n < nb && v < p.V) int4_store(p, b0 + n, v, y);
      } else {
        uint32_t dst;
        asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(dst) : "r"(smem_u32(join + (buf * p.split + rank) * kOut + j)));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(y) : "memory");
      }
    }
    if (p.split > 1) {
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      joined_tile = tile;
    }
    buf ^= 1;
  }
  if (p.split > 1 && joined_tile >= 0) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0) finish_join(joined_tile, buf ^ 1);
  }
  if (*abort_flag && lane == 0) {
    // a wait ran out: give copies still in flight a bounded chance to land before the CTA's memory is reused
    for (int i = 0; i < min(issued, p.stages); ++i) {
      const int last = ((issued - 1 - i) / p.stages) * p.stages + i;
      mbar_wait_plain(&full[i], (uint32_t)(last / p.stages) & 1u, 100000000ull);
    }
  }
}

}  // namespace fmms
