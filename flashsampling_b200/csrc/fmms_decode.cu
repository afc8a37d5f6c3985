// C ABI of the operators around a decode step (see include/fmms_b200.h): products with 4-bit weights, the beam-search
// step and the reordering of per-beam states.  Argument checks, launch plans and launches; no allocation, no
// synchronisation, no exceptions.
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/fmms_b200.h"
#include "fmms_beam.cuh"
#include "fmms_common.cuh"
#include "fmms_int4.cuh"
#include "fmms_reorder.cuh"

namespace fmms {

constexpr int kDecodeMaxDevices = 16;
constexpr int kInt4SmemLimit = 230000;  // of 232448 bytes a CTA may have; the rest: static shared memory

static int decode_num_sms(int* dev_out, int* sms_out) {
  static std::atomic<int> sms[kDecodeMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return kErrCuda;
  if (dev < 0 || dev >= kDecodeMaxDevices) return kErrUnsupported;
  int n = sms[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    int major = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess) return kErrCuda;
    if (major != 10) return kErrArch;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return kErrCuda;
    sms[dev].store(n, std::memory_order_relaxed);
  }
  *dev_out = dev;
  *sms_out = n;
  return kOk;
}

// ---- products with 4-bit weights ----------------------------------------------------------------
struct Int4Plan {
  int nt, split, warps, stages, stage_bytes, smem;
  int xs_off, ring_off, red_off, join_off, bar_off;
};

static int int4_smem(Int4Plan& pl, int cta_chunks, int group) {
  const int gran = group > 64 ? group / 64 : 1, per_chunk = group < 64 ? 64 / group : 1;
  pl.stage_bytes = kInt4StepChunks * 512 + kInt4StepChunks * per_chunk / gran * 48;
  int off = cta_chunks * pl.nt * 1024;
  pl.xs_off = off;
  off += (cta_chunks * per_chunk / gran * pl.nt * 32 + 127) / 128 * 128;
  pl.ring_off = off;
  off += pl.warps * pl.stages * pl.stage_bytes;
  pl.red_off = off;
  off += 2 * pl.warps * pl.nt * 512;
  pl.join_off = off;
  if (pl.split > 1) off += 2 * pl.split * pl.nt * 512;
  pl.bar_off = off;
  off += pl.warps * pl.stages * 8;
  pl.smem = off;
  return off;
}

// Blocks of eight rows of x per pass: all of x where shared memory holds it (a cluster of up to eight CTAs splits the
// columns between them), else as many as fit.
static bool int4_plan(Int4Plan& pl, int V, int D, int B, int group, int num_sms) {
  const int gran = group > 64 ? group / 64 : 1;
  const int chunks = (D + kInt4Chunk - 1) / kInt4Chunk, units = chunks / gran, tiles = (V + kInt4Tile - 1) / kInt4Tile;
  for (pl.nt = B <= 8 ? 1 : B <= 16 ? 2 : 4; pl.nt >= 1; pl.nt >>= 1) {
    pl.warps = pl.nt == 4 ? 8 : kInt4MaxWarps;
    for (pl.split = 1; pl.split <= 8 && pl.split <= units; pl.split *= 2) {
      const int cta_chunks = (units + pl.split - 1) / pl.split * gran;
      // few tiles: also split while that gives idle SMs work and every warp keeps a fetch of its own
      if (pl.split < 8 && tiles * pl.split * 2 <= num_sms && cta_chunks >= 2 * pl.warps * kInt4StepChunks) continue;
      for (pl.stages = kInt4MaxStages; pl.stages >= 2; --pl.stages)
        if (int4_smem(pl, cta_chunks, group) <= kInt4SmemLimit) return true;
    }
  }
  return false;
}

template <int NT, int GR, bool ZP>
static int int4_launch(const Int4Params& p, const Int4Plan& pl, int dev, int num_sms, cudaStream_t stream) {
  auto* kernel = int4_linear_kernel<NT, GR, ZP>;
  static std::atomic<bool> ready[kDecodeMaxDevices];
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kInt4SmemLimit) != cudaSuccess) {
      cudaGetLastError();
      return kErrCuda;
    }
    ready[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(min(p.tiles, num_sms / pl.split) * pl.split), (unsigned)((p.B + NT * 8 - 1) / (NT * 8)));
  cfg.blockDim = dim3((unsigned)pl.warps * 32);
  cfg.dynamicSmemBytes = (size_t)pl.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (pl.split > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)pl.split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) {
    cudaGetLastError();
    return kErrCuda;
  }
  return kOk;
}

template <int NT, bool ZP>
static int int4_launch_group(const Int4Params& p, const Int4Plan& pl, int group, int dev, int num_sms, cudaStream_t stream) {
  switch (group) {
    case 32: return int4_launch<NT, 32, ZP>(p, pl, dev, num_sms, stream);
    case 64: return int4_launch<NT, 64, ZP>(p, pl, dev, num_sms, stream);
    case 128: return int4_launch<NT, 128, ZP>(p, pl, dev, num_sms, stream);
    default: return int4_launch<NT, 256, ZP>(p, pl, dev, num_sms, stream);
  }
}

template <bool ZP>
static int int4_launch_rows(const Int4Params& p, const Int4Plan& pl, int group, int dev, int num_sms, cudaStream_t stream) {
  switch (pl.nt) {
    case 1: return int4_launch_group<1, ZP>(p, pl, group, dev, num_sms, stream);
    case 2: return int4_launch_group<2, ZP>(p, pl, group, dev, num_sms, stream);
    default: return int4_launch_group<4, ZP>(p, pl, group, dev, num_sms, stream);
  }
}

// ---- beam step ----------------------------------------------------------------------------------
static int beam_element_bytes(int dtype) { return dtype == FMMS_F32 ? 4 : 2; }

static int beam_splits(int V, int dtype) {
  const int es = beam_element_bytes(dtype), tile = kBeamThreads * kBeamVecs * (16 / es);
  return (V + 16 / es - 1 + tile - 1) / tile;  // a row may start anywhere within 16 bytes
}

static size_t beam_workspace(int R, int K, int V, int N, int dtype) {
  const size_t parts = (size_t)R * K * beam_splits(V, dtype);
  return parts * N * 8 + parts * 8 + parts * 4;
}

template <typename... KArgs, typename... Args>
static int launch_behind(void (*kernel)(KArgs...), dim3 grid, int threads, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return kErrCuda;
  }
  return kOk;
}

}  // namespace fmms

using namespace fmms;

extern "C" {

int fmms_int4_linear(const void* x, int x_dtype, long long x_stride, const void* qweight, const void* scales, int scale_dtype,
                     const void* zeros, int V, int D, int group, int B, void* out, int out_dtype, long long out_stride,
                     int* status_dev, void* stream) {
  if (!x || !qweight || !scales || !out || V <= 0 || D <= 0 || B <= 0) return FMMS_ERR_BAD_ARG;
  if ((x_dtype != FMMS_BF16 && x_dtype != FMMS_F16) || (scale_dtype != FMMS_BF16 && scale_dtype != FMMS_F16) ||
      out_dtype < FMMS_BF16 || out_dtype > FMMS_F32)
    return FMMS_ERR_BAD_ARG;
  if (x_stride < D || out_stride < V) return FMMS_ERR_BAD_ARG;
  if ((group != 32 && group != 64 && group != 128 && group != 256) || D % group != 0) return FMMS_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(qweight) | reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(zeros)) & 15)
    return FMMS_ERR_UNSUPPORTED;
  int dev = 0, num_sms = 0;
  const int rc = decode_num_sms(&dev, &num_sms);
  if (rc != kOk) return rc;
  Int4Plan pl;
  if (!int4_plan(pl, V, D, B, group, num_sms)) return FMMS_ERR_UNSUPPORTED;
  Int4Params p = {};
  p.x = x;
  p.x_stride = x_stride;
  p.q = reinterpret_cast<const uint8_t*>(qweight);
  p.scales = reinterpret_cast<const uint16_t*>(scales);
  p.zeros = reinterpret_cast<const uint8_t*>(zeros);
  p.out = out;
  p.out_stride = out_stride;
  p.V = V;
  p.D = D;
  p.B = B;
  p.tiles = (V + kInt4Tile - 1) / kInt4Tile;
  p.chunks = (D + kInt4Chunk - 1) / kInt4Chunk;
  p.groups = D / group;
  p.x_bf16 = x_dtype == FMMS_BF16;
  p.s_bf16 = scale_dtype == FMMS_BF16;
  p.out_kind = out_dtype - FMMS_BF16;
  p.x_vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && x_stride % 8 == 0;
  p.split = pl.split;
  p.stages = pl.stages;
  p.stage_bytes = pl.stage_bytes;
  p.xs_off = pl.xs_off;
  p.ring_off = pl.ring_off;
  p.red_off = pl.red_off;
  p.join_off = pl.join_off;
  p.bar_off = pl.bar_off;
  p.status_dev = status_dev;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return zeros ? int4_launch_rows<true>(p, pl, group, dev, num_sms, s) : int4_launch_rows<false>(p, pl, group, dev, num_sms, s);
}

int fmms_query_beam_workspace(int R, int K, int V, int N, int dtype, size_t* bytes) {
  if (!bytes || R <= 0 || K <= 0 || V <= 0 || N <= 0 || dtype < FMMS_BF16 || dtype > FMMS_F32) return FMMS_ERR_BAD_ARG;
  if (N > kBeamMaxN || K > kBeamMaxK) return FMMS_ERR_UNSUPPORTED;
  *bytes = beam_workspace(R, K, V, N, dtype);
  return FMMS_OK;
}

int fmms_beam_step(const void* logits, int dtype, long long stride_r, long long stride_k, const float* scores,
                   const unsigned char* finished, long long pad_token, int R, int K, int V, int N, float* out_scores,
                   long long* out_tokens, long long* out_parents, void* workspace, size_t workspace_bytes, void* stream) {
  if (!logits || !scores || !out_scores || !out_tokens || !out_parents) return FMMS_ERR_BAD_ARG;
  if (R <= 0 || K <= 0 || V <= 0 || N <= 0 || dtype < FMMS_BF16 || dtype > FMMS_F32) return FMMS_ERR_BAD_ARG;
  if (pad_token < 0 || pad_token >= V || N > (long long)K * V) return FMMS_ERR_BAD_ARG;
  if (reinterpret_cast<uintptr_t>(logits) % beam_element_bytes(dtype)) return FMMS_ERR_BAD_ARG;
  if (N > kBeamMaxN || K > kBeamMaxK || (long long)K * V >= (1ll << 31) || (long long)R * K > 65535) return FMMS_ERR_UNSUPPORTED;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < beam_workspace(R, K, V, N, dtype))
    return FMMS_ERR_WORKSPACE;
  int dev = 0, num_sms = 0;
  const int rc = decode_num_sms(&dev, &num_sms);
  if (rc != kOk) return rc;
  BeamParams p = {};
  p.logits = logits;
  p.stride_r = stride_r;
  p.stride_k = stride_k;
  p.scores = scores;
  p.finished = finished;
  p.R = R;
  p.K = K;
  p.V = V;
  p.N = N;
  p.splits = beam_splits(V, dtype);
  p.pad_token = pad_token;
  const size_t parts = (size_t)R * K * p.splits;
  p.keys = reinterpret_cast<unsigned long long*>(workspace);
  p.sums = reinterpret_cast<double*>(p.keys + parts * N);
  p.maxima = reinterpret_cast<float*>(p.sums + parts);
  p.out_scores = out_scores;
  p.out_tokens = out_tokens;
  p.out_parents = out_parents;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)p.splits, (unsigned)(R * K));
  if (dtype == FMMS_BF16)
    beam_part_kernel<__nv_bfloat16><<<grid, kBeamThreads, 0, s>>>(p);
  else if (dtype == FMMS_F16)
    beam_part_kernel<__half><<<grid, kBeamThreads, 0, s>>>(p);
  else
    beam_part_kernel<float><<<grid, kBeamThreads, 0, s>>>(p);
  if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  return launch_behind(beam_merge_kernel, dim3((unsigned)R), kBeamThreads, s, p);
}

int fmms_reorder_beams(const fmms_beam_state_t* states, int n_states, const void* parents, int parents_bytes, int R, int K,
                       const int* lengths, void* stream) {
  if (!states || n_states <= 0 || !parents || R <= 0 || K <= 0 || (parents_bytes != 4 && parents_bytes != 8)) return FMMS_ERR_BAD_ARG;
  if (K > kReorderMaxBeams) return FMMS_ERR_UNSUPPORTED;
  for (int i = 0; i < n_states; ++i) {
    const fmms_beam_state_t& s = states[i];
    if (!s.data || s.outer[0] <= 0 || s.outer[1] <= 0 || s.seg_bytes <= 0 || s.step_bytes < 0) return FMMS_ERR_BAD_ARG;
    if (s.step_bytes && s.seg_bytes % s.step_bytes) return FMMS_ERR_BAD_ARG;
  }
  int dev = 0, num_sms = 0;
  const int rc = decode_num_sms(&dev, &num_sms);
  if (rc != kOk) return rc;
  if (K == 1) return FMMS_OK;  // one beam: its own parent
  cudaStream_t stm = reinterpret_cast<cudaStream_t>(stream);
  for (int r0 = 0; r0 < R; r0 += kReorderMaxRequests) {
    for (int i0 = 0; i0 < n_states; i0 += kReorderMaxStates) {
      const int n = min(kReorderMaxStates, n_states - i0), nr = min(kReorderMaxRequests, R - r0);
      ReorderParams p;
      p.parents = reinterpret_cast<const uint8_t*>(parents) + (size_t)r0 * K * parents_bytes;
      p.parents_wide = parents_bytes == 8;
      p.lengths = lengths ? lengths + r0 : nullptr;
      p.R = nr;
      p.K = K;
      long long most = 1;  // units of the largest tensor
      const int U = K <= 4 ? 4 : K <= 8 ? 2 : 1;
      for (int i = 0; i < n; ++i) {
        const fmms_beam_state_t& s = states[i0 + i];
        ReorderState& d = p.st[i];
        d.data = reinterpret_cast<uint8_t*>(s.data) + (long long)r0 * K * s.beam_stride;
        d.beam_stride = s.beam_stride;
        d.outer_stride[0] = s.outer_stride[0];
        d.outer_stride[1] = s.outer_stride[1];
        d.outer[0] = s.outer[0];
        d.outer[1] = s.outer[1];
        d.seg_bytes = s.seg_bytes;
        d.step_bytes = s.step_bytes;
        unsigned long long bits = reinterpret_cast<uintptr_t>(s.data) | (unsigned long long)s.beam_stride |
                                  (unsigned long long)s.seg_bytes | (unsigned long long)s.step_bytes;
        for (int o = 0; o < 2; ++o)
          if (s.outer[o] > 1) bits |= (unsigned long long)s.outer_stride[o];
        int vec = K > 32 ? 8 : 16;
        while (bits & (unsigned long long)(vec - 1)) vec >>= 1;
        d.vec = vec;
        const long long cols = s.seg_bytes / vec, unit = kReorderThreads * U, outers = (long long)s.outer[0] * s.outer[1];
        if (nr * ((cols + unit - 1) / unit) >= (1ll << 31)) return FMMS_ERR_UNSUPPORTED;
        const long long units = cols >= unit / 2 ? outers * nr * ((cols + unit - 1) / unit) : (outers * nr * cols + unit - 1) / unit;
        if (units > most) most = units;
      }
      // CTAs: enough to fill the GPU eight times over all tensors together, not more than a tensor has work for
      long long per = ((long long)num_sms * 8 + n - 1) / n;
      if (per > most) per = most;
      const dim3 grid((unsigned)per, (unsigned)n);
      if (K <= 2)
        reorder_kernel<2, 4><<<grid, kReorderThreads, 0, stm>>>(p);
      else if (K <= 4)
        reorder_kernel<4, 4><<<grid, kReorderThreads, 0, stm>>>(p);
      else if (K <= 8)
        reorder_kernel<8, 2><<<grid, kReorderThreads, 0, stm>>>(p);
      else if (K <= 16)
        reorder_kernel<16, 1><<<grid, kReorderThreads, 0, stm>>>(p);
      else if (K <= 32)
        reorder_kernel<32, 1><<<grid, kReorderThreads, 0, stm>>>(p);
      else
        reorder_kernel<64, 1><<<grid, kReorderThreads, 0, stm>>>(p);
      if (cudaGetLastError() != cudaSuccess) return kErrCuda;
    }
  }
  return FMMS_OK;
}

}  // extern "C"
