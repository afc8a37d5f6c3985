// C ABI of the operators around a decode step (see include/fmms_b200.h): products with 4-bit weights, the beam-search
// step and the reordering of per-beam states.  Argument checks, launch plans and launches; no allocation, no
// synchronisation, no exceptions.
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/fmms_b200.h"
#include "fmms_beam.cuh"
#include "fmms_common.cuh"
#include "fmms_int4.cuh"
#include "fmms_int4_mma.cuh"
#include "fmms_reorder.cuh"

namespace fmms {

constexpr int kDecodeMaxDevices = 16;
constexpr int kInt4SmemLimit = 230000;  // of 232448 bytes a CTA may have; the rest: static shared memory and alignment

static bool on_boundary(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % (unsigned)bytes == 0; }

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

// A kernel that may start while the one before it on the stream still runs (and waits for it where it needs it).
template <typename... KArgs, typename... Args>
static int launch_behind(void (*kernel)(KArgs...), dim3 grid, int threads, int smem, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
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

// ---- products with 4-bit weights ----------------------------------------------------------------
struct Int4Plan {
  int phases, units, all_units, smem;
  int xs_off, xs32_off, ring_off, piece_off;
};

static int int4_smem(Int4Plan& pl, int group) {
  int off = pl.units * 2 * 1024;
  pl.xs_off = off;
  off += (pl.units * int4_unit_groups(group) * kInt4Rows * 4 + 127) / 128 * 128;
  pl.xs32_off = off;
  if (group > 32) off += pl.units * 4 * kInt4Rows * 4;
  pl.piece_off = off;
  off += kInt4Warps * 2 * 512;
  pl.ring_off = off;
  off += kInt4Warps * kInt4Stages * int4_stage_bytes(group);
  pl.smem = off;
  return off;
}

// As few phases as shared memory allows: rows of up to some 7000 columns take one.
static int int4_plan(Int4Plan& pl, int D, int group) {
  pl.all_units = (D + kInt4Unit - 1) / kInt4Unit;
  for (pl.phases = 1; pl.phases <= pl.all_units; ++pl.phases) {
    pl.units = (pl.all_units + pl.phases - 1) / pl.phases;
    if ((pl.phases - 1) * pl.units < pl.all_units &&  // the last phase is not empty
        int4_smem(pl, group) <= kInt4SmemLimit)
      return kOk;
  }
  return kErrUnsupported;
}

static bool int4_group_ok(int group, int D) { return (group == 32 || group == 64 || (group > 0 && group % kInt4Unit == 0)) && D % group == 0; }

// Sizes whose sums and rounded multiples stay within 32 bits in plans and kernels; at most 65535 passes of eight-plus rows.
static bool int4_sizes_ok(int V, int D, int group, int B) {
  return V <= 0x7fffffff - (kInt4Tile - 1) && D <= (1 << 30) && B <= 65535 * int4_mma_max_n(group);
}

static size_t int4_workspace(const Int4Plan& pl, int V) {
  return pl.phases == 1 ? 0 : (size_t)((V + kInt4Tile - 1) / kInt4Tile) * 512;
}

template <int GR, bool ZP>
static int int4_launch(const Int4Params& p, const Int4Plan& pl, int dev, int num_sms, cudaStream_t stream) {
  auto* kernel = int4_linear_kernel<GR, ZP>;
  static std::atomic<bool> ready[kDecodeMaxDevices];
  if (!ready[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kInt4SmemLimit) != cudaSuccess) {
      cudaGetLastError();
      return kErrCuda;
    }
    ready[dev].store(true, std::memory_order_release);
  }
  kernel<<<min(p.tiles, num_sms), kInt4Warps * 32, pl.smem, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

template <bool ZP>
static int int4_launch_group(const Int4Params& p, const Int4Plan& pl, int group, int dev, int num_sms, cudaStream_t stream) {
  switch (group) {
    case 32: return int4_launch<32, ZP>(p, pl, dev, num_sms, stream);
    case 64: return int4_launch<64, ZP>(p, pl, dev, num_sms, stream);
    default: return int4_launch<128, ZP>(p, pl, dev, num_sms, stream);
  }
}

// ---- more than eight rows: fmms_int4_mma.cuh.  Rows of x in a pass, and the stages of x that fit beside the rings.
struct Int4MmaPlan {
  int n, passes, row_steps, x_stages, ring_off, scale_off, smem;
};

static void int4_mma_plan(Int4MmaPlan& pl, int D, int B, int group, bool zeros) {
  const int gr = group < kInt4Unit ? group : kInt4Unit, most = int4_mma_max_n(gr);
  pl.passes = (B + most - 1) / most;
  pl.n = ((B + pl.passes - 1) / pl.passes + 15) / 16 * 16;
  const int units = int4_step_units(gr, pl.n);
  pl.row_steps = ((D + kInt4Unit - 1) / kInt4Unit + units - 1) / units;
  const int weights = kInt4MmaWeightWarps * kInt4MmaRing * (units * 1024 + (zeros ? 128 : 0));
  const int scales = kInt4MmaSumWarps * kInt4MmaScaleRing * int4_step_groups(gr, pl.n) * 64;
  pl.x_stages = min(kInt4MmaMaxX, (kInt4SmemLimit - weights - scales) / int4_x_bytes(pl.n, gr));
  pl.ring_off = pl.x_stages * int4_x_bytes(pl.n, gr);
  pl.scale_off = pl.ring_off + weights;
  pl.smem = pl.scale_off + scales + kInt4MmaAlign;
}

// staged x, then the exponents of its rows
static size_t int4_mma_workspace(int D, int B, int group) {
  Int4MmaPlan pl;
  int4_mma_plan(pl, D, B, group, true);
  return (size_t)pl.passes * (pl.row_steps * (size_t)int4_x_bytes(pl.n, group < kInt4Unit ? group : kInt4Unit) + kInt4MmaPass * 4);
}

template <int NC, int GR, bool ZP>
static int int4_mma_launch(const Int4MmaParams& p, const Int4MmaPlan& pl, int dev, int num_sms, uint8_t* staged, int* exponents, cudaStream_t stream) {
  if constexpr (NC <= int4_mma_max_n(GR)) {
    auto* kernel = int4_mma_kernel<NC, GR, ZP>;
    static std::atomic<bool> ready[kDecodeMaxDevices];
    if (!ready[dev].load(std::memory_order_acquire)) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kInt4SmemLimit + kInt4MmaAlign) != cudaSuccess) {
        cudaGetLastError();
        return kErrCuda;
      }
      ready[dev].store(true, std::memory_order_release);
    }
    int4_stage_x_kernel<GR><<<p.base.B, 256, 0, stream>>>(p, staged, exponents);
    if (cudaGetLastError() != cudaSuccess) return kErrCuda;
    return launch_behind(kernel, dim3((unsigned)min(p.base.tiles, num_sms), (unsigned)pl.passes), kInt4MmaThreads, pl.smem, stream, p);
  } else {
    return kErrUnsupported;  // the plan asks for no such pass
  }
}

template <int GR, bool ZP>
static int int4_mma_launch_rows(const Int4MmaParams& p, const Int4MmaPlan& pl, int dev, int num_sms, uint8_t* staged, int* exponents, cudaStream_t stream) {
  switch (pl.n) {
    case 16: return int4_mma_launch<16, GR, ZP>(p, pl, dev, num_sms, staged, exponents, stream);
    case 32: return int4_mma_launch<32, GR, ZP>(p, pl, dev, num_sms, staged, exponents, stream);
    case 48: return int4_mma_launch<48, GR, ZP>(p, pl, dev, num_sms, staged, exponents, stream);
    default: return int4_mma_launch<64, GR, ZP>(p, pl, dev, num_sms, staged, exponents, stream);
  }
}

template <bool ZP>
static int int4_mma_launch_group(const Int4MmaParams& p, const Int4MmaPlan& pl, int group, int dev, int num_sms, uint8_t* staged, int* exponents, cudaStream_t stream) {
  switch (group) {
    case 32: return int4_mma_launch_rows<32, ZP>(p, pl, dev, num_sms, staged, exponents, stream);
    case 64: return int4_mma_launch_rows<64, ZP>(p, pl, dev, num_sms, staged, exponents, stream);
    default: return int4_mma_launch_rows<128, ZP>(p, pl, dev, num_sms, staged, exponents, stream);
  }
}

// ---- beam step ----------------------------------------------------------------------------------
static int beam_element_bytes(int dtype) { return dtype == FMMS_F32 ? 4 : 2; }

static bool beam_sizes_ok(int R, int K, int V, int N) {
  return N <= kBeamMaxN && K <= kBeamMaxK && (long long)K * V < (1ll << 31) && (long long)R * K <= 65535;
}

// Vectors of a thread in a slice of a row, and slices of a row: as few slices as the list for their candidates allows,
// but enough that the rows together make some four CTAs for each of a B200's 148 SMs (a constant, for the workspace's size is
// asked for without a GPU, and sums must not depend on how many SMs there are); not below four vectors, which the bound is
// taken from.
static void beam_slices(int rows, int V, int dtype, int* iters, int* splits) {
  const long long per_iter = kBeamThreads * (16 / beam_element_bytes(dtype));
  const long long all = (V + per_iter - 1) / per_iter;
  long long want = (4 * 148 + rows - 1) / rows;
  long long it = (all + want - 1) / want;
  it = it < kBeamFirst ? kBeamFirst : it > kBeamMaxIters ? kBeamMaxIters : it;
  it += it & 1;
  *iters = (int)it;
  *splits = (int)((all + it - 1) / it);
}

static size_t beam_workspace(int R, int K, int V, int N, int dtype) {
  int iters, splits;
  beam_slices(R * K, V, dtype, &iters, &splits);
  const size_t parts = (size_t)R * K * splits;
  return parts * N * 8 + parts * 8 + parts * 4;
}

template <typename T>
static void beam_launch_part(const BeamParams& p, dim3 grid, cudaStream_t stream) {
  const long long between = (p.R > 1 ? p.stride_r : 0) | (p.K > 1 ? p.stride_k : 0);  // a set low bit: so has one of the strides
  if (reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && between % (16 / (int)sizeof(T)) == 0)
    beam_part_kernel<T, true><<<grid, kBeamThreads, 0, stream>>>(p);
  else
    beam_part_kernel<T, false><<<grid, kBeamThreads, 0, stream>>>(p);
}

int reorder_beams_rounded(int K) { return K <= 2 ? 2 : K <= 4 ? 4 : K <= 8 ? 8 : K <= 16 ? 16 : K <= 32 ? 32 : 64; }

// Bytes of a column: what divides the state's address and strides.
int reorder_vec(const fmms_beam_state_t& s, int K) {
  unsigned long long bits = reinterpret_cast<uintptr_t>(s.data) | (unsigned long long)s.beam_stride |
                            (unsigned long long)s.seg_bytes | (unsigned long long)s.step_bytes;
  for (int o = 0; o < 2; ++o)
    if (s.outer[o] > 1) bits |= (unsigned long long)s.outer_stride[o];
  int vec = K > 32 ? 8 : 16;
  while (bits & (unsigned long long)(vec - 1)) vec >>= 1;
  return vec;
}

template <int KM>
void launch_reorder_vec(const ReorderParams& p, int vec, dim3 grid, cudaStream_t stm) {
  switch (vec) {
    case 16:
      if constexpr (KM <= 32) reorder_kernel<KM, 16><<<grid, kReorderThreads, 0, stm>>>(p);  // 64 beams: columns of at most 8 bytes
      break;
    case 8: reorder_kernel<KM, 8><<<grid, kReorderThreads, 0, stm>>>(p); break;
    case 4: reorder_kernel<KM, 4><<<grid, kReorderThreads, 0, stm>>>(p); break;
    case 2: reorder_kernel<KM, 2><<<grid, kReorderThreads, 0, stm>>>(p); break;
    default: reorder_kernel<KM, 1><<<grid, kReorderThreads, 0, stm>>>(p); break;
  }
}

int launch_reorder(const ReorderParams& p, int vec, dim3 grid, cudaStream_t stm) {
  switch (reorder_beams_rounded(p.K)) {
    case 2: launch_reorder_vec<2>(p, vec, grid, stm); break;
    case 4: launch_reorder_vec<4>(p, vec, grid, stm); break;
    case 8: launch_reorder_vec<8>(p, vec, grid, stm); break;
    case 16: launch_reorder_vec<16>(p, vec, grid, stm); break;
    case 32: launch_reorder_vec<32>(p, vec, grid, stm); break;
    default: launch_reorder_vec<64>(p, vec, grid, stm); break;
  }
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace fmms

using namespace fmms;

extern "C" {

int fmms_query_int4_workspace(int V, int D, int group, int B, size_t* bytes) {
  if (!bytes || V <= 0 || D <= 0 || B <= 0) return FMMS_ERR_BAD_ARG;
  if (!int4_group_ok(group, D) || !int4_sizes_ok(V, D, group, B)) return FMMS_ERR_UNSUPPORTED;
  if (B > kInt4Rows) {
    *bytes = int4_mma_workspace(D, B, group);
    return FMMS_OK;
  }
  Int4Plan pl;
  const int rc = int4_plan(pl, D, group);
  if (rc == kOk) *bytes = int4_workspace(pl, V);
  return rc;
}

int fmms_int4_linear(const void* x, int x_dtype, long long x_stride, const void* qweight, const void* scales, int scale_dtype,
                     const void* zeros, int V, int D, int group, int B, void* out, int out_dtype, long long out_stride,
                     void* workspace, size_t workspace_bytes, int* status_dev, void* stream) {
  if (!x || !qweight || !scales || !out || V <= 0 || D <= 0 || B <= 0) return FMMS_ERR_BAD_ARG;
  if ((x_dtype != FMMS_BF16 && x_dtype != FMMS_F16) || (scale_dtype != FMMS_BF16 && scale_dtype != FMMS_F16) ||
      out_dtype < FMMS_BF16 || out_dtype > FMMS_F32)
    return FMMS_ERR_BAD_ARG;
  if (x_stride < D || out_stride < V) return FMMS_ERR_BAD_ARG;
  if (!on_boundary(x, 2) || !on_boundary(out, out_dtype == FMMS_F32 ? 4 : 2) || !on_boundary(status_dev, 4)) return FMMS_ERR_BAD_ARG;
  if (!int4_group_ok(group, D) || !int4_sizes_ok(V, D, group, B)) return FMMS_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(qweight) | reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(zeros)) & 15)
    return FMMS_ERR_UNSUPPORTED;
  const bool mma = B > kInt4Rows;
  Int4Plan pl = {};
  Int4MmaPlan mp = {};
  int rc = kOk;
  if (mma)
    int4_mma_plan(mp, D, B, group, zeros != nullptr);
  else
    rc = int4_plan(pl, D, group);
  if (rc != kOk) return rc;
  const size_t need = mma ? int4_mma_workspace(D, B, group) : int4_workspace(pl, V);
  if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need)) return FMMS_ERR_WORKSPACE;
  int dev = 0, num_sms = 0;
  rc = decode_num_sms(&dev, &num_sms);
  if (rc != kOk) return rc;
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
  p.x_pairs = (reinterpret_cast<uintptr_t>(x) & 3) == 0 && x_stride % 2 == 0;
  p.group_units = group > kInt4Unit ? group / kInt4Unit : 1;
  p.all_units = (D + kInt4Unit - 1) / kInt4Unit;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (mma) {
    Int4MmaParams m = {};
    m.base = p;
    uint8_t* staged = reinterpret_cast<uint8_t*>(workspace);
    int* exponents = reinterpret_cast<int*>(staged + (size_t)mp.passes * mp.row_steps * int4_x_bytes(mp.n, group < kInt4Unit ? group : kInt4Unit));
    m.staged = staged;
    m.exponents = exponents;
    m.n = mp.n;
    m.row_steps = mp.row_steps;
    m.x_stages = mp.x_stages;
    m.ring_off = mp.ring_off;
    m.scale_off = mp.scale_off;
    m.idesc = (1u << 4) | ((uint32_t)(mp.n >> 3) << 17) | ((128u >> 4) << 24);  // fp32 sums of fp16 products, 128 x n
    m.status_dev = status_dev;
    m.wait_ns = kWaitLimitNs;
    m.x_limit = 0x7fffffff;
    return zeros ? int4_mma_launch_group<true>(m, mp, group, dev, num_sms, staged, exponents, s)
                 : int4_mma_launch_group<false>(m, mp, group, dev, num_sms, staged, exponents, s);
  }
  for (p.log_rows = 0; (1 << p.log_rows) < B; ++p.log_rows) {
  }
  p.partial = reinterpret_cast<float*>(workspace);
  p.phases = pl.phases;
  p.units = pl.units;
  p.xs_off = pl.xs_off;
  p.xs32_off = pl.xs32_off;
  p.ring_off = pl.ring_off;
  p.piece_off = pl.piece_off;
  return zeros ? int4_launch_group<true>(p, pl, group, dev, num_sms, s) : int4_launch_group<false>(p, pl, group, dev, num_sms, s);
}

int fmms_query_beam_workspace(int R, int K, int V, int N, int dtype, size_t* bytes) {
  if (!bytes || R <= 0 || K <= 0 || V <= 0 || N <= 0 || dtype < FMMS_BF16 || dtype > FMMS_F32) return FMMS_ERR_BAD_ARG;
  if (!beam_sizes_ok(R, K, V, N)) return FMMS_ERR_UNSUPPORTED;
  *bytes = beam_workspace(R, K, V, N, dtype);
  return FMMS_OK;
}

int fmms_beam_step(const void* logits, int dtype, long long stride_r, long long stride_k, const float* scores,
                   const unsigned char* finished, long long pad_token, int R, int K, int V, int N, float* out_scores,
                   long long* out_tokens, long long* out_parents, void* workspace, size_t workspace_bytes, void* stream) {
  if (!logits || !scores || !out_scores || !out_tokens || !out_parents) return FMMS_ERR_BAD_ARG;
  if (R <= 0 || K <= 0 || V <= 0 || N <= 0 || dtype < FMMS_BF16 || dtype > FMMS_F32) return FMMS_ERR_BAD_ARG;
  if (pad_token < 0 || pad_token >= V || N > (long long)K * V) return FMMS_ERR_BAD_ARG;
  if (!on_boundary(logits, beam_element_bytes(dtype)) || !on_boundary(scores, 4) || !on_boundary(out_scores, 4) || !on_boundary(out_tokens, 8) ||
      !on_boundary(out_parents, 8))
    return FMMS_ERR_BAD_ARG;
  if (!beam_sizes_ok(R, K, V, N)) return FMMS_ERR_UNSUPPORTED;
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
  beam_slices(R * K, V, dtype, &p.iters, &p.splits);
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
    beam_launch_part<__nv_bfloat16>(p, grid, s);
  else if (dtype == FMMS_F16)
    beam_launch_part<__half>(p, grid, s);
  else
    beam_launch_part<float>(p, grid, s);
  if (cudaGetLastError() != cudaSuccess) return kErrCuda;
  return launch_behind(beam_merge_kernel, dim3((unsigned)R), kBeamThreads, 0, s, p);
}

int fmms_reorder_beams(const fmms_beam_state_t* states, int n_states, const void* parents, int parents_bytes, int R, int K,
                       const int* lengths, void* stream) {
  if (!states || n_states <= 0 || !parents || R <= 0 || K <= 0 || (parents_bytes != 4 && parents_bytes != 8)) return FMMS_ERR_BAD_ARG;
  if (!on_boundary(parents, parents_bytes) || !on_boundary(lengths, 4)) return FMMS_ERR_BAD_ARG;
  if (K > kReorderMaxBeams) return FMMS_ERR_UNSUPPORTED;
  for (int i = 0; i < n_states; ++i) {
    const fmms_beam_state_t& s = states[i];
    if (!s.data || s.outer[0] <= 0 || s.outer[1] <= 0 || s.seg_bytes <= 0 || s.step_bytes < 0) return FMMS_ERR_BAD_ARG;
    if (s.step_bytes && s.seg_bytes % s.step_bytes) return FMMS_ERR_BAD_ARG;
    const long long unit = kReorderThreads, cols = s.seg_bytes / reorder_vec(s, K);
    if (min(R, kReorderMaxRequests) * ((cols + unit - 1) / unit) >= (1ll << 31)) return FMMS_ERR_UNSUPPORTED;
  }
  int dev = 0, num_sms = 0;
  const int rc = decode_num_sms(&dev, &num_sms);
  if (rc != kOk) return rc;
  if (K == 1) return FMMS_OK;  // one beam: its own parent
  cudaStream_t stm = reinterpret_cast<cudaStream_t>(stream);
  // a launch for every width of columns that occurs (rarely more than one), so that each needs no more registers than its own
  for (int vec = K > 32 ? 8 : 16; vec >= 1; vec >>= 1)
    for (int r0 = 0; r0 < R; r0 += kReorderMaxRequests) {
      ReorderParams p;
      p.parents = reinterpret_cast<const uint8_t*>(parents) + (size_t)r0 * K * parents_bytes;
      p.parents_wide = parents_bytes == 8;
      p.lengths = lengths ? lengths + r0 : nullptr;
      p.R = min(kReorderMaxRequests, R - r0);
      p.K = K;
      int n = 0;
      long long most = 1;  // units of the largest tensor
      for (int i = 0; i < n_states; ++i) {
        const fmms_beam_state_t& s = states[i];
        if (reorder_vec(s, K) == vec) {
          ReorderState& d = p.st[n++];
          d.data = reinterpret_cast<uint8_t*>(s.data) + (long long)r0 * K * s.beam_stride;
          d.beam_stride = s.beam_stride;
          d.outer_stride[0] = s.outer_stride[0];
          d.outer_stride[1] = s.outer_stride[1];
          d.outer[0] = s.outer[0];
          d.outer[1] = s.outer[1];
          d.seg_bytes = s.seg_bytes;
          d.step_bytes = s.step_bytes;
          const long long cols = s.seg_bytes / vec, unit = kReorderThreads * reorder_columns_each(reorder_beams_rounded(K), vec);
          const long long outers = (long long)s.outer[0] * s.outer[1];
          const long long units = cols >= unit / 2 ? outers * p.R * ((cols + unit - 1) / unit) : (outers * p.R * cols + kReorderThreads - 1) / kReorderThreads;
          if (units > most) most = units;
        }
        if (n == kReorderMaxStates || (n > 0 && i == n_states - 1)) {
          // CTAs: enough to fill the GPU eight times over all tensors together, not more than a tensor has work for
          const long long per = min(((long long)num_sms * 8 + n - 1) / n, most);
          const int rc_launch = launch_reorder(p, vec, dim3((unsigned)per, (unsigned)n), stm);
          if (rc_launch != kOk) return rc_launch;
          n = 0;
          most = 1;
        }
      }
    }
  return FMMS_OK;
}

}  // extern "C"
