// A product of 16 rows with fewer steps of x fetched than it needs, and a short limit for its waits: what the kernel
// does when a wait runs out (test_gpu_int4_waits.py builds this; groups of 128, bf16, fp32 out, no zero points).
#include "fmms_int4_mma.cuh"

using namespace fmms;

extern "C" int int4_with_x_limit(const void* x, const void* qweight, const void* scales, int V, int D, int B, float* out, void* workspace,
                                 unsigned long long workspace_bytes, int* status, unsigned long long wait_ns, int x_limit, void* stream) {
  constexpr int n = 16, group = 128;
  constexpr int units = int4_step_units(group, n), x_bytes = int4_x_bytes(n, group);
  Int4MmaParams p = {};
  Int4Params& q = p.base;
  q.x = x;
  q.x_stride = D;
  q.q = static_cast<const uint8_t*>(qweight);
  q.scales = static_cast<const uint16_t*>(scales);
  q.out = out;
  q.out_stride = V;
  q.V = V;
  q.D = D;
  q.B = B;
  q.tiles = (V + kInt4Tile - 1) / kInt4Tile;
  q.chunks = (D + kInt4Chunk - 1) / kInt4Chunk;
  q.groups = D / group;
  q.x_bf16 = q.s_bf16 = q.x_pairs = 1;
  q.out_kind = 2;
  q.group_units = 1;
  q.all_units = (D + kInt4Unit - 1) / kInt4Unit;
  p.n = n;
  p.row_steps = (q.all_units + units - 1) / units;
  p.x_stages = 4;
  p.ring_off = p.x_stages * x_bytes;
  p.scale_off = p.ring_off + kInt4MmaWeightWarps * kInt4MmaRing * units * 1024;
  const int smem = p.scale_off + kInt4MmaSumWarps * kInt4MmaScaleRing * int4_step_groups(group, n) * 64 + kInt4MmaAlign;
  uint8_t* staged = static_cast<uint8_t*>(workspace);
  int* exponents = reinterpret_cast<int*>(staged + (size_t)p.row_steps * x_bytes);
  if (B < 1 || B > n || D % group || workspace_bytes < (size_t)p.row_steps * x_bytes + kInt4MmaPass * 4) return kErrBadArg;
  p.staged = staged;
  p.exponents = exponents;
  p.idesc = (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
  p.status_dev = status;
  p.wait_ns = wait_ns;
  p.x_limit = x_limit;
  int dev = 0, sms = 0;
  auto* kernel = int4_mma_kernel<n, group, false>;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return kErrCuda;
  int4_stage_x_kernel<group><<<B, 256, 0, static_cast<cudaStream_t>(stream)>>>(p, staged, exponents);
  kernel<<<q.tiles < sms ? q.tiles : sms, kInt4MmaThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}
