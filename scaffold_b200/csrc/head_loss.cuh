// What the kernels of the head's cross entropy share (head_loss.cu: up to 256 channels, head_wide.cu: more).
#pragma once
#include "common.cuh"
#include "host_api.h"

namespace sb {

int make_map_bf16(CUtensorMap* m, const void* base, int rank, const long long* dims, const long long* strides,
                  const int* box, int rowb);

constexpr int HD_PAD = 256;  // per-voxel and per-class arrays are padded to a multiple of this
constexpr float HD_LOG2E = 1.4426950408889634f;
constexpr float HD_LN2 = 0.6931471805599453f;

__device__ __forceinline__ float hd_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void hd_tma_2d(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}
// barrier of the 256 threads of the epilogue warps; the same answer in all of them: whether every one said `ok`
__device__ __forceinline__ bool hd_epi_vote(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred a, q;\n\t"
      "setp.ne.u32 a, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, 256, a;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(ok ? 1u : 0u)
      : "memory");
  return all != 0;
}

template <typename T> __device__ __forceinline__ T hd_cast(float v);
template <> __device__ __forceinline__ float hd_cast<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 hd_cast<__nv_bfloat16>(float v) { return __float2bfloat16(v); }

// head_wide.cu
int head_wide_splits(long long V, int K);
int head_wide_forward(const SbHeadArgs* a, float2* part, float* tl, int splits, cudaStream_t stream);
long long head_wide_scratch(const SbHeadArgs* a);
int head_wide_backward(const SbHeadArgs* a, cudaStream_t stream);

}  // namespace sb
