// What the kernels of the head's cross entropy share (head_loss.cu: up to 256 channels, head_wide.cu: more).
#pragma once
#include "common.cuh"
#include "host_api.h"

namespace sb {

int make_map_bf16(CUtensorMap* m, const void* base, int rank, const long long* dims, const long long* strides,
                  const int* box, int rowb);

constexpr int HD_PAD = 256;         // per-voxel and per-class arrays are padded to a multiple of this
constexpr int HD_FEW = 128;         // up to this many voxels, D's entries are kept in two bf16 (head_loss.cu)
constexpr int HD_SUM_BLOCKS = 1184;  // blocks of the loss's sums at most
constexpr float HD_LOG2E = 1.4426950408889634f;
constexpr float HD_LN2 = 0.6931471805599453f;
constexpr float HD_LOWEST = -1e30f;

static inline long long hd_pad(long long n) { return (n + HD_PAD - 1) / HD_PAD * HD_PAD; }

// What a call works on; arrays of voxels / classes are padded to HD_PAD.
struct HeadCall {
  const __nv_bfloat16* x;  // [V][C]
  const __nv_bfloat16* w;  // [K][C]
  const float* cw;         // optional class weights
  long long V;
  int K, C;
  // what the forward pass leaves for the backward pass
  double* total;  // [2] sums of u nll and of u
  float* den;     // [1] the second one, at least eps
  float* lse2;    // voxels: log2 of the sum of exponentials, +inf behind the last
  int* y;         // voxels: label, -1 where a voxel takes no part
  float* bias2;   // classes: bias log2(e), -inf behind the last
  uint4* w16;     // narrow heads, classes, twice: sixteen columns more of w
  uint32_t* hit;  // voxels, for both gradients at once (head_both): label (16 bits) and p - 1 of it (bf16)
  // of the backward pass
  const float* gout;  // [1] dL
  float* scale;   // [1] dL / den
  float* g;       // voxels: scale u, u the class weight of the label, 0 where a voxel takes no part
  uint4* x16;     // narrow heads, voxels: sixteen columns more of x
  float* u;       // wide heads, voxels: u
  float* lse2p;   // wide heads, voxels: lse2, +inf where u is 0
  __nv_bfloat16* dx;
  void* dw;
  int dw_kind;    // 0 bf16, 2 fp32
  void* db;
  int db_kind;
  float* scratch;
  uint32_t* status;
};

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
// a warp's wait, with the same answer in all lanes (one that gives up must not leave the others in a ballot)
__device__ __forceinline__ bool hd_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* status,
                                        int site) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, site));
}
// named barrier `id` of `threads` threads; the same answer in all of them: whether every one said `ok`
__device__ __forceinline__ bool hd_vote(int id, int threads, bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred a, q;\n\t"
      "setp.ne.u32 a, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, %2, %3, a;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(ok ? 1u : 0u), "r"(id), "r"(threads)
      : "memory");
  return all != 0;
}
// (v, i) in the place of (m, best) if it comes before it: NaN before numbers, larger ones first, then lower classes
__device__ __forceinline__ void hd_better(float& m, int& best, float v, int i) {
  const bool a = v != v, b = m != m;
  if ((a && !b) || (a == b && (v > m || ((v == m || a) && i < best)))) { m = v; best = i; }
}

// head_wide.cu
int head_wide_splits(long long V, int K);
int head_wide_forward(const HeadCall& a, float2* part, float* tl, cudaStream_t stream);
int head_wide_predict(const HeadCall& a, float2* part, cudaStream_t stream);
long long head_wide_scratch(const HeadCall& a);  // floats
int head_wide_backward(const HeadCall& a, cudaStream_t stream);

}  // namespace sb
