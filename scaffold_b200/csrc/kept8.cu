// Activations written to their 8-bit copy (kept8.cuh) and read back.
//
// Bound: memory. Per element keep8 reads 2 (4) bytes and writes 1.0625, restore8 the other way round; a thread owns one
// block of 16 elements, which it moves as one 32-byte (two for fp32) and one 16-byte access, and the largest magnitude
// needs no exchange between threads.
#include "common.cuh"
#include "host_api.h"
#include "kept8.cuh"

namespace sb {

constexpr int KEPT_THREADS = 256;

template <typename T> struct KeptType;
template <> struct KeptType<__nv_bfloat16> {
  static constexpr uint32_t top = KEPT_TOP_BF16;
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16(v); }
};
template <> struct KeptType<__half> {
  static constexpr uint32_t top = KEPT_TOP_FP16;
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half(v); }
};
template <> struct KeptType<float> {
  static constexpr uint32_t top = KEPT_TOP_BF16;
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};

template <typename T>
__global__ void __launch_bounds__(KEPT_THREADS) keep8_kernel(const T* __restrict__ x, long long n, long long blocks,
                                                             uint4* __restrict__ q, uint8_t* __restrict__ exps) {
  for (long long i = (long long)blockIdx.x * KEPT_THREADS + threadIdx.x; i < blocks;
       i += (long long)gridDim.x * KEPT_THREADS) {
    float f[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = i * 16 + j < n ? KeptType<T>::to(x[i * 16 + j]) : 0.f;
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) amax = max(amax, __float_as_uint(f[j]) & 0x7FFFFFFFu);  // a NaN's bits are the largest
    const uint32_t b = kept_exponent(amax);
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
    if (b != 255u) {
      const float inv = kept_inv(b);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        f[j] = fmaf(f[j], inv, KEPT_MAGIC);
        if (b >= KeptType<T>::top) f[j] = kept_cap(f[j]);
      }
      o.x = kept_pack4(f[0], f[1], f[2], f[3]);
      o.y = kept_pack4(f[4], f[5], f[6], f[7]);
      o.z = kept_pack4(f[8], f[9], f[10], f[11]);
      o.w = kept_pack4(f[12], f[13], f[14], f[15]);
    }
    q[i] = o;
    exps[i] = (uint8_t)b;
  }
}

template <typename T>
__global__ void __launch_bounds__(KEPT_THREADS) restore8_kernel(const uint4* __restrict__ q,
                                                                const uint8_t* __restrict__ exps, T* __restrict__ y,
                                                                long long n, long long blocks) {
  for (long long i = (long long)blockIdx.x * KEPT_THREADS + threadIdx.x; i < blocks;
       i += (long long)gridDim.x * KEPT_THREADS) {
    const uint4 w = q[i];
    const float step = kept_step(exps[i]);
    float f[4][4];
    kept_unpack4(w.x, f[0]);
    kept_unpack4(w.y, f[1]);
    kept_unpack4(w.z, f[2]);
    kept_unpack4(w.w, f[3]);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (i * 16 + j < n) y[i * 16 + j] = KeptType<T>::from(f[j / 4][j % 4] * step);
  }
}

static int kept_grid(long long blocks) {
  const long long need = (blocks + KEPT_THREADS - 1) / KEPT_THREADS;
  return (int)(need < 148 * 8 ? need : 148 * 8);
}

}  // namespace sb

using namespace sb;

// bytes of the copy of n elements: q, then the exponents
extern "C" long long sb_kept8_bytes(long long n) { return n < 0 ? -1 : (n + 15) / 16 * 17; }

// kind 0 bf16, 1 fp16, 2 fp32; `kept` 16-byte aligned, sb_kept8_bytes(n) bytes
extern "C" int sb_keep8(const void* x, int kind, long long n, void* kept, cudaStream_t stream) {
  if (n < 0 || kind < 0 || kind > 2) return SB_ERR_SHAPE;
  if (n == 0) return 0;
  if (x == nullptr || kept == nullptr) return SB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(kept) & 15) return SB_ERR_ALIGN;
  const long long blocks = (n + 15) / 16;
  uint4* q = (uint4*)kept;
  uint8_t* e = (uint8_t*)kept + blocks * 16;
  const int grid = kept_grid(blocks);
  if (kind == 0) keep8_kernel<<<grid, KEPT_THREADS, 0, stream>>>((const __nv_bfloat16*)x, n, blocks, q, e);
  else if (kind == 1) keep8_kernel<<<grid, KEPT_THREADS, 0, stream>>>((const __half*)x, n, blocks, q, e);
  else keep8_kernel<<<grid, KEPT_THREADS, 0, stream>>>((const float*)x, n, blocks, q, e);
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

extern "C" int sb_restore8(const void* kept, int kind, long long n, void* y, cudaStream_t stream) {
  if (n < 0 || kind < 0 || kind > 2) return SB_ERR_SHAPE;
  if (n == 0) return 0;
  if (y == nullptr || kept == nullptr) return SB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(kept) & 15) return SB_ERR_ALIGN;
  const long long blocks = (n + 15) / 16;
  const uint4* q = (const uint4*)kept;
  const uint8_t* e = (const uint8_t*)kept + blocks * 16;
  const int grid = kept_grid(blocks);
  if (kind == 0) restore8_kernel<<<grid, KEPT_THREADS, 0, stream>>>(q, e, (__nv_bfloat16*)y, n, blocks);
  else if (kind == 1) restore8_kernel<<<grid, KEPT_THREADS, 0, stream>>>(q, e, (__half*)y, n, blocks);
  else restore8_kernel<<<grid, KEPT_THREADS, 0, stream>>>(q, e, (float*)y, n, blocks);
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}
