// Activations written to their 8-bit copy (kept8.cuh) and read back.
//
// Bound: memory. Per element keep8 reads 2 (4) bytes and writes 1.0625, restore8 the other way round; a thread owns one
// block of 16 elements, which it moves as one 32-byte (two for fp32) and one 16-byte access, and the largest magnitude
// needs no exchange between threads. bf16 2 x 128^3 x 64: keep8 124 us (6.6 TB/s), restore8 138 (6.0).
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

// 32 bytes of read-only memory (needs a 32-byte aligned address)
__device__ __forceinline__ void kept_load_v8(const void* p, uint32_t (&v)[8]) {
  asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p));
}
template <typename T>
struct KeptRaw {  // a block as it lies in memory
  static constexpr int N = (int)sizeof(T) / 2;  // 32-byte words
  uint32_t v[N][8];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) kept_load_v8(reinterpret_cast<const uint8_t*>(p) + 32 * i, v[i]);
  }
  __device__ __forceinline__ void load_tail(const T* p, int n) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0u;
    T* t = reinterpret_cast<T*>(v);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < n) t[j] = p[j];
  }
};

template <typename T>
__device__ __forceinline__ void keep8_block(const KeptRaw<T>& raw, uint4& o, uint32_t& b) {
  float f[16];
  const T* t = reinterpret_cast<const T*>(raw.v);
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    f[j] = KeptType<T>::to(t[j]);
    amax = max(amax, __float_as_uint(f[j]) & 0x7FFFFFFFu);  // a NaN's bits are the largest
  }
  b = kept_exponent(amax);
  const float inv = b == 255u ? 0.f : kept_inv(b);
#pragma unroll
  for (int j = 0; j < 16; ++j) f[j] = fmaf(f[j], inv, KEPT_MAGIC);
  if (b >= KeptType<T>::top) {
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = b == 255u ? KEPT_MAGIC : kept_cap(f[j]);
  }
  o = make_uint4(kept_pack4(f[0], f[1], f[2], f[3]), kept_pack4(f[4], f[5], f[6], f[7]),
                 kept_pack4(f[8], f[9], f[10], f[11]), kept_pack4(f[12], f[13], f[14], f[15]));
}

// VEC: x starts on 32 bytes
template <typename T, bool VEC>
__global__ void __launch_bounds__(KEPT_THREADS) keep8_kernel(const T* __restrict__ x, long long n, long long blocks,
                                                             uint4* __restrict__ q, uint8_t* __restrict__ exps) {
  const long long stride = (long long)gridDim.x * KEPT_THREADS;
  const long long whole = VEC ? n / 16 : 0;  // blocks that one or two vector loads bring
  long long i = (long long)blockIdx.x * KEPT_THREADS + threadIdx.x;
  for (; i + stride < whole; i += 2 * stride) {  // two blocks in flight
    KeptRaw<T> r0, r1;
    r0.load(x + i * 16);
    r1.load(x + (i + stride) * 16);
    uint4 o;
    uint32_t b;
    keep8_block<T>(r0, o, b);
    q[i] = o;
    exps[i] = (uint8_t)b;
    keep8_block<T>(r1, o, b);
    q[i + stride] = o;
    exps[i + stride] = (uint8_t)b;
  }
  for (; i < blocks; i += stride) {
    KeptRaw<T> r;
    if (i < whole) r.load(x + i * 16);
    else r.load_tail(x + i * 16, n - i * 16 < 16 ? (int)(n - i * 16) : 16);
    uint4 o;
    uint32_t b;
    keep8_block<T>(r, o, b);
    q[i] = o;
    exps[i] = (uint8_t)b;
  }
}

template <typename T>
__device__ __forceinline__ void restore8_block(const uint4 w, uint32_t b, T* __restrict__ y, bool vec, int n) {
  const float step = kept_step(b);
  float f[4][4];
  kept_unpack4(w.x, f[0]);
  kept_unpack4(w.y, f[1]);
  kept_unpack4(w.z, f[2]);
  kept_unpack4(w.w, f[3]);
  __align__(16) T t[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) t[j] = KeptType<T>::from(f[j / 4][j % 4] * step);
  if (vec) {
    const uint4* v = reinterpret_cast<const uint4*>(t);
#pragma unroll
    for (int j = 0; j < (int)sizeof(T); j += 2) st_global_v8(reinterpret_cast<uint4*>(y) + j, v[j], v[j + 1]);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < n) y[j] = t[j];
  }
}

template <typename T>
__global__ void __launch_bounds__(KEPT_THREADS) restore8_kernel(const uint4* __restrict__ q,
                                                                const uint8_t* __restrict__ exps, T* __restrict__ y,
                                                                long long n, long long blocks, int vec) {
  const long long stride = (long long)gridDim.x * KEPT_THREADS;
  const long long whole = vec ? n / 16 : 0;
  long long i = (long long)blockIdx.x * KEPT_THREADS + threadIdx.x;
  for (; i + stride < whole; i += 2 * stride) {  // two blocks in flight
    const uint4 w0 = __ldg(q + i), w1 = __ldg(q + i + stride);
    const uint32_t b0 = __ldg(exps + i), b1 = __ldg(exps + i + stride);
    restore8_block<T>(w0, b0, y + i * 16, true, 16);
    restore8_block<T>(w1, b1, y + (i + stride) * 16, true, 16);
  }
  for (; i < blocks; i += stride)
    restore8_block<T>(__ldg(q + i), __ldg(exps + i), y + i * 16, i < whole, n - i * 16 < 16 ? (int)(n - i * 16) : 16);
}

static int kept_grid(long long blocks) {
  const long long need = (blocks + KEPT_THREADS - 1) / KEPT_THREADS;
  return (int)(need < 148 * 8 ? need : 148 * 8);
}

template <typename T>
static void keep8_launch(const T* x, long long n, long long blocks, uint4* q, uint8_t* e, cudaStream_t stream) {
  if (reinterpret_cast<uintptr_t>(x) & 31)
    keep8_kernel<T, false><<<kept_grid(blocks), KEPT_THREADS, 0, stream>>>(x, n, blocks, q, e);
  else
    keep8_kernel<T, true><<<kept_grid(blocks), KEPT_THREADS, 0, stream>>>(x, n, blocks, q, e);
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
  if (kind == 0) keep8_launch((const __nv_bfloat16*)x, n, blocks, q, e, stream);
  else if (kind == 1) keep8_launch((const __half*)x, n, blocks, q, e, stream);
  else keep8_launch((const float*)x, n, blocks, q, e, stream);
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
  const int vec = (reinterpret_cast<uintptr_t>(y) & 31) == 0;
  if (kind == 0) restore8_kernel<<<grid, KEPT_THREADS, 0, stream>>>(q, e, (__nv_bfloat16*)y, n, blocks, vec);
  else if (kind == 1) restore8_kernel<<<grid, KEPT_THREADS, 0, stream>>>(q, e, (__half*)y, n, blocks, vec);
  else restore8_kernel<<<grid, KEPT_THREADS, 0, stream>>>(q, e, (float*)y, n, blocks, vec);
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}
