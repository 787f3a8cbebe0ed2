// GroupNorm (+ ReLU) whose backward pass works on an 8-bit copy of its input (kept8.cuh), so that the bf16 input need
// not live until then: 1.0625 bytes per element instead of 2.
//
// Forward (gn8_apply_kernel, behind the statistics pass of group_norm.cu or a convolution's own partials):
//   y = relu(x a + c), a = rstd w, c = b - mean a, and the copy, in one pass over x.
//   A value that the rounding would move across the ReLU's border is kept one step further towards x instead (its error
//   is then up to a step): the backward pass takes the mask from the copy and finds the forward's own mask, and the
//   only thing that differs from the ordinary backward pass is xhat by at most a step.
// Backward: the two passes of group_norm.cu with the copy in the place of x:
//   gn8_bwd_partial  per (split, n) and channel: sum(dy') and sum(dy' xhat), dy' = dy gated by the mask
//   gn8_bwd_dx       dx = rstd (dy' w - c1 - xhat c2), c1 / c2 the group's means of dy' w and dy' w xhat
//
// Every thread owns 8 channels (half a block) of a voxel; the two halves find their largest magnitude by one shuffle.
// Channels are a multiple of 16, so a block never leaves its voxel. Bound: memory (forward 5.06 bytes an element behind
// the statistics, backward 3.06 + 5.06 against 4 + 6 of the bf16 kernels).
#include "common.cuh"
#include "host_api.h"
#include "kept8.cuh"

namespace sb {

constexpr int GN8_THREADS = 256;
// Blocks per SM (85 or 64 registers a thread) and voxels in flight per thread. 2 x 128^3 voxels x 64 channels: forward
// 370 us with its statistics (123), with 4 blocks 379, with 2 voxels 402; backward 372, with 4 blocks in the sums 399, with 2
// voxels in them 380, with 3 blocks in dx 386, with 4 voxels in dx 377. Alone: apply 244 us (5.6 TB/s), sums 156 (5.3), dx
// 212 (6.4).
constexpr int GN8_WAVE_APPLY = 3, GN8_WAVE_SUMS = 3, GN8_WAVE_DX = 4;
constexpr int GN8_U_APPLY = 4, GN8_U_SUMS = 4, GN8_U_DX = 2;

struct Gn8Params {
  const __nv_bfloat16* x;
  const __nv_bfloat16* dy;
  __nv_bfloat16* y;  // forward output / backward dx
  uint8_t* q;        // [N S C] int8
  uint8_t* exps;     // [N S C / 16]
  const float* w;
  const float* b;
  float* mean;
  float* rstd;
  const float* fin;  // forward: [N][G][3] statistics; dx: [N][C][2] sums
  float* part;       // [N][nsplit][C][2]
  float* dw;
  float* db;
  int N, C, G, nsplit, relu, accumulate;
  long long S;
  float eps, group_elems;
};

__device__ __forceinline__ void gn8_unpack(const uint4& v, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ uint4 gn8_pack(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void gn8_values(uint2 q, float step, float (&f)[8]) {
  float lo[4], hi[4];
  kept_unpack4(q.x, lo);
  kept_unpack4(q.y, hi);
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[i] = lo[i] * step; f[4 + i] = hi[i] * step; }
}
// The value's whole number t (plus KEPT_MAGIC) one step further towards the value where its kept form xq lies on the
// other side of the ReLU: y = x a + c there, and a step in the direction of a's sign makes y grow.
__device__ __forceinline__ void gn8_keep_side(float& t, float y, float xq, float a, float c) {
  // (predicated: half of the warps have such a value among a thread's eight)
  asm("{\n\t.reg .pred on, other;\n\t.reg .f32 k, d;\n\t"
      "fma.rn.f32 k, %2, %3, %4;\n\t"
      "setp.gt.f32 on, %1, 0f00000000;\n\t"
      "setp.gt.xor.f32 other, k, 0f00000000, on;\n\t"
      "copysign.f32 d, %3, 0f3F800000;\n\t"
      "@!on neg.f32 d, d;\n\t"
      "@other add.f32 %0, %0, d;\n\t}"
      : "+f"(t)
      : "f"(y), "f"(xq), "f"(a), "f"(c));
}

template <bool RELU>
__global__ void __launch_bounds__(GN8_THREADS, GN8_WAVE_APPLY) gn8_apply_kernel(const Gn8Params p) {
  __shared__ float s_mean[256], s_rstd[256];
  const int n = blockIdx.y;
  for (int g = threadIdx.x; g < p.G; g += GN8_THREADS) {
    const float* e = p.fin + ((long long)n * p.G + g) * 3;
    const float m = e[1], r = rsqrtf(e[2] / e[0] + p.eps);
    s_mean[g] = m;
    s_rstd[g] = r;
    if (blockIdx.x == 0) { p.mean[n * p.G + g] = m; p.rstd[n * p.G + g] = r; }
  }
  __syncthreads();
  const int tpv = p.C / 8, vpb = GN8_THREADS / tpv;
  const int oct = threadIdx.x % tpv, vl = threadIdx.x / tpv;
  const int cg = p.C / p.G;
  float a[8], c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int ch = oct * 8 + i, g = ch / cg;
    a[i] = s_rstd[g] * p.w[ch];
    c[i] = p.b[ch] - s_mean[g] * a[i];
  }
  // The loop is uniform over the block, for the shuffle: a thread without a voxel takes part with zeros. A thread counts
  // the voxels it has left and moves on by `row` elements a voxel (below 2^31: a row of voxels of the whole grid).
  const long long stride = (long long)gridDim.x * vpb, first = (long long)blockIdx.x * vpb;
  const int row = (int)(stride * p.C);
  int left = vl < vpb && first + vl < p.S ? (int)((p.S - first - vl + stride - 1) / stride) : 0;
  long long at = (long long)n * p.S * p.C + (first + vl) * p.C + oct * 8;
  for (int rounds = (int)((p.S - first + GN8_U_APPLY * stride - 1) / (GN8_U_APPLY * stride)); rounds > 0; --rounds) {
    uint4 raw[GN8_U_APPLY];
#pragma unroll
    for (int u = 0; u < GN8_U_APPLY; ++u) {
      raw[u] = make_uint4(0u, 0u, 0u, 0u);
      if (u < left) raw[u] = __ldg(reinterpret_cast<const uint4*>(p.x + at + u * row));
    }
#pragma unroll
    for (int u = 0; u < GN8_U_APPLY; ++u) {
      uint32_t m2 = kept_max2(kept_max2(raw[u].x, raw[u].y), kept_max2(raw[u].z, raw[u].w));
      m2 = kept_max2(m2, __shfl_xor_sync(0xffffffffu, m2, 1));
      const uint32_t b = kept_exponent(max(m2 << 16 & 0x7FFF0000u, m2 & 0x7FFF0000u));
      const float step = kept_step(b), inv = b == 255u ? 0.f : kept_inv(b);
      float f[8], t[8];
      gn8_unpack(raw[u], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        t[i] = fmaf(f[i], inv, KEPT_MAGIC);
        float yv = fmaf(f[i], a[i], c[i]);
        if (RELU) {
          gn8_keep_side(t[i], yv, (t[i] - KEPT_MAGIC) * step, a[i], c[i]);
          asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(yv));  // NaN propagates
        }
        f[i] = yv;
      }
      if (b >= KEPT_TOP_BF16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = b == 255u ? KEPT_MAGIC : kept_cap(t[i]);
      }
      if (u < left) {
        *reinterpret_cast<uint4*>(p.y + at) = gn8_pack(f);
        *reinterpret_cast<uint2*>(p.q + at) =
            make_uint2(kept_pack4(t[0], t[1], t[2], t[3]), kept_pack4(t[4], t[5], t[6], t[7]));
        if ((oct & 1) == 0) p.exps[at / KEPT_BLOCK] = (uint8_t)b;
      }
      at += row;
    }
    left -= GN8_U_APPLY;
  }
}

template <int GP, bool RELU>  // GP: groups that eight consecutive channels cover
__global__ void __launch_bounds__(GN8_THREADS, GN8_WAVE_SUMS) gn8_bwd_partial_kernel(const Gn8Params p) {
  __shared__ float s_a[GN8_THREADS * 8], s_b[GN8_THREADS * 8];
  const int split = blockIdx.x, n = blockIdx.y;
  const int tpv = p.C / 8, vpb = GN8_THREADS / tpv;
  const int oct = threadIdx.x % tpv, vl = threadIdx.x / tpv;
  const int cg = p.C / p.G;
  const long long chunk = (p.S + p.nsplit - 1) / p.nsplit;
  const long long v0 = (long long)split * chunk;
  const long long v1 = v0 + chunk < p.S ? v0 + chunk : p.S;
  float a[8], c[8], A[8], B[8], mu[GP];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int ch = oct * 8 + i, g = ch / cg;
    const float m = p.mean[n * p.G + g];
    if (i % (8 / GP) == 0) mu[i / (8 / GP)] = m;
    a[i] = p.rstd[n * p.G + g] * p.w[ch];
    c[i] = p.b[ch] - m * a[i];
    A[i] = 0.f;
    B[i] = 0.f;
  }
  const long long base = (long long)n * p.S * p.C + oct * 8;
  if (vl < vpb) {
    auto body = [&](const uint2 rq, uint32_t re, const uint4 rd) {
      float fx[8], fd[8];
      gn8_values(rq, kept_step(re), fx);
      gn8_unpack(rd, fd);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float dev = fx[i] - mu[i / (8 / GP)];
        if (RELU) {  // two predicated sums instead of a selection in front of them
          asm("{\n\t.reg .pred off;\n\t.reg .f32 y;\n\t"
              "fma.rn.f32 y, %2, %3, %4;\n\t"
              "setp.le.f32 off, y, 0f00000000;\n\t"
              "@!off add.f32 %0, %0, %5;\n\t"
              "@!off fma.rn.f32 %1, %5, %6, %1;\n\t}"
              : "+f"(A[i]), "+f"(B[i])
              : "f"(fx[i]), "f"(a[i]), "f"(c[i]), "f"(fd[i]), "f"(dev));
        } else {
          A[i] += fd[i];
          B[i] = fmaf(fd[i], dev, B[i]);
        }
      }
    };
    const long long row = (long long)vpb * p.C;
    long long v = v0 + vl, at = base + v * p.C;
    for (; v + (GN8_U_SUMS - 1) * vpb < v1; v += GN8_U_SUMS * vpb, at += GN8_U_SUMS * row) {
      uint2 rq[GN8_U_SUMS];
      uint32_t re[GN8_U_SUMS];
      uint4 rd[GN8_U_SUMS];
#pragma unroll
      for (int u = 0; u < GN8_U_SUMS; ++u) {
        const long long k = at + u * row;
        rq[u] = __ldg(reinterpret_cast<const uint2*>(p.q + k));
        re[u] = __ldg(p.exps + k / KEPT_BLOCK);
        rd[u] = __ldg(reinterpret_cast<const uint4*>(p.dy + k));
      }
#pragma unroll
      for (int u = 0; u < GN8_U_SUMS; ++u) body(rq[u], re[u], rd[u]);
    }
    for (; v < v1; v += vpb, at += row)
      body(__ldg(reinterpret_cast<const uint2*>(p.q + at)), __ldg(p.exps + at / KEPT_BLOCK),
           __ldg(reinterpret_cast<const uint4*>(p.dy + at)));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    s_a[threadIdx.x * 8 + i] = A[i];
    s_b[threadIdx.x * 8 + i] = B[i] * p.rstd[n * p.G + (oct * 8 + i) / cg];
  }
  __syncthreads();
  for (int ch = threadIdx.x; ch < p.C; ch += GN8_THREADS) {
    float sa = 0.f, sb = 0.f;
    for (int v = 0; v < vpb; ++v) {
      const int t = (v * tpv + ch / 8) * 8 + ch % 8;
      sa += s_a[t];
      sb += s_b[t];
    }
    float* dst = p.part + (((long long)n * p.nsplit + split) * p.C + ch) * 2;
    dst[0] = sa;
    dst[1] = sb;
  }
}

template <int GP, bool RELU>
__global__ void __launch_bounds__(GN8_THREADS, GN8_WAVE_DX) gn8_bwd_dx_kernel(const Gn8Params p) {
  __shared__ float s_c1[256], s_c2[256];
  const int n = blockIdx.y;
  const int tpv = p.C / 8, vpb = GN8_THREADS / tpv;
  const int oct = threadIdx.x % tpv, vl = threadIdx.x / tpv;
  const int cg = p.C / p.G;
  const float* fin = p.fin + (long long)n * p.C * 2;
  for (int g = threadIdx.x; g < p.G; g += GN8_THREADS) {
    float c1 = 0.f, c2 = 0.f;
    for (int ch = g * cg; ch < (g + 1) * cg; ++ch) {
      c1 = fmaf(p.w[ch], fin[2 * ch], c1);
      c2 = fmaf(p.w[ch], fin[2 * ch + 1], c2);
    }
    s_c1[g] = c1 / p.group_elems;
    s_c2[g] = c2 / p.group_elems;
  }
  // dweight / dbias: summed over samples in index order
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    for (int ch = threadIdx.x; ch < p.C; ch += GN8_THREADS) {
      float sa = 0.f, sb = 0.f;
      for (int nn = 0; nn < p.N; ++nn) {
        sa += p.fin[((long long)nn * p.C + ch) * 2];
        sb += p.fin[((long long)nn * p.C + ch) * 2 + 1];
      }
      p.db[ch] = p.accumulate ? p.db[ch] + sa : sa;
      p.dw[ch] = p.accumulate ? p.dw[ch] + sb : sb;
    }
  }
  __syncthreads();
  if (vl >= vpb) return;
  // dx = rstd (d w - c1 - xhat c2) = d a + (x - mean) q + r
  float a[8], c[8], mu[GP], q[GP], r[GP];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int ch = oct * 8 + i, g = ch / cg;
    const float rs = p.rstd[n * p.G + g], m = p.mean[n * p.G + g];
    a[i] = rs * p.w[ch];
    c[i] = p.b[ch] - m * a[i];
    if (i % (8 / GP) == 0) {
      mu[i / (8 / GP)] = m;
      q[i / (8 / GP)] = -rs * rs * s_c2[g];
      r[i / (8 / GP)] = -rs * s_c1[g];
    }
  }
  const long long base = (long long)n * p.S * p.C + oct * 8;
  auto body = [&](const uint2 rq, uint32_t re, const uint4 rd, long long at) {
    float fx[8], fd[8];
    gn8_values(rq, kept_step(re), fx);
    gn8_unpack(rd, fd);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float d = fd[i];
      if (RELU && fmaf(fx[i], a[i], c[i]) <= 0.f) d = 0.f;
      fx[i] = fmaf(d, a[i], fmaf(fx[i] - mu[i / (8 / GP)], q[i / (8 / GP)], r[i / (8 / GP)]));
    }
    *reinterpret_cast<uint4*>(p.y + at) = gn8_pack(fx);
  };
  const long long stride = (long long)gridDim.x * vpb, row = stride * p.C;
  long long v = (long long)blockIdx.x * vpb + vl, at = base + v * p.C;
  for (; v + (GN8_U_DX - 1) * stride < p.S; v += GN8_U_DX * stride, at += GN8_U_DX * row) {
    uint2 rq[GN8_U_DX];
    uint32_t re[GN8_U_DX];
    uint4 rd[GN8_U_DX];
#pragma unroll
    for (int u = 0; u < GN8_U_DX; ++u) {
      const long long k = at + u * row;
      rq[u] = __ldg(reinterpret_cast<const uint2*>(p.q + k));
      re[u] = __ldg(p.exps + k / KEPT_BLOCK);
      rd[u] = __ldg(reinterpret_cast<const uint4*>(p.dy + k));
    }
#pragma unroll
    for (int u = 0; u < GN8_U_DX; ++u) body(rq[u], re[u], rd[u], at + u * row);
  }
  for (; v < p.S; v += stride, at += row)
    body(__ldg(reinterpret_cast<const uint2*>(p.q + at)), __ldg(p.exps + at / KEPT_BLOCK),
         __ldg(reinterpret_cast<const uint4*>(p.dy + at)), at);
}

static bool gn8_ok(int N, long long S, int C, int G) {
  return sb_gn_supported(C, G) && C % KEPT_BLOCK == 0 && N >= 1 && N <= 65535 && S >= 1;
}
static void gn8_fill(Gn8Params& p, void* kept, const float* w, const float* b, float* stats, int N, long long S, int C,
                     int G, int relu) {
  memset(&p, 0, sizeof(p));
  p.q = (uint8_t*)kept;
  p.exps = p.q + (long long)N * S * C;
  p.w = w; p.b = b;
  p.mean = stats;
  p.rstd = stats + (long long)N * G;
  p.N = N; p.C = C; p.G = G; p.S = S;
  p.relu = relu;
  p.group_elems = (float)((double)S * (C / G));
}
static int gn8_blocks(const Gn8Params& p, int wave) {
  const int vpb = GN8_THREADS / (p.C / 8);
  const long long need = (p.S + vpb - 1) / vpb, cap = 148LL * wave / p.N;  // one wave
  const long long b = need < cap ? need : cap;
  return (int)(b < 1 ? 1 : b);
}

}  // namespace sb

using namespace sb;

static long long gn8_floats(long long n) { return (n + 63) / 64 * 64; }

// fp32 scratch of the forward (0) and the backward pass (1); -1: outside the kernels' range
extern "C" long long sb_gn8_scratch(int backward, int N, long long S, int C, int G) {
  if (!gn8_ok(N, S, C, G)) return -1;
  if (backward) return gn8_floats((long long)N * sb_gn_bwd_nsplit(N, S, C) * C * 2) + gn8_floats((long long)N * C * 2);
  return gn8_floats((long long)N * sb_gn_nsplit(N, S, C) * G * 3) + gn8_floats((long long)N * G * 3);
}

// fin: the statistics when the tensor's producer has them, else null; hand_over: the statistics kernel's last block
// collapses its partials (not inside a captured graph, see gn_kernels.py)
extern "C" int sb_gn8_forward(const void* x, const float* w, const float* b, int N, long long S, int C, int G, float eps,
                              int relu, const float* fin, int hand_over, void* y, void* kept, float* stats,
                              float* scratch, cudaStream_t stream) {
  if (!gn8_ok(N, S, C, G) || !x || !w || !b || !y || !kept || !stats || (!fin && !scratch)) return SB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(kept)) & 15)
    return SB_ERR_ALIGN;
  if (fin == nullptr) {
    SbGnArgs a;
    memset(&a, 0, sizeof(a));
    a.x = x; a.w = w; a.b = b;
    a.N = N; a.C = C; a.G = G; a.S = a.S_total = S;
    a.eps = eps; a.relu = relu;
    a.nsplit = sb_gn_nsplit(N, S, C);
    a.part = scratch;
    a.parts[0] = scratch;
    a.n_parts = 1;
    float* own = scratch + gn8_floats((long long)N * a.nsplit * G * 3);
    if (hand_over) a.fin = own;
    int rc = sb_gn_stats(&a, stream);
    if (rc == 0 && !hand_over) rc = sb_gn_stats_finalize(scratch, own, N, G, a.nsplit, stream);
    if (rc) return rc;
    fin = own;
  }
  Gn8Params p;
  gn8_fill(p, kept, w, b, stats, N, S, C, G, relu);
  p.x = (const __nv_bfloat16*)x;
  p.y = (__nv_bfloat16*)y;
  p.fin = fin;
  p.eps = eps;
  const dim3 grid(gn8_blocks(p, GN8_WAVE_APPLY), p.N);
  if (relu) gn8_apply_kernel<true><<<grid, GN8_THREADS, 0, stream>>>(p);
  else gn8_apply_kernel<false><<<grid, GN8_THREADS, 0, stream>>>(p);
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

template <int GP, bool RELU>
static int gn8_backward(Gn8Params& p, float* fin, cudaStream_t stream) {
  gn8_bwd_partial_kernel<GP, RELU><<<dim3(p.nsplit, p.N), GN8_THREADS, 0, stream>>>(p);
  sb_count_launch(1);
  const int rc = sb_gn_bwd_finalize(p.part, fin, p.N, p.C, p.nsplit, stream);
  if (rc) return rc;
  p.fin = fin;
  gn8_bwd_dx_kernel<GP, RELU><<<dim3(gn8_blocks(p, GN8_WAVE_DX), p.N), GN8_THREADS, 0, stream>>>(p);
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

extern "C" int sb_gn8_backward(const void* dy, const void* kept, const float* w, const float* b, const float* stats, int N,
                               long long S, int C, int G, int relu, void* dx, float* dw, float* db, int accumulate,
                               float* scratch, cudaStream_t stream) {
  if (!gn8_ok(N, S, C, G) || !dy || !kept || !w || !b || !stats || !dx || !dw || !db || !scratch) return SB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(kept)) & 15)
    return SB_ERR_ALIGN;
  Gn8Params p;
  gn8_fill(p, const_cast<void*>(kept), w, b, const_cast<float*>(stats), N, S, C, G, relu);
  p.dy = (const __nv_bfloat16*)dy;
  p.y = (__nv_bfloat16*)dx;
  p.dw = dw; p.db = db;
  p.accumulate = accumulate;
  p.nsplit = sb_gn_bwd_nsplit(N, S, C);
  p.part = scratch;
  float* fin = scratch + gn8_floats((long long)N * p.nsplit * C * 2);
  const int gp = C / G >= 8 ? 1 : 8 / (C / G);
  if (relu) return gp == 1 ? gn8_backward<1, true>(p, fin, stream) : gp == 2 ? gn8_backward<2, true>(p, fin, stream) : gn8_backward<4, true>(p, fin, stream);
  return gp == 1 ? gn8_backward<1, false>(p, fin, stream) : gp == 2 ? gn8_backward<2, false>(p, fin, stream) : gn8_backward<4, false>(p, fin, stream);
}
