// Cross entropy of a segmentation head with many classes, straight from the features in front of the head:
//   s_ij = x_i . w_j + b_j,  lse_i = log sum_j exp s_ij,  L = sum_i u_i (lse_i - s_i,y(i)) / sum_i u_i,  u_i = class weight
//   p_ij = exp(s_ij - lse_i),  D_ij = g_i (p_ij - [j = y_i]),  g_i = dL u_i / sum u
//   dX = D W,  dW = D^T X,  db_j = sum_i D_ij
// The logits (voxels x classes) are never written: every kernel multiplies the tiles of X and W again, keeps a 128 x 128
// tile of s in tensor memory and uses it up on the chip.
//
// Bias and log-sum-exp ride along the reduction: X and W have sixteen columns more (x16, w16), in which b_j, -lse_i and
// log u_i stand as three bf16 each (24 bits) against ones of the other side, so the tensor cores hand over
// s_ij + b_j - lse_i and an entry costs the epilogue a multiplication by log2(e) and an exponential. Column parameters
// out of shared memory cost it a data-pipe cycle per warp and column each, more than the exponential unit's share.
//
// A CTA keeps tiles of 128 ROWS resident and walks 128-wide tiles of COLUMNS, three kernels:
//   head_rows_kernel  rows = voxels, columns = classes: running maximum and sum of every row (one row per thread, no
//                     exchange between threads), or (ARG) the largest logit and its class
//   head_grad_kernel  HEAD_DX  rows = voxels, columns = classes: P = p - [j = y] in bf16 goes back to tensor memory over
//                     the tile of s it came from, and acc[128][C] += P W is the second MMA with P as its A operand (W's
//                     tile is the same shared memory, read MN-major); the row's g multiplies the finished sum
//                     HEAD_DW  rows = classes, columns = voxels: the same with X and W exchanged, P = u (p - [j = y]); a
//                     row of P^T is a class, so db is a sum inside a thread; dL / sum u multiplies the finished sums
//   head_both_kernel  both gradients from one P, where the weight and its gradient fit into a CTA
//
// Roundings. P has 8 significant bits, all sums are fp32. The target's one is taken off in fp32, before the rounding:
// behind it a confident voxel (p near 1) would keep nothing but the rounding of p. Common factors stay out of P, so that
// a target's entry is near -1 (exact when p is small) instead of -1 / V, whose rounding error all voxels would share.
// Where one rounding can make up a result (LO: up to HD_FEW voxels; class weights in HEAD_DW, whose rounding the voxels
// of a class share; head_both_kernel weighs X instead) P is kept as two bf16, value and remainder, and the second MMA runs once for each.
//
// Roles: warp 0 loads (TMA), warps 1 and 2 issue MMAs, warps 3-18 are the epilogue, four groups of four warps (a row per
// thread). All waits are bounded.
// Two issuing warps: one is never more than about an MMA ahead of the tensor pipe and loses some 100 clocks at each wait
// and some 300 at each commit, during which only the other one's MMAs can run. head_grad_kernel: warp 1 the first MMAs
// (as many tiles ahead as tensor memory holds), warp 2 the second ones; head_rows_kernel: two groups' tiles each. One
// warp for everything took 2150 clocks a tile at 64 channels, the exponentials left out or not.
#include <limits.h>

#include <atomic>

#include "head_loss.cuh"

namespace sb {

constexpr int HD_EPI_WARPS = 16;
constexpr int HD_FIRST_EPI = 3;
constexpr int HD_THREADS = 32 * (HD_FIRST_EPI + HD_EPI_WARPS);
constexpr int HD_TILE = 128;
constexpr int HD_BOX = HD_TILE * 128;  // bytes of a 128-row box of 64 channels
constexpr int HD_BOX16 = HD_TILE * 32; // and of the sixteen columns more
constexpr int HD_MAX_STAGES = 8;
// TMEM: two or three tiles of s and the accumulator in 512 columns. At that width head_wide.cu is slower still: dX of 131072
// voxels x 256 channels x 2048 classes 238 us here and 570 there.
constexpr int HD_MAX_C = 256;

enum HeadMode { HEAD_ROWS = 0, HEAD_DX = 1, HEAD_DW = 2, HEAD_BOTH = 3 };

struct HeadParams {
  CUtensorMap mapR, mapQ, mapR16, mapQ16;  // rows and columns, and their sixteen columns more
  CUtensorMap mapO;                        // both: dX
  const int* coly;      // DW: label (-1: none)
  const float* roww;    // DW: class weight of a row, or null
  const float* rowg;    // DX: g of a voxel
  // both: a column's label (16 bits, all ones: it takes no part) and p - 1 of it (bf16); its log2 of the sum of
  // exponentials; dL, the loss's denominator and where their quotient goes
  const uint32_t* colhit;
  const float* lse2;
  const float* gout;
  const float* den;
  float* scale;
  const int* rowy;      // ROWS / DX: label
  float2* part;         // ROWS: [splits, times four with `together` 1][rows padded] running maximum and sum
  float* tl;            // ROWS: [rows padded] s log2(e) at the label
  // ROWS, `whole`: a thread has all of a row, so what head_merge_kernel would make of it is made here (and cw, or null)
  int whole;
  float* lse2_out;
  uint32_t* hit_out;    // or null
  const float* cw;
  const void* bias;
  int bias_kind;
  double* sums;         // [CTAs][2]
  __nv_bfloat16* out;   // DX with one split: [rows][C]
  float* ws;            // DX / DW: [splits][rows padded][cpad]
  float* ws_b;          // DW: [4 splits][rows padded]
  uint32_t* status;
  long long rows, cols, rows_pad;
  int C, cpad, kboxes, ksteps;
  int row_tiles, col_tiles, splits, tiles_per_split;
  int stages, rbufs, bufs, accs;
  int row0;             // both: first class of this launch
  float4* part_x;       // both: dX of the launches so far, [voxel tiles][cpad / 4][128]
  int first, last;      // both: nothing to add, nothing to keep
  int together;         // ROWS: row tiles of a job, 4 or 1
};

// D[tmem] (+)= A[tmem] * B[smem]: A holds two bf16 of K per 32-bit column, one row per lane
__device__ __forceinline__ void hd_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void hd_tmem_st_x16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void hd_tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void hd_tma_store_2d(const CUtensorMap* m, const void* src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void bulk_wait_read_all() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void hd_sts4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float2 hd_lds2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void hd_sts16(uint32_t at, uint32_t v) {
  asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"((uint16_t)v) : "memory");
}
// two fp32 in one instruction
__device__ __forceinline__ float2 hd_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 hd_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// a number as three bf16 that add up to it (two in the first word, one in the second)
__device__ __forceinline__ uint2 hd_three(float v) {
  const __nv_bfloat16 a = __float2bfloat16(v);
  float rest = v - __bfloat162float(a);
  if (!isfinite(rest)) rest = 0.f;  // an infinity or a NaN is all in the first
  const __nv_bfloat16 b = __float2bfloat16(rest), c = __float2bfloat16(rest - __bfloat162float(b));
  return make_uint2((uint32_t)__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16,
                    (uint32_t)__bfloat16_as_ushort(c));
}
constexpr uint32_t HD_ONE = 0x3F80u;  // 1 in bf16

__device__ __forceinline__ float hd_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// A row's sum of powers of two, held finite (a NaN stays). Beyond |m| of some 1e9 (a run of classes that their biases turn
// off) m log2(e) less its nearest fp32, the exponent of the maximum itself, may be some hundred and more. Where other classes
// follow, what such a run left is multiplied by zero, which an infinity would not survive; else it is below m's rounding.
__device__ __forceinline__ void hd_hold(float& s) { asm("min.NaN.f32 %0, %0, 0f7149F2CA;" : "+f"(s)); }  // 1e30
// where `bits & bit`: v -= d; predicated, never a branch
__device__ __forceinline__ void hd_sub_if(float& v, float d, uint32_t bits, uint32_t bit) {
  asm("{\n\t.reg .pred q;\n\t.reg .b32 t;\n\tand.b32 t, %2, %3;\n\tsetp.ne.u32 q, t, 0;\n\t@q sub.f32 %0, %0, %1;\n\t}"
      : "+f"(v)
      : "f"(d), "r"(bits), "r"(bit));
}
// s = R Q^T of a tile: the sixteen columns more, then the channels
__device__ __forceinline__ void hd_first_mma(uint32_t d, uint32_t r, uint32_t r16, uint32_t q, uint32_t q16, int cols,
                                             int ksteps) {
  const uint32_t hi = desc_hi(8u * 128u, 2u), hi16 = desc_hi(8u * 32u, 6u);
  const uint32_t idesc = make_idesc_bf16(128, cols, 0, 0);
  const uint32_t a_lo = desc_lo(r, 16u), b_lo = desc_lo(q, 16u);
  tc_mma_bf16_pred(d, desc_lo(r16, 16u), hi16, desc_lo(q16, 16u), hi16, idesc, 0u);
  for (int k = 0; k < ksteps; ++k) {
    const uint32_t off = (uint32_t)(k >> 2) * (HD_BOX >> 4) + (uint32_t)(k & 3) * 2u;
    tc_mma_bf16_pred(d, a_lo + off, hi, b_lo + off, hi, idesc, 1u);
  }
}

struct HeadSum {
  double num, den;
};
// the sums over a block's warps, in thread 0; all its threads take part
template <int WARPS>
__device__ __forceinline__ HeadSum hd_block_sum(HeadSum a) {
  __shared__ double s_n[WARPS], s_d[WARPS];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.num += __shfl_xor_sync(0xffffffffu, a.num, o);
    a.den += __shfl_xor_sync(0xffffffffu, a.den, o);
  }
  if ((threadIdx.x & 31) == 0) { s_n[threadIdx.x >> 5] = a.num; s_d[threadIdx.x >> 5] = a.den; }
  __syncthreads();
  HeadSum t{0.0, 0.0};
  if (threadIdx.x == 0)
    for (int w = 0; w < WARPS; ++w) { t.num += s_n[w]; t.den += s_d[w]; }
  return t;
}

// bias: null, bf16 (kind 0) or fp32
__device__ __forceinline__ float hd_bias(const void* bias, int kind, long long i) {
  return bias == nullptr ? 0.f
         : kind == 0     ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(bias)[i])
                         : reinterpret_cast<const float*>(bias)[i];
}
// A voxel's log2 of the sum of exponentials, from maximum (log2) and sum; u nll and u are added, and the label's p - 1 and
// the label go to `hit`. i < V; y -1: takes no part. A label whose class its bias turns off (-inf, or the type's lowest
// number) was given HD_LOWEST or -inf as its logit: the bias itself takes that place, the products beside it are below its
// rounding.
__device__ __forceinline__ float hd_voxel(float m2, float sum, float tl, int y, const float* cw, const void* bias,
                                          int bias_kind, HeadSum& a, uint32_t& hit) {
  const float l = m2 < 0.1f * HD_LOWEST ? NAN : m2 + log2f(sum);  // every class is off: 0 / 0
  hit = 0xFFFFu;
  if (y >= 0) {
    const float u = cw == nullptr ? 1.f : cw[y], t = l - tl;
    double nll = (double)t * (double)HD_LN2;
    if (tl < 0.1f * HD_LOWEST) {
      const float b = hd_bias(bias, bias_kind, y);
      if (b < HD_LOWEST) nll = (double)l * (double)HD_LN2 - (double)b;
    }
    if (u != 0.f) a.num += (double)u * nll;  // (a class of weight zero takes no part: not 0 * inf)
    a.den += (double)u;
    hit = (uint32_t)__bfloat16_as_ushort(__float2bfloat16(expm1f(-t * HD_LN2))) << 16 | ((uint32_t)y & 0xFFFFu);
  }
  return l;
}

// Log-sum-exp of the rows (or ARG: their largest logit). Tensor memory holds four tiles of s, one for each epilogue group.
//   together = 4: a job is four row tiles by a run of column tiles; group g has row tile g all along, so a column tile is
//                 loaded once for 512 rows and a row's statistics stay in one thread: nothing is merged in the CTA
//   together = 1: a job is one row tile; group g takes every fourth column tile and leaves statistics of its own
// The second one is for calls that have no four row tiles for every SM, and for tiles of which shared memory holds few.
// `whole`: four row tiles and all columns in a job, so a thread ends with all of a row and makes the voxel's term of the loss
// and what the backward pass needs itself; else head_merge_kernel does, from the shares (2 x 128^3 voxels, 16 channels, 34
// classes: 136 instead of 215 us; 16^3: 14 instead of 25).
// Row tiles come in twice the number of a job, so that the next job's are there when this one ends (485 -> 427 us for the
// whole loss below). Bound: the exponential unit, 1024 clocks a tile of 128 x 128, at long runs of columns (75 % of it at
// 500 classes), and between jobs the way of a tile through tensor memory. 2 x 128^3 voxels, 64 channels and 257 classes: 381
// us (237 for the exponentials alone). Merging two halves of a tile's columns over two groups by tile parity instead (a
// barrier and an exchange in every job): 631.
template <bool ARG>
__global__ void __launch_bounds__(HD_THREADS, 1) head_rows_kernel(const __grid_constant__ HeadParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t r_full[8], r_empty[8], q_full[HD_MAX_STAGES], q_empty[HD_MAX_STAGES], s_full[4], s_done[4];
  __shared__ uint32_t tmem_base_s, abort_s;
  volatile uint32_t* abort_flag = &abort_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool four = p.together == 4;
  const int row_jobs = four ? (p.row_tiles + 3) / 4 : p.row_tiles, jobs = row_jobs * p.splits;
  const uint32_t box16 = (uint32_t)p.kboxes * HD_BOX, tile_bytes = box16 + HD_BOX16;
  uint8_t* smem_r = smem;
  uint8_t* smem_q = smem + (size_t)p.rbufs * box16;
  uint8_t* smem_r16 = smem_q + (size_t)p.stages * tile_bytes;  // the rows' columns more, of all rows the same

  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int i = 0; i < p.rbufs; ++i) {
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], four ? 1 : 2);  // a row tile of several is one issuing warp's, a single one both warps'
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_done[i], HD_EPI_WARPS / 4);
    }
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], four ? 2 : 1);
    }
    mbar_fence_init();
  }
  if (threadIdx.x < HD_TILE) {
    // ones against the three parts of the bias (32-byte rows, 16-byte halves exchanged in every second group of four rows:
    // the 32-byte swizzle)
    uint4* at = reinterpret_cast<uint4*>(smem_r16 + threadIdx.x * 32);
    const int half = (threadIdx.x >> 2) & 1;
    at[half] = make_uint4(0x3F803F80u, 0x00003F80u, 0u, 0u);
    at[half ^ 1] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_base_s, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  const int last_cols = ((int)(p.cols - (long long)(p.col_tiles - 1) * HD_TILE) + 31) & ~31;
  auto cols_of = [&](int t) -> int { return t + 1 < p.col_tiles ? HD_TILE : last_cols; };  // up to a multiple of 32

  HeadSum total{0.0, 0.0};
  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&p.mapR);
      tma_prefetch_desc(&p.mapQ);
      uint32_t rb = 0, rph = 0, st = 0, ph = 0;
      bool ok = true;
      for (int job = blockIdx.x; job < jobs && ok; job += gridDim.x) {
        const int rt = job % row_jobs * p.together, sp = job / row_jobs;
        const int t0 = sp * p.tiles_per_split;
        const int t1 = t0 + p.tiles_per_split < p.col_tiles ? t0 + p.tiles_per_split : p.col_tiles;
        for (int t = t0; t < t1 && ok; ++t) {
          // the column tile, and in front of the first one the row tiles (each as soon as its last one is done with)
          for (int g = 0; t == t0 && g < p.together; ++g) {
            if (!mbar_wait(&r_empty[rb], rph ^ 1u, abort_flag, p.status, 91)) { ok = false; break; }
            mbar_expect_tx(&r_full[rb], box16);
            for (int k = 0; k < p.kboxes; ++k)
              hd_tma_2d(smem_r + rb * box16 + k * HD_BOX, &p.mapR, &r_full[rb], k * 64, (rt + g) * HD_TILE);
            if (++rb == (uint32_t)p.rbufs) { rb = 0; rph ^= 1u; }
          }
          if (!ok || !mbar_wait(&q_empty[st], ph ^ 1u, abort_flag, p.status, 91)) { ok = false; break; }
          mbar_expect_tx(&q_full[st], tile_bytes);
          for (int k = 0; k < p.kboxes; ++k)
            hd_tma_2d(smem_q + st * tile_bytes + k * HD_BOX, &p.mapQ, &q_full[st], k * 64, t * HD_TILE);
          hd_tma_2d(smem_q + st * tile_bytes + box16, &p.mapQ16, &q_full[st], 0, t * HD_TILE);
          if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
        }
      }
    }
  } else if (warp <= 2) {
    const bool leader = elect_one();
    const uint32_t mine = (uint32_t)warp - 1u;
    const uint32_t r0 = smem_u32(smem_r), r16 = smem_u32(smem_r16), q0 = smem_u32(smem_q);
    uint32_t rb = 0, rph = 0, st = 0, ph = 0, fi = 0;  // fi: column tiles so far (together = 1)
    uint32_t uses[2] = {0u, 0u};                       // of this warp's two tiles of s
    bool ok = true;
    // one tile into buffer g: rows out of r_slot, columns out of the current stage
    auto tile = [&](uint32_t g, uint32_t r_slot, int t) -> bool {
      const uint32_t u = uses[g >> 1]++;
      if (!hd_wait(&s_done[g], (u & 1u) ^ 1u, abort_flag, p.status, 96)) return false;
      tc_fence_after();
      if (leader) {
        const uint32_t q = q0 + st * tile_bytes;
        hd_first_mma(tmem + g * HD_TILE, r0 + r_slot * box16, r16, q, q + box16, cols_of(t), p.ksteps);
        tc_commit(&s_full[g]);
      }
      __syncwarp();
      return true;
    };
    for (int job = blockIdx.x; job < jobs && ok; job += gridDim.x) {
      const int sp = job / row_jobs;
      const int t0 = sp * p.tiles_per_split;
      const int t1 = t0 + p.tiles_per_split < p.col_tiles ? t0 + p.tiles_per_split : p.col_tiles;
      bool used = false;
      if (!four && !hd_wait(&r_full[rb], rph, abort_flag, p.status, 94)) break;
      for (int t = t0; t < t1 && ok; ++t, ++fi) {
        if (four || (fi & 1u) == mine) {
          if (!hd_wait(&q_full[st], ph, abort_flag, p.status, 95)) { ok = false; break; }
          if (four) {
            for (uint32_t g = mine; g < 4u && ok; g += 2u) {
              if (t == t0) ok = hd_wait(&r_full[rb + g], rph, abort_flag, p.status, 94);
              ok = ok && tile(g, rb + g, t);
              if (ok && leader && t == t1 - 1) tc_commit(&r_empty[rb + g]);
              __syncwarp();
            }
          } else {
            ok = tile(fi & 3u, rb, t);
            used = true;
          }
          if (ok && leader) tc_commit(&q_empty[st]);
          __syncwarp();
        }
        if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
      }
      if (!four) {
        if (ok && leader) {  // this warp is done with the resident tile
          if (used) tc_commit(&r_empty[rb]);
          else mbar_arrive(&r_empty[rb]);
        }
        __syncwarp();
      }
      rb += p.together;
      if (rb == (uint32_t)p.rbufs) { rb = 0; rph ^= 1u; }
    }
  } else {
    const int quad = warp & 3, group = (warp - HD_FIRST_EPI) >> 2;
    const uint32_t tile = tmem + ((uint32_t)(quad * 32) << 16) + group * HD_TILE;
    uint32_t uses = 0, fi = 0;
    bool ok = true;
    int rt = blockIdx.x % row_jobs, sp = blockIdx.x / row_jobs;
    auto row_of = [&](int j) { return ((long long)(four ? j * 4 + group : j)) * HD_TILE + quad * 32 + lane; };
    auto label_of = [&](int j) { return !ARG && row_of(j) < p.rows_pad ? __ldg(p.rowy + row_of(j)) : -1; };
    int y_next = label_of(rt);
    while (sp < p.splits && ok) {
      const int t0 = sp * p.tiles_per_split;
      const int t1 = t0 + p.tiles_per_split < p.col_tiles ? t0 + p.tiles_per_split : p.col_tiles;
      const long long r = row_of(rt);
      const int y = y_next, slot = four ? sp : sp * 4 + group;
      rt += gridDim.x;
      if (rt >= row_jobs) {
        sp += rt / row_jobs;
        rt %= row_jobs;
      }
      if (sp < p.splits) y_next = label_of(rt);
      float m = ARG ? -INFINITY : HD_LOWEST, s = 0.f, tl = 0.f;
      bool met = false;
      int best = INT_MAX;
      int t = four ? t0 : t0 + (int)((group - fi) & 3u);
      fi += t1 - t0;
      for (; t < t1; t += four ? 1 : 4, ++uses) {
        if (!hd_wait(&s_full[group], uses & 1u, abort_flag, p.status, 98)) { ok = false; break; }
        tc_fence_after();
        const int nc = cols_of(t), c_abs = t * HD_TILE;
#pragma unroll 1
        for (int c0 = 0; c0 < nc; c0 += 32) {
          uint32_t v[32];
          tmem_ld_32x32(tile + c0, v);
          tmem_ld_wait();
          if (c0 + 32 >= nc) {  // read to the end: the next tile may come
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_done[group]);
          }
          float f[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]);
          if (ARG) {
            // columns behind the last class take no part: zeros of w there, and 0 * inf of a feature is a NaN
            const int left = (int)p.cols - (c_abs + c0);
            if (left < 32) {
#pragma unroll
              for (int j = 0; j < 32; ++j) f[j] = j < left ? f[j] : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (f[j] > m || (f[j] != f[j] && m == m)) { m = f[j]; best = c_abs + c0 + j; }
          } else {
            const int at = y - (c_abs + c0);
            const bool hit = (unsigned)at < 32u;
            if (__any_sync(0xffffffffu, hit)) {  // f[at], by halves
              float h[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) h[j] = at & 16 ? f[16 + j] : f[j];
#pragma unroll
              for (int n = 8; n > 0; n >>= 1)
#pragma unroll
                for (int j = 0; j < n; ++j) h[j] = at & n ? h[n + j] : h[j];
              if (hit) { tl = h[0]; met = true; }
            }
            float mx[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mx[j] = hd_max3(f[8 * j], f[8 * j + 1], f[8 * j + 2]);
              mx[j] = hd_max3(mx[j], f[8 * j + 3], f[8 * j + 4]);
              mx[j] = hd_max3(mx[j], f[8 * j + 5], f[8 * j + 6]);
              mx[j] = fmaxf(mx[j], f[8 * j + 7]);
            }
            const float top = hd_max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
            if (top > m) {
              s *= hd_ex2((m - top) * HD_LOG2E);
              m = top;
            }
            const float2 scale = make_float2(HD_LOG2E, HD_LOG2E), base = make_float2(-m * HD_LOG2E, -m * HD_LOG2E);
            float2 a[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float2 t = hd_fma2(make_float2(f[j], f[j + 1]), scale, base);
              a[j / 2 & 1] = hd_add2(a[j / 2 & 1], make_float2(hd_ex2(t.x), hd_ex2(t.y)));
            }
            a[0] = hd_add2(a[0], a[1]);
            s += a[0].x + a[0].y;
            hd_hold(s);
          }
        }
      }
      if (!ARG && p.whole) {
        if (ok && r < p.rows_pad) {
          uint32_t hit = 0xFFFFu;
          p.lse2_out[r] = r < p.rows ? hd_voxel(m * HD_LOG2E, s, tl * HD_LOG2E, y, p.cw, p.bias, p.bias_kind, total, hit)
                                       : INFINITY;
          if (p.hit_out != nullptr) p.hit_out[r] = hit;
        }
      } else if (ok && r < p.rows_pad) {
        p.part[(long long)slot * p.rows_pad + r] = ARG ? make_float2(m, __int_as_float(best)) : make_float2(m * HD_LOG2E, s);
        if (!ARG && met) p.tl[r] = tl * HD_LOG2E;
      }
    }
  }

  if (!ARG && p.whole) {
    __syncwarp();
    total = hd_block_sum<HD_THREADS / 32>(total);
    if (threadIdx.x == 0) { p.sums[2 * blockIdx.x] = total.num; p.sums[2 * blockIdx.x + 1] = total.den; }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 0) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One gradient (the header has the mathematics). Two or three tiles of s in tensor memory, whose P replaces it: two groups
// take a tile's halves, by tile parity. Bound: the instructions of the epilogue (about 8 an entry, 2300 clocks a tile of 128
// x 128, of which the exponential unit takes 1024), three of them for the target in its row. 2 x 128^3 voxels, 64 channels
// and 257 classes: 540 us each for dX and dW; 2^20 voxels and 512 classes 213 and 224 with all that stands around them.
template <int MODE, bool LO>
__global__ void __launch_bounds__(HD_THREADS, 1) head_grad_kernel(const __grid_constant__ HeadParams p) {
  constexpr int MAXB = 3;
  const uint32_t NB = (uint32_t)p.bufs;          // tiles of s in tensor memory
  const uint32_t ACC = NB * HD_TILE;             // column of the accumulators
  const uint32_t naccs = (uint32_t)p.accs;       // one or two, 64 columns apart: a job goes on while the last one's is read
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t r_full[2], r_empty[2], q_full[HD_MAX_STAGES], q_empty[HD_MAX_STAGES], s_full[MAXB], s_done[MAXB],
      acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base_s, abort_s;
  volatile uint32_t* abort_flag = &abort_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int jobs = p.row_tiles * p.splits;
  const uint32_t box16 = (uint32_t)p.kboxes * HD_BOX;  // where the sixteen columns more are
  const uint32_t tile_bytes = box16 + HD_BOX16;
  uint8_t* smem_r = smem;
  uint8_t* smem_q = smem + (size_t)p.rbufs * tile_bytes;

  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int i = 0; i < 2; ++i) { mbar_init(&r_full[i], 1); mbar_init(&r_empty[i], 1); }
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < MAXB; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_done[i], HD_EPI_WARPS / 2);
    }
    for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], HD_EPI_WARPS); }
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_base_s, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  const int last_cols = ((int)(p.cols - (long long)(p.col_tiles - 1) * HD_TILE) + 31) & ~31;
  auto cols_of = [&](int t) -> int { return t + 1 < p.col_tiles ? HD_TILE : last_cols; };  // up to a multiple of 32

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&p.mapR);
      tma_prefetch_desc(&p.mapQ);
      uint32_t rb = 0, rph = 0, st = 0, ph = 0;
      bool ok = true;
      for (int job = blockIdx.x; job < jobs && ok; job += gridDim.x) {
        const int rt = job % p.row_tiles, sp = job / p.row_tiles;
        const int t0 = sp * p.tiles_per_split;
        const int t1 = t0 + p.tiles_per_split < p.col_tiles ? t0 + p.tiles_per_split : p.col_tiles;
        if (!mbar_wait(&r_empty[rb], rph ^ 1u, abort_flag, p.status, 91)) break;
        mbar_expect_tx(&r_full[rb], tile_bytes);
        for (int k = 0; k < p.kboxes; ++k)
          hd_tma_2d(smem_r + rb * tile_bytes + k * HD_BOX, &p.mapR, &r_full[rb], k * 64, rt * HD_TILE);
        hd_tma_2d(smem_r + rb * tile_bytes + box16, &p.mapR16, &r_full[rb], 0, rt * HD_TILE);
        if (++rb == (uint32_t)p.rbufs) { rb = 0; rph ^= 1u; }
        for (int t = t0; t < t1; ++t) {
          if (!mbar_wait(&q_empty[st], ph ^ 1u, abort_flag, p.status, 91)) { ok = false; break; }
          mbar_expect_tx(&q_full[st], tile_bytes);
          for (int k = 0; k < p.kboxes; ++k)
            hd_tma_2d(smem_q + st * tile_bytes + k * HD_BOX, &p.mapQ, &q_full[st], k * 64, t * HD_TILE);
          hd_tma_2d(smem_q + st * tile_bytes + box16, &p.mapQ16, &q_full[st], 0, t * HD_TILE);
          if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t r0 = smem_u32(smem_r), q0 = smem_u32(smem_q);
    uint32_t rb = 0, rph = 0, st = 0, ph = 0, b = 0, tc = 0;
    uint32_t old_st = 0, old_ph = 0;  // the tile that had this one's buffer
    bool ok = true;
    for (int job = blockIdx.x; job < jobs && ok; job += gridDim.x) {
      const int sp = job / p.row_tiles;
      const int t0 = sp * p.tiles_per_split;
      const int t1 = t0 + p.tiles_per_split < p.col_tiles ? t0 + p.tiles_per_split : p.col_tiles;
      if (!hd_wait(&r_full[rb], rph, abort_flag, p.status, 94)) { ok = false; break; }
      for (int t = t0; t < t1; ++t, ++tc) {
        // the buffer is free: its P was read by the second MMA that used it
        if (tc >= NB) {
          if (!hd_wait(&q_empty[old_st], old_ph, abort_flag, p.status, 96)) { ok = false; break; }
          if (++old_st == (uint32_t)p.stages) { old_st = 0; old_ph ^= 1u; }
        }
        if (!hd_wait(&q_full[st], ph, abort_flag, p.status, 95)) { ok = false; break; }
        tc_fence_after();
        if (leader) {
          const uint32_t r = r0 + rb * tile_bytes, q = q0 + st * tile_bytes;
          hd_first_mma(tmem + b * HD_TILE, r, r + box16, q, q + box16, cols_of(t), p.ksteps);
          tc_commit(&s_full[b]);
          if (t == t1 - 1) tc_commit(&r_empty[rb]);
        }
        __syncwarp();
        if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
        if (++b == NB) b = 0;
      }
      if (++rb == (uint32_t)p.rbufs) { rb = 0; rph ^= 1u; }
    }
  } else if (warp == 2) {
    // acc += P Q of a tile, P out of the buffer of s
    const bool leader = elect_one();
    const uint32_t hi = desc_hi(8u * 128u, 2u);
    const uint32_t q0 = smem_u32(smem_q);
    const uint32_t idesc = make_idesc_bf16(128, p.cpad, 0, 1);
    const uint32_t lbo = p.kboxes > 1 ? (uint32_t)HD_BOX : 0u;
    uint32_t st = 0, ph = 0, b = 0, bph = 0, ab = 0, aph = 0;
    bool ok = true;
    for (int job = blockIdx.x; job < jobs && ok; job += gridDim.x) {
      const int sp = job / p.row_tiles;
      const int t0 = sp * p.tiles_per_split;
      const int t1 = t0 + p.tiles_per_split < p.col_tiles ? t0 + p.tiles_per_split : p.col_tiles;
      if (!hd_wait(&acc_empty[ab], aph ^ 1u, abort_flag, p.status, 92)) { ok = false; break; }
      const uint32_t acc = tmem + ACC + ab * 64u;
      for (int t = t0; t < t1; ++t) {
        const int ksteps = cols_of(t) / 16;
        const uint32_t lo = desc_lo(q0 + st * tile_bytes, lbo);
        const uint32_t a = tmem + b * HD_TILE;
        // (the other issuing warp has waited for the tile's loads; this one has to see them too)
        if (!(hd_wait(&q_full[st], ph, abort_flag, p.status, 95) &&
              hd_wait(&s_done[b], bph, abort_flag, p.status, 93))) { ok = false; break; }
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int part = 0; part < (LO ? 2 : 1); ++part)
            for (int k = 0; k < ksteps; ++k)
              hd_mma_ts(acc, a + 32 * (k >> 1) + 16 * part + 8 * (k & 1), lo + k * 128u, hi, idesc,
                        t == t0 && part == 0 && k == 0 ? 0u : 1u);
          tc_commit(&q_empty[st]);
          if (t == t1 - 1) tc_commit(&acc_full[ab]);
        }
        __syncwarp();
        if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
        if (++b == NB) { b = 0; bph ^= 1u; }
      }
      if (++ab == naccs) { ab = 0; aph ^= 1u; }
    }
  } else {
    const int quad = warp & 3, group = (warp - HD_FIRST_EPI) >> 2, half = group & 1;
    const uint32_t par = group >> 1;
    const int row = quad * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    uint32_t b = par, bph = 0, ab = 0, aph = 0, tc = 0;  // b: buffer of this group's next tile (two or more there are)
    bool ok = true, pending = false;
    int pend_rt = 0, pend_sp = 0;
    float pend_g = 0.f, pend_db = 0.f;
    uint32_t rank_bits[5];  // HEAD_DW: all ones where the lane's number has a zero
    if (MODE == HEAD_DW) {
#pragma unroll
      for (int k = 0; k < 5; ++k) rank_bits[k] = lane >> k & 1 ? 0u : ~0u;
    }
    // the accumulator of a finished job
    auto drain = [&]() -> bool {
      if (!hd_wait(&acc_full[ab], aph, abort_flag, p.status, 97)) return false;
      tc_fence_after();
      const long long r = (long long)pend_rt * HD_TILE + row;
      for (int c0 = group * 16; c0 < p.cpad; c0 += 64) {
        uint32_t v[16];
        tmem_ld_32x16(lane_base + ACC + ab * 64u + c0, v);
        tmem_ld_wait();
        float f[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = __uint_as_float(v[j]);
        if (MODE == HEAD_DX) {
          // a voxel that takes no part has no gradient, whatever its features hold
#pragma unroll
          for (int j = 0; j < 16; ++j) f[j] = pend_g == 0.f ? 0.f : f[j] * pend_g;
        }
        if (MODE == HEAD_DX && p.splits == 1) {
          if (r < p.rows) {
            uint4* dst = reinterpret_cast<uint4*>(p.out + r * p.C + c0);
            dst[0] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                                pack_bf16x2(f[6], f[7]));
            if (c0 + 8 < p.C)
              dst[1] = make_uint4(pack_bf16x2(f[8], f[9]), pack_bf16x2(f[10], f[11]), pack_bf16x2(f[12], f[13]),
                                  pack_bf16x2(f[14], f[15]));
          }
        } else {
          float4* dst = reinterpret_cast<float4*>(p.ws + ((long long)pend_sp * p.rows_pad + r) * p.cpad + c0);
#pragma unroll
          for (int j = 0; j < 4; ++j) dst[j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
        }
      }
      if (MODE == HEAD_DW) p.ws_b[((long long)pend_sp * 4 + group) * p.rows_pad + r] = pend_db;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[ab]);
      if (++ab == naccs) { ab = 0; aph ^= 1u; }
      return true;
    };
    // a row's own values; the next job's are read while this one runs
    int y_next = -1;
    float g_next = 1.f;
    auto fetch = [&](int rt) {
      const long long r = (long long)rt * HD_TILE + row;
      if (MODE == HEAD_DX) {
        y_next = __ldg(p.rowy + r);
        g_next = __ldg(p.rowg + r);
      }
      if (MODE == HEAD_DW && p.roww != nullptr && r < p.rows) g_next = __ldg(p.roww + r);
    };
    int rt = blockIdx.x % p.row_tiles, sp = blockIdx.x / p.row_tiles;
    fetch(rt);
    while (sp < p.splits && ok) {
      const int t0 = sp * p.tiles_per_split;
      const int t1 = t0 + p.tiles_per_split < p.col_tiles ? t0 + p.tiles_per_split : p.col_tiles;
      const long long r = (long long)rt * HD_TILE + row;
      const int y = y_next;
      const float g = g_next;
      int next_rt = rt + gridDim.x, next_sp = sp;
      if (next_rt >= p.row_tiles) {
        next_sp += next_rt / p.row_tiles;
        next_rt %= p.row_tiles;
      }
      if (next_sp < p.splits) fetch(next_rt);
      float db = 0.f;
      // this group's tiles of the job: every second one over all jobs
      int t = t0 + (int)((tc ^ par) & 1u);
      tc += t1 - t0;
      const int* labels = MODE == HEAD_DW ? p.coly + half * 64 + lane : nullptr;
      int label[2] = {-1, -1};  // HEAD_DW: of the tile's column `lane`, and 32 further; a tile ahead
      if (MODE == HEAD_DW && t < t1) {
        label[0] = __ldg(labels + (long long)t * HD_TILE);
        label[1] = __ldg(labels + (long long)t * HD_TILE + 32);
      }
      for (; t < t1; t += 2) {
        if (!hd_wait(&s_full[b], bph, abort_flag, p.status, 98)) { ok = false; break; }
        int rel[2] = {label[0] - (int)(r - lane), label[1] - (int)(r - lane)};
        if (MODE == HEAD_DW && t + 2 < t1) {
          label[0] = __ldg(labels + (long long)(t + 2) * HD_TILE);
          label[1] = __ldg(labels + (long long)(t + 2) * HD_TILE + 32);
        }
        tc_fence_after();
        const int nc = cols_of(t) - half * 64;  // this group's columns: none, 32 or (64 and more) 64
        const int c_abs = t * HD_TILE + half * 64;
        const uint32_t tile = lane_base + b * HD_TILE + half * 64;
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += 32) {
          if (c0 >= nc) break;
          uint32_t v[32];
          tmem_ld_32x32(tile + c0, v);
          tmem_ld_wait();
          float f[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]);
          // bit j: column j is the row's label
          uint32_t hits;
          if (MODE == HEAD_DX) {
            const int at = y - (c_abs + c0);
            hits = (unsigned)at < 32u ? 1u << at : 0u;
          } else {
            // lane c has the label of column c; a row's columns are those whose label has the row's five bits
            hits = __ballot_sync(0xffffffffu, (unsigned)rel[c0 / 32] < 32u);
#pragma unroll
            for (int k = 0; k < 5; ++k)
              hits &= __ballot_sync(0xffffffffu, rel[c0 / 32] >> k & 1) ^ rank_bits[k];
          }
          const bool any = __any_sync(0xffffffffu, hits != 0u);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 t = hd_fma2(make_float2(f[j], f[j + 1]), make_float2(HD_LOG2E, HD_LOG2E), make_float2(0.f, 0.f));
            f[j] = hd_ex2(t.x);
            f[j + 1] = hd_ex2(t.y);
          }
          if (any) {
            const float one = MODE == HEAD_DW ? g : 1.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) hd_sub_if(f[j], one, hits, 1u << j);
          }
          if (MODE == HEAD_DW) {
            float2 d[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int j = 0; j < 32; j += 2) d[j / 2 & 1] = hd_add2(d[j / 2 & 1], make_float2(f[j], f[j + 1]));
            d[0] = hd_add2(d[0], d[1]);
            db += d[0].x + d[0].y;
          }
          uint32_t o[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
          // over the 32 columns of s that this thread has just read: 16 columns of P, 16 of its remainder
          hd_tmem_st_x16(tile + c0, o);
          if (LO) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              o[j] = pack_bf16x2(f[2 * j] - __uint_as_float(o[j] << 16),
                                 f[2 * j + 1] - __uint_as_float(o[j] & 0xFFFF0000u));
            hd_tmem_st_x16(tile + c0 + 16, o);
          }
        }
        hd_tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_done[b]);
        if (pending) {
          if (!drain()) { ok = false; break; }
          pending = false;
        }
        b += 2;
        if (b >= NB) { b -= NB; bph ^= 1u; }
      }
      if (ok && pending) ok = drain();  // this job had no tile for this group
      pending = true;
      pend_rt = rt; pend_sp = sp; pend_g = g; pend_db = db;
      rt = next_rt;
      sp = next_sp;
    }
    if (ok && pending) drain();
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 0) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Both gradients from one matrix P^T = p - [j = y], rows = classes, columns = voxels (calls whose weight and whose dW fit
// into a CTA, or a part of them at a time: head_both). A CTA keeps all tiles of W in shared memory and dW's sums in tensor memory and walks tiles of
// 128 voxels; of each 128 x 128 tile of s^T the epilogue makes a tile of P^T in shared memory, [class][voxel], and two
// MMAs read it from there: dW += P^T X with the voxels along the reduction (K-major A), dX += P W with the classes along
// it (the same bytes as an MN-major A). An exponential serves both gradients, X is read once, and in shared memory the
// target's entry can be put right alone: every thread stores its row of p, then the lanes that hold the columns' labels
// store p - 1 of the target there (expm1 of the voxel's loss term, which keeps its relative precision). In tensor memory
// each of a row's entries has to be looked at for it, three instructions more than the three or so of the rest.
// Roles: warp 0 loads, warps 1 to 3 issue the MMAs of s, dW and dX (a warp loses some 300 clocks at each commit: dW and dX
// out of one warp 492 instead of 424 us at 128 classes, below), four groups of the epilogue (two take a tile's halves, by
// tile parity), and the last four warps take dX out of tensor memory, scale it and store it by TMA: row pieces stored by
// the epilogue itself, 16 bytes a row and instruction, kept the shared memory pipe from P's stores (860 us).
// WEIGHTED: P stays without the weights u, for dX, whose rows take g = k u at the end; for dW the last four warps put u X in
// the place of X as soon as the last product of s has read it. Its rounding goes by the feature, so the voxels of a class do
// not share it (u P would be off by the same for all of a class's targets), and db takes u in fp32.
// Bound: neither the exponential unit (1024 clocks a tile of 128 x 128, some 2100 are taken) nor the MMAs or the stores,
// but a tile's way through them, two tiles at a time: tensor memory holds no third one of s.
// 2 x 128^3 voxels, 64 channels, 257 classes: 690 us with the sums behind it, the two kernels above and what they need 1160;
// 128 classes 349 / 722; 16 channels and 34 classes 293 / 633; 32 channels and 500 classes 849 / 1456. Loss and gradients
// with class weights, in this kernel and in two: 64^3 x 64 x 147 92 / 113, 2 x 128^3 x 64 x 257 1510 / 1675, x 16 x 34 721 /
// 741, x 32 x 500 1829 / 2253.
constexpr int HB_FIRST_EPI = 4;
constexpr int HB_DX_WARPS = 4;  // behind the epilogue's
constexpr int HB_THREADS = 32 * (HB_FIRST_EPI + HD_EPI_WARPS + HB_DX_WARPS);
template <bool WEIGHTED>
__global__ void __launch_bounds__(HB_THREADS, 1) head_both_kernel(const __grid_constant__ HeadParams p) {
  constexpr uint32_t SB = 2, PB = 2;  // tiles of s in tensor memory and of P in shared memory: one for each pair of groups
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t w_full, x_full[HD_MAX_STAGES], x_empty[HD_MAX_STAGES], s_full[SB], s_empty[SB], p_full[PB],
      p_empty[PB], acc_full[2], acc_empty[2], dw_full, s_last[HD_MAX_STAGES], u_full[HD_MAX_STAGES];
  __shared__ uint32_t tmem_base_s, abort_s;
  volatile uint32_t* abort_flag = &abort_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kt = p.row_tiles;
  const uint32_t box16 = (uint32_t)p.kboxes * HD_BOX, tile_bytes = box16 + HD_BOX16;
  const uint32_t naccs = (uint32_t)p.accs;
  const uint32_t ACC_X = SB * HD_TILE, ACC_W = ACC_X + naccs * p.cpad;  // columns of the sums
  uint8_t* smem_p = smem;
  uint8_t* smem_w = smem_p + PB * 2 * HD_BOX;
  uint8_t* smem_x = smem_w + kt * tile_bytes;
  uint8_t* smem_o = smem_x + p.stages * tile_bytes;                     // [dX warps][kboxes][32 rows of 128 bytes]
  float* smem_db = reinterpret_cast<float*>(smem_o + p.kboxes * HD_BOX);  // [kt][groups][128]
  float* smem_cw = smem_db + kt * 4 * HD_TILE;                            // WEIGHTED: [kt][128], of the classes
  float* smem_u = smem_cw + kt * HD_TILE;                                 // and [stages][128], of the voxels

  if (threadIdx.x == 0) {
    abort_s = 0;
    mbar_init(&w_full, 1);
    mbar_init(&dw_full, 1);
    for (int i = 0; i < p.stages; ++i) { mbar_init(&x_full[i], 1 + HB_DX_WARPS); mbar_init(&x_empty[i], 1); }
    for (int i = 0; WEIGHTED && i < p.stages; ++i) { mbar_init(&s_last[i], 1); mbar_init(&u_full[i], HB_DX_WARPS); }
    for (uint32_t i = 0; i < SB; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], HD_EPI_WARPS / 2); }
    for (uint32_t i = 0; i < PB; ++i) { mbar_init(&p_full[i], HD_EPI_WARPS / 2); mbar_init(&p_empty[i], 2); }
    for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], HB_DX_WARPS); }
    mbar_fence_init();
  }
  if (WEIGHTED)
    for (int i = threadIdx.x; i < kt * HD_TILE; i += HB_THREADS) smem_cw[i] = i < p.rows ? __ldg(p.cw + i) : 0.f;
  if (warp == 0) {
    tmem_alloc(&tmem_base_s, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  // classes of a tile, up to a multiple of 32
  const int last_rows = ((int)(p.rows - (long long)(kt - 1) * HD_TILE) + 31) & ~31;
  auto rows_of = [&](int i) -> int { return i + 1 < kt ? HD_TILE : last_rows; };

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&p.mapR);
      tma_prefetch_desc(&p.mapQ);
      mbar_expect_tx(&w_full, kt * tile_bytes);
      for (int i = 0; i < kt; ++i) {
        for (int k = 0; k < p.kboxes; ++k)
          hd_tma_2d(smem_w + i * tile_bytes + k * HD_BOX, &p.mapR, &w_full, k * 64, p.row0 + i * HD_TILE);
        hd_tma_2d(smem_w + i * tile_bytes + box16, &p.mapR16, &w_full, 0, p.row0 + i * HD_TILE);
      }
      uint32_t st = 0, ph = 0;
      for (int v = blockIdx.x; v < p.col_tiles; v += gridDim.x) {
        if (!mbar_wait(&x_empty[st], ph ^ 1u, abort_flag, p.status, 91)) break;
        mbar_expect_tx(&x_full[st], box16);
        for (int k = 0; k < p.kboxes; ++k)
          hd_tma_2d(smem_x + st * tile_bytes + k * HD_BOX, &p.mapQ, &x_full[st], k * 64, v * HD_TILE);
        if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t w0 = smem_u32(smem_w), x0 = smem_u32(smem_x);
    uint32_t st = 0, ph = 0, b = 0, bph = 0;
    bool ok = hd_wait(&w_full, 0, abort_flag, p.status, 94);
    for (int v = blockIdx.x; v < p.col_tiles && ok; v += gridDim.x) {
      if (!hd_wait(&x_full[st], ph, abort_flag, p.status, 95)) break;
      for (int i = 0; i < kt; ++i) {
        if (!hd_wait(&s_empty[b], bph ^ 1u, abort_flag, p.status, 96)) { ok = false; break; }
        tc_fence_after();
        if (leader) {
          const uint32_t r = w0 + i * tile_bytes, q = x0 + st * tile_bytes;
          hd_first_mma(tmem + b * HD_TILE, r, r + box16, q, q + box16, HD_TILE, p.ksteps);
          tc_commit(&s_full[b]);
          if (WEIGHTED && i + 1 == kt) tc_commit(&s_last[st]);
        }
        __syncwarp();
        if (++b == SB) { b = 0; bph ^= 1u; }
      }
      if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
    }
  } else if (warp == 2) {
    // dW += P^T X
    const bool leader = elect_one();
    const uint32_t hi = desc_hi(8u * 128u, 2u), idesc = make_idesc_bf16(128, p.cpad, 0, 1);
    const uint32_t p0 = smem_u32(smem_p), x0 = smem_u32(smem_x), lbo = p.kboxes > 1 ? (uint32_t)HD_BOX : 0u;
    uint32_t st = 0, ph = 0, pb = 0, pph = 0;
    bool ok = true;
    for (int v = blockIdx.x; v < p.col_tiles && ok; v += gridDim.x) {
      // (the first issuing warp has waited for the loads; this one has to see them too, or their weighting)
      if (!hd_wait(WEIGHTED ? &u_full[st] : &x_full[st], ph, abort_flag, p.status, 95)) { ok = false; break; }
      const uint32_t x_lo = desc_lo(x0 + st * tile_bytes, lbo);
      for (int i = 0; i < kt; ++i) {
        if (!hd_wait(&p_full[pb], pph, abort_flag, p.status, 93)) { ok = false; break; }
        tc_fence_after();
        if (leader) {
          const uint32_t a_lo = desc_lo(p0 + pb * 2 * HD_BOX, 16u), d = tmem + ACC_W + i * p.cpad;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            tc_mma_bf16_pred(d, a_lo + (uint32_t)(k >> 2) * (HD_BOX >> 4) + (uint32_t)(k & 3) * 2u, hi, x_lo + k * 128u, hi,
                             idesc, v == (int)blockIdx.x && k == 0 ? 0u : 1u);
          tc_commit(&p_empty[pb]);
          if (i + 1 == kt) tc_commit(&x_empty[st]);
        }
        __syncwarp();
        if (++pb == PB) { pb = 0; pph ^= 1u; }
      }
      if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
    }
    if (ok && leader) tc_commit(&dw_full);
    __syncwarp();
  } else if (warp == 3) {
    // dX = P W
    const bool leader = elect_one();
    const uint32_t hi = desc_hi(8u * 128u, 2u), idesc = make_idesc_bf16(128, p.cpad, 1, 1);
    const uint32_t p0 = smem_u32(smem_p), w0 = smem_u32(smem_w), lbo = p.kboxes > 1 ? (uint32_t)HD_BOX : 0u;
    uint32_t pb = 0, pph = 0, ab = 0, aph = 0;
    bool ok = hd_wait(&w_full, 0, abort_flag, p.status, 94);
    for (int v = blockIdx.x; v < p.col_tiles && ok; v += gridDim.x) {
      if (!hd_wait(&acc_empty[ab], aph ^ 1u, abort_flag, p.status, 92)) break;
      for (int i = 0; i < kt; ++i) {
        if (!hd_wait(&p_full[pb], pph, abort_flag, p.status, 93)) { ok = false; break; }
        tc_fence_after();
        if (leader) {
          const uint32_t a_lo = desc_lo(p0 + pb * 2 * HD_BOX, HD_BOX), w_lo = desc_lo(w0 + i * tile_bytes, lbo);
          const int ksteps = rows_of(i) / 16;
          for (int k = 0; k < ksteps; ++k)
            tc_mma_bf16_pred(tmem + ACC_X + ab * p.cpad, a_lo + k * 128u, hi, w_lo + k * 128u, hi, idesc,
                             i == 0 && k == 0 ? 0u : 1u);
          tc_commit(&p_empty[pb]);
          if (i + 1 == kt) tc_commit(&acc_full[ab]);
        }
        __syncwarp();
        if (++pb == PB) { pb = 0; pph ^= 1u; }
      }
      if (++ab == naccs) { ab = 0; aph ^= 1u; }
    }
  } else if (warp >= HB_FIRST_EPI + HD_EPI_WARPS) {
    // A thread has a row of voxels: it writes the row's sixteen columns more when a stage is free, and takes dX of a
    // finished voxel tile; each warp stores its 32 rows.
    const int quad = warp & 3, row = quad * 32 + lane;
    const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + ACC_X;
    uint8_t* stage = smem_o + quad * p.kboxes * 4096;
    const float k = __ldg(p.gout) / __ldg(p.den);
    if (blockIdx.x == 0 && row == 0) p.scale[0] = k;
    uint32_t ab = 0, aph = 0, st = 0, ph = 0;
    int ahead = blockIdx.x;  // the next voxel tile whose columns are written; what they are of is read one more ahead
    float lse_next = __ldg(p.lse2 + (long long)ahead * HD_TILE + row);
    uint32_t hit_next = __ldg(p.colhit + (long long)ahead * HD_TILE + row);
    auto columns = [&]() -> bool {
      const float l = lse_next;
      const uint32_t label = hit_next & 0xFFFFu;
      const bool live = label != 0xFFFFu;
      const float u = WEIGHTED && live ? smem_cw[label] : 0.f;
      ahead += gridDim.x;
      if (ahead < p.col_tiles) {
        lse_next = __ldg(p.lse2 + (long long)ahead * HD_TILE + row);
        hit_next = __ldg(p.colhit + (long long)ahead * HD_TILE + row);
      }
      if (!hd_wait(&x_empty[st], ph ^ 1u, abort_flag, p.status, 91)) return false;
      const uint2 c = hd_three(live && (!WEIGHTED || u != 0.f) ? -l * HD_LN2 : HD_LOWEST);
      if (WEIGHTED) smem_u[st * HD_TILE + row] = u;  // (the epilogue is done with the stage's last one: its dX is out)
      const uint32_t at = smem_u32(smem_x) + st * tile_bytes + box16 + row * 32;
      const uint32_t second = (row >> 2) & 1;  // (32-byte rows, halves exchanged in every second group of four)
      hd_sts4(at + 16 * second, HD_ONE | HD_ONE << 16, HD_ONE | c.x << 16, c.x >> 16 | c.y << 16, 0u);
      hd_sts4(at + 16 * (second ^ 1u), 0u, 0u, 0u, 0u);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&x_full[st]);
      if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
      return true;
    };
    bool ok = true;
    for (int i = 0; i < p.stages && ahead < p.col_tiles && ok; ++i) ok = columns();
    uint32_t out_next = WEIGHTED ? 0u : __ldg(p.colhit + (long long)blockIdx.x * HD_TILE + row);
    uint32_t wst = 0, wph = 0;
    for (int v = blockIdx.x; v < p.col_tiles && ok; v += gridDim.x) {
      float g;
      if (WEIGHTED) {
        // u X in the place of X, as soon as the last product of s has read it
        const float u = smem_u[wst * HD_TILE + row];
        g = u == 0.f ? 0.f : k * u;
        if (!(hd_wait(&x_full[wst], wph, abort_flag, p.status, 95) &&
              hd_wait(&s_last[wst], wph, abort_flag, p.status, 93))) { ok = false; break; }
#pragma unroll 4
        for (int c = 0; c < p.cpad / 8; ++c) {
          uint4* at = reinterpret_cast<uint4*>(smem_x + wst * tile_bytes + (c >> 3) * HD_BOX + row * 128 +
                                               (((c & 7) ^ (row & 7)) << 4));
          uint4 x = *at;
          uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            w[j] = u == 0.f ? 0u : pack_bf16x2(__uint_as_float(w[j] << 16) * u, __uint_as_float(w[j] & 0xFFFF0000u) * u);
          *at = x;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&u_full[wst]);
        if (++wst == (uint32_t)p.stages) { wst = 0; wph ^= 1u; }
      } else {
        g = (out_next & 0xFFFFu) != 0xFFFFu ? k : 0.f;
        if (v + (int)gridDim.x < p.col_tiles) out_next = __ldg(p.colhit + ((long long)v + gridDim.x) * HD_TILE + row);
      }
      if (!hd_wait(&acc_full[ab], aph, abort_flag, p.status, 97)) break;
      tc_fence_after();
      if (lane == 0) bulk_wait_read_all();  // the last rows have left
      __syncwarp();
      for (int c0 = 0; c0 < p.cpad; c0 += 32) {
        uint32_t u[32];
        tmem_ld_32x32(acc + ab * p.cpad + c0, u);  // (past cpad: columns of the next sums, which nothing looks at)
        tmem_ld_wait();
        if (c0 + 32 >= p.cpad) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[ab]);
        }
        if (!p.first || !p.last) {
          float4* at = p.part_x + ((long long)v * (p.cpad / 4) + c0 / 4) * HD_TILE + quad * 32 + lane;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (c0 + 4 * j >= p.cpad) break;
            float4 f = make_float4(__uint_as_float(u[4 * j]), __uint_as_float(u[4 * j + 1]), __uint_as_float(u[4 * j + 2]),
                                   __uint_as_float(u[4 * j + 3]));
            if (!p.first) {
              const float4 before = at[j * HD_TILE];
              f.x += before.x; f.y += before.y; f.z += before.z; f.w += before.w;
            }
            if (!p.last) {
              at[j * HD_TILE] = f;
            } else {
              u[4 * j] = __float_as_uint(f.x); u[4 * j + 1] = __float_as_uint(f.y);
              u[4 * j + 2] = __float_as_uint(f.z); u[4 * j + 3] = __float_as_uint(f.w);
            }
          }
          if (!p.last) continue;
        }
        // a voxel that takes no part has no gradient, whatever its features hold
#pragma unroll
        for (int j = 0; j < 16; ++j)
          u[j] = g == 0.f ? 0u : pack_bf16x2(__uint_as_float(u[2 * j]) * g, __uint_as_float(u[2 * j + 1]) * g);
        uint8_t* dst = stage + (c0 >> 6) * 4096 + lane * 128;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(dst + (((((c0 & 32) >> 3) + j) ^ (lane & 7)) << 4)) =
              make_uint4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
      }
      fence_proxy_async();
      __syncwarp();
      const long long r = (long long)v * HD_TILE + quad * 32;
      if (lane == 0 && r < p.cols && p.last) {
        for (int k = 0; k < p.kboxes; ++k) hd_tma_store_2d(&p.mapO, stage + k * 4096, k * 64, (int)r);
        bulk_commit();
      }
      if (++ab == naccs) { ab = 0; aph ^= 1u; }
      if (ahead < p.col_tiles) ok = columns();
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  } else {
    const int quad = warp & 3, group = (warp - HB_FIRST_EPI) >> 2, half = group & 1;
    const uint32_t par = group >> 1;
    const int row = quad * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t swz = row * 128 + ((row & 7) << 4);  // the row's first 16 bytes of voxels in a 128-byte swizzled box
    const uint32_t s_tile = lane_base + par * HD_TILE + half * 64;
    uint32_t ph = 0, tc = 0;
    uint32_t st = kt == 1 ? par : 0u, xph = 0;  // WEIGHTED: stage of the voxel tile (there are two or more)
    bool ok = true;
    float* const db = smem_db + group * HD_TILE + row;  // this thread's alone
    for (int i = 0; i < kt; ++i) db[i * 4 * HD_TILE] = 0.f;
    // every second tile over all voxel tiles is this pair of groups'
    const int step = kt == 1 ? 2 * gridDim.x : gridDim.x;
    const int v0 = kt == 1 ? blockIdx.x + par * gridDim.x : blockIdx.x;
    for (int v = v0; v < p.col_tiles && ok; v += step) {
      // label and p - 1 of the columns `lane` and 32 further of its half; needed behind the first exponentials
      const uint32_t* at = p.colhit + (long long)v * HD_TILE + half * 64 + lane;
      const uint32_t hit[2] = {__ldg(at), __ldg(at + 32)};
      if (v + step < p.col_tiles) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + (long long)step * HD_TILE));
      int i = kt == 1 ? 0 : (int)((tc ^ par) & 1u);
      tc += kt;
      const uint32_t us = smem_u32(smem_u) + (st * HD_TILE + half * 64) * 4;
      if (WEIGHTED) {
        ok = hd_wait(&x_full[st], xph, abort_flag, p.status, 95);  // the weights of its columns are there
        st += kt == 1 ? 2u : 1u;
        if (st >= (uint32_t)p.stages) { st -= p.stages; xph ^= 1u; }
      }
      for (; i < kt && ok; i += 2) {
        if (!hd_wait(&s_full[par], ph, abort_flag, p.status, 98)) { ok = false; break; }
        tc_fence_after();
        const uint32_t out = smem_u32(smem_p) + par * 2 * HD_BOX + half * HD_BOX;
        float sum = 0.f;
        const bool live = quad * 32 < rows_of(i);
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += 32) {
          // WEIGHTED: 16 columns at a time, for their weights' registers (80 bytes spilled otherwise: 1789 us instead of 1510
          // for the loss and gradients of 2 x 128^3 voxels x 64 channels x 257 classes; without weights 1094 instead of 1072)
          constexpr int CH = WEIGHTED ? 16 : 32;
#pragma unroll
          for (int c1 = c0; c1 < c0 + 32; c1 += CH) {
            uint32_t u[CH];
            if (live) {
              if constexpr (WEIGHTED) tmem_ld_32x16(s_tile + c1, u);
              else tmem_ld_32x32(s_tile + c1, u);
              tmem_ld_wait();
            }
            if (c1 + CH == 64) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&s_empty[par]);
            }
            if (live) {
              float2 d[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
              for (int j = 0; j < CH / 2; ++j) {
                float2 f = hd_fma2(make_float2(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1])),
                                   make_float2(HD_LOG2E, HD_LOG2E), make_float2(0.f, 0.f));
                f.x = hd_ex2(f.x);
                f.y = hd_ex2(f.y);
                if constexpr (WEIGHTED) d[j & 1] = hd_fma2(f, hd_lds2(us + (c1 + 2 * j) * 4), d[j & 1]);
                else d[j & 1] = hd_add2(d[j & 1], f);
                u[j] = pack_bf16x2(f.x, f.y);
              }
              d[0] = hd_add2(d[0], d[1]);
              sum += d[0].x + d[0].y;
            }
            // the buffer is free: both products of its last tile are done
            if (c1 == 0) ok = hd_wait(&p_empty[par], ph ^ 1u, abort_flag, p.status, 96);
            if (live) {
#pragma unroll
              for (int j = 0; j < CH / 8; ++j)
                hd_sts4((out + swz) ^ (c1 / 8 + j) << 4, u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
            }
          }
          if (live) {
            __syncwarp();  // rows before single entries
            // lane c has the label of column c: a row's targets are the columns whose label has the row's five bits
            const int rel = (int)(hit[c0 / 32] & 0xFFFFu) - (p.row0 + i * HD_TILE + quad * 32);
            uint32_t hits = __ballot_sync(0xffffffffu, (unsigned)rel < 32u);
            if (hits != 0u) {
#pragma unroll
              for (int k = 0; k < 5; ++k) hits &= __ballot_sync(0xffffffffu, rel >> k & 1) ^ (lane >> k & 1 ? 0u : ~0u);
              sum -= (float)__popc(hits) * (WEIGHTED ? smem_cw[i * HD_TILE + row] : 1.f);
              if ((unsigned)rel < 32u) {
                const int c = c0 + lane, r = quad * 32 + rel;
                hd_sts16(out + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2, hit[c0 / 32] >> 16);
              }
            }
          }
        }
        if (!ok) break;
        if (live) db[i * 4 * HD_TILE] += sum;
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[par]);
        ph ^= 1u;
      }
    }
    // dW and db of this CTA's voxels
    if (hd_vote(1, 32 * HD_EPI_WARPS, ok) && hd_wait(&dw_full, 0, abort_flag, p.status, 97)) {
      tc_fence_after();
      for (int i = group; i < kt; i += 4) {  // the groups' sums, in order
        const float* all = smem_db + i * 4 * HD_TILE + row;
        p.ws_b[(long long)blockIdx.x * p.rows_pad + (long long)i * HD_TILE + row] =
            all[0] + all[HD_TILE] + all[2 * HD_TILE] + all[3 * HD_TILE];
      }
      for (int i = 0; i < kt; ++i) {
        const long long r = (long long)i * HD_TILE + row;
        for (int c0 = group * 16; c0 < p.cpad; c0 += 64) {
          uint32_t v[16];
          tmem_ld_32x16(lane_base + ACC_W + i * p.cpad + c0, v);
          tmem_ld_wait();
          float4* dst = reinterpret_cast<float4*>(p.ws + ((long long)blockIdx.x * p.rows_pad + r) * p.cpad + c0);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            dst[j] = make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 2]),
                                 __uint_as_float(v[4 * j + 3]));
        }
      }
      tc_fence_before();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 0) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// -- what stands around the three passes -----------------------------------------------------------------------------
__device__ __forceinline__ long long hd_label(const void* labels, int kind, long long i) {
  if (kind == 2) return reinterpret_cast<const short*>(labels)[i];
  if (kind == 4) return reinterpret_cast<const int*>(labels)[i];
  return reinterpret_cast<const long long*>(labels)[i];
}

// y[i]: the label, or -1 for a voxel that takes no part (the ignored label; one outside the classes, which is reported)
// and behind the last voxel; bias2[j] = bias_j log2(e), -inf behind the last class. w16 (narrow heads): a class's sixteen
// columns more, b in three parts against ones, then ones against -lse and (second array) log u. What is off stands as
// HD_LOWEST instead of -inf: zeros of the other side must not make a NaN of it.
__global__ void __launch_bounds__(256) head_prep_kernel(const void* __restrict__ labels, int kind, long long V,
                                                        long long v_pad, int K, int k_pad, int has_ignore,
                                                        long long ignore, int* __restrict__ y,
                                                        const void* __restrict__ bias, int bias_kind,
                                                        float* __restrict__ bias2, uint4* __restrict__ w16,
                                                        uint32_t* __restrict__ status) {
  const long long n = v_pad > k_pad ? v_pad : k_pad;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    if (i < v_pad && y != nullptr) {
      int v = -1;
      if (i < V) {
        const long long raw = hd_label(labels, kind, i);
        if (!(has_ignore && raw == ignore)) {
          if (raw >= 0 && raw < K) v = (int)raw;
          else report(status, ST_BAD_ARG, 63, (uint32_t)raw, (uint32_t)i);
        }
      }
      y[i] = v;
    }
    if (i < k_pad) {
      float b = -INFINITY;
      if (i < K) b = hd_bias(bias, bias_kind, i);
      bias2[i] = b * HD_LOG2E;
      if (w16 != nullptr) {
        const uint2 t = hd_three(b < HD_LOWEST ? HD_LOWEST : b);
        for (int k = 0; k < 2; ++k) {
          uint4* at = w16 + 2 * ((long long)k * k_pad + i);
          at[0] = make_uint4(t.x, t.y | HD_ONE << 16, HD_ONE | HD_ONE << 16, k ? HD_ONE | HD_ONE << 16 : 0u);
          at[1] = make_uint4(k ? HD_ONE : 0u, 0u, 0u, 0u);
        }
      }
    }
  }
}

// Shares of a row's statistics, merged. TEAM 1: by one thread, in order; TEAM 32: by a warp, each lane every 32nd one and
// then in a fixed tree: few voxels have many shares, and a thread would wait an L2 trip for a few of them at a time (512
// shares of one voxel: 45 us by one thread).
template <int TEAM>
__device__ __forceinline__ void hd_merge_best(const float2* part, int shares, long long v_pad, long long i, int lane,
                                              float& m, int& best) {
  m = -INFINITY;
  best = INT_MAX;
#pragma unroll 4
  for (int k = lane; k < shares; k += TEAM) {
    const float2 e = part[(long long)k * v_pad + i];
    hd_better(m, best, e.x, __float_as_int(e.y));
  }
#pragma unroll
  for (int o = TEAM / 2; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, m, o);
    const int j = __shfl_xor_sync(0xffffffffu, best, o);
    hd_better(m, best, v, j);
  }
}
template <int TEAM>
__device__ __forceinline__ float2 hd_merge_sums(const float2* part, int shares, long long v_pad, long long i, int lane) {
  constexpr int BATCH = TEAM == 1 ? 4 : 8;  // loads and exponentials that do not wait for one another
  float m = -INFINITY, s = 0.f;
  for (int k0 = lane; k0 < shares; k0 += BATCH * TEAM) {
    float2 e[BATCH];
    float mm = m;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      e[j] = k0 + j * TEAM < shares ? part[(long long)(k0 + j * TEAM) * v_pad + i] : make_float2(-INFINITY, 0.f);
      mm = fmaxf(mm, e[j].x);
    }
    const float base = mm == -INFINITY ? 0.f : mm;
    s *= hd_ex2(m - base);
#pragma unroll
    for (int j = 0; j < BATCH; ++j) s += e[j].y * hd_ex2(e[j].x - base);
    m = mm;
  }
#pragma unroll
  for (int o = TEAM / 2; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, m, o), t = __shfl_xor_sync(0xffffffffu, s, o);
    const float mm = fmaxf(m, v), base = mm == -INFINITY ? 0.f : mm;
    const float x = s * hd_ex2(m - base), y = t * hd_ex2(v - base);
    s = x + y;  // the same in both lanes
    m = mm;
  }
  return make_float2(m, s);
}

// the class of a voxel's largest logit
template <int TEAM>
__global__ void __launch_bounds__(256) head_arg_kernel(const float2* __restrict__ part, int shares, long long V,
                                                       long long v_pad, long long* __restrict__ out) {
  const int lane = threadIdx.x % TEAM;
  for (long long i = (long long)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM; i < V; i += (long long)gridDim.x * (256 / TEAM)) {
    float m;
    int best;
    hd_merge_best<TEAM>(part, shares, v_pad, i, lane, m, best);
    if (lane == 0) out[i] = best == INT_MAX ? 0 : best;  // nothing above -inf
  }
}

// loss = num / max(den, eps), den the clamped denominator
__device__ __forceinline__ void hd_loss(const HeadSum& a, double* total, float* loss, float* den) {
  const double eps = 1.1920928955078125e-7, d = a.den < eps ? eps : a.den;  // NaN stays
  total[0] = a.num;
  total[1] = a.den;
  loss[0] = (float)(a.num / d);
  den[0] = (float)d;
}

// lse2[i] from the shares of its statistics; block sums of u nll and u in double (a single block goes on to the loss)
template <int TEAM>
__global__ void __launch_bounds__(256) head_merge_kernel(const float2* __restrict__ part, const float* __restrict__ tl,
                                                         const int* __restrict__ y, const float* __restrict__ cw,
                                                         const void* __restrict__ bias, int bias_kind, int shares, long long V, long long v_pad,
                                                         float* __restrict__ lse2, uint32_t* __restrict__ hit,
                                                         double* __restrict__ sums, double* __restrict__ total, float* __restrict__ loss,
                                                         float* __restrict__ den) {
  HeadSum a{0.0, 0.0};
  const int lane = threadIdx.x % TEAM;
  for (long long i = (long long)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM; i < v_pad;
       i += (long long)gridDim.x * (256 / TEAM)) {
    float l = INFINITY;
    uint32_t h = 0xFFFFu;
    if (i < V) {  // (the same in a team's lanes)
      const float at_label = __ldg(tl + i);  // requested ahead of the shares
      const int label = __ldg(y + i);
      const float2 e = hd_merge_sums<TEAM>(part, shares, v_pad, i, lane);
      if (lane == 0) l = hd_voxel(e.x, e.y, at_label, label, cw, bias, bias_kind, a, h);
    }
    if (lane == 0) {
      lse2[i] = l;
      if (hit != nullptr) hit[i] = h;
    }
  }
  a = hd_block_sum<8>(a);
  if (threadIdx.x == 0) {
    if (gridDim.x == 1) hd_loss(a, total, loss, den);
    else { sums[2 * blockIdx.x] = a.num; sums[2 * blockIdx.x + 1] = a.den; }
  }
}

// total[2] = the blocks' sums in order, and the loss
__global__ void __launch_bounds__(256) head_total_kernel(const double* __restrict__ sums, int blocks,
                                                         double* __restrict__ total, float* __restrict__ loss,
                                                         float* __restrict__ den) {
  HeadSum a{0.0, 0.0};
  for (int i = threadIdx.x; i < blocks; i += 256) { a.num += sums[2 * i]; a.den += sums[2 * i + 1]; }
  a = hd_block_sum<8>(a);
  if (threadIdx.x == 0) hd_loss(a, total, loss, den);
}

// what the backward passes need of a voxel; x16 (narrow heads): its sixteen columns more
__global__ void __launch_bounds__(256) head_weights_kernel(HeadCall a, const float* __restrict__ gout, long long v_pad) {
  const float k = gout[0] / a.den[0];
  if (blockIdx.x == 0 && threadIdx.x == 0) a.scale[0] = k;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < v_pad; i += (long long)gridDim.x * 256) {
    const int c = a.y[i];
    const float u = c < 0 ? 0.f : a.cw == nullptr ? 1.f : a.cw[c], l = a.lse2[i];
    a.g[i] = u == 0.f ? 0.f : k * u;
    if (a.x16 == nullptr) {
      a.u[i] = u;
      a.lse2p[i] = u == 0.f ? INFINITY : l;
    } else {
      const uint2 t = hd_three(u == 0.f ? HD_LOWEST : -l * HD_LN2), v = hd_three(u == 0.f ? 0.f : logf(u));
      uint4* at = a.x16 + 2 * i;
      at[0] = make_uint4(HD_ONE | HD_ONE << 16, HD_ONE | t.x << 16, t.x >> 16 | t.y << 16, v.x);
      at[1] = make_uint4(v.y, 0u, 0u, 0u);
    }
  }
}

// One sum over slices: out[r][c] = scale * sum of ws[slice][rows_pad][ld] in slice order, r < rows, c < C.
struct HeadReduce {
  const float* ws;
  int slices, C, ld, kind, blocks;  // kind of out: 0 bf16, 2 fp32
  long long rows, rows_pad;
  void* out;
};
// The first a.blocks blocks take a, the others b (dw and db). Up to HD_FEW_SLICES a thread walks the slices of its outputs.
// More of them: a block takes 32 neighbouring outputs, each of its eight warps every eighth slice, since a thread would
// wait an L2 trip for a few of them at a time. (Loss and gradients of 1 voxel x 256 channels x 32768 classes,
// one slice: 105 us, in the second form 347; 300 x 64 x 20000 52 and 89; 2 x 128^3 x 64 x 257, 148 slices: 1152 us, in the
// first form 1162.)
constexpr int HD_FEW_SLICES = 4;
__global__ void __launch_bounds__(256) head_reduce_kernel(const HeadReduce a, const HeadReduce b,
                                                          const float* __restrict__ scale) {
  __shared__ float s_part[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool first = (int)blockIdx.x < a.blocks;
  const HeadReduce& p = first ? a : b;
  const int block = first ? blockIdx.x : blockIdx.x - a.blocks;
  const long long n = p.rows * p.C, slice = p.rows_pad * p.ld;
  const float k = scale != nullptr ? scale[0] : 1.f;
  if (p.slices <= HD_FEW_SLICES) {
    for (long long i = (long long)block * 256 + threadIdx.x; i < n; i += (long long)p.blocks * 256) {
      const float* src = p.ws + i / p.C * p.ld + i % p.C;
      float sum = 0.f;
      for (int s = 0; s < p.slices; ++s) sum += src[s * slice];
      sum *= k;
      if (p.kind == 2) reinterpret_cast<float*>(p.out)[i] = sum;
      else reinterpret_cast<__nv_bfloat16*>(p.out)[i] = __float2bfloat16(sum);
    }
    return;
  }
  for (long long i0 = (long long)block * 32; i0 < n; i0 += (long long)p.blocks * 32) {
    const long long i = i0 + lane;
    float sum = 0.f;
    if (i < n) {
      const float* src = p.ws + i / p.C * p.ld + i % p.C;
#pragma unroll 8
      for (int s = warp; s < p.slices; s += 8) sum += src[s * slice];
    }
    s_part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && i < n) {
      for (int w = 1; w < 8; ++w) sum += s_part[w][lane];
      sum *= k;
      if (p.kind == 2) reinterpret_cast<float*>(p.out)[i] = sum;
      else reinterpret_cast<__nv_bfloat16*>(p.out)[i] = __float2bfloat16(sum);
    }
    __syncthreads();
  }
}

static int hd_blocks(long long n, int per_sm) {
  const long long b = (n + 255) / 256;
  return (int)(b < 148LL * per_sm ? (b < 1 ? 1 : b) : 148LL * per_sm);
}

// How many ways the columns are cut: fewest rounds of (tiles per job + about one tile of fixed cost), fewest cuts first.
// Loss of 300 voxels x 64 channels x 20000 classes 19 us, without cuts 113; 1000 x 256 x 1000 17 and 25; loss and gradients
// of 40000 x 32 x 1001 130 and 318; 5000 x 64 x 300, whose row tiles are cut into few, 39 and 37.
static void head_split(int row_tiles, int col_tiles, int* splits, int* tps) {
  long long best = -1;
  for (int want = 1; want <= col_tiles && want <= 296; ++want) {
    const int per = (col_tiles + want - 1) / want, s = (col_tiles + per - 1) / per;
    const long long rounds = ((long long)row_tiles * s + 147) / 148, cost = rounds * (per + 1);
    if (best < 0 || cost < best) { best = cost; *splits = s; *tps = per; }
    if (row_tiles >= 148 * 4) break;
  }
}

static bool wide(const HeadCall& a) { return a.C > HD_MAX_C; }
constexpr int HD_BOXES = 54;  // of HD_BOX16 in shared memory; a tile of rows or columns is 4 kboxes + 1 of them

// Class tiles of one launch for both gradients, 0: two kernels. Shared memory holds the W of a launch next to two tiles of P
// and two of X, tensor memory its dW and a dX next to two tiles of s. Up to 32 channels more classes take several launches,
// which carry dX on in fp32, where a launch has four tiles, the voxels give every CTA four, and the sums stay about as large
// as L2. Loss and gradients of 401280 voxels x 32 channels x 1001 classes 366 us, in two kernels 431; 2^18 x 16 x 2000 420 and
// 514; 2^19 x 24 x 3000 1425 and 1549; but 2^20 x 32 x 600 (three tiles) 701 and 663, 40000 x 32 x 1500 119 and 111, and the
// gradients alone of 2^20 x 64 x 385 749 where 512 classes take 417 in two kernels; class weights 474 and 463 for 401280 x 32 x 1001. Few voxels want P
// in two parts; with class weights more are few, since the rounding of u X stands next to P's. Error of dW out of this
// kernel, class weights and 60 % of the voxels ignored, in parts of its norm (24 channels x 35 classes, 64 x 147, 16 x 257):
// 1.7 to 2.8e-3 at 129 voxels, up to 2.4e-3 at 500, up to 2.0e-3 at 2000, 0.7 to 1.3e-3 at 4000, 0.6 to 0.8e-3 at 8000 and
// falling; with P in two parts 4e-6. A bf16 dW's own rounding is 1.7e-3: the limit stands where the kernel's error is below
// it. What that costs (loss and gradients of 64 x 147, this kernel / P in two parts): 29 / 36 us at 200 voxels, 46 / 55 at 4000.
constexpr int HB_FEW_WEIGHTED = 4096;
static int head_both(const HeadCall& a) {
  if (a.V <= (a.cw == nullptr ? HD_FEW : HB_FEW_WEIGHTED) || a.K > 65000) return 0;
  const int cpad = (a.C + 15) / 16 * 16, kboxes = (a.C + 63) / 64, kt = (a.K + HD_TILE - 1) / HD_TILE;
  auto fits = [&](int n) {
    return (n + 1) * cpad <= 256 &&
           (n + 2) * (4 * kboxes + 1) + 16 + 4 * kboxes + (n + 1) / 2 + (a.cw != nullptr) <= HD_BOXES;
  };
  int most = 0;
  while (most < 4 && fits(most + 1)) ++most;
  if (most >= kt) return kt;
  if (a.cw != nullptr || cpad > 32 || a.V < 4 * 148 * HD_TILE || hd_pad(a.V) * cpad * 4 > (128LL << 20)) return 0;
  const int launches = (kt + most - 1) / most, each = (kt + launches - 1) / launches;
  return each == 4 ? 4 : 0;
}

static void head_geometry(const HeadCall& a, int mode, HeadParams& p) {
  memset(&p, 0, sizeof(p));
  p.C = a.C;
  p.cpad = (a.C + 15) / 16 * 16;
  p.kboxes = (a.C + 63) / 64;
  p.ksteps = p.cpad / 16;
  p.rows = mode >= HEAD_DW ? a.K : a.V;
  p.cols = mode >= HEAD_DW ? a.V : a.K;
  if (mode == HEAD_BOTH && p.rows > (long long)head_both(a) * HD_TILE) p.rows = (long long)head_both(a) * HD_TILE;  // of a launch
  p.row_tiles = (int)((p.rows + HD_TILE - 1) / HD_TILE);
  p.col_tiles = (int)((p.cols + HD_TILE - 1) / HD_TILE);
  p.rows_pad = hd_pad(p.rows);
  p.status = a.status;
  if (mode == HEAD_BOTH) {
    p.splits = p.col_tiles < 148 ? p.col_tiles : 148;  // CTAs, each with sums of its own
    p.accs = (p.row_tiles + 2) * p.cpad <= 256 ? 2 : 1;
    const int tile = 4 * p.kboxes + 1, left = HD_BOXES - p.row_tiles * tile - 4 * p.kboxes - (p.row_tiles + 1) / 2 -
                                              (a.cw != nullptr);
    p.stages = (left - 16) / tile;
    if (p.stages > 6) p.stages = 6;
    return;
  }
  head_split(p.row_tiles, p.col_tiles, &p.splits, &p.tiles_per_split);
  if (mode == HEAD_ROWS) {
    // With four row tiles a job the rounds have four tiles for each of theirs; with one, four of a job's tiles run side by
    // side, so one with fewer is as long. Four and one: 407 and 494 us for 2 x 128^3 voxels x 64 channels x 257 classes, 34
    // and 37 for 64^3 x 64 x 147; 37 and 35 for 100000 x 128 x 500, where it takes one.
    p.together = 1;
    if (p.kboxes <= 2) {
      int s4 = 1, per4 = 1;
      const int rows4 = (p.row_tiles + 3) / 4;
      head_split(rows4, p.col_tiles, &s4, &per4);
      const long long cost4 = (((long long)rows4 * s4 + 147) / 148) * (4 * per4 + 2);
      const long long cost1 = (((long long)p.row_tiles * p.splits + 147) / 148) * ((p.tiles_per_split > 4 ? p.tiles_per_split : 4) + 2);
      if (cost4 <= cost1) {
        p.together = 4;
        p.splits = s4;
        p.tiles_per_split = per4;
        p.whole = s4 == 1;
      }
    }
    p.rbufs = p.together == 4 ? (p.kboxes == 1 ? 8 : 4) : p.kboxes <= 2 ? 2 : 1;
    p.stages = p.kboxes == 1 ? (p.together == 4 ? 4 : 8) : p.kboxes == 2 ? (p.together == 4 ? 2 : 4) : p.kboxes == 3 ? 3 : 2;
    return;
  }
  p.bufs = p.cpad <= 128 ? 3 : 2;
  p.accs = p.cpad <= 64 ? 2 : 1;
  // One or two resident tiles, the rest in the ring. A tile stays until its second MMA, which is `bufs` tiles later, and
  // only what is left then hides the latency of a load.
  p.rbufs = p.kboxes == 1 ? 2 : 1;
  p.stages = p.kboxes == 1 ? 8 : p.kboxes == 2 ? 5 : p.kboxes == 3 ? 3 : 2;
}

template <int MODE, bool FLAG>
static int head_launch(const HeadCall& a, HeadParams& p, cudaStream_t stream) {
  constexpr bool rows = MODE == HEAD_ROWS, both = MODE == HEAD_BOTH, dw = MODE >= HEAD_DW;
  const long long dv[2] = {a.C, a.V}, dk[2] = {a.C, a.K}, st[2] = {1, a.C};
  const int box[2] = {64, HD_TILE};
  int rc = make_map_bf16(&p.mapR, dw ? a.w : a.x, 2, dw ? dk : dv, st, box, 128);
  if (rc) return rc;
  rc = make_map_bf16(&p.mapQ, dw ? a.x : a.w, 2, dw ? dv : dk, st, box, 128);
  if (rc) return rc;
  const long long st16[2] = {1, 16}, xv[2] = {16, hd_pad(a.V)}, wk[2] = {16, hd_pad(a.K)};
  const int box16[2] = {16, HD_TILE};
  const uint4* w16 = a.w16 + (MODE == HEAD_DW ? 2 * hd_pad(a.K) : 0);
  if (!rows) {
    rc = make_map_bf16(&p.mapR16, dw ? w16 : a.x16, 2, dw ? wk : xv, st16, box16, 32);
    if (rc) return rc;
  }
  if (!both) {
    rc = make_map_bf16(&p.mapQ16, dw ? a.x16 : w16, 2, dw ? xv : wk, st16, box16, 32);
    if (rc) return rc;
  } else {
    const int boxo[2] = {64, 32};
    rc = make_map_bf16(&p.mapO, a.dx, 2, dv, st, boxo, 128);
    if (rc) return rc;
  }
  void (*kernel)(HeadParams) = nullptr;
  if constexpr (rows) kernel = head_rows_kernel<FLAG>;
  else if constexpr (both) kernel = head_both_kernel<FLAG>;
  else kernel = head_grad_kernel<MODE, FLAG>;
  const size_t smem = 1024 + (size_t)((both ? p.row_tiles : p.rbufs) + p.stages) * p.kboxes * HD_BOX +
                      (size_t)((both ? p.row_tiles : rows ? 1 : p.rbufs) + p.stages) * HD_BOX16 +
                      (both ? 4 * HD_BOX + p.kboxes * HD_BOX + (p.row_tiles * 4 + (FLAG ? p.row_tiles + p.stages : 0)) * HD_TILE * 4 : 0);
  static std::atomic<unsigned long long> allowed{0};  // devices on which the kernel may have as much as it can need
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return SB_ERR_DRIVER;
  if (dev > 63 || !(allowed.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 1024 + HD_BOXES * HD_BOX16) != cudaSuccess)
      return SB_ERR_DRIVER;
    if (dev <= 63) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const long long jobs =
      both ? p.splits : (long long)(rows && p.together == 4 ? (p.row_tiles + 3) / 4 : p.row_tiles) * p.splits;
  kernel<<<(int)(jobs < 148 ? jobs : 148), both ? HB_THREADS : HD_THREADS, smem, stream>>>(p);
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}
// statistics that head_rows_kernel leaves of a row
static int head_shares(const HeadParams& p) { return p.splits * (p.together == 4 ? 1 : 4); }

static bool shape_ok(long long V, int K, int C) {
  return V >= 1 && V <= (1LL << 31) - 1024 && K >= 1 && K <= (1 << 30) && C >= 8 && C % 8 == 0 && C <= 32768;
}

// The forward pass's state and the scratch of each pass, in the caller's memory (256-byte aligned).
static long long head_state(HeadCall& a, void* base) {
  char* at = (char*)base;
  auto take = [&](long long bytes) { char* o = at; at += (bytes + 255) / 256 * 256; return o; };
  char* head = take(32);
  a.total = (double*)head;
  a.den = (float*)(head + 16);
  a.lse2 = (float*)take(4 * hd_pad(a.V));
  a.y = (int*)take(4 * hd_pad(a.V));
  a.bias2 = (float*)take(4 * hd_pad(a.K));
  if (!wide(a)) {
    a.w16 = (uint4*)take(64 * hd_pad(a.K));
    if (head_both(a)) a.hit = (uint32_t*)take(4 * hd_pad(a.V));
  }
  return at - (char*)base;
}
struct HeadFwdScratch {
  double* sums;
  float2* part;
  float* tl;
};
static long long head_fwd_scratch(const HeadCall& a, HeadFwdScratch& f, void* base) {
  HeadParams p;
  head_geometry(a, HEAD_ROWS, p);
  const long long splits = wide(a) ? head_wide_splits(a.V, a.K) : head_shares(p);
  char* at = (char*)base;
  auto take = [&](long long bytes) { char* o = at; at += (bytes + 255) / 256 * 256; return o; };
  f.sums = (double*)take(16LL * HD_SUM_BLOCKS);
  f.part = (float2*)take(8 * splits * p.rows_pad);
  f.tl = (float*)take(4 * p.rows_pad);
  return at - (char*)base;
}
// both gradients wanted, and one kernel makes them
static bool at_once(const HeadCall& a) {
  return !wide(a) && a.dx != nullptr && (a.dw != nullptr || a.db != nullptr) && head_both(a);
}
static long long head_bwd_scratch(HeadCall& a, void* base) {
  char* at = (char*)base;
  auto take = [&](long long bytes) { char* o = at; at += (bytes + 255) / 256 * 256; return o; };
  a.scale = (float*)take(4);
  if (at_once(a)) {
    HeadParams p;
    head_geometry(a, HEAD_BOTH, p);
    a.scratch = (float*)at;
    return at - (char*)base + 4 * (p.splits * p.rows_pad * (p.cpad + 1) + (p.rows < a.K ? hd_pad(a.V) * p.cpad : 0));
  }
  a.g = (float*)take(4 * hd_pad(a.V));
  if (wide(a)) {
    a.u = (float*)take(4 * hd_pad(a.V));
    a.lse2p = (float*)take(4 * hd_pad(a.V));
  } else {
    a.x16 = (uint4*)take(32 * hd_pad(a.V));
  }
  a.scratch = (float*)at;
  if (wide(a)) return at - (char*)base + 4 * head_wide_scratch(a);
  HeadParams p;
  head_geometry(a, HEAD_DX, p);
  const long long dx = p.splits == 1 ? 0 : p.splits * p.rows_pad * p.cpad;
  head_geometry(a, HEAD_DW, p);
  const long long dw = p.splits * p.rows_pad * (p.cpad + 4);
  return at - (char*)base + 4 * (dx > dw ? dx : dw);
}

static HeadReduce reduce_of(const float* ws, int slices, const HeadParams& p, int C, int ld, int kind, void* out) {
  HeadReduce r;
  r.ws = ws; r.slices = slices; r.C = C; r.ld = ld; r.kind = kind; r.out = out;
  r.rows = p.rows; r.rows_pad = p.rows_pad;
  const int each = slices <= HD_FEW_SLICES ? 256 : 32;  // outputs of a block
  const long long blocks = out == nullptr ? 0 : (p.rows * C + each - 1) / each;
  r.blocks = (int)(blocks < 148 * 8 ? blocks : 148 * 8);
  return r;
}
static void head_reduce(const HeadReduce& a, const HeadReduce& b, const float* scale, cudaStream_t stream) {
  head_reduce_kernel<<<a.blocks + b.blocks, 256, 0, stream>>>(a, b, scale);
  sb_count_launch(1);
}

static int head_narrow_backward(const HeadCall& a, cudaStream_t stream) {
  HeadParams p;
  int rc = 0;
  const bool few = a.V <= HD_FEW;
  if (at_once(a)) {
    head_geometry(a, HEAD_BOTH, p);
    p.colhit = a.hit;
    p.lse2 = a.lse2;
    p.gout = a.gout;
    p.den = a.den;
    p.scale = a.scale;
    p.cw = a.cw;
    p.out = a.dx;
    p.ws = a.scratch;
    p.ws_b = p.ws + p.splits * p.rows_pad * p.cpad;
    p.part_x = reinterpret_cast<float4*>(p.ws_b + p.splits * p.rows_pad);
    const long long most = p.rows;
    for (long long row0 = 0; row0 < a.K; row0 += most) {
      p.row0 = (int)row0;
      p.rows = a.K - row0 < most ? a.K - row0 : most;
      p.row_tiles = (int)((p.rows + HD_TILE - 1) / HD_TILE);
      p.first = row0 == 0;
      p.last = row0 + most >= a.K;
      rc = a.cw != nullptr ? head_launch<HEAD_BOTH, true>(a, p, stream) : head_launch<HEAD_BOTH, false>(a, p, stream);
      if (rc) return rc;
      auto from = [&](void* out, int kind, long long i) {
        return out == nullptr ? nullptr : (void*)((char*)out + i * (kind == 2 ? 4 : 2));
      };
      head_reduce(reduce_of(p.ws, p.splits, p, p.C, p.cpad, a.dw_kind, from(a.dw, a.dw_kind, row0 * a.C)),
                  reduce_of(p.ws_b, p.splits, p, 1, 1, a.db_kind, from(a.db, a.db_kind, row0)), a.scale, stream);
    }
    return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
  }
  if (a.dx != nullptr) {
    head_geometry(a, HEAD_DX, p);
    p.rowg = a.g;
    p.rowy = a.y;
    p.out = a.dx;
    p.ws = a.scratch;
    rc = few ? head_launch<HEAD_DX, true>(a, p, stream) : head_launch<HEAD_DX, false>(a, p, stream);
    if (rc) return rc;
    if (p.splits > 1)
      head_reduce(reduce_of(p.ws, p.splits, p, p.C, p.cpad, 0, a.dx), reduce_of(nullptr, 0, p, 1, 1, 0, nullptr), nullptr,
                  stream);
  }
  if (a.dw != nullptr || a.db != nullptr) {
    head_geometry(a, HEAD_DW, p);
    p.coly = a.y;
    p.roww = a.cw;
    p.ws = a.scratch;
    p.ws_b = a.scratch + p.splits * p.rows_pad * p.cpad;
    rc = few || a.cw != nullptr ? head_launch<HEAD_DW, true>(a, p, stream) : head_launch<HEAD_DW, false>(a, p, stream);
    if (rc) return rc;
    head_reduce(reduce_of(p.ws, p.splits, p, p.C, p.cpad, a.dw_kind, a.dw),
                reduce_of(p.ws_b, 4 * p.splits, p, 1, 1, a.db_kind, a.db), a.scale, stream);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

}  // namespace sb

using namespace sb;

// bytes of the state (0) and of the scratch of the forward (1) and the backward pass (2: one gradient, 3: of features and
// weight or bias); -1: outside the range
extern "C" long long sb_head_bytes(int what, long long V, int K, int C, int weighted) {
  if (!shape_ok(V, K, C) || what < 0 || what > 3) return -1;
  HeadCall a;
  memset(&a, 0, sizeof(a));
  a.V = V;
  a.K = K;
  a.C = C;
  a.cw = weighted ? (const float*)1 : nullptr;  // looked at, not followed
  if (what == 3) { a.dx = (__nv_bfloat16*)1; a.dw = (void*)1; }
  HeadFwdScratch f;
  return what == 0 ? head_state(a, nullptr) : what == 1 ? head_fwd_scratch(a, f, nullptr) : head_bwd_scratch(a, nullptr);
}

extern "C" int sb_head_forward(const void* x, const void* w, const void* bias, int bias_kind, const void* labels,
                               int label_kind, int has_ignore, long long ignore, const float* cw, long long V, int K,
                               int C, void* state, void* scratch, float* loss, uint32_t* status, cudaStream_t stream) {
  if (!shape_ok(V, K, C) || !x || !w || !labels || !state || !scratch || !loss) return SB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(scratch)) & 255) return SB_ERR_ALIGN;
  HeadCall a;
  memset(&a, 0, sizeof(a));
  a.x = (const __nv_bfloat16*)x;
  a.w = (const __nv_bfloat16*)w;
  a.cw = cw;
  a.V = V; a.K = K; a.C = C;
  a.status = status;
  head_state(a, state);
  HeadFwdScratch f;
  head_fwd_scratch(a, f, scratch);
  const long long v_pad = hd_pad(V);
  const int k_pad = (int)hd_pad(K);
  head_prep_kernel<<<hd_blocks(v_pad > k_pad ? v_pad : k_pad, 8), 256, 0, stream>>>(
      labels, label_kind, V, v_pad, K, k_pad, has_ignore, ignore, a.y, bias, bias_kind, a.bias2, a.w16, status);
  sb_count_launch(1);
  int rc, splits;
  if (wide(a)) {
    splits = head_wide_splits(V, K);
    rc = head_wide_forward(a, f.part, f.tl, stream);
  } else {
    HeadParams p;
    head_geometry(a, HEAD_ROWS, p);
    p.part = f.part;
    p.tl = f.tl;
    p.rowy = a.y;
    p.lse2_out = a.lse2;
    p.hit_out = a.hit;
    p.cw = cw;
    p.bias = bias;
    p.bias_kind = bias_kind;
    p.sums = f.sums;
    splits = head_shares(p);
    rc = head_launch<HEAD_ROWS, false>(a, p, stream);
    if (rc) return rc;
    if (p.whole) {
      const int jobs = (p.row_tiles + 3) / 4;
      head_total_kernel<<<1, 256, 0, stream>>>(f.sums, jobs < 148 ? jobs : 148, a.total, loss, a.den);
      sb_count_launch(1);
      return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
    }
  }
  if (rc) return rc;
  // a warp for a voxel: loss of 300 voxels x 64 channels x 20000 classes 19 us, a thread for each 90; of 40000 x 32 x 1001
  // (four shares) 45 and 33
  const bool team = splits > 4;
  // one block, which goes on to the loss, where its rounds cost less than another launch (18 us for 5000 x 64 x 300 both
  // ways on the device, and the launch's 3 us on the host)
  const int blocks = v_pad <= (team ? 256 : 4096) ? 1 : hd_blocks(team ? v_pad * 32 : v_pad, HD_SUM_BLOCKS / 148);
  if (team)
    head_merge_kernel<32><<<blocks, 256, 0, stream>>>(f.part, f.tl, a.y, cw, bias, bias_kind, splits, V, v_pad, a.lse2, a.hit,
                                                      f.sums, a.total, loss, a.den);
  else
    head_merge_kernel<1><<<blocks, 256, 0, stream>>>(f.part, f.tl, a.y, cw, bias, bias_kind, splits, V, v_pad, a.lse2, a.hit,
                                                     f.sums, a.total, loss, a.den);
  if (blocks > 1) head_total_kernel<<<1, 256, 0, stream>>>(f.sums, blocks, a.total, loss, a.den);
  sb_count_launch(blocks > 1 ? 2 : 1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

// scratch bytes of sb_head_predict; -1: outside the range
extern "C" long long sb_head_predict_bytes(long long V, int K, int C) {
  if (!shape_ok(V, K, C)) return -1;
  HeadCall a;
  memset(&a, 0, sizeof(a));
  a.V = V; a.K = K; a.C = C;
  HeadFwdScratch f;
  return head_state(a, nullptr) + head_fwd_scratch(a, f, nullptr);
}

// out [V]: the class of the largest logit, the lowest of several; a NaN is the largest
extern "C" int sb_head_predict(const void* x, const void* w, const void* bias, int bias_kind, long long V, int K, int C,
                               void* scratch, long long* out, uint32_t* status, cudaStream_t stream) {
  if (!shape_ok(V, K, C) || !x || !w || !scratch || !out) return SB_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(scratch) & 255) return SB_ERR_ALIGN;
  HeadCall a;
  memset(&a, 0, sizeof(a));
  a.x = (const __nv_bfloat16*)x;
  a.w = (const __nv_bfloat16*)w;
  a.V = V; a.K = K; a.C = C;
  a.status = status;
  HeadFwdScratch f;
  head_fwd_scratch(a, f, (char*)scratch + head_state(a, scratch));
  const int k_pad = (int)hd_pad(K);
  head_prep_kernel<<<hd_blocks(k_pad, 8), 256, 0, stream>>>(nullptr, 4, V, 0, K, k_pad, 0, 0, nullptr, bias, bias_kind,
                                                            a.bias2, a.w16, status);
  sb_count_launch(1);
  int rc, splits;
  if (wide(a)) {
    splits = head_wide_splits(V, K);
    rc = head_wide_predict(a, f.part, stream);
  } else {
    HeadParams p;
    head_geometry(a, HEAD_ROWS, p);
    p.part = f.part;
    splits = head_shares(p);
    rc = head_launch<HEAD_ROWS, true>(a, p, stream);
  }
  if (rc) return rc;
  if (splits > 4) head_arg_kernel<32><<<hd_blocks(V * 32, 8), 256, 0, stream>>>(f.part, splits, V, hd_pad(V), out);
  else head_arg_kernel<1><<<hd_blocks(V, 8), 256, 0, stream>>>(f.part, splits, V, hd_pad(V), out);
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

// the loss from the state's two sums (its first 16 bytes) after they were added over the shards
extern "C" int sb_head_total(void* state, float* loss, cudaStream_t stream) {
  if (!state || !loss) return SB_ERR_SHAPE;
  double* total = (double*)state;
  head_total_kernel<<<1, 256, 0, stream>>>(total, 1, total, loss, (float*)((char*)state + 16));
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

// dx, dw and db (each optional) from gout and the state; dw / db in fp32 when dw_kind / db_kind is 2, else bf16
extern "C" int sb_head_backward(const void* x, const void* w, const float* cw, long long V, int K, int C, void* state,
                                void* scratch, const float* gout, void* dx, void* dw, int dw_kind, void* db, int db_kind,
                                uint32_t* status, cudaStream_t stream) {
  if (!shape_ok(V, K, C) || !x || !w || !state || !scratch || !gout) return SB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(scratch)) & 255) return SB_ERR_ALIGN;
  if ((reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(dw)) & 15) return SB_ERR_ALIGN;
  HeadCall a;
  memset(&a, 0, sizeof(a));
  a.x = (const __nv_bfloat16*)x;
  a.w = (const __nv_bfloat16*)w;
  a.cw = cw;
  a.V = V; a.K = K; a.C = C;
  a.status = status;
  a.dx = (__nv_bfloat16*)dx;
  a.dw = dw; a.dw_kind = dw_kind;
  a.db = db; a.db_kind = db_kind;
  head_state(a, state);
  a.gout = gout;
  head_bwd_scratch(a, scratch);
  if (!at_once(a)) {
    const long long v_pad = hd_pad(V);
    head_weights_kernel<<<hd_blocks(v_pad, 8), 256, 0, stream>>>(a, gout, v_pad);
    sb_count_launch(1);
  }
  return wide(a) ? head_wide_backward(a, stream) : head_narrow_backward(a, stream);
}
