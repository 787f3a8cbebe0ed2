// Cross entropy of a head over features of more than 256 channels (head_loss.cuh): a tile of logits costs more on the
// tensor cores than its exponentials, so the passes are matrix products with something fused into their epilogue, on SM
// pairs (tcgen05 cta_group::2): a pair multiplies 256 rows by 256 columns, each CTA loads its own 128 rows and one half
// of the columns (64 bytes a clock and SM out of L2, half of what one CTA alone would read).
//   WIDE_LSE  rows = voxels, columns = classes: running maximum and sum of every row over the class tiles of a job
//   WIDE_ARG  the same with the largest logit and its class in their place
//   WIDE_D    rows = classes, columns = voxels: P^T = p - [j = y] in bf16, a piece of the classes by a piece of the
//             voxels at a time (HW_PIECE elements); db
//   WIDE_OUT  dX = g P W and dW = P^T (u X) of the piece (head_loss.cu for g and u). P^T is read K-major for dW and
//             MN-major for dX, W and X MN-major: nothing is transposed in memory. Long reductions are cut into slices
//             that are added in order.
// Roundings as in head_loss.cu; here the class weights go into a copy of X (whose roundings are independent of one
// another) and up to HD_FEW voxels P^T is followed by its remainder, along which the products' reductions go on.
// One thread holds a row of a tile, so a row's maximum, sum and db need no exchange.
// Bound: the tensor cores and, in long runs, the power. 8192 voxels x 1024 channels x 32771 classes: loss 339 us, loss and
// gradients 1796, which is 2.2 TFLOP with the logits' two times at 1.22 PFLOP/s.
#include <limits.h>

#include <atomic>

#include "head_loss.cuh"
#include "pair.cuh"

namespace sb {

constexpr int HW_THREADS = 320;
constexpr int HW_STAGES = 6;
constexpr int HW_STAGE = 32768;  // 64 of K for 128 rows of A and 128 columns of B
// 128 MB of P^T at a time. Larger pieces have fewer tails and fewer sums to carry on, smaller ones stay in L2: the gradients
// of 40000 voxels x 512 channels x 8000 classes take 2.02 ms with 64 MB, 1.87 with 128, 1.72 with 192; those of 8192 x 1024 x
// 32771 2.06, 1.96 and 1.89. The memory counts here: half of the last step for two thirds of its size.
constexpr long long HW_PIECE = 64LL << 20;

enum WideEpi { WIDE_LSE = 0, WIDE_D = 1, WIDE_OUT = 2, WIDE_ARG = 3 };

struct WideParams {
  CUtensorMap mapA, mapB;
  int row_tiles, col_tiles;     // of 256
  int splits, tiles_per_split;  // LSE / D: of the column tiles
  int kc, kslices, kc_per_slice;
  int cols;                     // real columns, for the last tile's width
  long long rows_pad;
  const int* y;                 // LSE: label of a row; D: of a column
  const float* colp;            // LSE: bias2; D: lse2p
  const float* colg;            // D: u
  const float* rowp;            // D: bias2
  int row0;                     // D: class of row 0
  float2* part;
  float* tl;
  __nv_bfloat16* dl;            // D: [rows][ldd]; the remainder lo_rows rows further
  long long ldd;
  int lo_rows;                  // 0: no remainder
  float* ws_b;                  // D: [2 splits][rows_pad]
  // OUT: [rows][C]; add: acc is added to the product; the sum goes, scaled, to out16 / out32, or back to acc
  int kc0;                      // blocks of the reduction behind which the remainder's begin
  const float* row_scale;       // of a row (0: the result is 0), or
  const float* scale;           // of all
  long long rows;
  float* acc;
  int add;
  __nv_bfloat16* out16;
  float* out32;
  float* slices;                // [kslices][rows][C] when kslices > 1
  uint32_t* status;
};

constexpr int HW_STRIDE = 20;  // floats of a staged row of 16

// rows x C sums: v = (add ? acc : 0) + product, then scaled to an output or back to acc; four columns
__device__ __forceinline__ void hw_sink(float* acc, int add, __nv_bfloat16* out16, float* out32, float scale, long long at,
                                        float4 f) {
  if (add) {
    const float4 a = *reinterpret_cast<const float4*>(acc + at);
    f.x += a.x; f.y += a.y; f.z += a.z; f.w += a.w;
  }
  if (out16 != nullptr || out32 != nullptr) {
    // a voxel that takes no part has no gradient, whatever its features hold
    f.x = scale == 0.f ? 0.f : f.x * scale;
    f.y = scale == 0.f ? 0.f : f.y * scale;
    f.z = scale == 0.f ? 0.f : f.z * scale;
    f.w = scale == 0.f ? 0.f : f.w * scale;
  }
  if (out16 != nullptr)
    *reinterpret_cast<uint2*>(out16 + at) = make_uint2(pack_bf16x2(f.x, f.y), pack_bf16x2(f.z, f.w));
  else
    *reinterpret_cast<float4*>((out32 != nullptr ? out32 : acc) + at) = f;
}

template <int EPI, int A_MN, int B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(HW_THREADS, 1)
    head_wide_kernel(const __grid_constant__ WideParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[HW_STAGES], empty[HW_STAGES], tfull[2], tempty[2];
  __shared__ float s_m[EPI == WIDE_OUT ? 1 : 128], s_s[EPI == WIDE_OUT ? 1 : 128], s_t[EPI == WIDE_OUT ? 1 : 128];
  __shared__ __align__(16) float s_stage[EPI == WIDE_OUT ? 8 : 1][EPI == WIDE_OUT ? 32 * HW_STRIDE : 1];
  __shared__ uint32_t tmem_base_s, abort_s;
  volatile uint32_t* abort_flag = &abort_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  // LSE and D: a job is a row tile and a run of column tiles; OUT: a row tile, a column tile and a slice of K
  const int jobs = EPI == WIDE_OUT ? p.row_tiles * p.col_tiles * p.kslices : p.row_tiles * p.splits;

  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int i = 0; i < HW_STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&tfull[i], 1); mbar_init(&tempty[i], 16); }  // 8 epilogue warps, both CTAs
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem2_alloc(&tmem_base_s, 512);
    tmem2_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers exist before any copy or arrive targets them
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;

  struct Job {
    int rt, t0, t1, k0, k1, sp;
  };
  auto job_at = [&](int job) {
    Job j;
    if (EPI == WIDE_OUT) {
      j.rt = job % p.row_tiles;
      const int t = job / p.row_tiles;
      j.t0 = t % p.col_tiles;
      j.t1 = j.t0 + 1;
      j.sp = t / p.col_tiles;
      j.k0 = j.sp * p.kc_per_slice;
      j.k1 = j.k0 + p.kc_per_slice < p.kc ? j.k0 + p.kc_per_slice : p.kc;
    } else {
      j.rt = job % p.row_tiles;
      j.sp = job / p.row_tiles;
      j.t0 = j.sp * p.tiles_per_split;
      j.t1 = j.t0 + p.tiles_per_split < p.col_tiles ? j.t0 + p.tiles_per_split : p.col_tiles;
      j.k0 = 0;
      j.k1 = p.kc;
    }
    return j;
  };
  auto cols_of = [&](int t) -> int {  // columns of tile t, up to a multiple of 32
    const int left = p.cols - t * 256;
    return left >= 256 ? 256 : (left + 31) / 32 * 32;
  };

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&p.mapA);
      tma_prefetch_desc(&p.mapB);
      uint32_t st = 0, ph = 0;
      bool ok = true;
      for (int job = pair; job < jobs && ok; job += npairs) {
        const Job j = job_at(job);
        const int row = j.rt * 256 + (int)rank * 128;
        for (int t = j.t0; t < j.t1 && ok; ++t) {
          const int nc = cols_of(t), col = t * 256 + (int)rank * (nc / 2);
          const int nb = B_MN ? (nc / 2 + 63) / 64 : 0;
          for (int k = j.k0; k < j.k1; ++k) {
            if (!mbar_wait_cl(&empty[st], ph ^ 1u, abort_flag, p.status, 101)) { ok = false; break; }
            const uint32_t bar = map_to_rank(smem_u32(&full[st]), 0);
            if (rank == 0) mbar_expect_tx(&full[st], 2u * (16384u + (B_MN ? nb * 8192u : 16384u)));  // both CTAs' bytes
            uint8_t* sa = smem + st * HW_STAGE;
            uint8_t* sb = sa + 16384;
            // behind block kc0 the reduction runs over the remainder, against the same B
            const bool lo = EPI == WIDE_OUT && k >= p.kc0;
            const int at = (lo ? k - p.kc0 : k) * 64, down = lo ? p.lo_rows : 0;
            if (A_MN) {
              for (int i = 0; i < 2; ++i) tma2_load_2d(sa + i * 8192, &p.mapA, bar, row + i * 64, at + down);
            } else {
              tma2_load_2d(sa, &p.mapA, bar, at, row + down);
            }
            if (B_MN) {
              for (int i = 0; i < nb; ++i) tma2_load_2d(sb + i * 8192, &p.mapB, bar, col + i * 64, at);
            } else {
              tma2_load_2d(sb, &p.mapB, bar, at, col);
            }
            if (++st == HW_STAGES) { st = 0; ph ^= 1u; }
          }
        }
      }
      // every release of a stage that this CTA filled has arrived before the CTA may leave
      for (int i = 0; i < HW_STAGES && ok; ++i) {
        if (!mbar_wait_cl(&empty[st], ph ^ 1u, abort_flag, p.status, 102)) ok = false;
        if (++st == HW_STAGES) { st = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leader = elect_one();
      const uint32_t hi = desc_hi(8u * 128u, 2u);
      const uint32_t s0 = smem_u32(smem);
      constexpr uint32_t A_STEP = A_MN ? 128u : 2u, B_STEP = B_MN ? 128u : 2u;  // 16 of K, in 16-byte units
      uint32_t st = 0, ph = 0, b = 0, bph = 0;
      bool ok = true;
      for (int job = pair; job < jobs && ok; job += npairs) {
        const Job j = job_at(job);
        for (int t = j.t0; t < j.t1 && ok; ++t) {
          if (!__all_sync(0xffffffffu, mbar_wait_cl(&tempty[b], bph ^ 1u, abort_flag, p.status, 103))) { ok = false; break; }
          tc_fence_after();
          const uint32_t idesc = make_idesc_bf16(256, cols_of(t), A_MN, B_MN);
          for (int k = j.k0; k < j.k1; ++k) {
            if (!__all_sync(0xffffffffu, mbar_wait_cl(&full[st], ph, abort_flag, p.status, 104))) { ok = false; break; }
            tc_fence_after();
            if (leader) {
              const uint32_t a_lo = desc_lo(s0 + st * HW_STAGE, A_MN ? 8192u : 16u);
              const uint32_t b_lo = desc_lo(s0 + st * HW_STAGE + 16384u, B_MN ? 8192u : 16u);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                tc2_mma_bf16_pred(tmem + b * 256u, a_lo + i * A_STEP, hi, b_lo + i * B_STEP, hi, idesc,
                                  k != j.k0 || i != 0 ? 1u : 0u);
              tc2_commit_both(&empty[st]);
            }
            __syncwarp();
            if (++st == HW_STAGES) { st = 0; ph ^= 1u; }
          }
          if (ok && leader) tc2_commit_both(&tfull[b]);
          __syncwarp();
          b ^= 1u;
          if (b == 0) bph ^= 1u;
        }
      }
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const int row = quad * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t release[2] = {map_to_rank(smem_u32(&tempty[0]), 0), map_to_rank(smem_u32(&tempty[1]), 0)};
    uint32_t b = 0, bph = 0;
    bool ok = true;
    for (int job = pair; job < jobs && ok; job += npairs) {
      const Job j = job_at(job);
      const long long r = (long long)j.rt * 256 + rank * 128 + row;
      const int y = EPI == WIDE_LSE ? p.y[r] : 0;
      const float rp = EPI == WIDE_D ? p.rowp[r] : 0.f;
      float scale = 1.f;  // OUT: of the row
      if (EPI == WIDE_OUT && p.row_scale != nullptr) scale = r < p.rows ? __ldg(p.row_scale + r) : 0.f;
      else if (EPI == WIDE_OUT && p.scale != nullptr) scale = __ldg(p.scale);
      // D: rows behind the piece's last class (up to the 64 that the products read) are left as they are
      const bool live = EPI != WIDE_D || r < p.rows;
      float m = -INFINITY, s = 0.f, tl = 0.f, db = 0.f;
      int best = INT_MAX;
      for (int t = j.t0; t < j.t1; ++t) {
        if (!__all_sync(0xffffffffu, mbar_wait_cl(&tfull[b], bph, abort_flag, p.status, 105))) { ok = false; break; }
        tc_fence_after();
        const int nc = live ? cols_of(t) : 0, c_abs = t * 256;
        for (int c0 = half * 32; c0 < nc; c0 += 64) {  // every second 32 columns are the other group's
          uint32_t v[32];
          tmem_ld_32x32(lane_base + b * 256 + c0, v);
          tmem_ld_wait();
          float f[32];
          if (EPI != WIDE_OUT) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 cp = __ldg(reinterpret_cast<const float4*>(p.colp + c_abs + c0 + i));
              const float cv[4] = {cp.x, cp.y, cp.z, cp.w};
#pragma unroll
              for (int e = 0; e < 4; ++e)
                f[i + e] = fmaf(__uint_as_float(v[i + e]), HD_LOG2E, EPI == WIDE_D ? rp - cv[e] : cv[e]);
            }
          }
          if (EPI == WIDE_ARG) {
            // columns behind the last class take no part: zeros of w there, and 0 * inf of a feature is a NaN
            const int left = p.cols - (c_abs + c0);
            if (left < 32) {
#pragma unroll
              for (int i = 0; i < 32; ++i) f[i] = i < left ? f[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (f[i] > m || (f[i] != f[i] && m == m)) { m = f[i]; best = c_abs + c0 + i; }
          } else if (EPI == WIDE_LSE) {
            const int at = y - (c_abs + c0);
            if ((unsigned)at < 32u) {
#pragma unroll
              for (int i = 0; i < 32; ++i) tl = i == at ? f[i] : tl;
            }
            float mx = f[0];
#pragma unroll
            for (int i = 1; i < 32; ++i) mx = fmaxf(mx, f[i]);
            if (mx > m) {
              s *= hd_ex2(m - mx);
              m = mx;
            }
            const float base = m == -INFINITY ? 0.f : m;
            float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              a0 += hd_ex2(f[i] - base);
              a1 += hd_ex2(f[i + 1] - base);
              a2 += hd_ex2(f[i + 2] - base);
              a3 += hd_ex2(f[i + 3] - base);
            }
            s += (a0 + a1) + (a2 + a3);
          } else if (EPI == WIDE_D) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            const int cls = p.row0 + (int)r;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 cu = __ldg(reinterpret_cast<const float4*>(p.colg + c_abs + c0 + i));
              const int4 cy = __ldg(reinterpret_cast<const int4*>(p.y + c_abs + c0 + i));
              f[i] = hd_ex2(f[i]) - (cy.x == cls ? 1.f : 0.f);
              f[i + 1] = hd_ex2(f[i + 1]) - (cy.y == cls ? 1.f : 0.f);
              f[i + 2] = hd_ex2(f[i + 2]) - (cy.z == cls ? 1.f : 0.f);
              f[i + 3] = hd_ex2(f[i + 3]) - (cy.w == cls ? 1.f : 0.f);
              d[0] = fmaf(cu.x, f[i], d[0]);
              d[1] = fmaf(cu.y, f[i + 1], d[1]);
              d[2] = fmaf(cu.z, f[i + 2], d[2]);
              d[3] = fmaf(cu.w, f[i + 3], d[3]);
            }
            db += (d[0] + d[1]) + (d[2] + d[3]);
            uint32_t o[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
            uint4* dst = reinterpret_cast<uint4*>(p.dl + r * p.ldd + c_abs + c0);
#pragma unroll
            for (int i = 0; i < 2; ++i)
              st_global_v8(dst + 2 * i, make_uint4(o[8 * i], o[8 * i + 1], o[8 * i + 2], o[8 * i + 3]),
                           make_uint4(o[8 * i + 4], o[8 * i + 5], o[8 * i + 6], o[8 * i + 7]));
            if (p.lo_rows) {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                o[i] = pack_bf16x2(f[2 * i] - __uint_as_float(o[i] << 16), f[2 * i + 1] - __uint_as_float(o[i] & 0xFFFF0000u));
              dst = reinterpret_cast<uint4*>(p.dl + (r + p.lo_rows) * p.ldd + c_abs + c0);
#pragma unroll
              for (int i = 0; i < 2; ++i)
                st_global_v8(dst + 2 * i, make_uint4(o[8 * i], o[8 * i + 1], o[8 * i + 2], o[8 * i + 3]),
                             make_uint4(o[8 * i + 4], o[8 * i + 5], o[8 * i + 6], o[8 * i + 7]));
            }
          } else {
            // A lane holds a row, and its stores would each be in another line: the warp's rows go through shared memory,
            // so that four lanes store 64 bytes of a row (bf16) or of half a row's 32 columns (fp32).
            float* stage = s_stage[warp - 2];
            const int rr = lane >> 2, piece = lane & 3;  // row rr + 8 i, quarter of it
            if (p.kslices == 1 && p.out16 != nullptr && !p.add) {
              uint32_t o[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                // a voxel that takes no part has no gradient, whatever its features hold
                const float lo = scale == 0.f ? 0.f : scale * __uint_as_float(v[2 * i]);
                const float hi = scale == 0.f ? 0.f : scale * __uint_as_float(v[2 * i + 1]);
                o[i] = pack_bf16x2(lo, hi);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint4*>(stage + lane * HW_STRIDE + 4 * i) =
                    make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
              __syncwarp();
              const int col = c_abs + c0 + piece * 8;
              __nv_bfloat16* dst = p.out16 + (r - lane + rr) * p.cols + col;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (r - lane + rr + 8 * i < p.rows && col < p.cols)
                  *reinterpret_cast<uint4*>(dst + (long long)(8 * i) * p.cols) =
                      *reinterpret_cast<const uint4*>(stage + (rr + 8 * i) * HW_STRIDE + piece * 4);
              __syncwarp();
            } else {
              float* acc = p.kslices > 1 ? p.slices + (long long)j.sp * p.rows * p.cols : p.acc;
              const bool whole = p.kslices == 1;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  *reinterpret_cast<uint4*>(stage + lane * HW_STRIDE + 4 * i) =
                      make_uint4(v[16 * h + 4 * i], v[16 * h + 4 * i + 1], v[16 * h + 4 * i + 2], v[16 * h + 4 * i + 3]);
                const int col = c_abs + c0 + h * 16 + piece * 4;
                const long long at = (r - lane + rr) * p.cols + col, step = 8LL * p.cols;
                float4 before[4];  // what is added to, requested ahead of everything
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  before[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                  if (whole && p.add && r - lane + rr + 8 * i < p.rows && col < p.cols)
                    before[i] = *reinterpret_cast<const float4*>(acc + at + i * step);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float k = __shfl_sync(0xffffffffu, scale, rr + 8 * i);
                  float4 f = *reinterpret_cast<const float4*>(stage + (rr + 8 * i) * HW_STRIDE + piece * 4);
                  f.x += before[i].x; f.y += before[i].y; f.z += before[i].z; f.w += before[i].w;
                  if (r - lane + rr + 8 * i < p.rows && col < p.cols)
                    hw_sink(acc, 0, whole ? p.out16 : nullptr, whole ? p.out32 : nullptr, k, at + i * step, f);
                }
                __syncwarp();
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(release[b]);
        b ^= 1u;
        if (b == 0) bph ^= 1u;
      }
      if (EPI == WIDE_ARG) {
        if (half == 1) { s_m[row] = m; s_s[row] = __int_as_float(best); }
        ok = hd_vote(1, 256, ok);
        if (half == 0 && ok) {
          hd_better(m, best, s_m[row], __float_as_int(s_s[row]));
          p.part[(long long)j.sp * p.rows_pad + r] = make_float2(m, __int_as_float(best));
        }
        hd_vote(1, 256, true);
      }
      if (EPI == WIDE_LSE) {
        if (half == 1) { s_m[row] = m; s_s[row] = s; s_t[row] = tl; }
        ok = hd_vote(1, 256, ok);
        if (half == 0 && ok) {
          const float m1 = s_m[row], mm = fmaxf(m, m1);
          const float base = mm == -INFINITY ? 0.f : mm;
          p.part[(long long)j.sp * p.rows_pad + r] = make_float2(mm, s * hd_ex2(m - base) + s_s[row] * hd_ex2(m1 - base));
          if (y >= j.t0 * 256 && y < j.t1 * 256) p.tl[r] = (y & 32) == 0 ? tl : s_t[row];
        }
        hd_vote(1, 256, true);  // the merge has read what the next job's will overwrite
      }
      if (EPI == WIDE_D && ok) p.ws_b[((long long)j.sp * 2 + half) * p.rows_pad + r] = db;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) __nanosleep(1000);
    __syncthreads();
  }
  cluster_sync_all();  // the leader's MMAs read the peer's shared memory; arrives target the other CTA
  if (warp == 0) {
    __syncwarp();
    tc_fence_after();
    tmem2_dealloc(tmem, 512);
  }
}

// Slices of a product [n][elems], added in order and handed on. (A team of warps for each output, as below, is no faster
// here: 166 us for the loss and gradients of 256 x 1024 x 32771 both ways.)
__global__ void __launch_bounds__(256) head_slices_kernel(const float* __restrict__ slices, int n, long long elems, int C,
                                                          float* acc, int add, __nv_bfloat16* out16, float* out32,
                                                          const float* __restrict__ row_scale,
                                                          const float* __restrict__ scale) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < elems / 4; i += (long long)gridDim.x * 256) {
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float4 a = __ldcs(reinterpret_cast<const float4*>(slices + (long long)k * elems) + i);
      f.x += a.x; f.y += a.y; f.z += a.z; f.w += a.w;
    }
    hw_sink(acc, add, out16, out32, row_scale != nullptr ? row_scale[i * 4 / C] : scale != nullptr ? scale[0] : 1.f, i * 4, f);
  }
}
// the same for the bias's sums: slices [n][ld], rows of them; a warp has 32 rows and every eighth slice
__global__ void __launch_bounds__(256) head_slices_b_kernel(const float* __restrict__ slices, int n, long long ld,
                                                            int rows, float* acc, int add, __nv_bfloat16* out16,
                                                            float* out32, const float* __restrict__ scale) {
  __shared__ float s_part[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, i = blockIdx.x * 32 + lane;
  float f = 0.f;
  if (i < rows) {
#pragma unroll 8
    for (int k = warp; k < n; k += 8) f += slices[(long long)k * ld + i];
  }
  s_part[warp][lane] = f;
  __syncthreads();
  if (warp != 0 || i >= rows) return;
  for (int k = 1; k < 8; ++k) f += s_part[k][lane];
  if (add) f += acc[i];
  if (out16 != nullptr) out16[i] = __float2bfloat16(f * scale[0]);
  else if (out32 != nullptr) out32[i] = f * scale[0];
  else acc[i] = f;
}
// out = u x, eight channels a thread (zeros for a voxel that takes no part, whatever its features hold)
__global__ void __launch_bounds__(256) head_weigh_kernel(const __nv_bfloat16* __restrict__ x, const float* __restrict__ u,
                                                         long long octets, int C, __nv_bfloat16* __restrict__ out) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < octets; i += (long long)gridDim.x * 256) {
    const float k = u[i * 8 / C];
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(x) + i);
    const uint32_t v[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = k == 0.f ? 0u : pack_bf16x2(k * __uint_as_float(v[j] << 16), k * __uint_as_float(v[j] & 0xFFFF0000u));
    reinterpret_cast<uint4*>(out)[i] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// SM pairs that can hold a cluster at the same time (a GPC with an odd SM count leaves one SM out)
template <int EPI, int A_MN, int B_MN>
static int wide_setup(int* pairs) {
  static std::atomic<int> known[64];  // by device; 0: not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return SB_ERR_DRIVER;
  if (dev < 64 && (*pairs = known[dev].load(std::memory_order_relaxed)) > 0) return 0;
  const int smem = 1024 + HW_STAGES * HW_STAGE;
  if (cudaFuncSetAttribute(head_wide_kernel<EPI, A_MN, B_MN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
      cudaSuccess)
    return SB_ERR_DRIVER;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(148);
  cfg.blockDim = dim3(HW_THREADS);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  const bool ok = cudaOccupancyMaxActiveClusters(&n, head_wide_kernel<EPI, A_MN, B_MN>, &cfg) == cudaSuccess;
  cudaGetLastError();
  *pairs = ok && n > 0 && n < 74 ? n : 74;
  if (dev < 64) known[dev].store(*pairs, std::memory_order_relaxed);
  return 0;
}

template <int EPI, int A_MN, int B_MN>
static int wide_launch(WideParams& p, cudaStream_t stream) {
  int most = 0;
  const int rc = wide_setup<EPI, A_MN, B_MN>(&most);
  if (rc) return rc;
  const long long jobs = EPI == WIDE_OUT ? (long long)p.row_tiles * p.col_tiles * p.kslices : (long long)p.row_tiles * p.splits;
  const int pairs = (int)(jobs < most ? jobs : most);
  head_wide_kernel<EPI, A_MN, B_MN><<<2 * pairs, HW_THREADS, 1024 + HW_STAGES * HW_STAGE, stream>>>(p);
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

static int map_rows(CUtensorMap* m, const void* base, long long rows, long long inner, long long ld, int box_rows) {
  const long long dims[2] = {inner, rows}, st[2] = {1, ld};
  const int box[2] = {64, box_rows};
  return make_map_bf16(m, base, 2, dims, st, box, 128);
}
static long long up(long long n, long long m) { return (n + m - 1) / m * m; }

// Cuts of the column tiles of LSE / D: fewest rounds of (tiles per job + a sixteenth of one), fewest cuts first. Loss of
// 256 voxels x 1024 channels x 32771 classes 72 us, without cuts 593; 8192 voxels 339 and 596.
static void wide_split(int row_tiles, int col_tiles, int* splits, int* per_out) {
  long long best = -1;
  for (int want = 1; want <= col_tiles && want <= 148; ++want) {
    const int per = (col_tiles + want - 1) / want, s = (col_tiles + per - 1) / per;
    const long long rounds = ((long long)row_tiles * s + 73) / 74, cost = rounds * (16 * per + 1);
    if (best < 0 || cost < best) { best = cost; *splits = s; *per_out = per; }
  }
}
// Slices of the reduction of a product rows x cols over kc blocks of 64: rounds of (blocks x 512 clocks + 1000), and the
// slices' way through memory at some 3500 bytes a clock. Loss and gradients of 256 voxels x 1024 channels x 32771 classes
// 166 us, in one slice 333; 20000 x 512 x 300 91 and 178; 8192 x 1024 x 32771 1796 and 1769, where it matters little.
static int wide_slices(long long rows, int C, int kc) {
  const long long tiles = up(rows, 256) / 256 * (up(C, 256) / 256);
  long long best = -1;
  int pick = 1;
  for (int s = 1; s <= 64 && s <= kc; ++s) {
    const int per = (kc + s - 1) / s;
    if ((kc + per - 1) / per != s) continue;
    long long cost = (tiles * s + 73) / 74 * (per * 512LL + 1000);
    if (s > 1) cost += 8LL * s * rows * C / 3500 + 4000;
    if (best < 0 || cost < best) { best = cost; pick = s; }
  }
  return pick;
}

struct Pieces {
  long long vc, kp;  // voxels and classes of a piece, multiples of 256
  int nv, nk;
  int sx, sw;        // slices of the two products
  int d_splits, d_per;
  int lo;            // P^T has a remainder
  long long dl, xu, acc_x, acc_w, acc_b, ws_b, slices, total;  // offsets in floats
};
static Pieces wide_pieces(const HeadCall& a) {
  Pieces q;
  const long long vp = up(a.V, 256), kp = up(a.K, 256);
  if (kp * (vp < 16384 ? vp : 16384) <= HW_PIECE) {  // all classes, as many voxels as fit
    q.kp = kp;
    q.vc = HW_PIECE / kp / 256 * 256;
    if (q.vc > vp) q.vc = vp;
  } else {
    q.vc = vp < 16384 ? vp : 16384;
    q.kp = HW_PIECE / q.vc / 256 * 256;
  }
  q.nv = (int)((vp + q.vc - 1) / q.vc);
  q.nk = (int)((kp + q.kp - 1) / q.kp);
  q.vc = up((vp + q.nv - 1) / q.nv, 256);
  q.kp = up((kp + q.nk - 1) / q.nk, 256);
  q.lo = a.V <= HD_FEW;
  q.sx = wide_slices(q.vc, a.C, (int)(q.kp / 64) * (1 + q.lo));
  q.sw = wide_slices(q.kp, a.C, (int)(q.vc / 64) * (1 + q.lo));
  wide_split((int)(q.kp / 256), (int)(q.vc / 256), &q.d_splits, &q.d_per);
  long long at = 0;
  auto take = [&](long long floats) { const long long o = at; at += up(floats, 64); return o; };
  q.dl = take(q.kp * q.vc / 2 * (1 + q.lo));
  q.xu = take(a.cw != nullptr ? q.vc * a.C / 2 : 0);
  q.acc_x = take(q.nk > 1 ? q.vc * a.C : 0);
  q.acc_w = take(q.nv > 1 ? (long long)a.K * a.C : 0);
  q.acc_b = take(q.nv > 1 ? a.K : 0);
  q.ws_b = take(2LL * q.d_splits * q.kp);
  const long long sx = q.sx > 1 ? q.sx * q.vc * a.C : 0, sw = q.sw > 1 ? q.sw * q.kp * a.C : 0;
  q.slices = take(sx > sw ? sx : sw);
  q.total = at;
  return q;
}

long long head_wide_scratch(const HeadCall& a) { return wide_pieces(a).total; }

int head_wide_splits(long long V, int K) {
  int s = 1, per = 1;
  wide_split((int)(up(V, 256) / 256), (int)(up(K, 256) / 256), &s, &per);
  return s;
}

template <int EPI>
static int wide_rows(const HeadCall& a, float2* part, float* tl, cudaStream_t stream) {
  WideParams p;
  memset(&p, 0, sizeof(p));
  p.row_tiles = (int)(up(a.V, 256) / 256);
  p.col_tiles = (int)(up(a.K, 256) / 256);
  wide_split(p.row_tiles, p.col_tiles, &p.splits, &p.tiles_per_split);
  p.kc = (a.C + 63) / 64;
  p.cols = a.K;
  p.rows_pad = up(a.V, HD_PAD);
  p.y = a.y;
  p.colp = a.bias2;
  p.part = part;
  p.tl = tl;
  p.status = a.status;
  int rc = map_rows(&p.mapA, a.x, a.V, a.C, a.C, 128);
  if (rc) return rc;
  rc = map_rows(&p.mapB, a.w, a.K, a.C, a.C, 128);
  if (rc) return rc;
  return wide_launch<EPI, 0, 0>(p, stream);
}

int head_wide_forward(const HeadCall& a, float2* part, float* tl, cudaStream_t stream) {
  return wide_rows<WIDE_LSE>(a, part, tl, stream);
}
int head_wide_predict(const HeadCall& a, float2* part, cudaStream_t stream) {
  return wide_rows<WIDE_ARG>(a, part, nullptr, stream);
}

// one product of a piece: rows x C over `kext` of the reduction
template <int A_MN>
static int wide_product(const HeadCall& a, const void* dl, long long ldd, long long vext, long long kext, int lo_rows,
                        const void* b, long long b_rows, long long rows, int slices, float* ws, float* acc, int add,
                        const float* row_scale, const float* scale, void* out16, void* out32, cudaStream_t stream) {
  WideParams p;
  memset(&p, 0, sizeof(p));
  const long long ext = A_MN ? up(b_rows, 64) : vext;  // of the reduction: the piece's classes, or its voxels
  p.kc0 = (int)(ext / 64);
  p.kc = lo_rows ? 2 * p.kc0 : p.kc0;
  p.lo_rows = lo_rows;
  p.row_scale = row_scale;
  p.scale = scale;
  p.kslices = slices < p.kc ? slices : p.kc;
  p.kc_per_slice = (p.kc + p.kslices - 1) / p.kslices;
  p.kslices = (p.kc + p.kc_per_slice - 1) / p.kc_per_slice;
  p.rows = rows;
  p.row_tiles = (int)(up(rows, 256) / 256);
  p.cols = a.C;
  p.col_tiles = (a.C + 255) / 256;
  p.acc = acc;
  p.add = add;
  p.out16 = (__nv_bfloat16*)out16;
  p.out32 = (float*)out32;
  p.slices = ws;
  p.status = a.status;
  int rc = map_rows(&p.mapA, dl, lo_rows + kext, vext, ldd, A_MN ? 64 : 128);
  if (rc) return rc;
  rc = map_rows(&p.mapB, b, b_rows, a.C, a.C, 64);
  if (rc) return rc;
  rc = wide_launch<WIDE_OUT, A_MN, 1>(p, stream);
  if (rc || p.kslices == 1) return rc;
  const long long elems = rows * a.C;
  const long long blocks = (elems / 4 + 255) / 256;
  const int grid = (int)(blocks < 148 * 8 ? blocks : 148 * 8);
  head_slices_kernel<<<grid, 256, 0, stream>>>(ws, p.kslices, elems, a.C, acc, add, p.out16, p.out32, row_scale, scale);
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

int head_wide_backward(const HeadCall& a, cudaStream_t stream) {
  const Pieces q = wide_pieces(a);
  __nv_bfloat16* dl = (__nv_bfloat16*)(a.scratch + q.dl);
  __nv_bfloat16* xu = (__nv_bfloat16*)(a.scratch + q.xu);
  float* ws_b = a.scratch + q.ws_b;
  for (int iv = 0; iv < q.nv; ++iv) {
    const long long v0 = iv * q.vc, vrows = a.V - v0 < q.vc ? a.V - v0 : q.vc, vext = up(vrows, 256);
    if (vrows <= 0) break;
    const bool v_last = v0 + q.vc >= a.V;
    const __nv_bfloat16* xv = a.x + v0 * a.C;
    const __nv_bfloat16* xw = xv;
    if (a.cw != nullptr && a.dw != nullptr) {
      const long long octets = vrows * a.C / 8, blocks = (octets + 255) / 256;
      head_weigh_kernel<<<(int)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, stream>>>(xv, a.u + v0, octets, a.C, xu);
      sb_count_launch(1);
      xw = xu;
    }
    for (int ik = 0; ik < q.nk; ++ik) {
      const long long k0 = ik * q.kp, krows = a.K - k0 < q.kp ? a.K - k0 : q.kp, kext = up(krows, 256);
      if (krows <= 0) break;
      const bool k_last = k0 + q.kp >= a.K;
      const __nv_bfloat16* wk = a.w + k0 * a.C;
      WideParams p;
      memset(&p, 0, sizeof(p));
      p.row_tiles = (int)(kext / 256);
      p.col_tiles = (int)(vext / 256);
      p.tiles_per_split = q.d_per;
      p.splits = (p.col_tiles + q.d_per - 1) / q.d_per;
      p.kc = (a.C + 63) / 64;
      p.cols = (int)vext;
      p.rows = up(krows, 64);
      p.rows_pad = q.kp;
      p.y = a.y + v0;
      p.colp = a.lse2p + v0;
      p.colg = a.u + v0;
      p.rowp = a.bias2 + k0;
      p.row0 = (int)k0;
      p.dl = dl;
      p.ldd = q.vc;
      p.lo_rows = q.lo ? (int)q.kp : 0;
      p.ws_b = ws_b;
      p.status = a.status;
      int rc = map_rows(&p.mapA, wk, krows, a.C, a.C, 128);
      if (rc) return rc;
      rc = map_rows(&p.mapB, xv, vrows, a.C, a.C, 128);
      if (rc) return rc;
      rc = wide_launch<WIDE_D, 0, 0>(p, stream);
      if (rc) return rc;
      if (a.db != nullptr) {
        head_slices_b_kernel<<<(int)((krows + 31) / 32), 256, 0, stream>>>(
            ws_b, 2 * p.splits, q.kp, (int)krows, a.scratch + q.acc_b + k0, iv > 0,
            v_last && a.db_kind == 0 ? (__nv_bfloat16*)a.db + k0 : nullptr,
            v_last && a.db_kind == 2 ? (float*)a.db + k0 : nullptr, a.scale);
        sb_count_launch(1);
      }
      if (a.dx != nullptr) {
        rc = wide_product<1>(a, dl, q.vc, vext, kext, p.lo_rows, wk, krows, vrows, q.sx, a.scratch + q.slices,
                             a.scratch + q.acc_x, ik > 0, a.g + v0, nullptr,
                             k_last ? a.dx + v0 * a.C : nullptr, nullptr, stream);
        if (rc) return rc;
      }
      if (a.dw != nullptr) {
        rc = wide_product<0>(a, dl, q.vc, vext, kext, p.lo_rows, xw, vrows, krows, q.sw, a.scratch + q.slices,
                             a.scratch + q.acc_w + k0 * a.C, iv > 0, nullptr, a.scale,
                             v_last && a.dw_kind == 0 ? (__nv_bfloat16*)a.dw + k0 * a.C : nullptr,
                             v_last && a.dw_kind == 2 ? (float*)a.dw + k0 * a.C : nullptr, stream);
        if (rc) return rc;
      }
    }
  }
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

}  // namespace sb
