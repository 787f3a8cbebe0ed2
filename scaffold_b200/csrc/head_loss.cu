// Cross entropy of a segmentation head with many classes, straight from the features in front of the head:
//   s_ij = x_i . w_j + b_j,  lse_i = log sum_j exp s_ij,  L = sum_i u_i (lse_i - s_i,y(i)) / sum_i u_i,  u_i = class weight
//   p_ij = exp(s_ij - lse_i),  D_ij = g_i (p_ij - [j = y_i]),  g_i = dL u_i / sum u
//   dX = D W,  dW = D^T X,  db_j = sum_i D_ij
// The logits (voxels x classes) are never written: each of the three kernels multiplies the tiles of X and W again, keeps
// a 128 x 128 tile of s in tensor memory and uses it up there. Everything is counted in powers of two: t = s log2(e).
//
// One kernel template, three modes. A CTA keeps 128 ROWS resident and walks 128-wide tiles of COLUMNS:
//   HEAD_FWD  rows = voxels, columns = classes: running maximum and sum of every row (one row per thread, no exchange)
//   HEAD_DX   rows = voxels, columns = classes: P = p - [j = y] in bf16 goes back to tensor memory over the tile of s it
//             came from, and acc[128][C] += P W is the second MMA with P as its A operand (W's tile is the same shared
//             memory, read MN-major)
//   HEAD_DW   rows = classes, columns = voxels: the same with X and W exchanged, P = g (p - [j = y]); a row of P^T is a
//             class, so db is a sum inside a thread
// The target's one is taken off in fp32, before the rounding to bf16: behind it a confident voxel (p near 1) would keep
// nothing but the rounding of p. Rounding: P has 8 significant bits, sums are fp32 everywhere.
//
// Roles: warp 0 loads (TMA), warp 1 issues MMAs, warps 2-9 are two epilogue groups that share a tile's 128 rows and
// take one half of its columns each. Column parameters (bias; log-sum-exp, weight and label of a voxel) travel with
// their tile as bulk copies. All waits are bounded.
#include "common.cuh"
#include "head_loss.cuh"

namespace sb {

constexpr int HD_THREADS = 320;
constexpr int HD_EPI_WARPS = 8;
constexpr int HD_TILE = 128;
constexpr int HD_BOX = HD_TILE * 128;  // bytes of a 128-row box of 64 channels
constexpr int HD_MAX_STAGES = 4;
constexpr int HD_MAX_C = 256;          // TMEM: two or three tiles of s and the accumulator in 512 columns
enum HeadMode { HEAD_FWD = 0, HEAD_DX = 1, HEAD_DW = 2 };

struct HeadParams {
  CUtensorMap mapR, mapQ;
  const float* colp;    // [cols, padded to 128] FWD / DX: bias log2(e) (-inf behind the last class); DW: log2-sum-exp less log2 g
  const float* colg;    // DW: g
  const int* coly;      // DW: label (-1: none)
  const float* rowp;    // DX: log2-sum-exp; DW: bias log2(e)
  const float* rowg;    // DX: g
  const int* rowy;      // FWD / DX: label
  float2* part;         // FWD: [splits][rows padded] running maximum and sum
  float* tl;            // FWD: [rows padded] t at the label
  __nv_bfloat16* out;   // DX with one split: [rows][C]
  float* ws;            // DX / DW: [splits][rows padded][cpad]
  float* ws_b;          // DW: [2 splits][rows padded]
  uint32_t* status;
  long long rows, cols, rows_pad;
  int C, cpad, kboxes, ksteps;
  int row_tiles, col_tiles, splits, tiles_per_split;
  int stages, rbufs, bufs;
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
__device__ __forceinline__ void hd_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
template <int MODE>
__global__ void __launch_bounds__(HD_THREADS, 1) head_kernel(const __grid_constant__ HeadParams p) {
  constexpr int MAXB = 4;
  constexpr int NPAR = MODE == HEAD_DW ? 3 : 1;  // column parameter arrays per tile
  const uint32_t NB = (uint32_t)p.bufs;          // tiles of s in tensor memory
  const uint32_t ACC = NB * HD_TILE;             // column of the accumulator
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t r_full[2], r_empty[2], q_full[HD_MAX_STAGES], q_empty[HD_MAX_STAGES], s_full[MAXB], s_done[MAXB],
      s_free[MAXB], acc_full, acc_empty;
  __shared__ float s_m[HD_TILE], s_s[HD_TILE], s_t[HD_TILE];
  __shared__ uint32_t tmem_base_s, abort_s;
  volatile uint32_t* abort_flag = &abort_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int jobs = p.row_tiles * p.splits;
  const uint32_t tile_bytes = (uint32_t)p.kboxes * HD_BOX;
  uint8_t* smem_r = smem;
  uint8_t* smem_q = smem + (size_t)p.rbufs * tile_bytes;
  float* smem_p = reinterpret_cast<float*>(smem_q + (size_t)p.stages * tile_bytes);  // [stages][NPAR][128]

  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int i = 0; i < 2; ++i) { mbar_init(&r_full[i], 1); mbar_init(&r_empty[i], 1); }
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], MODE == HEAD_FWD ? 1 + HD_EPI_WARPS : 1);
    }
    for (int i = 0; i < MAXB; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_done[i], HD_EPI_WARPS); mbar_init(&s_free[i], 1); }
    mbar_init(&acc_full, 1);
    mbar_init(&acc_empty, HD_EPI_WARPS);
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
  auto cols_of = [&](int t) -> int {  // columns of tile t, up to a multiple of 32
    const long long left = p.cols - (long long)t * HD_TILE;
    return left >= HD_TILE ? HD_TILE : (int)(left + 31) / 32 * 32;
  };

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
        if (++rb == (uint32_t)p.rbufs) { rb = 0; rph ^= 1u; }
        for (int t = t0; t < t1; ++t) {
          if (!mbar_wait(&q_empty[st], ph ^ 1u, abort_flag, p.status, 91)) { ok = false; break; }
          mbar_expect_tx(&q_full[st], tile_bytes + NPAR * HD_TILE * 4);
          for (int k = 0; k < p.kboxes; ++k)
            hd_tma_2d(smem_q + st * tile_bytes + k * HD_BOX, &p.mapQ, &q_full[st], k * 64, t * HD_TILE);
          float* par = smem_p + st * NPAR * HD_TILE;
          hd_bulk(par, p.colp + (long long)t * HD_TILE, HD_TILE * 4, &q_full[st]);
          if (MODE == HEAD_DW) {
            hd_bulk(par + HD_TILE, p.colg + (long long)t * HD_TILE, HD_TILE * 4, &q_full[st]);
            hd_bulk(par + 2 * HD_TILE, p.coly + (long long)t * HD_TILE, HD_TILE * 4, &q_full[st]);
          }
          if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t hi = desc_hi(8u * 128u, 2u);
    const uint32_t r0 = smem_u32(smem_r), q0 = smem_u32(smem_q);
    const uint32_t idesc2 = make_idesc_bf16(128, p.cpad, 0, 1);
    const uint32_t lbo = p.kboxes > 1 ? (uint32_t)HD_BOX : 0u;
    uint32_t rb = 0, rph = 0, st = 0, ph = 0, b = 0, bph = 0, aph = 0;
    // the tile whose P is still to be multiplied
    bool have = false, prev_first = false, prev_last = false;
    uint32_t prev_st = 0, prev_b = 0, prev_bph = 0;
    int prev_cols = 0;
    bool ok = true;
    auto second = [&]() -> bool {
      if (prev_first) {
        if (!__all_sync(0xffffffffu, mbar_wait(&acc_empty, aph ^ 1u, abort_flag, p.status, 92))) return false;
        aph ^= 1u;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&s_done[prev_b], prev_bph, abort_flag, p.status, 93))) return false;
      tc_fence_after();
      if (leader) {
        const uint32_t lo = desc_lo(q0 + prev_st * tile_bytes, lbo);
        const uint32_t a = tmem + prev_b * HD_TILE;
        for (int k = 0; k < prev_cols / 16; ++k)
          hd_mma_ts(tmem + ACC, a + (k < 4 ? 8 * k : 32 + 8 * k), lo + k * 128u, hi, idesc2,
                    prev_first && k == 0 ? 0u : 1u);
        tc_commit(&q_empty[prev_st]);
        tc_commit(&s_free[prev_b]);
        if (prev_last) tc_commit(&acc_full);
      }
      __syncwarp();
      return true;
    };
    for (int job = blockIdx.x; job < jobs && ok; job += gridDim.x) {
      const int sp = job / p.row_tiles;
      const int t0 = sp * p.tiles_per_split;
      const int t1 = t0 + p.tiles_per_split < p.col_tiles ? t0 + p.tiles_per_split : p.col_tiles;
      if (!__all_sync(0xffffffffu, mbar_wait(&r_full[rb], rph, abort_flag, p.status, 94))) { ok = false; break; }
      for (int t = t0; t < t1; ++t) {
        if (!__all_sync(0xffffffffu, mbar_wait(&q_full[st], ph, abort_flag, p.status, 95))) { ok = false; break; }
        // the buffer is free: read by the epilogue (FWD), or its P read by the second MMA that used it
        uint64_t* bar = MODE == HEAD_FWD ? &s_done[b] : &s_free[b];
        if (!__all_sync(0xffffffffu, mbar_wait(bar, bph ^ 1u, abort_flag, p.status, 96))) { ok = false; break; }
        tc_fence_after();
        const int nc = cols_of(t);
        if (leader) {
          const uint32_t idesc = make_idesc_bf16(128, nc, 0, 0);
          const uint32_t a_lo = desc_lo(r0 + rb * tile_bytes, 16u), b_lo = desc_lo(q0 + st * tile_bytes, 16u);
          for (int k = 0; k < p.ksteps; ++k) {
            const uint32_t off = (uint32_t)(k >> 2) * (HD_BOX >> 4) + (uint32_t)(k & 3) * 2u;
            tc_mma_bf16_pred(tmem + b * HD_TILE, a_lo + off, hi, b_lo + off, hi, idesc, k != 0 ? 1u : 0u);
          }
          tc_commit(&s_full[b]);
          if (MODE == HEAD_FWD) tc_commit(&q_empty[st]);
          if (t == t1 - 1) tc_commit(&r_empty[rb]);
        }
        __syncwarp();
        if (MODE != HEAD_FWD) {
          if (have && !second()) { ok = false; break; }
          have = true;
          prev_first = t == t0;
          prev_last = t == t1 - 1;
          prev_st = st; prev_b = b; prev_bph = bph; prev_cols = nc;
        }
        if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
        if (++b == NB) { b = 0; bph ^= 1u; }
      }
      if (++rb == (uint32_t)p.rbufs) { rb = 0; rph ^= 1u; }
    }
    if (MODE != HEAD_FWD && ok && have) second();
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const int row = quad * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
    uint32_t st = 0, ph = 0, b = 0, bph = 0, aph = 0;
    bool ok = true, pending = false;
    int pend_rt = 0, pend_sp = 0;
    float pend_g = 0.f, pend_db = 0.f;
    // the accumulator of a finished job
    auto drain = [&]() -> bool {
      if (!mbar_wait(&acc_full, aph, abort_flag, p.status, 97)) return false;
      aph ^= 1u;
      tc_fence_after();
      const long long r = (long long)pend_rt * HD_TILE + row;
      for (int c0 = half * 16; c0 < p.cpad; c0 += 32) {
        uint32_t v[16];
        tmem_ld_32x16(lane_base + ACC + c0, v);
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
      if (MODE == HEAD_DW) p.ws_b[((long long)pend_sp * 2 + half) * p.rows_pad + r] = pend_db;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty);
      return true;
    };
    for (int job = blockIdx.x; job < jobs && ok; job += gridDim.x) {
      const int rt = job % p.row_tiles, sp = job / p.row_tiles;
      const int t0 = sp * p.tiles_per_split;
      const int t1 = t0 + p.tiles_per_split < p.col_tiles ? t0 + p.tiles_per_split : p.col_tiles;
      const long long r = (long long)rt * HD_TILE + row;
      int y = -1;
      float rp = 0.f, g = 0.f, db = 0.f;
      if (MODE != HEAD_DW) y = p.rowy[r];
      if (MODE != HEAD_FWD) rp = p.rowp[r];
      if (MODE == HEAD_DX) g = p.rowg[r];
      float m = -INFINITY, s = 0.f, tl = 0.f;
      for (int t = t0; t < t1; ++t) {
        if (!mbar_wait(&q_full[st], ph, abort_flag, p.status, 98) ||
            !mbar_wait(&s_full[b], bph, abort_flag, p.status, 98)) { ok = false; break; }
        tc_fence_after();
        const float* par = smem_p + st * NPAR * HD_TILE + half * 64;
        const int nc = cols_of(t) - half * 64;  // this group's columns: none, 32 or (64 and more) 64
        const int c_abs = t * HD_TILE + half * 64;
#pragma unroll
        for (int c0 = 0; c0 < 64; c0 += 32) {
          if (c0 >= nc) break;
          uint32_t v[32];
          tmem_ld_32x32(lane_base + b * HD_TILE + half * 64 + c0, v);
          tmem_ld_wait();
          float f[32];
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 cp = *reinterpret_cast<const float4*>(par + c0 + j);
            const float cv[4] = {cp.x, cp.y, cp.z, cp.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float add = MODE == HEAD_FWD ? cv[i] : MODE == HEAD_DX ? cv[i] - rp : rp - cv[i];
              f[j + i] = fmaf(__uint_as_float(v[j + i]), HD_LOG2E, add);
            }
          }
          if (MODE == HEAD_FWD) {
            const int at = y - (c_abs + c0);
            if ((unsigned)at < 32u) {
#pragma unroll
              for (int j = 0; j < 32; ++j) tl = j == at ? f[j] : tl;
            }
            float mx = f[0];
#pragma unroll
            for (int j = 1; j < 32; ++j) mx = fmaxf(mx, f[j]);
            if (mx > m) {
              s *= hd_ex2(m - mx);  // m = -inf: 0 * 0
              m = mx;
            }
            const float base = m == -INFINITY ? 0.f : m;
            float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              a0 += hd_ex2(f[j] - base);
              a1 += hd_ex2(f[j + 1] - base);
              a2 += hd_ex2(f[j + 2] - base);
              a3 += hd_ex2(f[j + 3] - base);
            }
            s += (a0 + a1) + (a2 + a3);
          } else {
            uint32_t o[16];
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = hd_ex2(f[j]);
            if (MODE == HEAD_DX) {
              const int at = y - (c_abs + c0);
              if ((unsigned)at < 32u) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (j == at) f[j] -= 1.f;
              }
            } else {
              float d0 = 0.f, d1 = 0.f, d2 = 0.f, d3 = 0.f;
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 cg = *reinterpret_cast<const float4*>(par + HD_TILE + c0 + j);
                const int4 cy = *reinterpret_cast<const int4*>(par + 2 * HD_TILE + c0 + j);
                if (cy.x == (int)r) f[j] -= cg.x;
                if (cy.y == (int)r) f[j + 1] -= cg.y;
                if (cy.z == (int)r) f[j + 2] -= cg.z;
                if (cy.w == (int)r) f[j + 3] -= cg.w;
                d0 += f[j]; d1 += f[j + 1]; d2 += f[j + 2]; d3 += f[j + 3];
              }
              db += (d0 + d1) + (d2 + d3);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
            // over the columns of s that this thread has read: the second chunk's are still behind them
            hd_tmem_st_x16(lane_base + b * HD_TILE + half * 64 + c0 / 2, o);
          }
        }
        if (MODE != HEAD_FWD) hd_tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s_done[b]);
          if (MODE == HEAD_FWD) mbar_arrive(&q_empty[st]);
        }
        if (++st == (uint32_t)p.stages) { st = 0; ph ^= 1u; }
        if (++b == NB) { b = 0; bph ^= 1u; }
        if (MODE != HEAD_FWD && pending) {
          if (!drain()) { ok = false; break; }
          pending = false;
        }
      }
      if (MODE == HEAD_FWD) {
        // the two halves of the columns
        if (half == 1) { s_m[row] = m; s_s[row] = s; s_t[row] = tl; }
        ok = hd_epi_vote(ok);
        if (half == 0 && ok) {
          const float m1 = s_m[row], mm = fmaxf(m, m1);
          const float base = mm == -INFINITY ? 0.f : mm;
          const float ss = s * hd_ex2(m - base) + s_s[row] * hd_ex2(m1 - base);
          p.part[(long long)sp * p.rows_pad + r] = make_float2(mm, ss);
          const long long c_lo = (long long)t0 * HD_TILE, c_hi = (long long)t1 * HD_TILE;
          if (y >= c_lo && y < c_hi) p.tl[r] = (y & (HD_TILE - 1)) < 64 ? tl : s_t[row];
        }
        hd_epi_vote(true);  // the merge has read what the next job's will overwrite
      } else {
        pending = true;
        pend_rt = rt; pend_sp = sp; pend_g = g; pend_db = db;
      }
    }
    if (MODE != HEAD_FWD && ok && pending) drain();
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
// and behind the last voxel; bias2[j] = bias_j log2(e), -inf behind the last class
__global__ void __launch_bounds__(256) head_prep_kernel(const void* __restrict__ labels, int kind, long long V,
                                                        long long v_pad, int K, int k_pad, int has_ignore,
                                                        long long ignore, int* __restrict__ y,
                                                        const void* __restrict__ bias, int bias_kind,
                                                        float* __restrict__ bias2, uint32_t* __restrict__ status) {
  const long long n = v_pad > k_pad ? v_pad : k_pad;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    if (i < v_pad) {
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
      if (i < K)
        b = bias == nullptr ? 0.f
            : bias_kind == 0 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(bias)[i]) * HD_LOG2E
                             : reinterpret_cast<const float*>(bias)[i] * HD_LOG2E;
      bias2[i] = b;
    }
  }
}

struct HeadSum {
  double num, den;
};
__device__ __forceinline__ HeadSum hd_block_sum(HeadSum a) {
  __shared__ double s_n[8], s_d[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.num += __shfl_xor_sync(0xffffffffu, a.num, o);
    a.den += __shfl_xor_sync(0xffffffffu, a.den, o);
  }
  if ((threadIdx.x & 31) == 0) { s_n[threadIdx.x >> 5] = a.num; s_d[threadIdx.x >> 5] = a.den; }
  __syncthreads();
  HeadSum t{0.0, 0.0};
  if (threadIdx.x == 0)
    for (int w = 0; w < 8; ++w) { t.num += s_n[w]; t.den += s_d[w]; }
  return t;
}

// lse2[i] from the splits' running maxima and sums, merged in split order; block sums of u nll and u in double
__global__ void __launch_bounds__(256) head_merge_kernel(const float2* __restrict__ part, const float* __restrict__ tl,
                                                         const int* __restrict__ y, const float* __restrict__ cw,
                                                         int splits, long long V, long long v_pad,
                                                         float* __restrict__ lse2, double* __restrict__ sums) {
  HeadSum a{0.0, 0.0};
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < v_pad; i += (long long)gridDim.x * 256) {
    float l = INFINITY;
    if (i < V) {
      float m = -INFINITY, s = 0.f;
      for (int k = 0; k < splits; ++k) {
        const float2 e = part[(long long)k * v_pad + i];
        const float mm = fmaxf(m, e.x), base = mm == -INFINITY ? 0.f : mm;
        s = s * hd_ex2(m - base) + e.y * hd_ex2(e.x - base);
        m = mm;
      }
      l = m + log2f(s);
      const int c = y[i];
      if (c >= 0) {
        const float u = cw == nullptr ? 1.f : cw[c];
        a.num += (double)u * ((double)(l - tl[i]) * (double)HD_LN2);
        a.den += (double)u;
      }
    }
    lse2[i] = l;
  }
  a = hd_block_sum(a);
  if (threadIdx.x == 0) { sums[2 * blockIdx.x] = a.num; sums[2 * blockIdx.x + 1] = a.den; }
}

// total[2] = the blocks' sums in order; loss = num / max(den, eps), den the clamped denominator
__global__ void __launch_bounds__(256) head_total_kernel(const double* __restrict__ sums, int blocks,
                                                         double* __restrict__ total, float* __restrict__ loss,
                                                         float* __restrict__ den) {
  HeadSum a{0.0, 0.0};
  for (int i = threadIdx.x; i < blocks; i += 256) { a.num += sums[2 * i]; a.den += sums[2 * i + 1]; }
  a = hd_block_sum(a);
  if (threadIdx.x == 0) {
    const double eps = 1.1920928955078125e-7, d = a.den < eps ? eps : a.den;  // NaN stays
    total[0] = a.num;
    total[1] = a.den;
    loss[0] = (float)(a.num / d);
    den[0] = (float)d;
  }
}

// g[i] = dL u_i / den and lse2 - log2 g (so that exp2(t - it) = g p), 0 and +inf where a voxel takes no part
__global__ void __launch_bounds__(256) head_weights_kernel(const float* __restrict__ lse2, const int* __restrict__ y,
                                                           const float* __restrict__ cw, const float* __restrict__ gout,
                                                           const float* __restrict__ den, long long v_pad,
                                                           float* __restrict__ g, float* __restrict__ lse2g) {
  const float k = gout[0] / den[0];
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < v_pad; i += (long long)gridDim.x * 256) {
    const int c = y[i];
    const float gi = c < 0 ? 0.f : k * (cw == nullptr ? 1.f : cw[c]);
    g[i] = gi;
    lse2g[i] = gi == 0.f ? INFINITY : lse2[i] - log2f(gi);
  }
}

// out[r][c] = sum over the slices of ws[slice][rows_pad][ld], in slice order; r < rows, c < C
template <typename T>
__global__ void __launch_bounds__(256) head_reduce_kernel(const float* __restrict__ ws, int slices, long long rows,
                                                          long long rows_pad, int C, int ld, T* __restrict__ out) {
  const long long n = rows * C;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long r = i / C;
    const int c = (int)(i - r * C);
    const float* src = ws + r * ld + c;
    float a = 0.f;
#pragma unroll 4
    for (int k = 0; k < slices; ++k) a += src[(long long)k * rows_pad * ld];
    out[i] = hd_cast<T>(a);
  }
}

static int hd_blocks(long long n, int per_sm) {
  const long long b = (n + 255) / 256;
  return (int)(b < 148LL * per_sm ? (b < 1 ? 1 : b) : 148LL * per_sm);
}

// How many ways the columns are cut: fewest rounds of (tiles per job + about one tile of fixed cost), fewest cuts first.
static void head_split(int row_tiles, int col_tiles, int* splits, int* tps) {
  long long best = -1;
  for (int want = 1; want <= col_tiles && want <= 296; ++want) {
    const int per = (col_tiles + want - 1) / want, s = (col_tiles + per - 1) / per;
    const long long rounds = ((long long)row_tiles * s + 147) / 148, cost = rounds * (per + 1);
    if (best < 0 || cost < best) { best = cost; *splits = s; *tps = per; }
    if (row_tiles >= 148 * 4) break;
  }
}

static void head_geometry(const SbHeadArgs* a, int mode, HeadParams& p) {
  memset(&p, 0, sizeof(p));
  p.C = a->C;
  p.cpad = (a->C + 15) / 16 * 16;
  p.kboxes = (a->C + 63) / 64;
  p.ksteps = p.cpad / 16;
  p.rows = mode == HEAD_DW ? a->K : a->V;
  p.cols = mode == HEAD_DW ? a->V : a->K;
  p.row_tiles = (int)((p.rows + HD_TILE - 1) / HD_TILE);
  p.col_tiles = (int)((p.cols + HD_TILE - 1) / HD_TILE);
  p.rows_pad = (p.rows + HD_PAD - 1) / HD_PAD * HD_PAD;
  head_split(p.row_tiles, p.col_tiles, &p.splits, &p.tiles_per_split);
  p.bufs = mode == HEAD_FWD ? 4 : p.cpad <= 128 ? 3 : 2;
  // shared memory: 12 boxes of 16 KB (kboxes per tile); one or two resident tiles and two to four in the ring
  p.rbufs = p.kboxes <= 2 ? 2 : 1;
  p.stages = 12 / p.kboxes - p.rbufs;
  if (p.stages > HD_MAX_STAGES) p.stages = HD_MAX_STAGES;
  p.status = a->status;
}

template <int MODE>
static int head_launch(const SbHeadArgs* a, HeadParams& p, cudaStream_t stream) {
  const void* x = a->x;
  const void* w = a->w;
  const long long dv[2] = {a->C, a->V}, dk[2] = {a->C, a->K}, st[2] = {1, a->C};
  const int box[2] = {64, HD_TILE};
  int rc = make_map_bf16(&p.mapR, MODE == HEAD_DW ? w : x, 2, MODE == HEAD_DW ? dk : dv, st, box, 128);
  if (rc) return rc;
  rc = make_map_bf16(&p.mapQ, MODE == HEAD_DW ? x : w, 2, MODE == HEAD_DW ? dv : dk, st, box, 128);
  if (rc) return rc;
  const size_t smem = 1024 + (size_t)(p.rbufs + p.stages) * p.kboxes * HD_BOX + (size_t)p.stages * 3 * HD_TILE * 4;
  if (cudaFuncSetAttribute(head_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 4096) !=
      cudaSuccess)
    return SB_ERR_DRIVER;
  const long long jobs = (long long)p.row_tiles * p.splits;
  head_kernel<MODE><<<(int)(jobs < 148 ? jobs : 148), HD_THREADS, smem, stream>>>(p);
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

}  // namespace sb

using namespace sb;

static long long pad(long long n) { return (n + HD_PAD - 1) / HD_PAD * HD_PAD; }
static bool shape_ok(const SbHeadArgs* a) {
  return a->V >= 1 && a->V <= (1LL << 31) - 512 && a->K >= 1 && a->K <= (1 << 30) && a->C >= 8 && a->C % 8 == 0 &&
         a->C <= 32768;
}
static bool wide(const SbHeadArgs* a) { return a->C > HD_MAX_C; }
constexpr int HD_SUM_BLOCKS = 148 * 4;

// fp32 scratch of the forward (mode 0) and the backward pass (1); -1: outside the kernels' range
extern "C" long long sb_head_scratch(const SbHeadArgs* a, int mode) {
  if (mode < 0 || mode > 1 || !shape_ok(a)) return -1;
  HeadParams p;
  if (mode == 0) {
    head_geometry(a, HEAD_FWD, p);
    const int splits = wide(a) ? head_wide_splits(a->V, a->K) : p.splits;
    return 4LL * HD_SUM_BLOCKS + (2LL * splits + 1) * p.rows_pad;
  }
  if (wide(a)) return head_wide_scratch(a);
  head_geometry(a, HEAD_DX, p);
  const long long dx = p.splits == 1 ? 0 : p.splits * p.rows_pad * p.cpad;
  head_geometry(a, HEAD_DW, p);
  const long long dw = p.splits * p.rows_pad * (p.cpad + 2);
  return dx > dw ? dx : dw;
}

// labels, bias -> y, bias2, lse2, total, loss, den
extern "C" int sb_head_forward(const SbHeadArgs* a, cudaStream_t stream) {
  if (!shape_ok(a) || !a->x || !a->w || !a->labels || !a->y || !a->bias2 || !a->lse2 || !a->total || !a->loss ||
      !a->den || !a->scratch)
    return SB_ERR_SHAPE;
  if (a->scratch_floats < sb_head_scratch(a, 0)) return SB_ERR_TOO_LARGE;
  HeadParams p;
  head_geometry(a, HEAD_FWD, p);
  const long long v_pad = pad(a->V);
  const int k_pad = (int)pad(a->K);
  head_prep_kernel<<<hd_blocks(v_pad > k_pad ? v_pad : k_pad, 8), 256, 0, stream>>>(
      a->labels, a->label_kind, a->V, v_pad, a->K, k_pad, a->has_ignore, a->ignore, a->y, a->bias, a->bias_kind, a->bias2,
      a->status);
  sb_count_launch(1);
  // scratch: block sums (double), running maxima and sums, t at the labels
  double* sums = (double*)a->scratch;
  const int splits = wide(a) ? head_wide_splits(a->V, a->K) : p.splits;
  p.part = (float2*)(a->scratch + 4LL * HD_SUM_BLOCKS);
  p.tl = (float*)(p.part + splits * p.rows_pad);
  p.colp = a->bias2;
  p.rowy = a->y;
  const int rc = wide(a) ? head_wide_forward(a, p.part, p.tl, splits, stream) : head_launch<HEAD_FWD>(a, p, stream);
  if (rc) return rc;
  const int blocks = hd_blocks(v_pad, 4);
  head_merge_kernel<<<blocks, 256, 0, stream>>>(p.part, p.tl, a->y, a->cw, splits, a->V, v_pad, a->lse2, sums);
  sb_count_launch(1);
  return sb_head_total(sums, blocks, a->total, a->loss, a->den, stream);
}

extern "C" int sb_head_total(const double* sums, int blocks, double* total, float* loss, float* den,
                             cudaStream_t stream) {
  head_total_kernel<<<1, 256, 0, stream>>>(sums, blocks, total, loss, den);
  sb_count_launch(1);
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}

template <typename T>
static void head_reduce(const float* ws, int slices, long long rows, long long rows_pad, int C, int ld, void* out,
                        cudaStream_t stream) {
  head_reduce_kernel<T><<<hd_blocks(rows * C, 8), 256, 0, stream>>>(ws, slices, rows, rows_pad, C, ld, (T*)out);
  sb_count_launch(1);
}

// dx, dw and db (each optional) from gout and what the forward pass left; dw / db in fp32 when dw_kind / bias_kind is 2
extern "C" int sb_head_backward(const SbHeadArgs* a, const float* gout, cudaStream_t stream) {
  if (!shape_ok(a) || !a->x || !a->w || !a->y || !a->bias2 || !a->lse2 || !a->den || !a->g || !a->lse2g || !gout)
    return SB_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(a->dx) | reinterpret_cast<uintptr_t>(a->dw) | reinterpret_cast<uintptr_t>(a->scratch)) & 15)
    return SB_ERR_ALIGN;
  if (a->scratch_floats < sb_head_scratch(a, 1)) return SB_ERR_TOO_LARGE;
  const long long v_pad = pad(a->V);
  head_weights_kernel<<<hd_blocks(v_pad, 8), 256, 0, stream>>>(a->lse2, a->y, a->cw, gout, a->den, v_pad, a->g, a->lse2g);
  sb_count_launch(1);
  if (wide(a)) return head_wide_backward(a, stream);
  HeadParams p;
  int rc = 0;
  if (a->dx != nullptr) {
    head_geometry(a, HEAD_DX, p);
    p.colp = a->bias2;
    p.rowp = a->lse2;
    p.rowg = a->g;
    p.rowy = a->y;
    p.out = (__nv_bfloat16*)a->dx;
    p.ws = a->scratch;
    rc = head_launch<HEAD_DX>(a, p, stream);
    if (rc) return rc;
    if (p.splits > 1) head_reduce<__nv_bfloat16>(p.ws, p.splits, p.rows, p.rows_pad, p.C, p.cpad, a->dx, stream);
  }
  if (a->dw != nullptr || a->db != nullptr) {
    head_geometry(a, HEAD_DW, p);
    p.colp = a->lse2g;
    p.colg = a->g;
    p.coly = a->y;
    p.rowp = a->bias2;
    p.ws = a->scratch;
    p.ws_b = a->scratch + p.splits * p.rows_pad * p.cpad;
    rc = head_launch<HEAD_DW>(a, p, stream);
    if (rc) return rc;
    if (a->dw != nullptr) {
      if (a->dw_kind == 2) head_reduce<float>(p.ws, p.splits, p.rows, p.rows_pad, p.C, p.cpad, a->dw, stream);
      else head_reduce<__nv_bfloat16>(p.ws, p.splits, p.rows, p.rows_pad, p.C, p.cpad, a->dw, stream);
    }
    if (a->db != nullptr) {
      if (a->bias_kind == 2) head_reduce<float>(p.ws_b, 2 * p.splits, p.rows, p.rows_pad, 1, 1, a->db, stream);
      else head_reduce<__nv_bfloat16>(p.ws_b, 2 * p.splits, p.rows, p.rows_pad, 1, 1, a->db, stream);
    }
  }
  return cudaGetLastError() == cudaSuccess ? 0 : SB_ERR_LAUNCH;
}
