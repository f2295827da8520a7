// gated_ffn.cuh -- the gated feed-forward block and its backward pass on the
// 5th-generation tensor cores (bf16 operands, fp32 accumulation in TMEM).
//
//   z = x W^T, W = [Wg; Wu] [2F, d], z = [g | u]       a = act(g) * u
//   y = a Wd^T (+ residual)
//   da = dy Wd     dg = da u act'(g)    du = da act(g)    dz = [dg | du]
//   dx = dz W      dW = dz^T x          dWd = dy^T a
// (teenyformers' FFN: src/layers/ffn.rs:47-56 around src/kernels/swiglu.rs:56-136.)
//
// Rounding: z leaves the accumulators in fp32 when it is saved for the
// backward pass, which recomputes a from it bit for bit (so a need not be
// kept); a, dz and every result are rounded once to bf16, as operands of the
// next product or as outputs.  With z in bf16 the gradients' error against
// the formulas in 64 bits grows from 1.4 to 1.8 output roundings.
//
// Two kernels:
//   ffn_pair_kernel    persistent CTA pairs (cta_group::2), 256 x 256 tiles;
//                      the structure of gemm_sm100.cuh's kernel with operands
//                      of either major and several products in one launch.
//                      Tensor-bound: 4096 x 4096 x 4096 takes 185 us for the up
//                      product with z saved (tensor pipe 79%), 120 us for da and
//                      its epilogue, 438 us for the three products of the
//                      gradients together (88%)
//   ffn_tile_kernel    small products (few tokens above all): 128 x 16..128
//                      tiles, K split over a cluster and joined through
//                      distributed shared memory
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "gemm_sm100.cuh"
#include "norm_act.cuh"
#include "sm100.cuh"

namespace tfb {

enum FfnAct : int { FFN_ACT_SILU = 0, FFN_ACT_GELU = 1, FFN_ACT_GELU_TANH = 2 };

// Phi(g), the normal distribution function, and E = exp(-g^2 / 2).  With x =
// |g| / sqrt(2) and t = 1 / (1 + 3/8 x), Phi(-|g|) = erfc(x) / 2 = t P(t) E, where P is
// the polynomial of degree 6 with the least largest relative error of t P(t) against
// erfc(x) exp(x^2) / 2 over x = 0 .. 10 (6.0e-7; fitted by linear programming).  The error
// is relative, so that the tail keeps its digits: with t, E and the sum in fp32 it stays
// below 5e-6 to g = -13, where E leaves fp32 (7.1.26 of Abramowitz and Stegun's Handbook,
// whose bound is on the absolute error, is off by 0.25 % at g = -5.5 and 1 % at -8, more
// than the bf16 rounding behind it).  It shares its exponential with the slope's density and has no branch.
__device__ __forceinline__ float ffn_phi(float g, float& E) {
  const float x = fabsf(g) * 0.70710678118654752f;
  const float t = __fdividef(1.0f, fmaf(0.375f, x, 1.0f));
  float q = fmaf(t, -0.0675347522f, 0.193916559f);
  q = fmaf(t, q, -0.064717561f);
  q = fmaf(t, q, 0.141468897f);
  q = fmaf(t, q, 0.0833564177f);
  q = fmaf(t, q, 0.107840098f);
  q = fmaf(t, q, 0.105670035f) * t;
  E = __expf(-0.5f * g * g);
  q *= E;  // Phi(-|g|)
  return g < 0.0f ? q : 1.0f - q;
}

// 1 / (1 + exp(-v)).  __fdividef (2 ulp) gives 0 for a divisor above 2^126, where
// the quotient is below 1e-37: a full fp32 division is a dozen instructions, and
// the epilogue of a short product is bound by its own.
__device__ __forceinline__ float ffn_sigmoid(float v) {
  return __fdividef(1.0f, 1.0f + __expf(-v));
}

// act(g) and act'(g).  The forward pass and the backward pass, which computes a
// again, take the value from the same expression: the same bits.
template <int ACT>
__device__ __forceinline__ void ffn_act_grad(float g, float& value, float& slope) {
  if constexpr (ACT == FFN_ACT_SILU) {
    const float s = ffn_sigmoid(g);
    value = g * s;
    slope = fmaf(value, 1.0f - s, s);
  } else if constexpr (ACT == FFN_ACT_GELU) {
    float E;
    const float phi = ffn_phi(g, E);
    value = g * phi;
    slope = fmaf(g * 0.39894228040143268f, E, phi);
  } else {
    // (1 + tanh v) / 2 = sigmoid(2 v), v = sqrt(2 / pi) (g + 0.044715 g^3)
    // (past |g| = 1e5 s is 0 or 1, and an infinite g^2 would make 0 x inf of the slope)
    const float g2 = fminf(g * g, 1e10f);
    const float s = ffn_sigmoid(1.5957691216057308f * g * fmaf(0.044715f, g2, 1.0f));
    value = g * s;
    slope = fmaf(value * (1.0f - s), 1.5957691216057308f * fmaf(0.134145f, g2, 1.0f), s);
  }
}
template <int ACT>
__device__ __forceinline__ float ffn_act(float g) {
  float value, slope;
  ffn_act_grad<ACT>(g, value, slope);
  return value;
}

__device__ __forceinline__ float ffn_act_rt(int act, float g) {  // (uniform branches)
  if (act == FFN_ACT_SILU) return ffn_act<FFN_ACT_SILU>(g);
  if (act == FFN_ACT_GELU) return ffn_act<FFN_ACT_GELU>(g);
  return ffn_act<FFN_ACT_GELU_TANH>(g);
}

// ===================================================================== CTA pairs
enum FfnMode : int {
  FFN_GLU = 0,    // A = x, B = W (gate rows to the even CTA, up rows to the odd one): a (, z)
  FFN_DGLU = 1,   // A = dy, B = Wd read MN-major: dz and a from z and the product da
  FFN_STORE = 2,  // up to three products, each rounded to bf16 (+ residual)
  FFN_DGLU_LONG = 3,  // FFN_DGLU for a long K: its z, dz and a by the lanes' loads and stores
};

constexpr int kFfnMaxProblems = 3;

// One product D[M, N] = A[M, K] B[N, K]^T.  Either operand may be stored with
// its M / N index innermost (a_mn / b_mn: rows of the stored matrix are K).
struct FfnProblem {
  int M, N, n_mblk, n_nblk, n_kblk, group_m;
  int bn;       // columns of a tile: 256, or 128 (FFN_DGLU)
  int ks;       // runs of k-blocks that a tile's K is split into (FFN_STORE; each gives fp32
                // partial sums, joined by ffn_sum_kernel)
  int n_items;  // ks times the tiles
  int a_mn, b_mn;
  __nv_bfloat16* out;             // FFN_STORE: [M, N]
  const __nv_bfloat16* residual;  // FFN_STORE: [M, N] or null
};

struct FfnPairParams {
  FfnProblem prob[kFfnMaxProblems];
  int n_prob;
  int pdl;  // launched with programmatic stream serialization
  // static schedule (ffn_next): items of the longer K, then `light` items
  int heavy, light, bal_rounds;
  // FFN_GLU / FFN_DGLU
  int F;
  __nv_bfloat16* a;   // [M, F]
  float* z;           // [M, 2F]; null in FFN_GLU: not saved
  __nv_bfloat16* dz;  // [M, 2F]
};

struct FfnMaps {
  CUtensorMap a[kFfnMaxProblems], b[kFfnMaxProblems];
  // FFN_STORE: each product's output; FFN_GLU: a, z; FFN_DGLU: a, dz, z
  CUtensorMap out[3];
};

constexpr int kFfnEpiWarps = 8;
constexpr int kFfnThreads = 64 + kFfnEpiWarps * 32;

// The pair kernel's shared memory: a ring of 32 KB stages, and each epilogue
// warp's part.  A long K wants the sixth stage (8192 x 2048 x 5632 forward 450
// us, with five 470; z saved 483, with five 524); FFN_DGLU's epilogue is the
// longer part of a tile with a short K, and there has 8 KB a warp.
template <int MODE>
struct FfnPairCfg {
  static constexpr int STAGES = MODE == FFN_DGLU ? 5 : 6;
  static constexpr int EPI_BYTES = MODE == FFN_DGLU ? 8192 : 4096;  // a warp's
  static constexpr int A_BYTES = 128 * kGemmBK * 2;  // this CTA's 128 rows of A
  static constexpr int B_BYTES = 128 * kGemmBK * 2;  // and of B
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int OFF_EPI = STAGES * STAGE_BYTES;
  static constexpr int OFF_BAR = OFF_EPI + kFfnEpiWarps * EPI_BYTES;
  static constexpr int SMEM_ALLOC = OFF_BAR + 512 + 1024;
  static constexpr int TM_COLS = 2 * kGemmBN;
  static_assert(SMEM_ALLOC <= 232448, "the pair kernel's shared memory exceeds the limit");
  // barriers
  static constexpr int FULL = 0, EMPTY = STAGES, AFULL = 2 * STAGES, AEMPTY = AFULL + 2,
                       DRAIN = AEMPTY + 2, Z = DRAIN + 1 /* FFN_DGLU: one a warp */,
                       COUNT = Z + kFfnEpiWarps;
  static_assert((COUNT + 1) * 8 <= 512, "barriers");
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t smem_src, int c0,
                                             int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(smem_src), "r"(c0), "r"(c1)
      : "memory");
}

// The i-th item of a pair, in the concatenated list of all products' items
// (those with the longer K first); -1 at the end.  Heavy items go round robin;
// the pairs that get one fewer of them (those from heavy % n_pairs on) then
// take bal_rounds light items each, about one heavy item's work, before the
// round robin over all pairs goes on.
__device__ __forceinline__ int ffn_next(const FfnPairParams& p, int pair, int n_pairs, int i) {
  const int mine = pair < p.heavy ? (p.heavy - 1 - pair) / n_pairs + 1 : 0;
  if (i < mine) return pair + i * n_pairs;
  int j = i - mine;
  const int r = p.heavy % n_pairs, q = n_pairs - r;
  int first = 0;
  if (p.bal_rounds > 0) {
    first = p.bal_rounds * q;
    if (pair >= r) {
      if (j < p.bal_rounds) return p.heavy + j * q + (pair - r);
      j -= p.bal_rounds;
    }
  }
  const long long l = (long long)first + pair + (long long)j * n_pairs;
  return l < p.light ? p.heavy + (int)l : -1;
}

// Item of the list -> product k, run of k-blocks, row block and column block
// (grouped order).
struct FfnItem {
  int k, split, mb, nb, kb0, kb1;
};
__device__ __forceinline__ FfnItem ffn_item(const FfnPairParams& p, int t) {
  FfnItem it;
  it.k = 0;
  while (it.k + 1 < p.n_prob && t >= p.prob[it.k].n_items) t -= p.prob[it.k++].n_items;
  const FfnProblem& q = p.prob[it.k];
  const int tiles = q.n_mblk * q.n_nblk;
  it.split = t / tiles;
  t -= it.split * tiles;
  it.kb0 = (int)((long long)q.n_kblk * it.split / q.ks);
  it.kb1 = (int)((long long)q.n_kblk * (it.split + 1) / q.ks);
  const int per_group = q.group_m * q.n_nblk;
  const int g = t / per_group;
  const int m_first = g * q.group_m;
  const int gm = min(q.group_m, q.n_mblk - m_first);
  const int local = t - g * per_group;
  it.mb = m_first + local % gm;
  it.nb = local / gm;
  return it;
}

__device__ __forceinline__ uint2 ffn_pack4(const float (&v)[4]) {
  return make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// Reads 32 staged rows of 32 fp32 (128-byte rows, 16-byte chunks XOR-swizzled by
// row) 4 columns a lane: iteration `it` gives row it * 4 + lane / 8, columns
// 4 (lane % 8)..
__device__ __forceinline__ float4 ffn_unstage32(uint32_t stg, int it, int lane) {
  const int rr = it * 4 + (lane >> 3);
  const uint4 v = gemm_lds128(stg + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
  return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z),
                     __uint_as_float(v.w));
}

// Epilogue of one accumulator tile for one warp: TMEM columns acc.. of this
// warp's lane quarter, output rows row0..row0+31, column block nb, the half
// `hf` of the tile's columns (two warps share a lane quarter: the epilogue of
// a tile with a short K, bound by its instructions, then takes half the time).
// A lane works on its own row.  Values leave through the warp's shared memory
// `stg` as bulk tensor stores (and FFN_DGLU's z comes in as bulk tensor loads):
// with global loads and stores of the lanes, the load/store unit bound the
// epilogues of short products (FFN_DGLU 17 us a tile).  Bulk stores clip rows
// past M and columns past the output's.  wait_acc() blocks until the
// accumulator is complete; what does not depend on it is loaded first.
// zbar: this warp's barrier, zn: its z chunks so far (FFN_DGLU).
template <int MODE, int ACT, class Wait, class Release>
__device__ __forceinline__ bool ffn_epilogue_warp(const FfnPairParams& p, const FfnProblem& q,
                                                  const FfnMaps& maps, int k, int split,
                                                  uint32_t acc, int row0, int nb, int hf, int lane,
                                                  uint32_t stg, uint32_t zbar, int& zn,
                                                  Wait&& wait_acc,
                                                  Release&& release_acc) {
  if (row0 >= q.M) {
    if (!wait_acc()) return false;
    release_acc();
    return true;
  }
  // stg is free again once the store before has read it
  auto free_stg = [&]() {
    if (lane == 0) bulk_wait_group_read0();
    __syncwarp();
  };
  // a lane's 32 fp32 as a 128-byte row, chunks XOR-swizzled by row
  auto stage32 = [&](uint32_t buf, const uint32_t (&r)[32]) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      gemm_sts128(buf + lane * 128 + ((j ^ (lane & 7)) << 4), r[4 * j], r[4 * j + 1], r[4 * j + 2],
                  r[4 * j + 3]);
  };
  auto staged = [&]() {  // this warp's shared memory writes, before a bulk store reads them
    fence_proxy_async_smem();
    __syncwarp();
  };
  if constexpr (MODE == FFN_GLU) {
    // columns 0..127 of the accumulator are gate, 128..255 up of outputs 128 nb..
    if (!wait_acc()) return false;
    for (int hh = 0; hh < 2; ++hh) {
      const int c0 = hf * 64 + hh * 32;
      const int col0 = nb * 128 + c0;
      uint32_t gr[32], ur[32];
      tmem_ld32(acc + c0, gr);
      tmem_ld32(acc + 128 + c0, ur);
      tmem_wait_ld();
      if (hh == 1) release_acc();
      // a: 64-byte rows of 16-byte chunks, XOR-swizzled by pairs of rows
      free_stg();
#pragma unroll
      for (int jc = 0; jc < 4; ++jc) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 8 * jc + 2 * e;
          w[e] = pack_bf16x2(ffn_act<ACT>(__uint_as_float(gr[i])) * __uint_as_float(ur[i]),
                             ffn_act<ACT>(__uint_as_float(gr[i + 1])) * __uint_as_float(ur[i + 1]));
        }
        gemm_sts128(stg + lane * 64 + ((jc ^ ((lane >> 1) & 3)) << 4), w[0], w[1], w[2], w[3]);
      }
      staged();
      const bool inside = lane == 0 && col0 < p.F;  // (a box wholly past the edge is not stored)
      if (inside) tma_store_2d(&maps.out[0], stg, col0, row0);
      if (lane == 0) bulk_commit_group();
      if (p.z) {
        free_stg();
        stage32(stg, gr);
        staged();
        if (inside) tma_store_3d(&maps.out[1], stg, col0, 0, row0);
        if (lane == 0) bulk_commit_group();
        free_stg();
        stage32(stg, ur);
        staged();
        if (inside) tma_store_3d(&maps.out[1], stg, col0, 1, row0);
        if (lane == 0) bulk_commit_group();
      }
    }
  } else if constexpr (MODE == FFN_DGLU_LONG) {
    // under a long main loop the time of this does not show, but its bulk copies
    // did, which wait for one another with the operands' (4096 x 4096 x 4096: 127
    // us, so 120): here the lanes load and store themselves, 4 columns each of
    // rows of 32
    const int rows_valid = q.M - row0;
    const int r4 = lane >> 3, c4 = (lane & 7) * 4;  // ffn_unstage32: row in a group of 4, column
    float4 g[8], u[8];
    auto load_z = [&](int c) {
      const int col = nb * kGemmBN + hf * 128 + c * 32 + c4;
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int rr = it * 4 + r4;
        if (rr < rows_valid && col < p.F) {
          const float* zr = p.z + (long long)(row0 + rr) * 2 * p.F + col;
          g[it] = *reinterpret_cast<const float4*>(zr);
          u[it] = *reinterpret_cast<const float4*>(zr + p.F);
        }
      }
    };
    load_z(0);
    if (!wait_acc()) return false;
    for (int c = 0; c < 4; ++c) {
      uint32_t r[32];
      tmem_ld32(acc + hf * 128 + c * 32, r);
      tmem_wait_ld();
      if (c == 3) release_acc();
      stage32(stg, r);
      __syncwarp();
      const int col = nb * kGemmBN + hf * 128 + c * 32 + c4;
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const float4 d4 = ffn_unstage32(stg, it, lane);
        const int rr = it * 4 + r4;
        if (rr < rows_valid && col < p.F) {
          const float d[4] = {d4.x, d4.y, d4.z, d4.w};
          const float gv[4] = {g[it].x, g[it].y, g[it].z, g[it].w};
          const float uv[4] = {u[it].x, u[it].y, u[it].z, u[it].w};
          float dg[4], du[4], av[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float value, slope;
            ffn_act_grad<ACT>(gv[e], value, slope);
            av[e] = value * uv[e];
            du[e] = d[e] * value;
            dg[e] = d[e] * uv[e] * slope;
          }
          __nv_bfloat16* dz = p.dz + (long long)(row0 + rr) * 2 * p.F + col;
          *reinterpret_cast<uint2*>(dz) = ffn_pack4(dg);
          *reinterpret_cast<uint2*>(dz + p.F) = ffn_pack4(du);
          *reinterpret_cast<uint2*>(p.a + (long long)(row0 + rr) * p.F + col) = ffn_pack4(av);
        }
      }
      if (c < 3) load_z(c + 1);
      __syncwarp();
    }
  } else if constexpr (MODE == FFN_DGLU) {
    // chunks of 16 columns: z comes in through the first 4 KB (gate 2 KB, up 2 KB:
    // 64-byte rows), the next chunk's as soon as a chunk's is in registers; dg,
    // du and a go out through the second (1 KB each: 32-byte rows)
    const int half_cols = q.bn / 2, chunks = q.bn / 32;
    const int col_h = nb * q.bn + hf * half_cols;
    const uint32_t out = stg + 4096;
    auto load_z = [&](int c) {  // (lane 0)
      mbar_arrive_expect_tx(zbar, 4096);
      tma_load_3d(stg, &maps.out[2], zbar, col_h + c * 16, 0, row0);
      tma_load_3d(stg + 2048, &maps.out[2], zbar, col_h + c * 16, 1, row0);
    };
    if (lane == 0) load_z(0);
    __syncwarp();
    // a load of z needs nothing of the other roles: its wait does not look at
    // their giving up, and the load has landed when this warp does
    auto wait_z = [&]() { return mbar_wait_warp(zbar, zn++ & 1, nullptr, 927); };
    if (!wait_acc()) {
      (void)wait_z();
      return false;
    }
    for (int c = 0; c < chunks; ++c) {
      uint32_t r[16];
      tmem_ld16(acc + hf * half_cols + c * 16, r);
      if (!wait_z()) return false;
      uint4 g4[4], u4[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t at = stg + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4);
        g4[j] = gemm_lds128(at), u4[j] = gemm_lds128(at + 2048);
      }
      tmem_wait_ld();
      if (c == chunks - 1) release_acc();
      __syncwarp();  // every lane has read its z
      if (lane == 0) {
        if (c + 1 < chunks) load_z(c + 1);
        bulk_wait_group_read0();  // the chunk before has left `out`
      }
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t dg[4], du[4], av[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint4 gq = g4[2 * h + j], uq = u4[2 * h + j];
          const uint32_t gw[4] = {gq.x, gq.y, gq.z, gq.w}, uw[4] = {uq.x, uq.y, uq.z, uq.w};
          float x[4], y[4], w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float value, slope;
            const float d = __uint_as_float(r[8 * h + 4 * j + e]), u = __uint_as_float(uw[e]);
            ffn_act_grad<ACT>(__uint_as_float(gw[e]), value, slope);
            w[e] = value * u;
            y[e] = d * value;
            x[e] = d * u * slope;
          }
          dg[2 * j] = pack_bf16x2(x[0], x[1]), dg[2 * j + 1] = pack_bf16x2(x[2], x[3]);
          du[2 * j] = pack_bf16x2(y[0], y[1]), du[2 * j + 1] = pack_bf16x2(y[2], y[3]);
          av[2 * j] = pack_bf16x2(w[0], w[1]), av[2 * j + 1] = pack_bf16x2(w[2], w[3]);
        }
        const uint32_t at = out + lane * 32 + ((h ^ ((lane >> 2) & 1)) << 4);
        gemm_sts128(at, dg[0], dg[1], dg[2], dg[3]);
        gemm_sts128(at + 1024, du[0], du[1], du[2], du[3]);
        gemm_sts128(at + 2048, av[0], av[1], av[2], av[3]);
      }
      staged();
      if (lane == 0) {
        const int col = col_h + c * 16;
        if (col < p.F) {
          tma_store_3d(&maps.out[1], out, col, 0, row0);
          tma_store_3d(&maps.out[1], out + 1024, col, 1, row0);
          tma_store_2d(&maps.out[0], out + 2048, col, row0);
        }
        bulk_commit_group();
      }
    }
  } else if (q.residual) {
    // the residual is added to the fp32 product: one rounding
    const int r4 = lane >> 3, c4 = (lane & 7) * 4;  // ffn_unstage32: row in a group of 4, column
    const int rows_valid = q.M - row0;
    uint2 res[8];
    auto load_res = [&](int c) {
      const int col = nb * kGemmBN + hf * 128 + c * 32 + c4;
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int rr = it * 4 + r4;
        if (rr < rows_valid && col < q.N)
          res[it] = *reinterpret_cast<const uint2*>(q.residual + (long long)(row0 + rr) * q.N + col);
      }
    };
    load_res(0);
    if (!wait_acc()) return false;
    for (int c = 0; c < 4; ++c) {
      uint32_t r[32];
      tmem_ld32(acc + hf * 128 + c * 32, r);
      tmem_wait_ld();
      if (c == 3) release_acc();
      stage32(stg, r);
      __syncwarp();
      const int col = nb * kGemmBN + hf * 128 + c * 32 + c4;
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const float4 v = ffn_unstage32(stg, it, lane);
        const int rr = it * 4 + r4;
        if (rr < rows_valid && col < q.N) {
          const uint2 w = res[it];
          *reinterpret_cast<uint2*>(q.out + (long long)(row0 + rr) * q.N + col) = make_uint2(
              pack_bf16x2(v.x + __uint_as_float(w.x << 16),
                          v.y + __uint_as_float(w.x & 0xFFFF0000u)),
              pack_bf16x2(v.z + __uint_as_float(w.y << 16),
                          v.w + __uint_as_float(w.y & 0xFFFF0000u)));
        }
      }
      if (c < 3) load_res(c + 1);
      __syncwarp();
    }
  } else if (q.ks > 1) {
    // fp32 partial sums of this run of k-blocks: [ks, M, N]
    if (!wait_acc()) return false;
    for (int c = 0; c < 4; ++c) {
      const int col0 = nb * kGemmBN + hf * 128 + c * 32;
      uint32_t r[32];
      tmem_ld32(acc + hf * 128 + c * 32, r);
      tmem_wait_ld();
      if (c == 3) release_acc();
      free_stg();
      stage32(stg, r);
      staged();
      if (lane == 0) {
        if (col0 < q.N) tma_store_3d(&maps.out[k], stg, col0, row0, split);
        bulk_commit_group();
      }
    }
  } else {
    if (!wait_acc()) return false;
    for (int c = 0; c < 2; ++c) {
      const int col0 = nb * kGemmBN + hf * 128 + c * 64;
      uint32_t r0[32], r1[32];
      tmem_ld32(acc + hf * 128 + c * 64, r0);
      tmem_ld32(acc + hf * 128 + c * 64 + 32, r1);
      tmem_wait_ld();
      if (c == 1) release_acc();
      free_stg();
#pragma unroll
      for (int jc = 0; jc < 8; ++jc) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 8 * jc + 2 * e;
          w[e] = pack_bf16x2(__uint_as_float(i < 32 ? r0[i] : r1[i - 32]),
                             __uint_as_float(i + 1 < 32 ? r0[i + 1] : r1[i + 1 - 32]));
        }
        gemm_sts128(stg + lane * 128 + ((jc ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
      }
      staged();
      if (lane == 0) {
        if (col0 < q.N) tma_store_2d(&maps.out[k], stg, col0, row0);
        bulk_commit_group();
      }
    }
  }
  return true;
}

// Roles, barriers, ring and TMEM as in gemm_bf16_sm100_pair_kernel.  A k-block
// of an operand with its M / N index innermost arrives as two 64 (K) x 64
// (M / N) boxes: 128-byte rows of K, swizzled, which the MMA reads MN-major
// (8 KB between the 64-column halves, 1 KB between groups of 8 K rows, 2 KB a
// K step of 16).
template <int MODE, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFfnThreads, 1)
    ffn_pair_kernel(const __grid_constant__ FfnMaps maps,
                    const __grid_constant__ FfnPairParams p) {
  using C = FfnPairCfg<MODE>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;  // same offset in both CTAs
  uint8_t* sptr = smem_raw + (sbase - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sptr + C::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::COUNT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const bool leader = crank == 0;
  const int pair = (int)cluster_id_x(), n_pairs = (int)cluster_count_x();

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(bar(C::FULL + s), 1);
      mbar_init(bar(C::EMPTY + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(C::AFULL + b), 1);
      mbar_init(bar(C::AEMPTY + b), 2 * kFfnEpiWarps);  // both CTAs'
    }
    mbar_init(bar(C::DRAIN), 1);
    for (int i = 0; i < kFfnEpiWarps; ++i) mbar_init(bar(C::Z + i), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), C::TM_COLS);
    tmem_relinquish_pair();
  }
  if (warp == 0 && lane < p.n_prob) {
    tma_prefetch_desc(&maps.a[lane]);
    tma_prefetch_desc(&maps.b[lane]);
  }
  if (warp == 2 && lane < (MODE == FFN_GLU     ? 1 + (p.z != nullptr)
                             : MODE == FFN_STORE ? p.n_prob
                             : MODE == FFN_DGLU  ? 3
                                                 : 0))
    tma_prefetch_desc(&maps.out[lane]);
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers initialised before any remote signal
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();  // (a tile kernel behind this one may set itself up)

  // (every role: the bounded waits below start when the kernel before has ended)
  if (p.pdl) pdl_wait();

  if (warp == 0) {
    // ===================== TMA producer (both CTAs) =====================
    const uint32_t full0 = mapa_cta(bar(C::FULL), 0);  // the even CTA's FULL[0]
    int g = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      const int t = ffn_next(p, pair, n_pairs, i);
      if (t < 0) break;
      const FfnItem item = ffn_item(p, t);
      const FfnProblem& q = p.prob[item.k];
      const CUtensorMap* tm_a = &maps.a[item.k];
      const CUtensorMap* tm_b = &maps.b[item.k];
      const int m0 = item.mb * 256 + (int)crank * 128;  // this CTA's rows of A
      const int n0 = MODE == FFN_GLU ? item.nb * 128 + (int)crank * p.F  // gate rows | up rows
                                     : item.nb * q.bn + (int)crank * (q.bn / 2);
      const uint32_t bytes = 2 * (C::A_BYTES + q.bn * kGemmBK);  // both CTAs'
      const bool a_mn = q.a_mn, b_mn = q.b_mn;
      for (int kb = item.kb0; kb < item.kb1; ++kb, ++g) {
        const int s = g % C::STAGES, u = g / C::STAGES;
        if (u > 0) ok = mbar_wait_warp(bar(C::EMPTY + s), (u - 1) & 1, abort_flag, 921);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t sa = sbase + s * C::STAGE_BYTES;
          const uint32_t fb = full0 + s * 8;
          if (leader) mbar_arrive_expect_tx(bar(C::FULL + s), bytes);
          if (a_mn) {
            tma_load_2d_pair(sa, tm_a, fb, m0, kb * kGemmBK);
            tma_load_2d_pair(sa + 8192, tm_a, fb, m0 + 64, kb * kGemmBK);
          } else {
            tma_load_2d_pair(sa, tm_a, fb, kb * kGemmBK, m0);
          }
          if (b_mn) {
            tma_load_2d_pair(sa + C::A_BYTES, tm_b, fb, n0, kb * kGemmBK);
            if (MODE != FFN_DGLU || q.bn == 256)
              tma_load_2d_pair(sa + C::A_BYTES + 8192, tm_b, fb, n0 + 64, kb * kGemmBK);
          } else {
            tma_load_2d_pair(sa + C::A_BYTES, tm_b, fb, kb * kGemmBK, n0);
          }
        }
        __syncwarp();
      }
    }
    if (!ok) {
      if (leader) {
        // the last copies counted on each stage (both CTAs') land first
        for (int s = 0; s < C::STAGES; ++s) {
          const int n_s = g > s ? (g - s - 1) / C::STAGES + 1 : 0;
          if (n_s) (void)mbar_wait(bar(C::FULL + s), (n_s - 1) & 1, nullptr, 922);
        }
      } else {
        // the odd CTA cannot see the even CTA's barrier: give copies in flight
        // into its own shared memory time to land
        __nanosleep(200000);
      }
    }
  } else if (warp == 1) {
    // ===================== MMA issuer (even CTA only) ===================
    if (leader) {
      int g = 0;
      bool ok = true;
      for (int i = 0; ok; ++i) {
        const int t = ffn_next(p, pair, n_pairs, i);
        if (t < 0) break;
        const FfnItem item = ffn_item(p, t);
        const FfnProblem& q = p.prob[item.k];
        const int a_mn = q.a_mn, b_mn = q.b_mn, n_kblk = item.kb1 - item.kb0;
        const uint32_t idesc = make_idesc_bf16(256, q.bn, a_mn, b_mn);
        const uint64_t da0 = make_sdesc_sw128(sbase, a_mn ? 8192 : 16, 1024);
        const uint64_t db0 = make_sdesc_sw128(sbase + C::A_BYTES, b_mn ? 8192 : 16, 1024);
        const uint32_t a_step = a_mn ? 2048 : 32, b_step = b_mn ? 2048 : 32;
        const int b = i & 1, use = i >> 1;
        if (use > 0) ok = mbar_wait_warp(bar(C::AEMPTY + b), (use - 1) & 1, abort_flag, 923);
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = tmem + b * kGemmBN;
        for (int kb = 0; kb < n_kblk; ++kb, ++g) {
          const int s = g % C::STAGES;
          ok = mbar_wait_warp(bar(C::FULL + s), (g / C::STAGES) & 1, abort_flag, 924);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t off = s * C::STAGE_BYTES;
#pragma unroll
            for (int kk = 0; kk < kGemmBK / 16; ++kk)
              mma_ss_pair(acc, desc_adv(da0, off + kk * a_step), desc_adv(db0, off + kk * b_step),
                          idesc, (kb | kk) != 0 ? 1u : 0u);
            tc_commit_pair_mc(bar(C::EMPTY + s), 0x3);  // the stage is free in both CTAs
          }
          __syncwarp();
        }
        if (!ok) break;
        if (elect_one()) tc_commit_pair_mc(bar(C::AFULL + b), 0x3);
        __syncwarp();
      }
      // every pair MMA has completed before either CTA frees TMEM or exits
      if (elect_one()) tc_commit_pair(bar(C::DRAIN));
      __syncwarp();
      (void)mbar_wait(bar(C::DRAIN), 0, nullptr, 925);
    }
  } else {
    // ===================== epilogue (both CTAs) =========================
    const int quarter = warp & 3, hf = (warp - 2) >> 2;
    const uint32_t stg = sbase + C::OFF_EPI + (warp - 2) * C::EPI_BYTES;
    const uint32_t aempty0 = mapa_cta(bar(C::AEMPTY), 0);
    int zn = 0;
    for (int i = 0;; ++i) {
      const int t = ffn_next(p, pair, n_pairs, i);
      if (t < 0) break;
      const FfnItem item = ffn_item(p, t);
      const FfnProblem& q = p.prob[item.k];
      const int b = i & 1, use = i >> 1;
      const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + b * kGemmBN;
      const int row0 = item.mb * 256 + (int)crank * 128 + quarter * 32;
      auto wait_acc = [&]() {
        const bool ok = mbar_wait_warp(bar(C::AFULL + b), use & 1, abort_flag, 926);
        tc_fence_after();
        return ok;
      };
      auto release_acc = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(aempty0 + b * 8);
      };
      if (!ffn_epilogue_warp<MODE, ACT>(p, q, maps, item.k, item.split, acc, row0, item.nb, hf,
                                        lane, stg, bar(C::Z + warp - 2), zn, wait_acc, release_acc))
        break;
    }
    if (lane == 0) bulk_wait_group0();  // the stores, before the shared memory goes away
    __syncwarp();
  }

  tc_fence_before();
  __syncwarp();
  cluster_sync_all();  // no CTA frees TMEM or leaves while the pair still uses it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, C::TM_COLS);
  }
}

// Joins the partial sums of products whose K was split: out = sum over the runs,
// in order, rounded once.
struct FfnSumParams {
  const float* part[kFfnMaxProblems];  // [ks, n]
  __nv_bfloat16* out[kFfnMaxProblems];
  long long n[kFfnMaxProblems];  // a multiple of 8
  int ks[kFfnMaxProblems];
  int n_prob;
};

__global__ void __launch_bounds__(256) ffn_sum_kernel(const __grid_constant__ FfnSumParams p) {
  pdl_wait();
  for (int k = 0; k < p.n_prob; ++k) {
    const long long n4 = p.n[k] / 4;
    const float4* part = reinterpret_cast<const float4*>(p.part[k]);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n4;
         i += (long long)gridDim.x * 256) {
      float4 v = part[i];
#pragma unroll 4
      for (int s = 1; s < p.ks[k]; ++s) {
        const float4 w = part[s * n4 + i];
        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
      }
      reinterpret_cast<uint2*>(p.out[k])[i] =
          make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    }
  }
}

// ===================================================================== small products
// out[t, j] over tiles of 128 weight rows j (FFN_GLU: 64 gate rows and the 64 up
// rows of the same outputs) and NT tokens t: D[128, NT] = W[128, K] X[NT, K]^T.
// With few tokens the product is bound by reading the weights once (1 token x
// 4096 x 14336: 41.5 us for the 235 MB of the up product, 5.7 TB/s, and 25.2 us
// for the 117 MB of the down one); with more, these tiles fill the SMs where
// 256 x 256 ones are too few.  A cluster of S CTAs takes one tile, each a
// contiguous run of k-blocks through its own TMA ring; the S partial tiles are
// summed through distributed shared memory, always in rank order, so results
// repeat bit for bit.
//   warp 0 TMA producer, warp 1 MMA issuer, warps 2-9 move the accumulator
//   from TMEM to shared memory (two a lane quarter, half the columns each);
//   all warps join the partials.
constexpr int kTileThreads = 320;

template <int NT, bool DEEP>
struct TileCfg {
  static constexpr int A_BYTES = 128 * 64 * 2;
  static constexpr int B_BYTES = NT * 64 * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // two CTAs an SM, or a ring twice as deep where there is one
  static constexpr int STAGES = (NT <= 32 ? 5 : NT == 64 ? 4 : 3) * (DEEP ? 2 : 1);
  static constexpr int OFF_BAR = STAGES * STAGE_BYTES;
  static constexpr int SMEM_ALLOC = OFF_BAR + 256 + 1024;
  static constexpr int TM_COLS = NT < 32 ? 32 : NT;
  static_assert(NT * 128 * 4 <= OFF_BAR, "the partial tile exceeds the ring");
  static_assert(SMEM_ALLOC <= (DEEP ? 232448 : 115712), "shared memory");
  static_assert((2 * STAGES + 2) * 8 <= 256, "barriers");
};

struct FfnTileParams {
  int J, T;  // outputs of a token, tokens
  int n_tt, n_kblk;
  int act;   // FFN_GLU
  int pdl;   // launched with programmatic stream serialization
  __nv_bfloat16* out;             // [T, J]
  float* z;                       // FFN_GLU: [T, 2 J] or null
  const __nv_bfloat16* residual;  // FFN_STORE: [T, J] or null
};

__device__ __forceinline__ void tma_load_2d(uint32_t smem_dst, const CUtensorMap* map, uint32_t bar,
                                            int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

// What is done with four joined outputs v (FFN_GLU: and the four u beside
// them; FFN_STORE: the four of the residual in w) at row `row` of the output and
// column `col`.
template <int MODE>
__device__ __forceinline__ void ffn_tile_store(const FfnTileParams& p, long long row, int col,
                                               float (&v)[4], float (&u)[4], uint2 w) {
  if constexpr (MODE == FFN_GLU) {
    if (p.z) {
      float* z = p.z + row * 2 * p.J + col;
      *reinterpret_cast<float4*>(z) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(z + p.J) = make_float4(u[0], u[1], u[2], u[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = ffn_act_rt(p.act, v[i]) * u[i];
  } else if (p.residual) {
    v[0] += __uint_as_float(w.x << 16);
    v[1] += __uint_as_float(w.x & 0xFFFF0000u);
    v[2] += __uint_as_float(w.y << 16);
    v[3] += __uint_as_float(w.y & 0xFFFF0000u);
  }
  *reinterpret_cast<uint2*>(p.out + row * p.J + col) = ffn_pack4(v);
}

// Joins this CTA's share of a tile: ROWS / S outputs of every token, four at a
// time, summed over the S partial tiles in rank order.  A thread has 8 loads
// of other CTAs' memory in flight, and the residual's before its first store
// (which may be to the residual itself): one after the other, they were half
// of a small launch's time.
template <int MODE, int S>
__device__ __forceinline__ void ffn_join(const FfnTileParams& p, uint32_t part, int rank, int j0,
                                         int t0, int tokens) {
  constexpr int ROWS = MODE == FFN_GLU ? 64 : 128;
  constexpr int R4 = ROWS / S / 4, U = 8 / S;
  const int n = R4 * tokens;
  for (int e0 = threadIdx.x; e0 < n; e0 += kTileThreads * U) {
    float4 a[U][S], b[U][S];
    uint2 res[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int e = min(e0 + k * kTileThreads, n - 1);
      if constexpr (MODE == FFN_STORE) {
        const int col = j0 + (rank * R4 + e % R4) * 4;
        if (p.residual && col < p.J)
          res[k] = *reinterpret_cast<const uint2*>(p.residual +
                                                   ((long long)t0 + e / R4) * p.J + col);
      }
      const uint32_t mine = part + (uint32_t)((e / R4) * 128 + (rank * R4 + e % R4) * 4) * 4;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const uint32_t at = mapa_cta(mine, s);
        a[k][s] = ld_cluster_f32x4(at);
        if constexpr (MODE == FFN_GLU) b[k][s] = ld_cluster_f32x4(at + 64 * 4);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int e = e0 + k * kTileThreads;
      const int col = j0 + (rank * R4 + e % R4) * 4;
      if (e >= n || col >= p.J) continue;
      float v[4] = {a[k][0].x, a[k][0].y, a[k][0].z, a[k][0].w}, u[4];
      if constexpr (MODE == FFN_GLU)
        u[0] = b[k][0].x, u[1] = b[k][0].y, u[2] = b[k][0].z, u[3] = b[k][0].w;
#pragma unroll
      for (int s = 1; s < S; ++s) {
        v[0] += a[k][s].x, v[1] += a[k][s].y, v[2] += a[k][s].z, v[3] += a[k][s].w;
        if constexpr (MODE == FFN_GLU)
          u[0] += b[k][s].x, u[1] += b[k][s].y, u[2] += b[k][s].z, u[3] += b[k][s].w;
      }
      ffn_tile_store<MODE>(p, (long long)t0 + e / R4, col, v, u, res[k]);
    }
  }
}

template <int NT, int MODE, bool DEEP>
__global__ void __launch_bounds__(kTileThreads)
    ffn_tile_kernel(const __grid_constant__ CUtensorMap tm_a,
                    const __grid_constant__ CUtensorMap tm_b, const FfnTileParams p) {
  using C = TileCfg<NT, DEEP>;
  constexpr int ROWS = MODE == FFN_GLU ? 64 : 128;  // outputs of a tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;  // same offset in every CTA of the cluster
  uint8_t* sptr = smem_raw + (sbase - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sptr + C::OFF_BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * C::STAGES + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto full = [&](int s) { return smem_u32(bars + s); };
  auto empty = [&](int s) { return smem_u32(bars + C::STAGES + s); };
  const uint32_t done = smem_u32(bars + 2 * C::STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = (int)gridDim.y, rank = (int)cluster_ctarank();  // shares of this tile's K
  // row tiles are slow, token tiles fast: tiles that share rows of A run
  // together, so those come from memory once
  const int j0 = (int)blockIdx.x / p.n_tt * ROWS, t0 = (int)blockIdx.x % p.n_tt * NT;
  const int kb0 = (int)((long long)p.n_kblk * rank / S);
  const int n_kb = (int)((long long)p.n_kblk * (rank + 1) / S) - kb0;  // at least 1
  // Row tiles start at different k-blocks of their run and wrap: all at the same
  // one read the same lines of X at once (1, 64, 128 tokens x 4096 x 14336:
  // 59.8, 67.6, 80.2 us without, 57.3, 64.7, 75.8 with).
  const int first_kb = (int)blockIdx.x / p.n_tt * 5 % n_kb;
  auto k_of = [&](int kb) {
    kb += first_kb;
    return (kb0 + (kb < n_kb ? kb : kb - n_kb)) * 64;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), C::TM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();  // (a kernel behind this one may set itself up)
  // the bounded waits of the other roles start when the kernel before has ended;
  // warp 0 asks for weights first
  if (p.pdl && warp != 0) pdl_wait();

  if (warp == 0) {
    auto load_a = [&](int kb, int s) {
      const uint32_t sa = sbase + s * C::STAGE_BYTES;
      const int k = k_of(kb);
      tma_load_2d(sa, &tm_a, full(s), k, j0);
      if (MODE == FFN_GLU) tma_load_2d(sa + 8192, &tm_a, full(s), k, p.J + j0);
    };
    // the weights do not depend on the kernel before this one: the ring's first
    // stages of them are requested before its result is waited for
    const int early = min(n_kb, C::STAGES);
    if (elect_one())
      for (int kb = 0; kb < early; ++kb) {
        mbar_arrive_expect_tx(full(kb), C::STAGE_BYTES);
        load_a(kb, kb);
      }
    __syncwarp();
    if (p.pdl) pdl_wait();
    int issued = 0;
    bool ok = true;
    for (int kb = 0; kb < n_kb; ++kb) {
      const int s = kb % C::STAGES, u = kb / C::STAGES;
      if (u > 0) ok = mbar_wait_warp(empty(s), (u - 1) & 1, abort_flag, 931);
      if (!ok) break;
      if (elect_one()) {
        if (kb >= early) {
          mbar_arrive_expect_tx(full(s), C::STAGE_BYTES);
          load_a(kb, s);
        }
        tma_load_2d(sbase + s * C::STAGE_BYTES + C::A_BYTES, &tm_b, full(s), k_of(kb), t0);
      }
      __syncwarp();
      issued = kb + 1;
    }
    if (!ok)  // copies in flight land before the shared memory goes away
      for (int s = 0; s < C::STAGES; ++s) {
        const int n_s = issued > s ? (issued - s - 1) / C::STAGES + 1 : 0;
        if (n_s) (void)mbar_wait(full(s), (n_s - 1) & 1, nullptr, 932);
      }
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc_bf16(128, NT, 0, 0);
    const uint64_t da0 = make_sdesc_sw128(sbase, 16, 1024);
    const uint64_t db0 = make_sdesc_sw128(sbase + C::A_BYTES, 16, 1024);
    bool ok = true;
    for (int kb = 0; kb < n_kb; ++kb) {
      const int s = kb % C::STAGES;
      ok = mbar_wait_warp(full(s), (kb / C::STAGES) & 1, abort_flag, 933);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t off = s * C::STAGE_BYTES;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_ss(tmem, desc_adv(da0, off + kk * 32), desc_adv(db0, off + kk * 32), idesc,
                 (kb | kk) != 0 ? 1u : 0u);
        tc_commit(empty(s));
      }
      __syncwarp();
    }
    // completes when every MMA issued above has, whether or not all were
    if (elect_one()) tc_commit(done);
    __syncwarp();
  }
  // Every thread: the accumulator is complete (or the CTA gave up).
  (void)mbar_wait(done, 0, nullptr, 934);
  tc_fence_after();
  __syncthreads();  // the ring's shared memory is free: it now holds the partial tile
  float* part = reinterpret_cast<float*>(sptr);  // [NT][128]
  if (warp >= 2) {
    const int quarter = warp & 3;
    const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
    for (int c = ((warp - 2) >> 2) * 16; c < NT; c += 32) {
      if (t0 + c >= p.T) break;
      uint32_t r[16];
      tmem_ld16(acc + c, r);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; ++e)
        part[(c + e) * 128 + quarter * 32 + lane] = __uint_as_float(r[e]);
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TM_COLS);
  }
  if (!*abort_flag) {
    const int tokens = min(NT, p.T - t0);
    switch (S) {
      case 1: ffn_join<MODE, 1>(p, sbase, 0, j0, t0, tokens); break;
      case 2: ffn_join<MODE, 2>(p, sbase, rank, j0, t0, tokens); break;
      case 4: ffn_join<MODE, 4>(p, sbase, rank, j0, t0, tokens); break;
      default: ffn_join<MODE, 8>(p, sbase, rank, j0, t0, tokens); break;
    }
  }
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while another reads its partial tile
}

}  // namespace tfb
