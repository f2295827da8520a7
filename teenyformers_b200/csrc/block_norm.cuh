// block_norm.cuh -- the norms on either side of a block's residual sum, fused
// with the branch's gate, scales and dropout:
//
//   n = RMSNorm(f) * w_post            (w_post null: n = f)
//   v = dropout(gate * n)              (gate null: 1; drop.rng null: no dropout)
//   y = residual_scale * x + branch_scale * v        (f null: y = x, not written)
//   h = RMSNorm(y) * w_pre             (w_pre null: no h)
//
// RMSNorm(v) = v * rsqrt(mean(v^2) + eps) over the row.  f is a block's output,
// x the residual stream, h what the next block reads.  The gate has one row
// for every rows / gate_rows consecutive rows of x (one for all, one a
// sequence, one a token).  h is computed from y before y is rounded.
//
// Backward, with t the whole gradient of y and r_f, r_y the inverse RMS of the
// saved bf16 rows (recomputed: the rows are read anyway):
//   t      = dy + r_y (dh w_pre - y r_y^2 mean(dh w_pre y))
//   dx     = residual_scale t          dw_pre = sum_rows dh y r_y
//   dv     = branch_scale mask t       dgate  = sum_(its rows) dv n
//   q      = dv gate                   dw_post = sum_rows q f r_f
//   df     = r_f (q w_post - f r_f^2 mean(q w_post f))
//
// Both passes are HBM-bound: 8 bytes an element forward (x, f, y, h), 12
// backward (f, y, dy, dh, dx, df), everything else stays on the chip.  A row
// belongs to a team of WPR warps; all statistics and sums are fp32.  The
// column sums of the backward pass are accumulated in registers over a team's
// contiguous rows, written as fp32 partials and summed in a fixed order by a
// second kernel, so results repeat bit for bit.
#pragma once

#include "norm_act.cuh"
#include "philox.cuh"
#include "sm100.cuh"

namespace tfb {

constexpr int kBnThreads = 256;
constexpr int kBnWarps = kBnThreads / 32;
constexpr int kBnMaxCols = 8192;

struct BlockNormParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* f;
  const __nv_bfloat16* w_post;
  const __nv_bfloat16* gate;
  const __nv_bfloat16* w_pre;
  __nv_bfloat16* y;
  __nv_bfloat16* h;
  int rows, cols, rows_per_gate;
  float eps, residual_scale, branch_scale;
  DropoutParams drop;
};

// Sums NV values over a team's threads.  `buf` alternates between calls: a
// thread can only write buffer b again after the team's barrier of the call
// in between, which every thread reaches after its reads of b.
template <int WPR, int NV>
__device__ __forceinline__ void team_sum(float (&v)[NV], float (*red)[2][kBnWarps][4], int& buf,
                                         int team, int warp_in_team) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (WPR > 1) {
    float(*r)[4] = (*red)[buf] + team * WPR;
    buf ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < NV; ++k) r[warp_in_team][k] = v[k];
    named_bar_sync(1 + team, WPR * 32);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      v[k] = r[0][k];
#pragma unroll
      for (int w = 1; w < WPR; ++w) v[k] += r[w][k];
    }
  }
}

template <int WPR, int VPT>
__global__ void __launch_bounds__(kBnThreads) block_norm_fwd_kernel(const BlockNormParams p) {
  constexpr int TEAMS = kBnWarps / WPR, TT = WPR * 32;
  __shared__ float red[2][kBnWarps][4];
  const int team = (int)threadIdx.x / TT, tid = (int)threadIdx.x % TT;
  const long long row = (long long)blockIdx.x * TEAMS + team;
  if (row >= p.rows) return;  // whole teams leave: their barriers are their own
  const int nvec = p.cols / 8;
  const long long base = row * p.cols;
  int buf = 0;
  uint4 xv[VPT], fv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * TT;
    if (v < nvec) {
      xv[i] = reinterpret_cast<const uint4*>(p.x + base)[v];
      if (p.f) fv[i] = reinterpret_cast<const uint4*>(p.f + base)[v];
    }
  }
  float r_f = 1.0f;
  if (p.f && p.w_post) {
    float ss[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (tid + i * TT < nvec) {
        float a[8];
        bf16x8_to_f32(fv[i], a);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss[0] = fmaf(a[e], a[e], ss[0]);
      }
    team_sum<WPR, 1>(ss, &red, buf, team, tid >> 5);
    r_f = rsqrtf(ss[0] / (float)p.cols + p.eps);
  }
  PhiloxState rng = {};
  if (p.drop.rng) rng = philox_state(p.drop);
  const __nv_bfloat16* gate_row =
      p.gate ? p.gate + (row / p.rows_per_gate) * (long long)p.cols : nullptr;
  float y[VPT][8];
  float ssy[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * TT;
    if (v < nvec) {
      bf16x8_to_f32(xv[i], y[i]);
      if (p.f) {
        float b[8], w[8];
        bf16x8_to_f32(fv[i], b);
        if (p.w_post) {
          bf16x8_to_f32(reinterpret_cast<const uint4*>(p.w_post)[v], w);
#pragma unroll
          for (int e = 0; e < 8; ++e) b[e] = b[e] * r_f * w[e];
        }
        if (gate_row) {
          bf16x8_to_f32(reinterpret_cast<const uint4*>(gate_row)[v], w);
#pragma unroll
          for (int e = 0; e < 8; ++e) b[e] *= w[e];
        }
        if (p.drop.rng) dropout8(p.drop, rng, (uint32_t)(base / 8 + v), b);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = p.residual_scale * y[i][e] + p.branch_scale * b[e];
        reinterpret_cast<uint4*>(p.y + base)[v] = f32_to_bf16x8(y[i]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) ssy[0] = fmaf(y[i][e], y[i][e], ssy[0]);
    }
  }
  if (!p.w_pre) return;
  team_sum<WPR, 1>(ssy, &red, buf, team, tid >> 5);
  const float r_y = rsqrtf(ssy[0] / (float)p.cols + p.eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * TT;
    if (v < nvec) {
      float w[8];
      bf16x8_to_f32(reinterpret_cast<const uint4*>(p.w_pre)[v], w);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = y[i][e] * r_y * w[e];
      reinterpret_cast<uint4*>(p.h + base)[v] = f32_to_bf16x8(w);
    }
  }
}

// ------------------------------------------------------------------ backward
struct BlockNormBwdParams {
  const __nv_bfloat16* f;       // read when w_post or gate is set
  const __nv_bfloat16* w_post;
  const __nv_bfloat16* gate;
  const __nv_bfloat16* y;       // read when w_pre is set
  const __nv_bfloat16* w_pre;
  const __nv_bfloat16* dy;      // null: zero
  const __nv_bfloat16* dh;      // with w_pre
  __nv_bfloat16* dx;
  __nv_bfloat16* df;            // null: no branch
  __nv_bfloat16* dgate;
  float* part_post;             // [n_teams, cols]
  float* part_pre;              // [n_teams, cols]
  float* part_gate;             // [n_teams, 2, cols]
  int rows, cols, rows_per_gate, rows_per_team, n_teams;
  float eps, residual_scale, branch_scale;
  DropoutParams drop;
};

// The teams of a call: two 256-thread CTAs on each of 148 SMs, contiguous
// rows to each team.  A pure function of the shape, so that the workspace
// query and the launch agree.
constexpr int kBnBwdCtas = 296;

struct BlockNormTeams {
  int wpr, vpt, rows_per_team, n_teams;
};
inline BlockNormTeams block_norm_teams(int rows, int cols) {
  BlockNormTeams t;
  const int nvec = cols / 8;
  t.vpt = nvec <= 32 ? 1 : nvec <= 512 ? 2 : 4;
  t.wpr = nvec <= 64 ? 1 : nvec <= 128 ? 2 : nvec <= 256 ? 4 : 8;
  const int want = kBnBwdCtas * (kBnWarps / t.wpr);
  t.rows_per_team = rows > 0 ? (int)(((long long)rows + want - 1) / want) : 1;
  t.n_teams = (int)(((long long)rows + t.rows_per_team - 1) / t.rows_per_team);
  return t;
}

// Simple form: one row at a time, straight from global memory.
template <int WPR, int VPT>
__global__ void __launch_bounds__(kBnThreads) block_norm_bwd_kernel(const BlockNormBwdParams p) {
  constexpr int TEAMS = kBnWarps / WPR, TT = WPR * 32;
  __shared__ float red[2][kBnWarps][4];
  const int team_in_cta = (int)threadIdx.x / TT, tid = (int)threadIdx.x % TT;
  const int team = (int)blockIdx.x * TEAMS + team_in_cta;
  if (team >= p.n_teams) return;
  const int nvec = p.cols / 8;
  const int row0 = team * p.rows_per_team;
  const int row1 = (int)min((long long)p.rows, (long long)row0 + p.rows_per_team);
  int buf = 0;
  PhiloxState rng = {};
  if (p.drop.rng) rng = philox_state(p.drop);
  const bool has_f = p.df && (p.w_post || p.gate);
  float a_post[VPT][8], a_pre[VPT][8], a_gate[VPT][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) a_post[i][e] = a_pre[i][e] = a_gate[i][e] = 0.0f;

  int gate_row = row0 / p.rows_per_gate, gate_first = row0;  // this segment of the gate's rows
  for (int row = row0; row < row1; ++row) {
    const long long base = (long long)row * p.cols;
    float s3[3] = {0.0f, 0.0f, 0.0f};  // y^2, dh w_pre y, f^2
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * TT;
      if (v < nvec) {
        if (p.w_pre) {
          float y8[8], d8[8], w8[8];
          bf16x8_to_f32(reinterpret_cast<const uint4*>(p.y + base)[v], y8);
          bf16x8_to_f32(reinterpret_cast<const uint4*>(p.dh + base)[v], d8);
          bf16x8_to_f32(reinterpret_cast<const uint4*>(p.w_pre)[v], w8);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            s3[0] = fmaf(y8[e], y8[e], s3[0]);
            s3[1] = fmaf(d8[e] * w8[e], y8[e], s3[1]);
          }
        }
        if (has_f && p.w_post) {
          float f8[8];
          bf16x8_to_f32(reinterpret_cast<const uint4*>(p.f + base)[v], f8);
#pragma unroll
          for (int e = 0; e < 8; ++e) s3[2] = fmaf(f8[e], f8[e], s3[2]);
        }
      }
    }
    team_sum<WPR, 3>(s3, &red, buf, team_in_cta, tid >> 5);
    const float inv_c = 1.0f / (float)p.cols;
    const float r_y = rsqrtf(s3[0] * inv_c + p.eps);
    const float m_y = s3[1] * inv_c * r_y * r_y;  // mean(dh w_pre y) r_y^2
    const float r_f = p.w_post ? rsqrtf(s3[2] * inv_c + p.eps) : 1.0f;
    float q[VPT][8];
    float s1[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * TT;
      if (v < nvec) {
        float t[8];
        if (p.dy) {
          bf16x8_to_f32(reinterpret_cast<const uint4*>(p.dy + base)[v], t);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) t[e] = 0.0f;
        }
        if (p.w_pre) {
          float y8[8], d8[8], w8[8];
          bf16x8_to_f32(reinterpret_cast<const uint4*>(p.y + base)[v], y8);
          bf16x8_to_f32(reinterpret_cast<const uint4*>(p.dh + base)[v], d8);
          bf16x8_to_f32(reinterpret_cast<const uint4*>(p.w_pre)[v], w8);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            a_pre[i][e] = fmaf(d8[e], y8[e] * r_y, a_pre[i][e]);
            t[e] += r_y * (d8[e] * w8[e] - y8[e] * m_y);
          }
        }
        if (p.df) {
          float b[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) b[e] = p.branch_scale * t[e];
          if (p.drop.rng) dropout8(p.drop, rng, (uint32_t)(base / 8 + v), b);
          if (has_f) {
            float n[8], w8[8], g8[8];
            bf16x8_to_f32(reinterpret_cast<const uint4*>(p.f + base)[v], n);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              n[e] *= r_f;
              w8[e] = g8[e] = 1.0f;
            }
            if (p.w_post) bf16x8_to_f32(reinterpret_cast<const uint4*>(p.w_post)[v], w8);
            if (p.gate) {
              bf16x8_to_f32(
                  reinterpret_cast<const uint4*>(p.gate + (long long)gate_row * p.cols)[v], g8);
#pragma unroll
              for (int e = 0; e < 8; ++e) a_gate[i][e] = fmaf(b[e], n[e] * w8[e], a_gate[i][e]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              b[e] *= g8[e];
              a_post[i][e] = fmaf(b[e], n[e], a_post[i][e]);
              b[e] *= w8[e];
              s1[0] = fmaf(b[e], n[e], s1[0]);
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) q[i][e] = b[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] *= p.residual_scale;
        reinterpret_cast<uint4*>(p.dx + base)[v] = f32_to_bf16x8(t);
      }
    }
    if (p.df) {
      if (p.w_post) team_sum<WPR, 1>(s1, &red, buf, team_in_cta, tid >> 5);
      const float m_f = s1[0] * inv_c * r_f;  // mean(q w_post n) r_f
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = tid + i * TT;
        if (v < nvec) {
          if (p.w_post) {
            float f8[8];
            bf16x8_to_f32(reinterpret_cast<const uint4*>(p.f + base)[v], f8);
#pragma unroll
            for (int e = 0; e < 8; ++e) q[i][e] = r_f * (q[i][e] - f8[e] * m_f);
          }
          reinterpret_cast<uint4*>(p.df + base)[v] = f32_to_bf16x8(q[i]);
        }
      }
    }
    if (p.gate && p.df) {
      // the last row of the gate's rows, or of this team's: hand over the sum
      const long long gate_end = ((long long)gate_row + 1) * p.rows_per_gate;
      if (row + 1 == gate_end || row + 1 == row1) {
        const bool whole =
            gate_first == (long long)gate_row * p.rows_per_gate && row + 1 == gate_end;
        // a segment that starts at the team's first row goes to slot 0
        float* part = p.part_gate +
                      ((long long)team * 2 + (gate_first == row0 ? 0 : 1)) * p.cols;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int v = tid + i * TT;
          if (v < nvec) {
            if (whole) {
              reinterpret_cast<uint4*>(p.dgate + (long long)gate_row * p.cols)[v] =
                  f32_to_bf16x8(a_gate[i]);
            } else {
              reinterpret_cast<float4*>(part)[2 * v] =
                  make_float4(a_gate[i][0], a_gate[i][1], a_gate[i][2], a_gate[i][3]);
              reinterpret_cast<float4*>(part)[2 * v + 1] =
                  make_float4(a_gate[i][4], a_gate[i][5], a_gate[i][6], a_gate[i][7]);
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) a_gate[i][e] = 0.0f;
        }
        ++gate_row;
        gate_first = row + 1;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * TT;
    if (v < nvec) {
      if (p.df && p.w_post) {
        float4* d = reinterpret_cast<float4*>(p.part_post + (long long)team * p.cols);
        d[2 * v] = make_float4(a_post[i][0], a_post[i][1], a_post[i][2], a_post[i][3]);
        d[2 * v + 1] = make_float4(a_post[i][4], a_post[i][5], a_post[i][6], a_post[i][7]);
      }
      if (p.w_pre) {
        float4* d = reinterpret_cast<float4*>(p.part_pre + (long long)team * p.cols);
        d[2 * v] = make_float4(a_pre[i][0], a_pre[i][1], a_pre[i][2], a_pre[i][3]);
        d[2 * v + 1] = make_float4(a_pre[i][4], a_pre[i][5], a_pre[i][6], a_pre[i][7]);
      }
    }
  }
}

// Sums the teams' partials: output 0 is dw_post, 1 is dw_pre, 2 + g the gate's
// row g where more than one team has rows of it.  32 columns a block, eight
// strided partial sums a column, joined in a fixed order.
struct BlockNormSumParams {
  const float* part_post;
  const float* part_pre;
  const float* part_gate;
  __nv_bfloat16* dw_post;
  __nv_bfloat16* dw_pre;
  __nv_bfloat16* dgate;  // null: no gate, or every gate row is one team's
  int cols, n_teams, rows_per_team, rows_per_gate, gate_rows;
};

__global__ void __launch_bounds__(256) block_norm_sum_kernel(const BlockNormSumParams p) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int col = (int)blockIdx.x * 32 + lane;
  const int outs = 2 + (p.dgate ? p.gate_rows : 0);
  for (int o = blockIdx.y; o < outs; o += gridDim.y) {
    const float* src;
    __nv_bfloat16* dst;
    int t0 = 0, t1 = p.n_teams - 1;
    const int g = o - 2;
    if (o == 0) {
      src = p.part_post, dst = p.dw_post;
    } else if (o == 1) {
      src = p.part_pre, dst = p.dw_pre;
    } else {
      src = p.part_gate, dst = p.dgate + (long long)g * p.cols;
      t0 = (int)((long long)g * p.rows_per_gate / p.rows_per_team);
      t1 = (int)((((long long)g + 1) * p.rows_per_gate - 1) / p.rows_per_team);
      if (t0 == t1) dst = nullptr;  // written whole by its team
    }
    if (!dst) continue;  // the same for every thread of the block
    float acc = 0.0f;
    if (col < p.cols) {
#pragma unroll 4
      for (int t = t0 + part; t <= t1; t += 8) {
        long long at = t;
        if (o >= 2) {
          // slot 0 unless the segment starts inside the team's rows
          const bool inside =
              (long long)g * p.rows_per_gate > (long long)t * p.rows_per_team;
          at = 2LL * t + (inside ? 1 : 0);
        }
        acc += src[at * p.cols + col];
      }
    }
    s[part][lane] = acc;
    __syncthreads();
    if (part == 0 && col < p.cols) {
#pragma unroll
      for (int k = 1; k < 8; ++k) acc += s[k][lane];
      dst[col] = __float2bfloat16_rn(acc);
    }
    __syncthreads();
  }
}

}  // namespace tfb
