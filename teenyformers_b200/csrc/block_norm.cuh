// block_norm.cuh -- the norms on either side of a block's residual sum, fused
// with the branch's gate, scales and dropout:
//
//   n = RMSNorm(f) * w_post            (w_post null: n = f)
//   v = dropout(gate * n)              (gate null: 1; drop.rng null: no dropout)
//   y = residual_scale * x + branch_scale * v        (f null: y = x, not written)
//   h = RMSNorm(y) * w_pre             (w_pre null: no h)
//
// A NaN of f under w_post makes its row's inverse RMS and so the whole row of y NaN, the
// dropped places included; without w_post what is dropped leaves nothing behind.
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
// backward (f, y, dy, dh, dx, df), everything else stays on the chip (16384 x
// 4096, whole calls on inputs from memory: 90 us, 5.9 TB/s, with 8 gate rows and 102
// with one or none; backward 138-144, 5.7 TB/s, and with dropout 164-169, when the
// generator's rounds stand between a row's loads and its stores: 58 % of the issue
// slots are taken, it is latency).  A row belongs to a team of WPR
// warps; all statistics and sums are fp32.  The column sums of the backward pass
// are accumulated in registers over a team's rows, written as fp32 partials and
// summed in a fixed order by a second kernel, so results repeat bit for bit.
#pragma once

#include "norm_act.cuh"
#include "philox.cuh"
#include "sm100.cuh"

namespace tfb {

constexpr int kBnMaxCols = 8192;
// A CTA's warps and teams, for teams of WPR warps
__host__ __device__ constexpr int bn_warps(int wpr) { return wpr > 8 ? wpr : 8; }
__host__ __device__ constexpr int bn_teams(int wpr) { return bn_warps(wpr) / wpr; }

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

// ---------------------------------------------------------------- teams and rings
// A row is worked on by a team of WPR warps (the smallest of 1, 2, 4, 8, 16 that
// holds it at VPT 16-byte vectors a thread); a CTA of 256 threads has 8 / WPR
// teams, one of 512 a team of 16 warps.  The rows' tensors arrive through
// a ring of shared-memory stages, filled by bulk copies of one or several
// whole rows (rows are contiguous), so the loads of the next rows run under
// the arithmetic and the two reductions of this one: with plain loads the
// forward pass of 16384 x 4096 took 100 us and the backward pass 370 us, bound
// by load latency (4.7 and more stalled cycles an instruction).
constexpr int kBnStages = 3;
constexpr int kBnRed = 4 * 24;       // team_sum: at most 4 teams of several warps
constexpr int kBnCtas = 296;  // two CTAs on each of 148 SMs (of 512 threads: one)
constexpr int kBnRingBytes = 98304;  // a CTA's stages, where a row is not longer

struct BlockNormTeams {
  int wpr, vpt, threads, rows_per_team, n_teams, n_ctas;
  int rows_per_stage, smem;
};
// A pure function of the shape, so that the workspace query and the launch
// agree.  `tensors`: the most that a row's stage holds (2 forward, 4 backward).
// A thread has two vectors where a row allows it (the reductions are then a
// smaller part of its work), and one in the backward pass up to 2048 columns:
// with two, the teams of fewer than 8 warps spill registers (16384 x 2048 with
// dropout 121 us, with one 98 us).  Rows past 4096 columns take 16 warps: with 8
// and four vectors a thread, one CTA an SM had too few warps (16384 x 8192 backward
// 311 us, with dropout 367, so 258 and 314; forward 166, so 161; on inputs from memory
// the latter are 276-290, 333 and 174).
inline BlockNormTeams block_norm_teams(int rows, int cols, int tensors) {
  BlockNormTeams t;
  const int nvec = cols / 8;
  if (tensors == 4) {
    t.vpt = nvec <= 256 ? 1 : 2;
    t.wpr = nvec <= 32 ? 1 : nvec <= 64 ? 2 : nvec <= 128 ? 4 : nvec <= 512 ? 8 : 16;
  } else {
    t.vpt = nvec <= 32 ? 1 : 2;
    t.wpr = nvec <= 64 ? 1 : nvec <= 128 ? 2 : nvec <= 256 ? 4 : nvec <= 512 ? 8 : 16;
  }
  t.threads = bn_warps(t.wpr) * 32;
  const int teams = bn_teams(t.wpr);
  const int want = (t.wpr == 16 ? kBnCtas / 2 : kBnCtas) * teams;
  t.rows_per_team = rows > 0 ? (int)(((long long)rows + want - 1) / want) : 1;
  t.n_teams = (int)(((long long)rows + t.rows_per_team - 1) / t.rows_per_team);
  t.n_ctas = (t.n_teams + teams - 1) / teams;
  const int row_stage = teams * kBnStages * tensors * cols * 2;
  int r = kBnRingBytes / row_stage;
  r = r < 1 ? 1 : r > 8 ? 8 : r;
  t.rows_per_stage = r < t.rows_per_team ? r : t.rows_per_team;
  t.smem = t.rows_per_stage * row_stage;
  return t;
}

__device__ __forceinline__ uint4 bn_lds(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Eight bf16 as four packed fp32 pairs, and back.
__device__ __forceinline__ void bn_unpack(const uint4& v, uint64_t (&f)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    f[i] = f2_make(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
}
__device__ __forceinline__ uint4 bn_pack(const uint64_t (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    f2_split(f[i], lo, hi);
    w[i] = pack_bf16x2(lo, hi);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float bn_hsum(uint64_t v) {
  float lo, hi;
  f2_split(v, lo, hi);
  return lo + hi;
}
// dropout_select8 of elements held as pairs.
__device__ __forceinline__ void bn_select(const DropoutParams& d, const PhiloxState& s,
                                          uint32_t group, uint64_t (&f)[4]) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_split(f[i], v[2 * i], v[2 * i + 1]);
  dropout_select8(d, s, group, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = f2_make(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void bn_store_f32(float* dst, int v, const uint64_t (&f)[4]) {
  float a[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_split(f[i], a[2 * i], a[2 * i + 1]);
  reinterpret_cast<float4*>(dst)[2 * v] = make_float4(a[0], a[1], a[2], a[3]);
  reinterpret_cast<float4*>(dst)[2 * v + 1] = make_float4(a[4], a[5], a[6], a[7]);
}

// One team's ring of row stages.  Chunk k is the rows from row0 + k * step on,
// rows_per_stage of them or as many as there are before row1.
template <int TENSORS>
struct BnRing {
  const __nv_bfloat16* src[TENSORS];  // null: absent
  uint32_t bar, data;                 // kBnStages mbarriers; the team's stages
  uint32_t slot, stage;               // bytes of one tensor's rows, and of a stage
  int rows_per_stage, row0, row1, cols, present;
  long long step;

  // (the team's first thread)
  __device__ __forceinline__ void issue(int k) const {
    const long long r = row0 + k * step;
    if (r >= row1) return;
    const uint32_t bytes = (uint32_t)min((long long)rows_per_stage, row1 - r) * cols * 2;
    const int s = k % kBnStages;
    mbar_arrive_expect_tx(bar + s * 8, bytes * present);
#pragma unroll
    for (int i = 0; i < TENSORS; ++i)
      if (src[i])
        bulk_load(data + s * stage + i * slot, src[i] + r * cols, bytes, bar + s * 8);
  }
  // Every thread of the team.  A wait that runs out (a fault) is recorded and
  // makes the later ones return at once; the outputs are then invalid.
  __device__ __forceinline__ void wait(int k, volatile int* abort_flag, int site) const {
    (void)mbar_wait(bar + (k % kBnStages) * 8, (k / kBnStages) & 1, abort_flag, site);
  }
  __device__ __forceinline__ uint32_t at(int k, int i, int row_in_stage) const {
    return data + (k % kBnStages) * stage + i * slot + (uint32_t)row_in_stage * cols * 2;
  }
};

template <int WPR>
__device__ __forceinline__ void team_sync(int team) {
  if constexpr (WPR == 1)
    __syncwarp();
  else
    named_bar_sync(1 + team, WPR * 32);
}

// Sums NV (1 or 3) values over a team's threads.  `buf` alternates between
// calls: a thread can only write buffer b again after the team's barrier of
// the call in between, which every thread reaches after its reads of b.
// Instruction counts matter here (an eighth of the backward pass): three
// values over a warp in 6 shuffles (lanes 0, 8, 16 end with one value each),
// and the warps' sums in one load, 3 shuffles and a broadcast a value.
template <int WPR, int NV>
__device__ __forceinline__ void team_sum(float (&v)[NV], float (*red)[kBnRed], int& buf, int team,
                                         int warp_in_team) {
  static_assert(NV == 1 || NV == 3, "one or three values");
  constexpr unsigned ALL = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  if constexpr (WPR == 1) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < NV; ++k) v[k] += __shfl_xor_sync(ALL, v[k], o);
  } else {
    float t;
    if constexpr (NV == 3) {
      const bool up = lane & 16, mid = lane & 8;
      // the lower half keeps values 0 and 1, the upper half value 2
      float a = up ? v[2] : v[0];
      a += __shfl_xor_sync(ALL, up ? v[0] : v[2], 16);
      float b = up ? 0.0f : v[1];
      b += __shfl_xor_sync(ALL, up ? v[1] : 0.0f, 16);
      t = mid ? b : a;
      t += __shfl_xor_sync(ALL, mid ? a : b, 8);
    } else {
      t = v[0] + __shfl_xor_sync(ALL, v[0], 16);
      t += __shfl_xor_sync(ALL, t, 8);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) t += __shfl_xor_sync(ALL, t, o);
    // 8 slots a value and team, WPR of them used (16 warps: two runs of 8 slots a value)
    float* r = red[buf] + team * 24;
    buf ^= 1;
    float* slot = r + (warp_in_team & 7) + (warp_in_team >> 3) * 24;
    if constexpr (NV == 3) {
      if ((lane & 7) == 0 && lane < 24) slot[lane] = t;
      named_bar_sync(1 + team, WPR * 32);
      t = (lane < 24 && (lane & 7) < WPR) ? r[lane] : 0.0f;
      if (WPR == 16 && lane < 24) t += r[24 + lane];
    } else {
      if (lane == 0) slot[0] = t;
      named_bar_sync(1 + team, WPR * 32);
      t = (lane & 7) < WPR ? r[lane & 7] : 0.0f;
      if (WPR == 16) t += r[24 + (lane & 7)];
    }
#pragma unroll
    for (int o = (WPR < 8 ? WPR : 8) / 2; o > 0; o >>= 1) t += __shfl_xor_sync(ALL, t, o);
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] = NV == 1 && WPR >= 8 ? t : __shfl_sync(ALL, t, 8 * k);
  }
}

// ---------------------------------------------------------------- forward
// VPT vectors a thread; a vector past the row's end reads zeros from `zero`, so
// that nothing but the stores is predicated.  ALL: f, w_post and w_pre are given
// (a block's usual case: no branches on them).  The weights stay in registers over
// the team's rows (gate * w_post as their fp32 product, renewed where the gate's
// row changes).
template <int WPR, int VPT, bool ALL>
__global__ void __launch_bounds__(bn_warps(WPR) * 32, WPR <= 8 ? 2 : 1)
    block_norm_fwd_kernel(const BlockNormParams p, const BlockNormTeams tm) {
  constexpr int TT = WPR * 32;
  extern __shared__ uint4 bn_stages[];
  __shared__ float red[2][kBnRed];
  __shared__ uint4 zero_cell;
  __shared__ uint64_t bars[8 * kBnStages];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int team_in_cta = (int)threadIdx.x / TT, tid = (int)threadIdx.x % TT;
  const int team = (int)blockIdx.x * bn_teams(WPR) + team_in_cta;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 8 * kBnStages; ++i) mbar_init(smem_u32(bars + i), 1);
    abort_word = 0;
    zero_cell = make_uint4(0, 0, 0, 0);
    fence_mbar_init();
  }
  __syncthreads();
  if (team >= tm.n_teams) return;  // whole teams leave: their barriers are their own
  const int nvec = p.cols / 8;
  const bool has_f = ALL || p.f, post = ALL || (p.f && p.w_post), pre = ALL || p.w_pre;
  const uint32_t zero = smem_u32(&zero_cell);
  auto lds = [&](uint32_t row, int i) {
    const int v = tid + i * TT;
    return bn_lds(v < nvec ? row + v * 16 : zero);
  };
  BnRing<2> ring;
  ring.src[0] = p.f, ring.src[1] = p.x;
  ring.present = p.f ? 2 : 1;
  ring.cols = p.cols, ring.rows_per_stage = tm.rows_per_stage;
  ring.row0 = team * tm.rows_per_stage;
  ring.row1 = p.rows;
  ring.step = (long long)tm.n_teams * tm.rows_per_stage;
  ring.slot = (uint32_t)tm.rows_per_stage * p.cols * 2;
  ring.stage = 2 * ring.slot;
  ring.bar = smem_u32(bars + team_in_cta * kBnStages);
  ring.data = smem_u32(bn_stages) + team_in_cta * kBnStages * ring.stage;
  if (tid == 0)
    for (int k = 0; k < kBnStages; ++k) ring.issue(k);
  int buf = 0;
  PhiloxState rng = {};
  if (p.drop.rng) rng = philox_state(p.drop);
  const float inv_c = 1.0f / (float)p.cols;
  const uint64_t rs2 = f2_make(p.residual_scale, p.residual_scale);

  uint64_t wg[VPT][4];  // gate * w_post
  uint4 wn[VPT];        // w_pre
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * TT;
    wn[i] = p.w_pre && v < nvec ? reinterpret_cast<const uint4*>(p.w_pre)[v] : make_uint4(0, 0, 0, 0);
  }
  const float branch = p.branch_scale * (p.drop.rng ? p.drop.scale : 1.0f);
  long long gate_end = 0;  // the first row of the next gate row
  auto load_gate = [&](int g) {
    gate_end = ((long long)g + 1) * p.rows_per_gate;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * TT;
#pragma unroll
      for (int e = 0; e < 4; ++e) wg[i][e] = f2_make(1.0f, 1.0f);
      if (v >= nvec) continue;
      if (p.w_post) bn_unpack(reinterpret_cast<const uint4*>(p.w_post)[v], wg[i]);
      if (p.gate) {
        uint64_t g4[4];
        bn_unpack(reinterpret_cast<const uint4*>(p.gate + (long long)g * p.cols)[v], g4);
#pragma unroll
        for (int e = 0; e < 4; ++e) wg[i][e] = f2_mul(wg[i][e], g4[e]);
      }
    }
  };
  if (has_f) load_gate(ring.row0 / p.rows_per_gate);

  int k = 0;
  for (long long r = ring.row0; r < ring.row1; r += ring.step, ++k) {
    ring.wait(k, abort_flag, 941);
    const int here = (int)min((long long)tm.rows_per_stage, ring.row1 - r);
    for (int j = 0; j < here; ++j) {
      const int row = (int)r + j;
      const long long base = (long long)row * p.cols;
      const uint32_t fa = ring.at(k, 0, j), xa = ring.at(k, 1, j);
      float r_f = 1.0f;
      if (post) {
        uint64_t ss = 0;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          uint64_t a[4];
          bn_unpack(lds(fa, i), a);
#pragma unroll
          for (int e = 0; e < 4; ++e) ss = f2_fma(a[e], a[e], ss);
        }
        float s1[1] = {bn_hsum(ss)};
        team_sum<WPR, 1>(s1, red, buf, team_in_cta, tid >> 5);
        r_f = rsqrtf(s1[0] * inv_c + p.eps);
      }
      if (p.gate && row >= gate_end) load_gate(row / p.rows_per_gate);
      const float bf = branch * r_f;
      const uint64_t bf2 = f2_make(bf, bf);
      uint64_t y[VPT][4], ssy = 0;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = tid + i * TT;
        bn_unpack(lds(xa, i), y[i]);
        if (has_f) {
          uint64_t b[4];
          bn_unpack(lds(fa, i), b);
#pragma unroll
          for (int e = 0; e < 4; ++e) b[e] = f2_mul(b[e], wg[i][e]);
          if (p.drop.rng) bn_select(p.drop, rng, (uint32_t)(base / 8 + v), b);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[i][e] = f2_fma(b[e], bf2, f2_mul(y[i][e], rs2));
          if (v < nvec) reinterpret_cast<uint4*>(p.y + base)[v] = bn_pack(y[i]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) ssy = f2_fma(y[i][e], y[i][e], ssy);
      }
      if (pre) {
        float s1[1] = {bn_hsum(ssy)};
        team_sum<WPR, 1>(s1, red, buf, team_in_cta, tid >> 5);
        const float r_y = rsqrtf(s1[0] * inv_c + p.eps);
        const uint64_t ry2 = f2_make(r_y, r_y);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int v = tid + i * TT;
          uint64_t w[4];
          bn_unpack(wn[i], w);
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = f2_mul(f2_mul(y[i][e], ry2), w[e]);
          if (v < nvec) reinterpret_cast<uint4*>(p.h + base)[v] = bn_pack(w);
        }
      }
    }
    team_sync<WPR>(team_in_cta);  // every thread has read the stage
    if (tid == 0) ring.issue(k + kBnStages);
  }
  if (*abort_flag && tid == 0)  // copies in flight land before the shared memory goes away
    for (int u = max(0, k - kBnStages); u < k; ++u) ring.wait(u, nullptr, 942);
}

// ---------------------------------------------------------------- backward
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
  float* part_post;             // [n_ctas, cols]
  float* part_pre;              // [n_ctas, cols]
  float* part_gate;             // [n_teams, 2, cols]
  int rows, cols, rows_per_gate;
  int cyclic;  // teams take rows in turn; 0: contiguous rows
  float eps, residual_scale, branch_scale;
  DropoutParams drop;
};

// The column sums need one product a row and element: with c = sum over a
// gate row's rows of dv f r_f, the gate's gradient is w_post c, and c times
// the gate's row adds to dw_post.
template <int WPR, int VPT, bool ALL>
__global__ void __launch_bounds__(bn_warps(WPR) * 32, WPR <= 8 ? 2 : 1)
    block_norm_bwd_kernel(const BlockNormBwdParams p, const BlockNormTeams tm) {
  constexpr int TT = WPR * 32, TEAMS = bn_teams(WPR);
  extern __shared__ uint4 bn_stages[];
  __shared__ float red[2][kBnRed];
  __shared__ uint4 zero_cell;
  __shared__ uint64_t bars[8 * kBnStages];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int team_in_cta = (int)threadIdx.x / TT, tid = (int)threadIdx.x % TT;
  const int team = (int)blockIdx.x * TEAMS + team_in_cta;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 8 * kBnStages; ++i) mbar_init(smem_u32(bars + i), 1);
    abort_word = 0;
    zero_cell = make_uint4(0, 0, 0, 0);
    fence_mbar_init();
  }
  __syncthreads();
  pdl_launch_dependents();  // (the sums behind this kernel wait for it themselves)
  const int nvec = p.cols / 8;
  const bool branch = ALL || p.df, post = ALL || p.w_post, pre = ALL || p.w_pre;
  const bool has_f = ALL || (p.df && (p.w_post || p.gate)), has_dy = ALL || p.dy;
  const uint32_t zero = smem_u32(&zero_cell);
  auto lds = [&](uint32_t row, int i) {
    const int v = tid + i * TT;
    return bn_lds(v < nvec ? row + v * 16 : zero);
  };
  BnRing<4> ring;
  ring.src[0] = has_f ? p.f : nullptr;
  ring.src[1] = p.w_pre ? p.y : nullptr;
  ring.src[2] = p.dy;
  ring.src[3] = p.w_pre ? p.dh : nullptr;
  ring.present = (has_f ? 1 : 0) + (p.w_pre ? 2 : 0) + (p.dy ? 1 : 0);
  ring.cols = p.cols, ring.rows_per_stage = tm.rows_per_stage;
  // teams past the last have no rows
  const long long start = (long long)team * (p.cyclic ? tm.rows_per_stage : tm.rows_per_team);
  ring.row0 = team < tm.n_teams ? (int)start : p.rows;
  ring.row1 = p.cyclic ? p.rows : (int)min((long long)p.rows, (long long)ring.row0 + tm.rows_per_team);
  ring.step = p.cyclic ? (long long)tm.n_teams * tm.rows_per_stage : tm.rows_per_stage;
  ring.slot = (uint32_t)tm.rows_per_stage * p.cols * 2;
  ring.stage = 4 * ring.slot;
  ring.bar = smem_u32(bars + team_in_cta * kBnStages);
  ring.data = smem_u32(bn_stages) + team_in_cta * kBnStages * ring.stage;
  if (tid == 0)
    for (int k = 0; k < kBnStages; ++k) ring.issue(k);
  int buf = 0;
  PhiloxState rng = {};
  if (p.drop.rng) rng = philox_state(p.drop);
  const float inv_c = 1.0f / (float)p.cols;
  const uint64_t rs2 = f2_make(p.residual_scale, p.residual_scale);
  const float bs = p.branch_scale * (p.drop.rng ? p.drop.scale : 1.0f);
  const uint64_t bs2 = f2_make(bs, bs);

  uint64_t a_post[VPT][4], a_pre[VPT][4], a_c[VPT][4];
  uint64_t wg[VPT][4];  // gate * w_post
  uint4 wn[VPT];        // w_pre
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * TT;
    wn[i] = p.w_pre && v < nvec ? reinterpret_cast<const uint4*>(p.w_pre)[v] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) a_post[i][e] = a_pre[i][e] = a_c[i][e] = 0;
  }
  int gate_row = 0, seg_first = 0, seg_end = 0;  // this team's rows in the gate's row so far
  long long gate_end = 0;                        // the first row of the next gate row
  auto load_gate = [&](int row) {
    const int g = row / p.rows_per_gate;
    gate_row = g, seg_first = row;
    gate_end = ((long long)g + 1) * p.rows_per_gate;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * TT;
#pragma unroll
      for (int e = 0; e < 4; ++e) wg[i][e] = f2_make(1.0f, 1.0f);
      if (v >= nvec) continue;
      if (p.w_post) bn_unpack(reinterpret_cast<const uint4*>(p.w_post)[v], wg[i]);
      if (p.gate) {
        uint64_t g4[4];
        bn_unpack(reinterpret_cast<const uint4*>(p.gate + (long long)g * p.cols)[v], g4);
#pragma unroll
        for (int e = 0; e < 4; ++e) wg[i][e] = f2_mul(wg[i][e], g4[e]);
      }
    }
  };
  if (has_f && ring.row0 < ring.row1) load_gate(ring.row0);
  // Hands over the sums of a gate row's rows seg_first .. seg_end - 1.
  auto flush = [&]() {
    // (rows in turn with one gate for all: every team has a part of it)
    const bool whole = p.gate && (!p.cyclic || p.rows_per_gate == 1) &&
                       seg_first == (long long)gate_row * p.rows_per_gate && seg_end == gate_end;
    // a segment that starts at the team's first row goes to slot 0
    float* part = p.part_gate + ((long long)team * 2 + (seg_first == ring.row0 ? 0 : 1)) * p.cols;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * TT;
      if (v < nvec) {
        uint64_t c4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) c4[e] = a_c[i][e];
        if (p.gate) {
          uint64_t g4[4], d4[4];
          bn_unpack(reinterpret_cast<const uint4*>(p.gate + (long long)gate_row * p.cols)[v], g4);
#pragma unroll
          for (int e = 0; e < 4; ++e) d4[e] = c4[e];
          if (p.w_post) {
            uint64_t w4[4];
            bn_unpack(reinterpret_cast<const uint4*>(p.w_post)[v], w4);
#pragma unroll
            for (int e = 0; e < 4; ++e) d4[e] = f2_mul(d4[e], w4[e]);
          }
          if (whole)
            reinterpret_cast<uint4*>(p.dgate + (long long)gate_row * p.cols)[v] = bn_pack(d4);
          else
            bn_store_f32(part, v, d4);
#pragma unroll
          for (int e = 0; e < 4; ++e) c4[e] = f2_mul(c4[e], g4[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) a_post[i][e] = f2_add(a_post[i][e], c4[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) a_c[i][e] = 0;
    }
  };

  int k = 0;
  for (long long r = ring.row0; r < ring.row1; r += ring.step, ++k) {
    ring.wait(k, abort_flag, 943);
    const int here = (int)min((long long)tm.rows_per_stage, ring.row1 - r);
    for (int j = 0; j < here; ++j) {
      const int row = (int)r + j;
      const long long base = (long long)row * p.cols;
      const uint32_t fa = ring.at(k, 0, j), ya = ring.at(k, 1, j), ga = ring.at(k, 2, j),
                     ha = ring.at(k, 3, j);
      if (p.gate && has_f && row >= gate_end) {
        flush();
        load_gate(row);
      }
      seg_end = row + 1;
      float s3[3];  // y^2, dh w_pre y, f^2
      {
        uint64_t a0 = 0, a1 = 0, a2 = 0;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          if (pre) {
            uint64_t y4[4], d4[4], w4[4];
            bn_unpack(lds(ya, i), y4);
            bn_unpack(lds(ha, i), d4);
            bn_unpack(wn[i], w4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              a0 = f2_fma(y4[e], y4[e], a0);
              a1 = f2_fma(f2_mul(d4[e], w4[e]), y4[e], a1);
            }
          }
          if (has_f && post) {
            uint64_t f4[4];
            bn_unpack(lds(fa, i), f4);
#pragma unroll
            for (int e = 0; e < 4; ++e) a2 = f2_fma(f4[e], f4[e], a2);
          }
        }
        s3[0] = bn_hsum(a0), s3[1] = bn_hsum(a1), s3[2] = bn_hsum(a2);
      }
      if (pre || post) team_sum<WPR, 3>(s3, red, buf, team_in_cta, tid >> 5);
      const float r_y = rsqrtf(s3[0] * inv_c + p.eps);
      const float m_y = -(s3[1] * inv_c) * r_y * r_y * r_y;  // -r_y^3 mean(dh w_pre y)
      const float r_f = post ? rsqrtf(s3[2] * inv_c + p.eps) : 1.0f;
      const uint64_t ry2 = f2_make(r_y, r_y), my2 = f2_make(m_y, m_y), rf2 = f2_make(r_f, r_f);
      uint64_t q[VPT][4], s1p = 0;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = tid + i * TT;
        uint64_t t[4] = {0, 0, 0, 0};
        if (has_dy) bn_unpack(lds(ga, i), t);
        if (pre) {
          uint64_t y4[4], d4[4], w4[4];
          bn_unpack(lds(ya, i), y4);
          bn_unpack(lds(ha, i), d4);
          bn_unpack(wn[i], w4);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint64_t dr = f2_mul(d4[e], ry2);
            a_pre[i][e] = f2_fma(dr, y4[e], a_pre[i][e]);
            t[e] = f2_fma(dr, w4[e], f2_fma(y4[e], my2, t[e]));
          }
        }
        if (branch) {
          uint64_t b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) b[e] = f2_mul(t[e], bs2);
          if (p.drop.rng) bn_select(p.drop, rng, (uint32_t)(base / 8 + v), b);
          if (has_f) {
            uint64_t n[4];
            bn_unpack(lds(fa, i), n);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              n[e] = f2_mul(n[e], rf2);
              a_c[i][e] = f2_fma(b[e], n[e], a_c[i][e]);
              b[e] = f2_mul(b[e], wg[i][e]);
              s1p = f2_fma(b[e], n[e], s1p);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) q[i][e] = b[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = f2_mul(t[e], rs2);
        if (v < nvec) reinterpret_cast<uint4*>(p.dx + base)[v] = bn_pack(t);
      }
      if (branch) {
        if (post) {
          float s1[1] = {bn_hsum(s1p)};
          team_sum<WPR, 1>(s1, red, buf, team_in_cta, tid >> 5);
          const float m_f = -(s1[0] * inv_c) * r_f * r_f;  // -r_f mean(q w_post n), times r_f f
          const uint64_t mf2 = f2_make(m_f, m_f);
#pragma unroll
          for (int i = 0; i < VPT; ++i) {
            uint64_t f4[4];
            bn_unpack(lds(fa, i), f4);
#pragma unroll
            for (int e = 0; e < 4; ++e) q[i][e] = f2_fma(q[i][e], rf2, f2_mul(f4[e], mf2));
          }
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i)
          if (tid + i * TT < nvec)
            reinterpret_cast<uint4*>(p.df + base)[tid + i * TT] = bn_pack(q[i]);
      }
    }
    team_sync<WPR>(team_in_cta);  // every thread has read the stage
    if (tid == 0) ring.issue(k + kBnStages);
  }
  if (*abort_flag && tid == 0)  // copies in flight land before the shared memory goes away
    for (int u = max(0, k - kBnStages); u < k; ++u) ring.wait(u, nullptr, 944);
  if (has_f && ring.row0 < ring.row1) flush();

  // the weights' sums: the CTA's teams joined in order through the (idle) stages
  if constexpr (TEAMS > 1) {
    float* sums = reinterpret_cast<float*>(bn_stages);  // [TEAMS][cols]
    for (int which = 0; which < 2; ++which) {
      if (which == 0 ? !(p.df && p.w_post) : !p.w_pre) continue;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = tid + i * TT;
        if (v < nvec)
          bn_store_f32(sums + (long long)team_in_cta * p.cols, v, which == 0 ? a_post[i] : a_pre[i]);
      }
      __syncthreads();
      float* dst = (which == 0 ? p.part_post : p.part_pre) + (long long)blockIdx.x * p.cols;
      for (int c = threadIdx.x; c < p.cols; c += TEAMS * TT) {
        float t = sums[c];
#pragma unroll
        for (int w = 1; w < TEAMS; ++w) t += sums[w * p.cols + c];
        dst[c] = t;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * TT;
      if (v < nvec) {
        if (p.df && p.w_post) bn_store_f32(p.part_post + (long long)blockIdx.x * p.cols, v, a_post[i]);
        if (p.w_pre) bn_store_f32(p.part_pre + (long long)blockIdx.x * p.cols, v, a_pre[i]);
      }
    }
  }
}

// Sums the partials: output 0 is dw_post, 1 is dw_pre (a partial a CTA), 2 + g
// the gate's row g where more than one team has rows of it (a partial a team).
// 64 columns a block, four a thread; each of 32 groups of 16 threads takes every
// 32nd partial, and the groups' sums are joined in order.  Bound by the latency of
// a thread's loads: with 128 columns a block, and so twice as many, 4096 x 4096
// takes 51.1 us for 49.4 and 1037 x 1000 10.4 for 9.5.
constexpr int kBnSumThreads = 512;
constexpr int kBnSumCols = 64;
struct BlockNormSumParams {
  const float* part_post;
  const float* part_pre;
  const float* part_gate;
  __nv_bfloat16* dw_post;
  __nv_bfloat16* dw_pre;
  __nv_bfloat16* dgate;  // null: no gate, or every gate row is one team's
  int cols, n_ctas, rows_per_team, rows_per_gate, gate_rows;
};

__global__ void __launch_bounds__(kBnSumThreads)
    block_norm_sum_kernel(const BlockNormSumParams p) {
  constexpr int LANES = kBnSumCols / 4, PARTS = kBnSumThreads / LANES;
  __shared__ float4 s[PARTS][LANES];
  const int lane = threadIdx.x % LANES, part = threadIdx.x / LANES;
  const int col = (int)blockIdx.x * kBnSumCols + lane * 4;
  const int outs = 2 + (p.dgate ? p.gate_rows : 0);
  pdl_wait();
  for (int o = blockIdx.y; o < outs; o += gridDim.y) {
    const float* src;
    __nv_bfloat16* dst;
    int t0 = 0, t1 = p.n_ctas - 1, inside = -1;
    long long step = p.cols;
    const int g = o - 2;
    if (o == 0) {
      src = p.part_post, dst = p.dw_post;
    } else if (o == 1) {
      src = p.part_pre, dst = p.dw_pre;
    } else {
      // a team's slot 0, or 1 where the gate row starts inside its rows: only
      // the first team can have that
      const long long row = (long long)g * p.rows_per_gate;
      src = p.part_gate, dst = p.dgate + (long long)g * p.cols;
      step = 2LL * p.cols;
      t0 = (int)(row / p.rows_per_team);
      t1 = (int)((row + p.rows_per_gate - 1) / p.rows_per_team);
      if (row > (long long)t0 * p.rows_per_team) inside = t0;
      if (t0 == t1) dst = nullptr;  // written whole by its team
    }
    if (!dst) continue;  // the same for every thread of the block
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (col < p.cols) {
      const float* at = src + col;
#pragma unroll 8
      for (int t = t0 + part; t <= t1; t += PARTS) {
        const float4 v =
            *reinterpret_cast<const float4*>(at + t * step + (t == inside ? p.cols : 0));
        acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
      }
    }
    s[part][lane] = acc;
    __syncthreads();
    const int c = (int)blockIdx.x * kBnSumCols + (int)threadIdx.x;
    if (threadIdx.x < kBnSumCols && c < p.cols) {
      const float* f = reinterpret_cast<const float*>(s) + threadIdx.x;
      float v = f[0];
#pragma unroll
      for (int w = 1; w < PARTS; ++w) v += f[w * kBnSumCols];
      dst[c] = __float2bfloat16_rn(v);
    }
    __syncthreads();
  }
}

}  // namespace tfb
