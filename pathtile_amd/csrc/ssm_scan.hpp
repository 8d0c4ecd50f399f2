// ssm_scan.hpp — the selective state space scan, channels last, for MI355X
// (gfx950, wave64).
//
//   v = dt + dt_bias,  d = softplus(v) or v
//   s[n] <- exp(d A[h,n]) s[n] + d x B[n],   y = sum_n C[n] s[n] + D x
// for each sequence b and channel h, over its tokens; B and C belong to a
// token and a group of channels, states are FP32.
//
// A workgroup owns 64 channels of one sequence, a lane each; its four waves
// share the channels and split the states, so that B and C are the same for
// all lanes of a wave and come through the scalar cache. Tokens go by tiles of
// 16: every thread loads four channels of one token and puts d and d x into
// LDS, the waves run the recurrence on them, and the same threads add the four
// waves' parts of y.

#pragma once

#include "ssm_common.hpp"

namespace pt {

constexpr int kScanTile = 16;      // tokens between two barriers, and between two saved states
constexpr int kScanCh = 64;        // channels of a workgroup
constexpr int kScanWaves = 4;
constexpr int kScanThreads = 256;
constexpr int kScanMaxN = 64;

struct ScanArgs {
  const void *x, *dt;           // [B, L, H]
  const void *bm, *cm;          // B, C: [B, L, G, N]
  long long x_batch, x_row, dt_batch, dt_row;  // strides in elements
  long long b_batch, b_row, c_batch, c_row;
  int b_group, c_group;
  const float *a, *d, *dt_bias; // [H, N]; [H] or null
  const float* state;           // [B, H, N] or null
  const int* lengths;           // [B] or null
  int B, L, H, N, G, softplus;
  int hg, blocks_g;             // channels of a group; workgroups that cover them
  int np;                       // N rounded up to what the kernels hold
  int ntiles;                   // tiles of a sequence
};

__device__ __forceinline__ int scan_length(const ScanArgs& a, int b) {
  if (!a.lengths) return a.L;
  const int n = a.lengths[b];
  return n < 0 ? 0 : n < a.L ? n : a.L;
}

// softplus(v) = log(1 + e^v) and its derivative. log(u) e / (u - 1) with the
// rounded u = 1 + e keeps the result's relative precision at small e, where
// log(u) alone would lose it.
__device__ __forceinline__ float softplus_f32(float v, float* grad) {
  const float e = exp_f32(v > 20.0f ? 20.0f : v), u = 1.0f + e;  // a NaN stays one
  const float l = __builtin_amdgcn_logf(u) * kLn2;
  *grad = v > 20.0f ? 1.0f : e * __builtin_amdgcn_rcpf(u);
  return v > 20.0f ? v : u == 1.0f ? e : l * (e * __builtin_amdgcn_rcpf(u - 1.0f));
}

// N values that all lanes share, through the scalar cache.
typedef const __attribute__((address_space(4))) uint32_t* scalar_ptr;
template <int NS>
__device__ __forceinline__ void load_uniform(const float* p, float (&v)[NS]) {
  scalar_ptr q = (scalar_ptr)(uintptr_t)p;
#pragma unroll
  for (int i = 0; i < NS; ++i) v[i] = __uint_as_float(q[i]);
}
template <int NS>
__device__ __forceinline__ void load_uniform(const __bf16* p, float (&v)[NS]) {
  scalar_ptr q = (scalar_ptr)(uintptr_t)p;
#pragma unroll
  for (int i = 0; i < NS; i += 2) {
    const uint32_t u = q[i / 2];
    v[i] = bf16_lo(u), v[i + 1] = bf16_hi(u);
  }
}

// Four channels of one token, those below `n` (0 elsewhere).
template <bool VEC, typename T>
__device__ __forceinline__ void load_four(const T* p, int n, float (&v)[4]) {
  if constexpr (VEC) {
    if (n > 0) {
      load_vec<4>(p, v);
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 0.0f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? load1(p + i) : 0.0f;
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store_four(T* p, int n, const float (&v)[4]) {
  if constexpr (VEC) {
    if (n > 0) store_vec<4>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) store1(p + i, v[i]);
  }
}

// B and C as FP32 [B, L, G, 2, np], zeros from state N on: for layouts that
// the scalar loads cannot take as they are.
template <typename T>
__global__ __launch_bounds__(256) void scan_bc_kernel(ScanArgs a, float* __restrict__ out) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = id / (2 * a.np);  // (b L + t) G + g
  if (row >= (long long)a.B * a.L * a.G) return;
  const int r = (int)(id - row * 2 * a.np), half = r / a.np, n = r - half * a.np;
  const int g = (int)(row % a.G);
  const long long bt = row / a.G;
  const long long b = bt / a.L, t = bt - b * a.L;
  float v = 0.0f;
  if (n < a.N)
    v = half ? load1(static_cast<const T*>(a.cm) + b * a.c_batch + t * a.c_row + (long long)g * a.c_group + n)
             : load1(static_cast<const T*>(a.bm) + b * a.b_batch + t * a.b_row + (long long)g * a.b_group + n);
  out[id] = v;
}

// Where a workgroup works: blocks of channels are fastest.
struct ScanPlace {
  int blk, g, h0, nh, b;  // block, group, first channel, channels, sequence
};
__device__ __forceinline__ ScanPlace scan_place(const ScanArgs& a, uint32_t id) {
  ScanPlace p;
  const int blocks = a.blocks_g * a.G;
  p.b = (int)(id / (uint32_t)blocks);
  p.blk = (int)(id - (uint32_t)p.b * blocks);
  p.g = p.blk / a.blocks_g;
  const int k = p.blk - p.g * a.blocks_g;
  p.h0 = p.g * a.hg + k * kScanCh;
  p.nh = a.hg - k * kScanCh < kScanCh ? a.hg - k * kScanCh : kScanCh;
  return p;
}

struct ScanFwdArgs {
  ScanArgs s;
  void* y;           // [B, L, H] contiguous
  float* state_out;  // [B, H, N] or null
  float* saved;      // [B, ntiles, np, H]: the state before each tile, or null
};

template <typename T, typename BCT, int NS, bool VEC>
__global__ __launch_bounds__(kScanThreads) void scan_fwd_kernel(ScanFwdArgs f) {
  __shared__ float2 du[2][kScanTile][kScanCh];
  __shared__ float yp[2][kScanWaves][kScanTile][kScanCh];
  const ScanArgs& a = f.s;
  const ScanPlace p = scan_place(a, blockIdx.x);
  const int len = scan_length(a, p.b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool mine = lane < p.nh;
  const int h = p.h0 + lane, n0 = wave * NS;

  float a2[NS], s[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const bool in = mine && n0 + i < a.N;
    a2[i] = in ? a.a[(long long)h * a.N + n0 + i] * kLog2E : 0.0f;
    s[i] = in && a.state ? a.state[((long long)p.b * a.H + h) * a.N + n0 + i] : 0.0f;
  }

  // Loading and storing: token tid / 16 of a tile, four channels.
  const int row = tid >> 4, c0 = (tid & 15) * 4, cn = p.nh - c0;
  const T* xp = static_cast<const T*>(a.x) + (long long)p.b * a.x_batch + p.h0 + c0;
  const T* dp = static_cast<const T*>(a.dt) + (long long)p.b * a.dt_batch + p.h0 + c0;
  T* yo = static_cast<T*>(f.y) + (long long)p.b * a.L * a.H + p.h0 + c0;
  float bias[4], dskip[4], xv[4], dv[4], xk[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bias[i] = a.dt_bias && i < cn ? a.dt_bias[p.h0 + c0 + i] : 0.0f;
    dskip[i] = a.d && i < cn ? a.d[p.h0 + c0 + i] : 0.0f;
  }
  auto fetch = [&](int tile) {
    const int t = tile * kScanTile + row;
    const int n = t < len ? cn : 0;
    load_four<VEC>(xp + (n > 0 ? t * a.x_row : 0), n, xv);
    load_four<VEC>(dp + (n > 0 ? t * a.dt_row : 0), n, dv);
  };
  auto put = [&](int tile) {
    const bool in = tile * kScanTile + row < len;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float g, d = dv[i] + bias[i];
      if (a.softplus) d = softplus_f32(d, &g);
      xk[i] = xv[i];
      du[tile & 1][row][c0 + i] = in ? make_float2(d, d * xv[i]) : make_float2(0.0f, 0.0f);
    }
  };

  const int tiles = (len + kScanTile - 1) / kScanTile;
  const BCT* bp = static_cast<const BCT*>(a.bm) + p.b * a.b_batch + (long long)p.g * a.b_group + n0;
  const BCT* cp = static_cast<const BCT*>(a.cm) + p.b * a.c_batch + (long long)p.g * a.c_group + n0;
  if (tiles > 0) {
    fetch(0);
    put(0);
    if (tiles > 1) fetch(1);
  }
  __syncthreads();
  for (int tile = 0; tile < tiles; ++tile) {
    if (f.saved && mine) {
      float* sp = f.saved + (((long long)p.b * a.ntiles + tile) * a.np + n0) * a.H + h;
#pragma unroll
      for (int i = 0; i < NS; ++i) sp[(long long)i * a.H] = s[i];
    }
    const int count = len - tile * kScanTile < kScanTile ? len - tile * kScanTile : kScanTile;
    const int buf = tile & 1;
    auto step = [&](int t) {
      const float2 q = du[buf][t][lane];
      float bv[NS], cv[NS], y = 0.0f;
      load_uniform<NS>(bp, bv);
      load_uniform<NS>(cp, cv);
      bp += a.b_row, cp += a.c_row;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        s[i] = fmaf(__builtin_amdgcn_exp2f(q.x * a2[i]), s[i], q.y * bv[i]);
        y = fmaf(cv[i], s[i], y);
      }
      yp[buf][wave][t][lane] = y;
    };
    if (count == kScanTile) {
#pragma unroll 4
      for (int t = 0; t < kScanTile; ++t) step(t);
    } else {
      for (int t = 0; t < count; ++t) step(t);
    }
    float xr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) xr[i] = xk[i];
    if (tile + 1 < tiles) {
      put(tile + 1);
      if (tile + 2 < tiles) fetch(tile + 2);
    }
    __syncthreads();
    const int t = tile * kScanTile + row;
    if (t < a.L) {
      float out[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float y = dskip[i] * xr[i];
#pragma unroll
        for (int w = 0; w < kScanWaves; ++w) y += yp[buf][w][row][c0 + i];
        out[i] = row < count ? y : 0.0f;
      }
      store_four<VEC>(yo + (long long)t * a.H, cn, out);
    }
  }
  const float zero[4] = {};
  for (int t = tiles * kScanTile + row; t < a.L; t += kScanTile)
    store_four<VEC>(yo + (long long)t * a.H, cn, zero);
  if (f.state_out && mine) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (n0 + i < a.N) f.state_out[((long long)p.b * a.H + h) * a.N + n0 + i] = s[i];
  }
}

// ---------------------------------------------------------------------------
// Backward. With G the gradient of a state, a = exp(d A) and q = a G:
//   G_t = C_t gy_t + q_{t+1},  dC = sum_h gy s_t,  dB = sum_h G d x,
//   dx = D gy + d sum_n G B,   dd = x sum_n G B + sum_n q s_{t-1} A,
//   dA = sum_{b,t} q s_{t-1} d,  and q at the first token is the state's.
// A workgroup goes through its tiles from the last to the first. For each it
// runs the tile forward again from the state saved before it, with a and s of
// all 16 tokens in registers, then backward. Sums over the states go through
// LDS as y does; sums over the channels are butterflies over the lanes that
// halve the number of values at each level, so that a value costs about two
// instructions, and leave one (token, state) in each lane.
// ---------------------------------------------------------------------------
struct ScanBwdArgs {
  ScanArgs s;
  const void* gy;           // [B, L, H] contiguous
  const float* saved;       // of the forward
  const float* gstate_out;  // gradient of the final state [B, H, N], or null
  void *gx, *gdt;           // [B, L, H] contiguous
  float* gstate;            // [B, H, N] or null
  float* part_bc;           // [blocks][B][L][2][np]
  float* part_a;            // [B][np][H]
  float* part_d;            // [B][2][H]: dD, ddt_bias
};

typedef uint32_t u2s __attribute__((ext_vector_type(2)));
// (lanes 0-31: u + u of lanes 32-63; lanes 32-63: the same of v)
__device__ __forceinline__ float fold32(float u, float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(u), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// the same over rows of 16 lanes: even rows u, odd rows v
__device__ __forceinline__ float fold16(float u, float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(u), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// within rows: lanes whose `bit` is 0 u, the others v, each plus its partner's
template <int CTRL>
__device__ __forceinline__ float fold_row(float u, float v, bool bit) {
  const float keep = bit ? v : u, send = bit ? u : v;
  return keep + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(send), CTRL, 0xf, 0xf, true));
}
constexpr int kDppRor8 = 0x128, kDppHalfMirror = 0x141, kDppXor2 = 0x4e, kDppXor1 = 0xb1;

template <typename T, typename BCT, int R, bool VEC>
__global__ __launch_bounds__(kScanThreads) void scan_bwd_kernel(ScanBwdArgs f) {
  constexpr int NS = 4;  // states of a wave in a round; R rounds
  __shared__ float2 du[kScanTile][kScanCh];
  __shared__ float gys[kScanTile][kScanCh];
  __shared__ float p1[kScanWaves][kScanTile][kScanCh], p2[kScanWaves][kScanTile][kScanCh];
  const ScanArgs& a = f.s;
  const ScanPlace p = scan_place(a, blockIdx.x);
  const int len = scan_length(a, p.b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool mine = lane < p.nh;
  const int h = p.h0 + lane;

  float a2[R][NS], q[R][NS], ga[R][NS];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int n = (r * kScanWaves + wave) * NS + i;
      const bool in = mine && n < a.N;
      a2[r][i] = in ? a.a[(long long)h * a.N + n] * kLog2E : 0.0f;
      q[r][i] = in && f.gstate_out ? f.gstate_out[((long long)p.b * a.H + h) * a.N + n] : 0.0f;
      ga[r][i] = 0.0f;
    }

  const int row = tid >> 4, c0 = (tid & 15) * 4, cn = p.nh - c0;
  const T* xp = static_cast<const T*>(a.x) + (long long)p.b * a.x_batch + p.h0 + c0;
  const T* dp = static_cast<const T*>(a.dt) + (long long)p.b * a.dt_batch + p.h0 + c0;
  const long long yb = (long long)p.b * a.L * a.H + p.h0 + c0;
  const T* gp = static_cast<const T*>(f.gy) + yb;
  T* gxp = static_cast<T*>(f.gx) + yb;
  T* gdp = static_cast<T*>(f.gdt) + yb;
  float bias[4], dskip[4], gd[4] = {}, gbias[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bias[i] = a.dt_bias && i < cn ? a.dt_bias[p.h0 + c0 + i] : 0.0f;
    dskip[i] = a.d && i < cn ? a.d[p.h0 + c0 + i] : 0.0f;
  }
  const int tiles = (len + kScanTile - 1) / kScanTile;
  const float zero[4] = {};
  for (int t = tiles * kScanTile + row; t < a.L; t += kScanTile) {
    store_four<VEC>(gxp + (long long)t * a.H, cn, zero);
    store_four<VEC>(gdp + (long long)t * a.H, cn, zero);
  }
  float xv[4], dv[4], gv[4];
  auto fetch = [&](int tile) {
    const int t = tile * kScanTile + row;
    const int n = t < len ? cn : 0;
    load_four<VEC>(xp + (n > 0 ? t * a.x_row : 0), n, xv);
    load_four<VEC>(dp + (n > 0 ? t * a.dt_row : 0), n, dv);
    load_four<VEC>(gp + (n > 0 ? (long long)t * a.H : 0), n, gv);
  };
  if (tiles > 0) fetch(tiles - 1);
  for (int tile = tiles - 1; tile >= 0; --tile) {
    const int t0 = tile * kScanTile, count = len - t0 < kScanTile ? len - t0 : kScanTile;
    float x[4], d[4], sg[4], gy[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = xv[i], gy[i] = gv[i], sg[i] = 1.0f, d[i] = dv[i] + bias[i];
      if (a.softplus) d[i] = softplus_f32(d[i], &sg[i]);
      du[row][c0 + i] = row < count ? make_float2(d[i], d[i] * x[i]) : make_float2(0.0f, 0.0f);
      gys[row][c0 + i] = gy[i];
    }
    if (tile > 0) fetch(tile - 1);
    __syncthreads();
    float s1[R > 1 ? kScanTile : 1], s2[R > 1 ? kScanTile : 1];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int n0 = (r * kScanWaves + wave) * NS;
      const BCT* bp = static_cast<const BCT*>(a.bm) + p.b * a.b_batch + t0 * a.b_row +
                      (long long)p.g * a.b_group + n0;
      const BCT* cp = static_cast<const BCT*>(a.cm) + p.b * a.c_batch + t0 * a.c_row +
                      (long long)p.g * a.c_group + n0;
      const float* sp = f.saved + (((long long)p.b * a.ntiles + tile) * a.np + n0) * a.H + h;
      float s[kScanTile + 1][NS], e[kScanTile][NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) s[0][i] = mine ? sp[(long long)i * a.H] : 0.0f;
#pragma unroll
      for (int t = 0; t < kScanTile; ++t) {
        if (t < count) {
          const float2 w = du[t][lane];
          float bv[NS];
          load_uniform<NS>(bp + t * a.b_row, bv);
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            e[t][i] = __builtin_amdgcn_exp2f(w.x * a2[r][i]);
            s[t + 1][i] = fmaf(e[t][i], s[t][i], w.y * bv[i]);
          }
        }
      }
      float rb[kScanTile], rc[kScanTile], gat[NS] = {};
#pragma unroll
      for (int t = kScanTile - 1; t >= 0; --t) {
        rb[t] = rc[t] = 0.0f;
        if (t < count) {
          const float2 w = du[t][lane];
          const float gyt = gys[t][lane];
          float bv[NS], cv[NS], vb[NS], vc[NS], u1 = 0.0f, u2 = 0.0f;
          load_uniform<NS>(bp + t * a.b_row, bv);
          load_uniform<NS>(cp + t * a.c_row, cv);
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            const float g = fmaf(cv[i], gyt, q[r][i]);
            u1 = fmaf(g, bv[i], u1);
            vb[i] = g * w.y;
            vc[i] = gyt * s[t + 1][i];
            q[r][i] = g * e[t][i];
            const float k = q[r][i] * s[t][i];
            u2 = fmaf(k, a2[r][i], u2);
            gat[i] = fmaf(k, w.x, gat[i]);
          }
          rb[t] = fold16(fold32(vb[0], vb[2]), fold32(vb[1], vb[3]));
          rc[t] = fold16(fold32(vc[0], vc[2]), fold32(vc[1], vc[3]));
          if constexpr (R > 1) {
            s1[t] = r == 0 ? u1 : s1[t] + u1;
            s2[t] = r == 0 ? u2 : s2[t] + u2;
          }
          if (r == R - 1) {
            p1[wave][t][lane] = R > 1 ? s1[R > 1 ? t : 0] : u1;
            p2[wave][t][lane] = R > 1 ? s2[R > 1 ? t : 0] : u2;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NS; ++i) ga[r][i] += gat[i];
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        rb[t] = fold_row<kDppRor8>(rb[t], rb[t + 8], lane & 8);
        rc[t] = fold_row<kDppRor8>(rc[t], rc[t + 8], lane & 8);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        rb[t] = fold_row<kDppHalfMirror>(rb[t], rb[t + 4], lane & 4);
        rc[t] = fold_row<kDppHalfMirror>(rc[t], rc[t + 4], lane & 4);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        rb[t] = fold_row<kDppXor2>(rb[t], rb[t + 2], lane & 2);
        rc[t] = fold_row<kDppXor2>(rc[t], rc[t + 2], lane & 2);
      }
      rb[0] = fold_row<kDppXor1>(rb[0], rb[1], lane & 1);
      rc[0] = fold_row<kDppXor1>(rc[0], rc[1], lane & 1);
      // lane: token lane % 16, state lane / 16
      const int t = t0 + (lane & 15);
      if (t < len) {
        float* bc = f.part_bc + (((long long)p.blk * a.B + p.b) * a.L + t) * 2 * a.np + n0 + (lane >> 4);
        bc[0] = rb[0];
        bc[a.np] = rc[0];
      }
    }
    __syncthreads();
    const int t = t0 + row;
    if (t < a.L) {
      float ox[4], od[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float g1 = 0.0f, g2 = 0.0f;
#pragma unroll
        for (int w = 0; w < kScanWaves; ++w) g1 += p1[w][row][c0 + i], g2 += p2[w][row][c0 + i];
        ox[i] = od[i] = 0.0f;
        if (row < count) {
          ox[i] = fmaf(d[i], g1, dskip[i] * gy[i]);
          od[i] = fmaf(x[i], g1, kLn2 * g2) * sg[i];
          gd[i] = fmaf(gy[i], x[i], gd[i]);
          gbias[i] += od[i];
        }
      }
      store_four<VEC>(gxp + (long long)t * a.H, cn, ox);
      store_four<VEC>(gdp + (long long)t * a.H, cn, od);
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int n = (r * kScanWaves + wave) * NS + i;
      if (!mine) continue;
      f.part_a[((long long)p.b * a.np + n) * a.H + h] = ga[r][i];
      if (f.gstate && n < a.N) f.gstate[((long long)p.b * a.H + h) * a.N + n] = q[r][i];
    }
  // The sums over the tokens of a tile's rows.
  p1[0][row][c0] = gd[0], p1[0][row][c0 + 1] = gd[1], p1[0][row][c0 + 2] = gd[2], p1[0][row][c0 + 3] = gd[3];
  p2[0][row][c0] = gbias[0], p2[0][row][c0 + 1] = gbias[1], p2[0][row][c0 + 2] = gbias[2], p2[0][row][c0 + 3] = gbias[3];
  __syncthreads();
  if (tid < 2 * kScanCh && mine) {
    float v = 0.0f;
    for (int t = 0; t < kScanTile; ++t) v += wave ? p2[0][t][lane] : p1[0][t][lane];
    f.part_d[((long long)p.b * 2 + wave) * a.H + h] = v;
  }
}

// gB, gC [B, L, G, N] from the blocks' parts.
template <typename T>
__global__ __launch_bounds__(256) void scan_bc_reduce_kernel(ScanArgs a, const float* __restrict__ part,
                                                             T* __restrict__ gb, T* __restrict__ gc) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = id / (2 * a.np);  // (b L + t) G + g
  if (row >= (long long)a.B * a.L * a.G) return;
  const int r = (int)(id - row * 2 * a.np), half = r / a.np, n = r - half * a.np;
  if (n >= a.N) return;
  const int g = (int)(row % a.G);
  const long long bt = row / a.G;
  const int b = (int)(bt / a.L), t = (int)(bt - (long long)b * a.L);
  float v = 0.0f;
  if (t < scan_length(a, b)) {
    const float* q = part + ((long long)g * a.blocks_g * a.B * a.L + bt) * 2 * a.np + r;
    for (int k = 0; k < a.blocks_g; ++k, q += (long long)a.B * a.L * 2 * a.np) v += *q;
  }
  store1((half ? gc : gb) + row * a.N + n, v);
}

// One token of each of B sequences, states of a pool updated in place. PER
// lanes share a channel, four states each. slots as in the convolution's step.
template <typename T, int PER, bool VEC>
__global__ __launch_bounds__(256) void scan_step_kernel(
    const T* __restrict__ x, const T* __restrict__ dt, const float* __restrict__ A,
    const T* __restrict__ bm, const T* __restrict__ cm, float* __restrict__ state,
    const float* __restrict__ dskip, const float* __restrict__ dt_bias,
    const int* __restrict__ slots, T* __restrict__ y, long long x_row, long long dt_row,
    long long b_row, long long c_row, int b_group, int c_group, int B, int H, int N, int G, int pool,
    int softplus, int blocks) {
  const int b = (int)(blockIdx.x / (uint32_t)blocks);
  const int h = (int)(blockIdx.x - (uint32_t)b * blocks) * (256 / PER) + (int)threadIdx.x / PER;
  const int n0 = ((int)threadIdx.x & (PER - 1)) * 4;
  if (h >= H) return;  // all lanes of a channel together
  const int slot = slots ? slots[b] : b;
  if (slot < 0 || slot >= pool) {
    if (n0 == 0) store1(y + (long long)b * H + h, 0.0f);
    return;
  }
  const int g = h / (H / G);
  const float xv = load1(x + b * x_row + h);
  float d = load1(dt + b * dt_row + h) + (dt_bias ? dt_bias[h] : 0.0f), grad;
  if (softplus) d = softplus_f32(d, &grad);
  const float* ap = A + (long long)h * N + n0;
  float* sp = state + ((long long)slot * H + h) * N + n0;
  const T* bp = bm + b * b_row + (long long)g * b_group + n0;
  const T* cp = cm + b * c_row + (long long)g * c_group + n0;
  float s[4], av[4], bv[4], cv[4], out = 0.0f;
  load_four<VEC>(sp, N - n0, s);
  load_four<VEC>(ap, N - n0, av);
  load_four<VEC>(bp, N - n0, bv);
  load_four<VEC>(cp, N - n0, cv);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[i] = fmaf(__builtin_amdgcn_exp2f(d * (av[i] * kLog2E)), s[i], d * xv * bv[i]);
    out = fmaf(cv[i], s[i], out);
  }
  store_four<VEC>(sp, N - n0, s);
#pragma unroll
  for (int k = 1; k < PER; k *= 2) out += __shfl_xor(out, k);
  if (n0 == 0) store1(y + (long long)b * H + h, fmaf(dskip ? dskip[h] : 0.0f, xv, out));
}

}  // namespace pt
