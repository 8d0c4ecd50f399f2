// ssm_conv.hpp — the short causal depthwise convolution of a selective state
// space block, channels last, for MI355X (gfx950, wave64).
//
//   p[b,t,h] = bias[h] + sum_{j<K} w[h,j] x[b, t - (K-1) + j, h],  K <= 8
//   y = silu(p) or p;  y = 0 from the sequence's length on
// with x[b, -(K-1) .. -1] the state [B, K-1, H] of earlier tokens (or 0).
//
// Bound by HBM: 2 K + 5 FLOP for one element read and one written. A lane owns
// V neighbouring channels (16 bytes) and walks a run of tokens with the last
// K - 1 of them in registers, so each element is loaded once but for the K - 1
// before a run, which neighbouring runs share through L2.

#pragma once

#include "ssm_common.hpp"

namespace pt {

constexpr int kCausalMaxK = 8;
constexpr int kCausalThreads = 256;

struct CausalArgs {
  const void* x;      // [B, L, H], rows of H contiguous channels
  const float* w;     // [H, K]
  const float* bias;  // [H] or null
  const void* state;  // [B, K-1, H] or null
  const int* lengths; // [B] or null
  void* y;            // [B, L, H] contiguous
  void* state_out;    // [B, K-1, H] or null
  long long x_batch, x_row;  // strides of x in elements
  int B, L, H, silu;
  int run, nruns;     // tokens of a run, runs of a sequence
  int cols;           // lanes that cover a row: ceil(H / V)
};

// A lane's channels at `p`: V of them, or its one.
template <int V, typename T>
__device__ __forceinline__ void load_cols(const T* p, float (&v)[V]) {
  if constexpr (V == 1)
    v[0] = load1(p);
  else
    load_vec<V>(p, v);
}
template <int V, typename T>
__device__ __forceinline__ void store_cols(T* p, const float (&v)[V]) {
  if constexpr (V == 1)
    store1(p, v[0]);
  else
    store_vec<V>(p, v);
}

// Lane `id` of the grid: its first channel, sequence and run. Channels are
// fastest, so that a workgroup's lanes read whole rows.
struct CausalPlace {
  int h, b, r;
};
__device__ __forceinline__ bool causal_place(long long id, const CausalArgs& a, int V,
                                             CausalPlace* o) {
  const long long row = id / a.cols;
  if (row >= (long long)a.B * a.nruns) return false;
  o->h = (int)(id - row * a.cols) * V;
  o->b = (int)(row / a.nruns);
  o->r = (int)(row - (long long)o->b * a.nruns);
  return true;
}

__device__ __forceinline__ int clamped_length(const int* lengths, int b, int L) {
  if (!lengths) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : n < L ? n : L;
}

// The token `t` of a sequence (its state's for t < 0) at channels h .. h + V - 1.
template <typename T, int V, int K>
__device__ __forceinline__ void load_token(const CausalArgs& a, const T* xb, int b, int h, int t,
                                           float (&v)[V]) {
  if (t >= 0) {
    load_cols<V>(xb + (long long)t * a.x_row + h, v);
  } else if (a.state) {
    load_cols<V>(static_cast<const T*>(a.state) + ((long long)b * (K - 1) + (K - 1) + t) * a.H + h, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.0f;
  }
}

template <typename T, int V, int K>
__global__ __launch_bounds__(kCausalThreads) void causal_fwd_kernel(CausalArgs a) {
  CausalPlace at;
  if (!causal_place((long long)blockIdx.x * kCausalThreads + threadIdx.x, a, V, &at)) return;
  const int len = clamped_length(a.lengths, at.b, a.L);
  const T* xb = static_cast<const T*>(a.x) + (long long)at.b * a.x_batch;
  T* yb = static_cast<T*>(a.y) + (long long)at.b * a.L * a.H + at.h;
  const int t0 = at.r * a.run, t1 = t0 + a.run < a.L ? t0 + a.run : a.L;
  const int te = t1 < len ? t1 : len;  // tokens from te on are past the sequence's end

  // The run that the sequence ends in writes the state: the last K - 1 tokens.
  if (K > 1 && a.state_out && at.r == (len > 0 ? (len - 1) / a.run : 0)) {
    T* so = static_cast<T*>(a.state_out) + (long long)at.b * (K - 1) * a.H + at.h;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      float v[V];
      load_token<T, V, K>(a, xb, at.b, at.h, len - (K - 1) + j, v);
      store_cols<V>(so + (long long)j * a.H, v);
    }
  }

  float w[K][V], bias[V], win[K][V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias ? a.bias[at.h + i] : 0.0f;
#pragma unroll
    for (int j = 0; j < K; ++j) w[j][i] = a.w[(long long)(at.h + i) * K + j];
  }
  if (t0 < te) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) load_token<T, V, K>(a, xb, at.b, at.h, t0 - (K - 1) + j, win[j]);
  }
  const T* xp = xb + (long long)t0 * a.x_row + at.h;
  for (int t = t0; t < te; ++t, xp += a.x_row) {
    load_cols<V>(xp, win[K - 1]);
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float p = bias[i];
#pragma unroll
      for (int j = 0; j < K; ++j) p = fmaf(w[j][i], win[j][i], p);
      y[i] = a.silu ? p * sigmoid_f32(p) : p;
#pragma unroll
      for (int j = 0; j + 1 < K; ++j) win[j][i] = win[j + 1][i];
    }
    store_cols<V>(yb + (long long)t * a.H, y);
  }
  float zero[V] = {};
  for (int t = te > t0 ? te : t0; t < t1; ++t) store_cols<V>(yb + (long long)t * a.H, zero);
}

struct CausalGradArgs {
  CausalArgs f;       // y and state_out unused
  const void* gy;     // [B, L, H] contiguous
  const void* gstate; // gradient of the final state [B, K-1, H], or null
  void* gx;           // [B, L, H] contiguous
  void* gstate_in;    // gradient of the initial state [B, K-1, H], or null
  float* part;        // [B nruns][H][K + 1]: sums of dw and dbias of a run
};

// Backward. With dp = gy silu'(p) at the sequence's tokens and 0 elsewhere:
//   gx[t] = sum_j w[j] dp[t + (K-1) - j],  dw[j] = sum dp[t] x[t-(K-1)+j].
// A run walks its tokens and K - 1 further ones, with windows of x and of dp;
// it sums dw over its own tokens alone, and writes gx K - 1 tokens behind. The
// first run also writes the initial state's gradient, gx at t < 0. A final
// state's gradient adds to gx at the last K - 1 tokens.
template <typename T, int V, int K>
__global__ __launch_bounds__(kCausalThreads) void causal_bwd_kernel(CausalGradArgs g) {
  const CausalArgs& a = g.f;
  CausalPlace at;
  if (!causal_place((long long)blockIdx.x * kCausalThreads + threadIdx.x, a, V, &at)) return;
  const int len = clamped_length(a.lengths, at.b, a.L);
  const T* xb = static_cast<const T*>(a.x) + (long long)at.b * a.x_batch;
  const T* gyb = static_cast<const T*>(g.gy) + (long long)at.b * a.L * a.H + at.h;
  const T* gsb = static_cast<const T*>(g.gstate) + (long long)at.b * (K - 1) * a.H + at.h;
  T* gxb = static_cast<T*>(g.gx) + (long long)at.b * a.L * a.H + at.h;
  T* gib = static_cast<T*>(g.gstate_in) + (long long)at.b * (K - 1) * a.H + at.h;
  const int t0 = at.r * a.run, t1 = t0 + a.run < a.L ? t0 + a.run : a.L;

  float w[K][V], bias[V], win[K][V], dp[K][V], dw[K][V] = {}, db[V] = {};
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias ? a.bias[at.h + i] : 0.0f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      w[j][i] = a.w[(long long)(at.h + i) * K + j];
      dp[j][i] = win[j][i] = 0.0f;
    }
  }
  // The first run starts K - 1 tokens early, where dp is 0: the gradients of
  // the state's tokens come out there.
  const int first = at.r == 0 && K > 1 ? t0 - (K - 1) : t0;
  if (t0 < len) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) load_token<T, V, K>(a, xb, at.b, at.h, t0 - (K - 1) + j, win[j]);
  }
  for (int t = t0; t < t1 + K - 1; ++t) {
#pragma unroll
    for (int j = 0; j + 1 < K; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) dp[j][i] = dp[j + 1][i];
    if (t < len) {
      float gy[V];
      load_cols<V>(xb + (long long)t * a.x_row + at.h, win[K - 1]);
      load_cols<V>(gyb + (long long)t * a.H, gy);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float d = gy[i];
        if (a.silu) {
          float p = bias[i];
#pragma unroll
          for (int j = 0; j < K; ++j) p = fmaf(w[j][i], win[j][i], p);
          d *= silu_grad_f32(p, sigmoid_f32(p));
        }
        dp[K - 1][i] = d;
        if (t < t1) {
          db[i] += d;
#pragma unroll
          for (int j = 0; j < K; ++j) dw[j][i] = fmaf(d, win[j][i], dw[j][i]);
        }
#pragma unroll
        for (int j = 0; j + 1 < K; ++j) win[j][i] = win[j + 1][i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) dp[K - 1][i] = 0.0f;
    }
    const int s = t - (K - 1);  // dp holds tokens s .. t
    if (s < first) continue;
    float out[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      out[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < K; ++j) out[i] = fmaf(w[j][i], dp[K - 1 - j][i], out[i]);
    }
    if (K > 1 && g.gstate && s >= len - (K - 1) && s < len) {
      float v[V];
      load_cols<V>(gsb + (long long)(s - (len - (K - 1))) * a.H, v);
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] += v[i];
    }
    if (s >= 0)
      store_cols<V>(gxb + (long long)s * a.H, out);
    else if (g.gstate_in)
      store_cols<V>(gib + (long long)(s + K - 1) * a.H, out);
  }
  float* part = g.part + (((long long)at.b * a.nruns + at.r) * a.H + at.h) * (K + 1);
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j < K; ++j) part[i * (K + 1) + j] = dw[j][i];
    part[i * (K + 1) + K] = db[i];
  }
}

// One token of each of B sequences: the pool's states shift by it in place.
// slots (null: sequence b has state b): a slot outside the pool marks a row
// without a sequence, whose y is 0.
template <typename T, int V, int K>
__global__ __launch_bounds__(kCausalThreads) void causal_step_kernel(
    const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ bias,
    T* __restrict__ state, const int* __restrict__ slots, T* __restrict__ y, long long x_row,
    int B, int H, int pool, int silu, int cols) {
  const long long id = (long long)blockIdx.x * kCausalThreads + threadIdx.x;
  const int b = (int)(id / cols), h = (int)(id - (long long)b * cols) * V;
  if (b >= B) return;
  const int s = slots ? slots[b] : b;
  float out[V] = {};
  if (s >= 0 && s < pool) {
    T* sp = state + (long long)s * (K - 1) * H + h;
    float win[K][V];
#pragma unroll
    for (int j = 0; j + 1 < K; ++j) load_cols<V>(sp + (long long)j * H, win[j]);
    load_cols<V>(x + (long long)b * x_row + h, win[K - 1]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float p = bias ? bias[h + i] : 0.0f;
#pragma unroll
      for (int j = 0; j < K; ++j) p = fmaf(w[(long long)(h + i) * K + j], win[j][i], p);
      out[i] = silu ? p * sigmoid_f32(p) : p;
    }
#pragma unroll
    for (int j = 0; j + 1 < K; ++j) store_cols<V>(sp + (long long)j * H, win[j + 1]);
  }
  store_cols<V>(y + (long long)b * H + h, out);
}

}  // namespace pt
