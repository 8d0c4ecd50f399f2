// ssm_conv.hip — entry points of the short causal convolution.

#include "ssm_conv.hpp"
#include "ssm_host.hpp"

namespace pt {

// The causal_*_kernel of (type, vector or single channels, taps, silu), vectors
// of VB BF16 or four FP32.
template <template <typename, int, int, bool> class F, typename T, int V, int K = 1>
static const void* causal_of(int k, bool silu) {
  if constexpr (K <= kCausalMaxK) {
    if (k == K) return silu ? F<T, V, K, true>::fn() : F<T, V, K, false>::fn();
    return causal_of<F, T, V, K + 1>(k, silu);
  }
  return nullptr;
}
template <template <typename, int, int, bool> class F, int VB>
static const void* causal_fn(int dtype, int v, int k, int silu) {
  if (dtype == PT_F32)
    return v > 1 ? causal_of<F, float, 4>(k, silu != 0) : causal_of<F, float, 1>(k, silu != 0);
  return v > 1 ? causal_of<F, __bf16, VB>(k, silu != 0) : causal_of<F, __bf16, 1>(k, silu != 0);
}
template <typename T, int V, int K, bool SILU>
struct CausalFwd {
  static const void* fn() { return (const void*)&causal_fwd_kernel<T, V, K, SILU>; }
};
template <typename T, int V, int K, bool SILU>
struct CausalBwd {
  static const void* fn() { return (const void*)&causal_bwd_kernel<T, V, K, SILU>; }
};
template <typename T, int V, int K, bool SILU>
struct CausalStep {
  static const void* fn() { return (const void*)&causal_step_kernel<T, V, K, SILU>; }
};

// gw [H, K] and gbias [H] from the runs' parts [parts][K + 1][H].
__global__ __launch_bounds__(kSumThreads) void causal_reduce_kernel(const float* __restrict__ part,
                                                                    float* __restrict__ gw,
                                                                    float* __restrict__ gbias,
                                                                    long long parts, int H, int K) {
  const long long cols = (long long)H * (K + 1);
  sum_columns((long long)blockIdx.x * kSumCols, parts,
              [&](long long c, long long* stride) {
                *stride = cols;
                return c < cols ? part + c : nullptr;
              },
              [&](long long c, float v) {
                const int j = (int)(c / H), h = (int)(c - (long long)j * H);
                if (c >= cols) return;
                if (j < K)
                  gw[(long long)h * K + j] = v;
                else if (gbias)
                  gbias[h] = v;
              });
}

static int check_causal(int dtype, int B, int L, int H, int K) {
  if (dtype != PT_F32 && dtype != PT_BF16) return PT_ERR_CONFIG;
  if (B < 0 || L < 1 || L > kCausalMaxL || H < 1 || K < 1 || K > kCausalMaxK) return PT_ERR_SHAPE;
  return PT_OK;
}

// Channels of 16 bytes.
static int causal_vector(int dtype) { return dtype == PT_F32 ? 4 : 8; }

// Channels a lane takes: v of them where rows and pointers allow.
static int causal_lanes(int dtype, int v, int H, long long batch, long long row,
                        const void* const* ptrs, int n) {
  bool ok = H % v == 0 && batch % v == 0 && row % v == 0;
  for (int i = 0; i < n; ++i) ok = ok && ssm_aligned(ptrs[i], (uintptr_t)v * (dtype == PT_F32 ? 4 : 2));
  return ok ? v : 1;
}

// Tokens of a run: as long as the grid still has `lanes` lanes, from `most`
// down to `least` (a run reads K - 1 tokens of the one before it again, and in
// the backward writes H (K + 1) sums). At 8 x 2048 x 4096 BF16 runs of 32, 64
// and 128 tokens take 52, 57 and 59 us forward and 125, 105 and 94 us backward.
static int causal_run(long long rows, int L, int cols, long long lanes, int most, int least) {
  int run = most;
  while (run > least && rows * cols * ssm_ceil(L, run) < lanes) run /= 2;
  return run;
}

static int causal_run_bwd(int B, int L, int H) {
  return causal_run(B, L, (int)ssm_ceil(H, 4), 131072, 128, 16);
}

}  // namespace pt

extern "C" {

int pt_causal_conv_fwd(int dtype, const void* x, long long x_batch, long long x_row, const float* w,
                       const float* bias, const void* state, const int* lengths, void* y,
                       void* state_out, int B, int L, int H, int K, int silu, void* stream) {
  const int st = pt::check_causal(dtype, B, L, H, K);
  if (st != PT_OK) return st;
  if (B == 0) return PT_OK;
  if (!x || !w || !y) return PT_ERR_NULL;
  const void* ptrs[] = {x, state, y, state_out};
  const int v = pt::causal_lanes(dtype, 4, H, x_batch, x_row, ptrs, 4);
  const int cols = (int)pt::ssm_ceil(H, v), run = pt::causal_run(B, L, cols, 524288, 32, 8);
  pt::CausalArgs a = {x, w, bias, state, lengths, y, state_out, x_batch, x_row, B, L, H,
                      run, (int)pt::ssm_ceil(L, run), cols};
  void* args[] = {&a};
  return pt::ssm_launch(pt::causal_fn<pt::CausalFwd, 4>(dtype, v, K, silu),
                        pt::ssm_ceil((long long)B * a.nruns * cols, pt::kCausalThreads),
                        pt::kCausalThreads, stream, args);
}

int pt_causal_conv_bwd_workspace_bytes(int dtype, int B, int L, int H, int K, size_t* bytes) {
  if (!bytes) return PT_ERR_NULL;
  const int st = pt::check_causal(dtype, B, L, H, K);
  if (st == PT_OK)
    *bytes = (size_t)B * pt::ssm_ceil(L, pt::causal_run_bwd(B, L, H)) * H * (K + 1) * 4;
  return st;
}

int pt_causal_conv_bwd(int dtype, const void* x, long long x_batch, long long x_row, const float* w,
                       const float* bias, const void* state, const int* lengths, const void* gy,
                       const void* gstate_out, void* gx, float* gw, float* gbias, void* gstate,
                       void* workspace, size_t workspace_bytes, int B, int L, int H, int K, int silu,
                       void* stream) {
  size_t need = 0;
  int st = pt_causal_conv_bwd_workspace_bytes(dtype, B, L, H, K, &need);
  if (st != PT_OK) return st;
  if (!gw) return PT_ERR_NULL;
  if (B > 0) {
    if (!x || !w || !gy || !gx) return PT_ERR_NULL;
    if (!workspace || workspace_bytes < need) return PT_ERR_WORKSPACE;
    if (!pt::ssm_aligned(workspace, 16)) return PT_ERR_ALIGN;  // sums are stored by fours
  }
  const void* ptrs[] = {x, state, gy, gstate_out, gx, gstate};
  const int v = pt::causal_lanes(dtype, 4, H, x_batch, x_row, ptrs, 6);
  const int cols = (int)pt::ssm_ceil(H, v), run = pt::causal_run_bwd(B, L, H);
  pt::CausalGradArgs g = {{x, w, bias, state, lengths, nullptr, nullptr, x_batch, x_row, B, L, H, run,
                           (int)pt::ssm_ceil(L, run), cols},
                          gy, gstate_out, gx, gstate, static_cast<float*>(workspace)};
  void* args[] = {&g};
  st = pt::ssm_launch(pt::causal_fn<pt::CausalBwd, 4>(dtype, v, K, silu),
                      pt::ssm_ceil((long long)B * g.f.nruns * cols, pt::kCausalThreads),
                      pt::kCausalThreads, stream, args);
  if (st != PT_OK) return st;
  long long parts = (long long)B * g.f.nruns;
  void* rargs[] = {&g.part, &gw, &gbias, &parts, &H, &K};
  return pt::ssm_launch((const void*)&pt::causal_reduce_kernel,
                        pt::ssm_ceil((long long)H * (K + 1), pt::kSumCols), pt::kSumThreads, stream,
                        rargs);
}

int pt_causal_conv_step(int dtype, const void* x, long long x_row, const float* w, const float* bias,
                        void* state, const int* slots, void* y, int B, int H, int K, int pool,
                        int silu, void* stream) {
  const int st = pt::check_causal(dtype, B, 1, H, K);
  if (st != PT_OK) return st;
  if (pool < 0) return PT_ERR_SHAPE;
  if (B == 0) return PT_OK;
  if (!x || !w || !y || (K > 1 && pool > 0 && !state)) return PT_ERR_NULL;
  const void* ptrs[] = {x, state, y};
  const int v = pt::causal_lanes(dtype, pt::causal_vector(dtype), H, 0, x_row, ptrs, 3);
  int cols = (int)pt::ssm_ceil(H, v);
  void* args[] = {&x, &w, &bias, &state, &slots, &y, &x_row, &B, &H, &pool, &cols};
  return pt::ssm_launch(pt::causal_fn<pt::CausalStep, 8>(dtype, v, K, silu),
                        pt::ssm_ceil((long long)B * cols, pt::kCausalThreads), pt::kCausalThreads,
                        stream, args);
}

}  // extern "C"
