// ssm_scan.hip — entry points of the selective scan.

#include "ssm_host.hpp"
#include "ssm_scan.hpp"
#include "ssm_tables.hpp"

namespace pt {

// gA [H, N], gD and gdt_bias [H] from the sequences' parts: 64 columns (a
// channel of one of the np + 2 sums) by 4 ranges of sequences a workgroup.
__global__ __launch_bounds__(256) void scan_param_reduce_kernel(ScanArgs a, const float* __restrict__ part_a,
                                                                const float* __restrict__ part_d,
                                                                float* __restrict__ ga, float* __restrict__ gd,
                                                                float* __restrict__ gbias, int parts) {
  __shared__ float sums[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const long long col = (long long)blockIdx.x * 64 + lane;
  const long long na = (long long)a.np * a.H, cols = na + 2LL * a.H;
  float v = 0.0f;
  if (col < cols) {
    const float* q = col < na ? part_a + col : part_d + (col - na);
    const long long stride = col < na ? na : 2LL * a.H;
    for (int k = w; k < parts; k += 4) v += q[k * stride];
  }
  sums[w][lane] = v;
  __syncthreads();
  if (w || col >= cols) return;
  v = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
  if (col < na) {
    const int n = (int)(col / a.H), h = (int)(col - (long long)n * a.H);
    if (n < a.N) ga[(long long)h * a.N + n] = v;
  } else {
    const int h = (int)((col - na) % a.H);
    float* o = col - na < a.H ? gd : gbias;
    if (o) o[h] = v;
  }
}

// States that the kernels hold: 16, 32 or 64.
static int scan_index(int N) { return N <= 16 ? 0 : N <= 32 ? 1 : 2; }

static int check_scan(const pt_scan_inputs* in, int L) {
  if (in->dtype != PT_F32 && in->dtype != PT_BF16) return PT_ERR_CONFIG;
  if (in->B < 0 || L < 1 || in->H < 1 || in->N < 1 || in->N > kScanMaxN || in->G < 1 || in->H % in->G)
    return PT_ERR_SHAPE;
  if (in->b_group < 0 || in->c_group < 0 || in->b_group >= (1LL << 31) || in->c_group >= (1LL << 31))
    return PT_ERR_SHAPE;
  if (in->B == 0) return PT_OK;
  return in->x && in->dt && in->a && in->b && in->c ? PT_OK : PT_ERR_NULL;
}

static ScanArgs scan_args(const pt_scan_inputs* in) {
  ScanArgs a;
  a.x = in->x, a.dt = in->dt, a.bm = in->b, a.cm = in->c;
  a.x_batch = in->x_batch, a.x_row = in->x_row, a.dt_batch = in->dt_batch, a.dt_row = in->dt_row;
  a.b_batch = in->b_batch, a.b_row = in->b_row, a.c_batch = in->c_batch, a.c_row = in->c_row;
  a.b_group = (int)in->b_group, a.c_group = (int)in->c_group;
  a.a = in->a, a.d = in->d, a.dt_bias = in->dt_bias, a.state = in->state, a.lengths = in->lengths;
  a.B = in->B, a.L = in->L, a.H = in->H, a.N = in->N, a.G = in->G, a.softplus = in->softplus;
  a.hg = in->H / in->G;
  a.blocks_g = (int)ssm_ceil(a.hg, kScanCh);
  a.np = 16 << scan_index(in->N);
  a.ntiles = (int)ssm_ceil(in->L, kScanTile);
  return a;
}

// Whether the scalar loads can take B and C as they are: whole registers of
// states, and pairs of BF16 on 4-byte boundaries.
static bool scan_direct(const pt_scan_inputs* in) {
  if (in->N != 16 << scan_index(in->N)) return false;
  if (!ssm_aligned(in->b, 4) || !ssm_aligned(in->c, 4)) return false;
  if (in->dtype == PT_F32) return true;
  return ((in->b_batch | in->b_row | in->b_group | in->c_batch | in->c_row | in->c_group) & 1) == 0;
}

static size_t scan_bc_floats(const pt_scan_inputs* in) {
  return scan_direct(in) ? 0
                         : ssm_round((size_t)in->B * in->L * in->G * 2 * (16 << scan_index(in->N)));
}

// Loads and stores of four channels: 16 bytes of FP32, 8 of BF16.
static bool scan_vector(const ScanArgs& a, int dtype, const void* const* ptrs, int n) {
  bool ok = a.hg % 4 == 0 && ((a.x_batch | a.x_row | a.dt_batch | a.dt_row) & 3) == 0;
  for (int i = 0; i < n; ++i) ok = ok && ssm_aligned(ptrs[i], dtype == PT_F32 ? 16 : 8);
  return ok;
}

// B and C into the workspace where they are not taken as they are.
static int scan_lay_out(const pt_scan_inputs* in, ScanArgs* a, float* ws, void* stream) {
  if (scan_direct(in)) return PT_OK;
  void* args[] = {a, &ws};
  const void* fn = in->dtype == PT_F32 ? (const void*)&scan_bc_kernel<float>
                                       : (const void*)&scan_bc_kernel<__bf16>;
  const int st = ssm_launch(fn, ssm_ceil((long long)in->B * in->L * in->G * 2 * a->np, 256), 256,
                            stream, args);
  a->bm = ws, a->cm = ws + a->np;
  a->b_group = a->c_group = 2 * a->np;
  a->b_row = a->c_row = (long long)in->G * 2 * a->np;
  a->b_batch = a->c_batch = a->b_row * in->L;
  return st;
}

struct ScanBwdLayout {
  size_t bc, part_a, part_d, total;
};
static ScanBwdLayout scan_bwd_layout(const pt_scan_inputs* in, const ScanArgs& a) {
  ScanBwdLayout o;
  o.bc = scan_bc_floats(in);
  o.part_a = o.bc + ssm_round((size_t)a.blocks_g * a.G * a.B * a.L * 2 * a.np);
  o.part_d = o.part_a + ssm_round((size_t)a.B * a.np * a.H);
  o.total = (o.part_d + (size_t)a.B * 2 * a.H) * sizeof(float);
  return o;
}

static long long scan_blocks(const ScanArgs& a) { return (long long)a.B * a.blocks_g * a.G; }

// [FP32; BF16; BF16 with B and C laid out as FP32]
static int scan_types(const pt_scan_inputs* in) {
  return in->dtype == PT_F32 ? 0 : scan_direct(in) ? 1 : 2;
}

template <typename T, int PER>
static const void* step_fn(bool vec) {
  return vec ? (const void*)&scan_step_kernel<T, PER, true> : (const void*)&scan_step_kernel<T, PER, false>;
}

}  // namespace pt

extern "C" {

int pt_selective_scan_sizes(const pt_scan_inputs* in, size_t* fwd_workspace, size_t* saved,
                            size_t* bwd_workspace) {
  if (!in) return PT_ERR_NULL;
  const int st = pt::check_scan(in, in->L);
  if (st != PT_OK) return st;
  const pt::ScanArgs a = pt::scan_args(in);
  if (fwd_workspace) *fwd_workspace = pt::scan_bc_floats(in) * sizeof(float);
  if (saved) *saved = (size_t)a.B * a.ntiles * a.np * a.H * sizeof(float);
  if (bwd_workspace) *bwd_workspace = pt::scan_bwd_layout(in, a).total;
  return PT_OK;
}

int pt_selective_scan_fwd(const pt_scan_inputs* in, void* y, float* state_out, float* saved,
                          void* workspace, size_t workspace_bytes, void* stream) {
  if (!in) return PT_ERR_NULL;
  int st = pt::check_scan(in, in->L);
  if (st != PT_OK) return st;
  if (in->B == 0) return PT_OK;
  if (!y) return PT_ERR_NULL;
  const size_t need = pt::scan_bc_floats(in) * sizeof(float);
  if (need && (!workspace || workspace_bytes < need)) return PT_ERR_WORKSPACE;
  pt::ScanFwdArgs f = {pt::scan_args(in), y, state_out, saved};
  const void* ptrs[] = {in->x, in->dt, y};
  const bool vec = pt::scan_vector(f.s, in->dtype, ptrs, 3);
  st = pt::scan_lay_out(in, &f.s, static_cast<float*>(workspace), stream);
  if (st != PT_OK) return st;
  void* args[] = {&f};
  return pt::ssm_launch((const void*)pt::kScanFwd[pt::scan_types(in)][pt::scan_index(in->N)][vec],
                        pt::scan_blocks(f.s), pt::kScanThreads, stream, args);
}

int pt_selective_scan_bwd(const pt_scan_inputs* in, const void* gy, const float* saved,
                          const float* gstate_out, void* gx, void* gdt, float* ga, void* gb,
                          void* gc, float* gd, float* gdt_bias, float* gstate, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (!in) return PT_ERR_NULL;
  int st = pt::check_scan(in, in->L);
  if (st != PT_OK) return st;
  if (!ga) return PT_ERR_NULL;
  if (in->B > 0 && (!gy || !saved || !gx || !gdt || !gb || !gc)) return PT_ERR_NULL;
  pt::ScanArgs a = pt::scan_args(in);
  const pt::ScanBwdLayout o = pt::scan_bwd_layout(in, a);
  if (in->B > 0 && (!workspace || workspace_bytes < o.total)) return PT_ERR_WORKSPACE;
  float* ws = static_cast<float*>(workspace);
  const void* ptrs[] = {in->x, in->dt, gy, gx, gdt};
  const bool vec = pt::scan_vector(a, in->dtype, ptrs, 5);
  float *part_bc = ws + o.bc, *part_a = ws + o.part_a, *part_d = ws + o.part_d;
  if (in->B > 0) {
    st = pt::scan_lay_out(in, &a, ws, stream);
    if (st != PT_OK) return st;
    pt::ScanBwdArgs f = {a, gy, saved, gstate_out, gx, gdt, gstate, part_bc, part_a, part_d};
    void* args[] = {&f};
    st = pt::ssm_launch((const void*)pt::kScanBwd[pt::scan_types(in)][pt::scan_index(in->N)][vec],
                        pt::scan_blocks(a), pt::kScanThreads, stream, args);
    if (st != PT_OK) return st;
    const float* cpart = part_bc;
    void* bargs[] = {&a, &cpart, &gb, &gc};
    st = pt::ssm_launch(in->dtype == PT_F32 ? (const void*)&pt::scan_bc_reduce_kernel<float>
                                            : (const void*)&pt::scan_bc_reduce_kernel<__bf16>,
                        pt::ssm_ceil((long long)a.B * a.L * a.G * 2 * a.np, 256), 256, stream, bargs);
    if (st != PT_OK) return st;
  }
  void* pargs[] = {&a, &part_a, &part_d, &ga, &gd, &gdt_bias, &a.B};
  return pt::ssm_launch((const void*)&pt::scan_param_reduce_kernel,
                        pt::ssm_ceil((long long)(a.np + 2) * a.H, 64), 256, stream, pargs);
}

int pt_selective_scan_step(const pt_scan_inputs* in, float* state, const int* slots, int pool,
                           void* y, void* stream) {
  if (!in) return PT_ERR_NULL;
  const int st = pt::check_scan(in, 1);
  if (st != PT_OK) return st;
  if (pool < 0) return PT_ERR_SHAPE;
  if (in->B == 0) return PT_OK;
  if (!y || (pool > 0 && !state)) return PT_ERR_NULL;
  const uintptr_t four = in->dtype == PT_F32 ? 16 : 8;
  const bool vec = in->N % 4 == 0 && ((in->b_batch | in->c_batch | in->b_group | in->c_group) & 3) == 0 &&
                   pt::ssm_aligned(state, 16) && pt::ssm_aligned(in->a, 16) &&
                   pt::ssm_aligned(in->b, four) && pt::ssm_aligned(in->c, four);
  const int per = in->N <= 4 ? 1 : in->N <= 8 ? 2 : in->N <= 16 ? 4 : in->N <= 32 ? 8 : 16;
  const int at = per == 1 ? 0 : per == 2 ? 1 : per == 4 ? 2 : per == 8 ? 3 : 4;
  const void* const fns[2][5] = {
      {pt::step_fn<float, 1>(vec), pt::step_fn<float, 2>(vec), pt::step_fn<float, 4>(vec),
       pt::step_fn<float, 8>(vec), pt::step_fn<float, 16>(vec)},
      {pt::step_fn<__bf16, 1>(vec), pt::step_fn<__bf16, 2>(vec), pt::step_fn<__bf16, 4>(vec),
       pt::step_fn<__bf16, 8>(vec), pt::step_fn<__bf16, 16>(vec)}};
  int B = in->B, H = in->H, N = in->N, G = in->G, softplus = in->softplus;
  int b_group = (int)in->b_group, c_group = (int)in->c_group;
  int blocks = (int)pt::ssm_ceil(H, 256 / per);
  long long xr = in->x_batch, dr = in->dt_batch, br = in->b_batch, cr = in->c_batch;
  const void *x = in->x, *dt = in->dt, *b = in->b, *c = in->c;
  const float *A = in->a, *d = in->d, *bias = in->dt_bias;
  void* args[] = {&x, &dt, &A, &b, &c, &state, &d, &bias, &slots, &y, &xr, &dr, &br, &cr,
                  &b_group, &c_group, &B, &H, &N, &G, &pool, &softplus, &blocks};
  return pt::ssm_launch(fns[in->dtype == PT_BF16][at], (long long)B * blocks, 256, stream, args);
}

}  // extern "C"
