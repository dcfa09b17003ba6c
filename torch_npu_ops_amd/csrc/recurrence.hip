// Gated linear recurrence for gfx950: forward over ragged sequences, the
// decode step on a pool of states, and the backward pass.
//
//   r = sigmoid(a), i = sigmoid(b), l = -c softplus(lam) r, alpha = exp(l),
//   s = sqrt(1 - alpha^2), h_t = alpha h_{t-1} + s i x_t, y_t = h_t
//
// per channel, in fp32.  alpha - 1 is formed as expm1(l) and 1 - alpha^2 as
// -(alpha - 1)(2 + (alpha - 1)), so neither loses digits where a channel
// keeps nearly all of its state (alpha near 1, the case that matters).
#include <math.h>

#include "xk_common.h"

namespace xk {
namespace {

constexpr int kWin = XK_GLR_WINDOW;

// Per-channel constants: k = -c softplus(lam), so that l = k r.
__device__ __forceinline__ float softplus_f32(float v) {
  return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v)));
}

// The decay of a token for l <= 0: alpha = exp(l) and alpha - 1, each to its
// own last digits.  Above -1/4 the power series to l^6 / 720 (the next term is
// 5e-8 of the sum) gives alpha - 1, below it the exponential gives alpha.
struct Decay {
  float alpha, em1;
};
__device__ __forceinline__ Decay decay_of(float l) {
  float p = fmaf(l, 1.f / 720.f, 1.f / 120.f);
  p = fmaf(p, l, 1.f / 24.f);
  p = fmaf(p, l, 1.f / 6.f);
  p = fmaf(p, l, 0.5f);
  p = fmaf(p, l, 1.f) * l;
  const float e = __expf(l);
  const bool near = l > -0.25f;
  return {near ? 1.f + p : e, near ? p : e - 1.f};
}

struct Gate {
  float alpha, em1;
  float s;  // sqrt(1 - alpha^2)
};
__device__ __forceinline__ Gate gate_of(float k, float r) {
  const Decay d = decay_of(k * r);
  return {d.alpha, d.em1, __builtin_amdgcn_sqrtf(-d.em1 * (1.f + d.alpha))};
}

// alpha v from alpha - 1: one rounding, of the product, where alpha is near 1
// (thousands of tokens may lie between a state and its use); 2^-24 |v| at most
// where it is not.
__device__ __forceinline__ float decayed(float em1, float v) { return fmaf(em1, v, v); }

struct FwdParams {
  const void* x;
  const void* a;
  const void* b;
  void* y;
  int64_t sx, sa, sb, sy;
  const float* lam;
  float c;
  const float* h0;
  float* fin;
  float* states;
  const void* cu;
  int cu64;
  int64_t N, T, total, D;
};

// First token of sequence n (N: the end); without cu_seqlens, N equal runs.
__device__ __forceinline__ int64_t cu_at(const void* cu, int cu64, int64_t n, int64_t run,
                                         int64_t total) {
  if (!cu) return n * run;
  const int64_t v = cu64 ? static_cast<const int64_t*>(cu)[n]
                         : static_cast<int64_t>(static_cast<const int32_t*>(cu)[n]);
  return v < 0 ? 0 : (v > total ? total : v);
}

// One lane per (sequence, channel), token by token.
template <typename T>
__global__ void __launch_bounds__(64) glr_fwd_kernel(FwdParams p) {
  const int64_t ch = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x;
  const int64_t n = blockIdx.y;
  if (ch >= p.D) return;
  const int64_t t0 = cu_at(p.cu, p.cu64, n, p.T, p.total), t1 = cu_at(p.cu, p.cu64, n + 1, p.T, p.total);
  const float k = -p.c * softplus_f32(p.lam[ch]);
  float h = p.h0 ? p.h0[n * p.D + ch] : 0.f;
  for (int64_t t = t0; t < t1; ++t) {
    const float x = to_f32(static_cast<const T*>(p.x)[t * p.sx + ch]);
    const float r = sigmoid(to_f32(static_cast<const T*>(p.a)[t * p.sa + ch]));
    const float i = sigmoid(to_f32(static_cast<const T*>(p.b)[t * p.sb + ch]));
    const Gate g = gate_of(k, r);
    if (p.states && t % kWin == 0 && t != t0) p.states[t / kWin * p.D + ch] = h;
    h = decayed(g.em1, h) + g.s * (i * x);
    static_cast<T*>(p.y)[t * p.sy + ch] = from_f32<T>(h);
  }
  if (p.fin) p.fin[n * p.D + ch] = h;
}

struct UpdateParams {
  const void* x;
  const void* a;
  const void* b;
  void* y;
  int64_t sx, sa, sb, sy;
  const float* lam;
  float c;
  float* state;
  int64_t slot_pitch, num_slots;
  const int32_t* idx;
  int64_t cols;
  const int32_t* acc;
  const void* cu;
  int cu64;
  int64_t N, T, total, D;
};

template <typename T>
__global__ void __launch_bounds__(64) glr_update_kernel(UpdateParams p) {
  const int64_t ch = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x;
  const int64_t n = blockIdx.y;
  if (ch >= p.D) return;
  const int64_t t0 = cu_at(p.cu, p.cu64, n, p.T, p.total);
  const int64_t t1 = cu_at(p.cu, p.cu64, n + 1, p.T, p.total);
  const float k = -p.c * softplus_f32(p.lam[ch]);
  const int64_t width = p.cols > 0 ? p.cols : 1;
  int64_t col = p.acc ? static_cast<int64_t>(p.acc[n]) - 1 : 0;
  col = col < 0 ? 0 : (col >= width ? width - 1 : col);
  auto slot_at = [&](int64_t c) -> int64_t { return p.idx ? p.idx[n * width + c] : n; };
  const int64_t first = slot_at(col);
  const bool in = first >= 0 && first < p.num_slots;
  float h = in ? p.state[first * p.slot_pitch + ch] : 0.f;
  for (int64_t t = t0; t < t1; ++t) {
    const float x = to_f32(static_cast<const T*>(p.x)[t * p.sx + ch]);
    const float r = sigmoid(to_f32(static_cast<const T*>(p.a)[t * p.sa + ch]));
    const float i = sigmoid(to_f32(static_cast<const T*>(p.b)[t * p.sb + ch]));
    const Gate g = gate_of(k, r);
    h = decayed(g.em1, h) + g.s * (i * x);
    static_cast<T*>(p.y)[t * p.sy + ch] = from_f32<T>(h);
    if (p.cols > 0 && t - t0 < p.cols) {
      const int64_t s = slot_at(t - t0);
      if (s >= 0 && s < p.num_slots) p.state[s * p.slot_pitch + ch] = h;
    }
  }
  if (p.cols == 0 && in && t1 > t0) p.state[first * p.slot_pitch + ch] = h;
}

struct BwdParams {
  const void* dy;
  const void* x;
  const void* a;
  const void* b;
  void* dx;
  void* da;
  void* db;
  int64_t sdy, sx, sa, sb, sdx, sda, sdb;
  const float* lam;
  float c;
  const float* states;
  const float* h0;
  const float* dfin;
  float* dh0;
  float* part;  // dlam's parts, [N, D]
  const void* cu;
  int cu64;
  int64_t N, T, total, D;
};

// sigmoid(lam) / softplus(lam), 1 in the limit lam -> -inf.
__device__ __forceinline__ float slope_ratio(float lam) {
  if (lam < -17.f) return 1.f;  // 1 - e^lam / 2 rounds to 1
  return 1.f / ((1.f + expf(-lam)) * softplus_f32(lam));
}

template <typename T>
__global__ void __launch_bounds__(64) glr_bwd_kernel(BwdParams p) {
  const int64_t ch = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x;
  const int64_t n = blockIdx.y;
  if (ch >= p.D) return;
  const int64_t t0 = cu_at(p.cu, p.cu64, n, p.T, p.total), t1 = cu_at(p.cu, p.cu64, n + 1, p.T, p.total);
  const float k = -p.c * softplus_f32(p.lam[ch]);
  float q = p.dfin ? p.dfin[n * p.D + ch] : 0.f;  // gradient of the state after token t
  float sum = 0.f;
  for (int64_t hi = t1; hi > t0;) {
    int64_t lo = (hi - 1) / kWin * kWin;
    lo = lo < t0 ? t0 : lo;
    float h = lo == t0 ? (p.h0 ? p.h0[n * p.D + ch] : 0.f) : p.states[lo / kWin * p.D + ch];
    float before[kWin];
#pragma unroll
    for (int j = 0; j < kWin; ++j) {
      const int64_t t = lo + j;
      if (t < hi) {
        before[j] = h;
        const float x = to_f32(static_cast<const T*>(p.x)[t * p.sx + ch]);
        const float r = sigmoid(to_f32(static_cast<const T*>(p.a)[t * p.sa + ch]));
        const float i = sigmoid(to_f32(static_cast<const T*>(p.b)[t * p.sb + ch]));
        const Gate g = gate_of(k, r);
        h = decayed(g.em1, h) + g.s * (i * x);
      }
    }
#pragma unroll
    for (int j = kWin - 1; j >= 0; --j) {
      const int64_t t = lo + j;
      if (t < hi) {
        const float x = to_f32(static_cast<const T*>(p.x)[t * p.sx + ch]);
        const float av = to_f32(static_cast<const T*>(p.a)[t * p.sa + ch]);
        const float bv = to_f32(static_cast<const T*>(p.b)[t * p.sb + ch]);
        const float r = sigmoid(av), i = sigmoid(bv);
        const Gate g = gate_of(k, r);
        const float l = k * r;
        const float G = to_f32(static_cast<const T*>(p.dy)[t * p.sdy + ch]) + q;
        const float l_s = g.s > 0.f ? l / g.s : 0.f;
        const float e = G * g.alpha * (before[j] * l - i * x * g.alpha * l_s);
        static_cast<T*>(p.dx)[t * p.sdx + ch] = from_f32<T>(G * g.s * i);
        static_cast<T*>(p.da)[t * p.sda + ch] = from_f32<T>(e * sigmoid(-av));
        static_cast<T*>(p.db)[t * p.sdb + ch] = from_f32<T>(G * g.s * i * x * sigmoid(-bv));
        sum += e;
        q = decayed(g.em1, G);
      }
    }
    hi = lo;
  }
  if (p.dh0) p.dh0[n * p.D + ch] = q;
  if (p.part) p.part[n * p.D + ch] = sum;
}

// dlam = sum over parts of (sum dl l) sigmoid(lam) / softplus(lam).
__global__ void __launch_bounds__(64) glr_dlam_kernel(const float* part, int64_t parts,
                                                      const float* lam, float* dlam, int64_t D) {
  const int64_t ch = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x;
  if (ch >= D) return;
  float s = 0.f;
  for (int64_t j = 0; j < parts; ++j) s += part[j * D + ch];
  dlam[ch] = s * slope_ratio(lam[ch]);
}

bool pitch_ok(int64_t pitch, int64_t D) { return pitch >= D; }

// cu_seqlens of a readable type, or none and N equal runs.
bool seqs_ok(const void* cu, xk_dtype dt, int64_t N, int64_t total) {
  return cu ? dt == XK_I32 || dt == XK_I64 : total % N == 0;
}

}  // namespace
}  // namespace xk

using namespace xk;

extern "C" int64_t xk_gated_linear_recurrence_workspace_bytes(int64_t, int64_t) { return 0; }

extern "C" int xk_gated_linear_recurrence(
    const void* x, int64_t stride_x_tok, const void* a, int64_t stride_a_tok, const void* b,
    int64_t stride_b_tok, xk_dtype dtype, const float* lam, float c, void* y,
    int64_t stride_y_tok, const float* initial_state, float* final_state, float* states,
    const void* cu_seqlens, xk_dtype cu_dtype, int64_t N, int64_t total_tokens, int64_t D,
    void* workspace, size_t workspace_bytes, void* stream) {
  if (N < 0 || total_tokens < 0 || D <= 0 || !(c >= 0.f)) return XK_ERR_INVALID;
  if (!is_float_dtype(dtype)) return XK_ERR_UNSUPPORTED;
  if (N == 0) return XK_OK;
  if (!seqs_ok(cu_seqlens, cu_dtype, N, total_tokens) || !lam) return XK_ERR_INVALID;
  if (total_tokens > 0 &&
      (!x || !a || !b || !y || !pitch_ok(stride_x_tok, D) || !pitch_ok(stride_a_tok, D) ||
       !pitch_ok(stride_b_tok, D) || !pitch_ok(stride_y_tok, D)))
    return XK_ERR_INVALID;
  FwdParams p{x, a, b, y, stride_x_tok, stride_a_tok, stride_b_tok, stride_y_tok, lam, c,
              initial_state, final_state, states, cu_seqlens, cu_dtype == XK_I64, N,
              total_tokens / N, total_tokens, D};
  const dim3 grid(cdiv(D, 64), N);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case XK_F32: hipLaunchKernelGGL(glr_fwd_kernel<float>, grid, dim3(64), 0, s, p); break;
    case XK_BF16: hipLaunchKernelGGL(glr_fwd_kernel<bf16>, grid, dim3(64), 0, s, p); break;
    default: hipLaunchKernelGGL(glr_fwd_kernel<f16>, grid, dim3(64), 0, s, p); break;
  }
  return launch_status();
}

extern "C" int xk_gated_linear_recurrence_update(
    const void* x, int64_t stride_x_tok, const void* a, int64_t stride_a_tok, const void* b,
    int64_t stride_b_tok, xk_dtype dtype, const float* lam, float c, void* y,
    int64_t stride_y_tok, float* state, int64_t stride_state_slot, int64_t num_slots,
    const int32_t* state_indices, int64_t num_cols, const int32_t* num_accepted_tokens,
    const void* cu_seqlens, xk_dtype cu_dtype, int64_t N, int64_t T, int64_t total_tokens,
    int64_t D, void* stream) {
  if (N < 0 || total_tokens < 0 || D <= 0 || num_slots < 0 || num_cols < 0 || !(c >= 0.f))
    return XK_ERR_INVALID;
  if (!is_float_dtype(dtype)) return XK_ERR_UNSUPPORTED;
  if (N == 0 || total_tokens == 0) return XK_OK;
  if (cu_seqlens ? cu_dtype != XK_I32 && cu_dtype != XK_I64 : T <= 0 || T > total_tokens / N)
    return XK_ERR_INVALID;
  if (!x || !a || !b || !y || !lam || (num_slots > 0 && !state) || stride_state_slot < D ||
      (num_cols > 0 && !state_indices) || !pitch_ok(stride_x_tok, D) ||
      !pitch_ok(stride_a_tok, D) || !pitch_ok(stride_b_tok, D) || !pitch_ok(stride_y_tok, D))
    return XK_ERR_INVALID;
  UpdateParams p{x, a, b, y, stride_x_tok, stride_a_tok, stride_b_tok, stride_y_tok, lam, c,
                 state, stride_state_slot, num_slots, state_indices, num_cols,
                 num_accepted_tokens, cu_seqlens, cu_dtype == XK_I64, N, T, total_tokens, D};
  const dim3 grid(cdiv(D, 64), N);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case XK_F32: hipLaunchKernelGGL(glr_update_kernel<float>, grid, dim3(64), 0, s, p); break;
    case XK_BF16: hipLaunchKernelGGL(glr_update_kernel<bf16>, grid, dim3(64), 0, s, p); break;
    default: hipLaunchKernelGGL(glr_update_kernel<f16>, grid, dim3(64), 0, s, p); break;
  }
  return launch_status();
}

extern "C" int64_t xk_gated_linear_recurrence_bwd_workspace_bytes(int64_t, int64_t N,
                                                                  int64_t D) {
  return N * D * 4;
}

extern "C" int xk_gated_linear_recurrence_bwd(
    const void* dy, int64_t stride_dy_tok, const void* x, int64_t stride_x_tok, const void* a,
    int64_t stride_a_tok, const void* b, int64_t stride_b_tok, xk_dtype dtype, const float* lam,
    float c, const float* states, const float* initial_state, const float* d_final_state,
    void* dx, int64_t stride_dx_tok, void* da, int64_t stride_da_tok, void* db,
    int64_t stride_db_tok, float* dlam, float* d_initial_state, const void* cu_seqlens,
    xk_dtype cu_dtype, int64_t N, int64_t total_tokens, int64_t D, void* workspace,
    size_t workspace_bytes, void* stream) {
  if (N < 0 || total_tokens < 0 || D <= 0 || !(c >= 0.f)) return XK_ERR_INVALID;
  if (!is_float_dtype(dtype)) return XK_ERR_UNSUPPORTED;
  if (!lam || (N > 0 && !seqs_ok(cu_seqlens, cu_dtype, N, total_tokens))) return XK_ERR_INVALID;
  if (total_tokens > 0 &&
      (!dy || !x || !a || !b || !states || !dx || !da || !db || !pitch_ok(stride_dy_tok, D) ||
       !pitch_ok(stride_x_tok, D) || !pitch_ok(stride_a_tok, D) || !pitch_ok(stride_b_tok, D) ||
       !pitch_ok(stride_dx_tok, D) || !pitch_ok(stride_da_tok, D) || !pitch_ok(stride_db_tok, D)))
    return XK_ERR_INVALID;
  const int64_t need = xk_gated_linear_recurrence_bwd_workspace_bytes(total_tokens, N, D);
  if (need > 0 && (!workspace || workspace_bytes < static_cast<size_t>(need) ||
                   !aligned(workspace, 256)))
    return XK_ERR_WORKSPACE;
  BwdParams p{dy, x, a, b, dx, da, db, stride_dy_tok, stride_x_tok, stride_a_tok, stride_b_tok,
              stride_dx_tok, stride_da_tok, stride_db_tok, lam, c, states, initial_state,
              d_final_state, d_initial_state, static_cast<float*>(workspace), cu_seqlens,
              cu_dtype == XK_I64, N, N > 0 ? total_tokens / N : 0, total_tokens, D};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (N > 0) {
    const dim3 grid(cdiv(D, 64), N);
    switch (dtype) {
      case XK_F32: hipLaunchKernelGGL(glr_bwd_kernel<float>, grid, dim3(64), 0, s, p); break;
      case XK_BF16: hipLaunchKernelGGL(glr_bwd_kernel<bf16>, grid, dim3(64), 0, s, p); break;
      default: hipLaunchKernelGGL(glr_bwd_kernel<f16>, grid, dim3(64), 0, s, p); break;
    }
  }
  if (dlam)
    hipLaunchKernelGGL(glr_dlam_kernel, dim3(cdiv(D, 64)), dim3(64), 0, s,
                       static_cast<const float*>(workspace), N, lam, dlam, D);
  return launch_status();
}
