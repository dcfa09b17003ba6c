// Entry points of the block-to-block norm, its sums over rows, and the
// kernels for rows that no block holds (residual_norm.h has the others).
#include "residual_norm.h"

namespace xk {
namespace resnorm {
namespace {

__device__ __forceinline__ void put(void* p, int64_t i, xk_dtype dt, float v) {
  switch (dt) {
    case XK_BF16: static_cast<bf16*>(p)[i] = from_f32<bf16>(v); break;
    case XK_F16: static_cast<f16*>(p)[i] = from_f32<f16>(v); break;
    default: static_cast<float*>(p)[i] = v;
  }
}

// Sum over a block of 1024; a barrier on both sides.
__device__ __forceinline__ float block_sum(float v, float* red) {
  __syncthreads();
  return team_sum<1024>(v, red, 0);
}

__global__ void __launch_bounds__(1024) stream_fwd_kernel(FwdParams p) {
  __shared__ float red[16];
  const float inv_n = 1.f / static_cast<float>(p.N);
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    float r1 = 1.f, ss = 0.f;
    if (p.post) {
      for (int64_t e = threadIdx.x; e < p.N; e += 1024) {
        const float f = load_as_f32(p.x, row * p.sx + e, p.dt);
        ss = fmaf(f, f, ss);
      }
      r1 = 1.f / sqrtf(block_sum(ss, red) * inv_n + p.eps);
      if (p.r1 && threadIdx.x == 0) p.r1[row] = r1;
    }
    auto at = [&](int64_t e) {
      float v = load_as_f32(p.x, row * p.sx + e, p.dt);
      if (p.post) v *= r1 * (load_as_f32(p.post, e, p.wdt) + p.off);
      if (p.gate) v *= silu(load_as_f32(p.gate, row * p.sgate + e, p.dt));
      if (p.scale) v *= load_as_f32(p.scale, e, p.wdt);
      return v + load_as_f32(p.res, row * p.sres + e, p.rdt);
    };
    float r2 = 0.f;
    if (p.pre) {
      ss = 0.f;
      for (int64_t e = threadIdx.x; e < p.N; e += 1024) {
        const float f = at(e);
        ss = fmaf(f, f, ss);
      }
      r2 = 1.f / sqrtf(block_sum(ss, red) * inv_n + p.eps);
      if (p.r2 && threadIdx.x == 0) p.r2[row] = r2;
    }
    // An element's inputs are read before its outputs (which may lie over
    // them) are written.
    for (int64_t e = threadIdx.x; e < p.N; e += 1024) {
      const float f = at(e);
      put(p.h, row * p.sh + e, p.rdt, f);
      if (p.pre)
        put(p.y, row * p.sy + e, p.dt, f * r2 * (load_as_f32(p.pre, e, p.wdt) + p.off));
    }
  }
}

__global__ void __launch_bounds__(1024) stream_bwd_kernel(BwdParams p) {
  __shared__ float red[16];
  const float inv_n = 1.f / static_cast<float>(p.N);
  const int64_t pitch = part_pitch(p.N);
  float* part = p.part + static_cast<int64_t>(blockIdx.x) * 3 * pitch;
  for (int64_t row = blockIdx.x; row < p.M; row += p.parts) {
    const bool first = row == blockIdx.x;  // this part's sums start here
    const float r1 = p.post ? p.r1[row] : 1.f, r2 = p.dy ? p.r2[row] : 0.f;
    struct El {
      float xh, n, z, sg, v, s, h;
    };
    auto at = [&](int64_t e) {
      El o;
      o.xh = load_as_f32(p.x, row * p.sx + e, p.dt) * r1;
      o.n = p.post ? o.xh * (load_as_f32(p.post, e, p.wdt) + p.off) : o.xh;
      o.z = p.gate ? load_as_f32(p.gate, row * p.sgate + e, p.dt) : 0.f;
      o.sg = p.gate ? sigmoid(o.z) : 1.f;
      o.v = p.gate ? o.n * o.z * o.sg : o.n;
      o.s = p.scale ? load_as_f32(p.scale, e, p.wdt) : 1.f;
      o.h = fmaf(o.s, o.v, load_as_f32(p.res, row * p.sres + e, p.rdt));
      return o;
    };
    float ss = 0.f, dot = 0.f;
    if (p.dy) {
      for (int64_t e = threadIdx.x; e < p.N; e += 1024)
        ss = fmaf(load_as_f32(p.dy, row * p.sdy + e, p.dt) *
                      (load_as_f32(p.pre, e, p.wdt) + p.off),
                  at(e).h * r2, ss);
      ss = block_sum(ss, red) * inv_n;
    }
    auto grad_h = [&](int64_t e, const El& o) {
      float g = 0.f;
      if (p.dy)
        g = r2 * (load_as_f32(p.dy, row * p.sdy + e, p.dt) *
                      (load_as_f32(p.pre, e, p.wdt) + p.off) -
                  o.h * r2 * ss);
      if (p.dh) g += load_as_f32(p.dh, row * p.sdh + e, p.rdt);
      return g;
    };
    if (p.post) {
      for (int64_t e = threadIdx.x; e < p.N; e += 1024) {
        const El o = at(e);
        float g = grad_h(e, o) * o.s;
        if (p.gate) g *= o.z * o.sg;
        dot = fmaf(g * (load_as_f32(p.post, e, p.wdt) + p.off), o.xh, dot);
      }
      dot = block_sum(dot, red) * inv_n;
    }
    auto add = [&](int k, int64_t e, float v) {
      float* q = part + k * pitch + e;
      *q = first ? v : *q + v;
    };
    for (int64_t e = threadIdx.x; e < p.N; e += 1024) {
      const El o = at(e);
      float g = grad_h(e, o);
      if (p.sums & 4)
        add(2, e, p.dy ? load_as_f32(p.dy, row * p.sdy + e, p.dt) * o.h * r2 : 0.f);
      if (p.sums & 2) add(1, e, g * o.v);
      if (p.dres) put(p.dres, row * p.sdres + e, p.rdt, g);
      g *= o.s;
      if (p.gate) {
        if (p.dgate)
          put(p.dgate, row * p.sdgate + e, p.dt,
              g * o.n * o.sg * fmaf(o.z, 1.f - o.sg, 1.f));
        g *= o.z * o.sg;
      }
      if (p.post) {
        if (p.sums & 1) add(0, e, g * o.xh);
        g = r1 * (g * (load_as_f32(p.post, e, p.wdt) + p.off) - o.xh * dot);
      }
      if (p.dx) put(p.dx, row * p.sdx + e, p.dt, g);
    }
  }
}

// Column sums of the parts in their order: a block takes 16 columns, each of
// its 16 rows of lanes every 16th part.
constexpr int kSumCols = 16;
__global__ void __launch_bounds__(256)
    sums_kernel(const float* part, int64_t parts, int64_t N, void* dpost, void* dscale,
                void* dpre, xk_dtype wdt) {
  __shared__ float red[16][kSumCols + 1];
  const int k = blockIdx.y, lane = threadIdx.x % kSumCols, first = threadIdx.x / kSumCols;
  void* out = k == 0 ? dpost : (k == 1 ? dscale : dpre);
  if (!out) return;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kSumCols + lane;
  const int64_t pitch = part_pitch(N);
  float s = 0.f;
  if (col < N) {
#pragma unroll 8
    for (int64_t q = first; q < parts; q += 16) s += part[(q * 3 + k) * pitch + col];
  }
  red[first][lane] = s;
  __syncthreads();
  if (first == 0 && col < N) {
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += red[w][lane];
    put(out, col, wdt, s);
  }
}

// 16 elements of a row take 256 lanes of sums_kernel, fewer than 2^32 of them.
constexpr int64_t kMostRow = int64_t{1} << 28;
bool pitch_bad(const void* p, int64_t pitch, int64_t N) { return p && pitch < N; }

}  // namespace

int stream_fwd(const FwdParams& p, hipStream_t s) {
  const int64_t grid = std::min<int64_t>(p.M, int64_t{2} * num_cus());
  hipLaunchKernelGGL(stream_fwd_kernel, dim3(grid), dim3(1024), 0, s, p);
  return launch_status();
}
int stream_bwd(const BwdParams& p, hipStream_t s) {
  hipLaunchKernelGGL(stream_bwd_kernel, dim3(p.parts), dim3(1024), 0, s, p);
  return launch_status();
}

}  // namespace resnorm
}  // namespace xk

using namespace xk;

extern "C" int xk_gated_residual_rms_norm(
    const void* x, int64_t stride_x_row, const void* residual, int64_t stride_res_row,
    const void* gate, int64_t stride_gate_row, const void* post_weight, const void* scale,
    const void* pre_weight, void* h, int64_t stride_h_row, void* y, int64_t stride_y_row,
    float* rstd_post, float* rstd_pre, int64_t M, int64_t N, float eps, int unit_offset,
    xk_dtype dtype, xk_dtype rdtype, xk_dtype wdtype, void* stream) {
  using namespace resnorm;
  if (M < 0 || N <= 0 || N >= kMostRow || !(eps >= 0.f)) return XK_ERR_INVALID;
  if (!is_float_dtype(dtype) || (rdtype != dtype && rdtype != XK_F32) ||
      (wdtype != dtype && wdtype != XK_F32))
    return XK_ERR_UNSUPPORTED;
  if (M == 0) return XK_OK;
  if (!x || !residual || !h || (pre_weight && !y)) return XK_ERR_INVALID;
  if (M > 1 && (pitch_bad(x, stride_x_row, N) || pitch_bad(residual, stride_res_row, N) ||
                pitch_bad(gate, stride_gate_row, N) || pitch_bad(h, stride_h_row, N) ||
                pitch_bad(pre_weight ? y : nullptr, stride_y_row, N)))
    return XK_ERR_INVALID;
  FwdParams p{x, residual, gate, post_weight, scale, pre_weight, h, y, rstd_post, rstd_pre,
              stride_x_row, stride_res_row, stride_gate_row, stride_h_row, stride_y_row, M, N,
              eps, unit_offset ? 1.f : 0.f, dtype, rdtype, wdtype};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case XK_F32: return run_fwd_f32(p, s);
    case XK_BF16: return run_fwd_bf16(p, s);
    default: return run_fwd_f16(p, s);
  }
}

extern "C" int64_t xk_gated_residual_rms_norm_bwd_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0 || N >= resnorm::kMostRow) return 0;
  // The parts of the types with 4 and 8 elements a lane.
  return std::max(resnorm::sum_parts(M, N, 4), resnorm::sum_parts(M, N, 8)) * 3 *
         resnorm::part_pitch(N) * 4;
}

extern "C" int xk_gated_residual_rms_norm_bwd(
    const void* dh, int64_t stride_dh_row, const void* dy, int64_t stride_dy_row, const void* x,
    int64_t stride_x_row, const void* residual, int64_t stride_res_row, const void* gate,
    int64_t stride_gate_row, const void* post_weight, const void* scale, const void* pre_weight,
    const float* rstd_post, const float* rstd_pre, void* dx, int64_t stride_dx_row,
    void* dresidual, int64_t stride_dres_row, void* dgate, int64_t stride_dgate_row,
    void* dpost_weight, void* dscale, void* dpre_weight, int64_t M, int64_t N, int unit_offset,
    xk_dtype dtype, xk_dtype rdtype, xk_dtype wdtype, void* workspace, size_t workspace_bytes,
    void* stream) {
  using namespace resnorm;
  if (M < 0 || N <= 0 || N >= kMostRow) return XK_ERR_INVALID;
  if (!is_float_dtype(dtype) || (rdtype != dtype && rdtype != XK_F32) ||
      (wdtype != dtype && wdtype != XK_F32))
    return XK_ERR_UNSUPPORTED;
  if ((dpost_weight && !post_weight) || (dscale && !scale) || (dpre_weight && !pre_weight) ||
      (dgate && !gate) || (dy && !pre_weight))
    return XK_ERR_INVALID;
  const int sums = (dpost_weight ? 1 : 0) | (dscale ? 2 : 0) | (dpre_weight ? 4 : 0);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t parts = sum_parts(M, N, 16 / elem_bytes(dtype));
  if (M > 0) {
    if (!x || !residual || (!dh && !dy) || (post_weight && !rstd_post) || (dy && !rstd_pre))
      return XK_ERR_INVALID;
    if (M > 1 &&
        (pitch_bad(dh, stride_dh_row, N) || pitch_bad(dy, stride_dy_row, N) ||
         pitch_bad(x, stride_x_row, N) || pitch_bad(residual, stride_res_row, N) ||
         pitch_bad(gate, stride_gate_row, N) || pitch_bad(dx, stride_dx_row, N) ||
         pitch_bad(dresidual, stride_dres_row, N) || pitch_bad(dgate, stride_dgate_row, N)))
      return XK_ERR_INVALID;
    if (sums && (!workspace || !aligned(workspace, 256) ||
                 workspace_bytes <
                     static_cast<size_t>(xk_gated_residual_rms_norm_bwd_workspace_bytes(M, N))))
      return XK_ERR_WORKSPACE;
    BwdParams p{dh, dy, x, residual, gate, post_weight, scale, pre_weight, rstd_post, rstd_pre,
                dx, dresidual, dgate, static_cast<float*>(workspace), parts, sums,
                stride_dh_row, stride_dy_row, stride_x_row, stride_res_row, stride_gate_row,
                stride_dx_row, stride_dres_row, stride_dgate_row, M, N,
                unit_offset ? 1.f : 0.f, dtype, rdtype, wdtype};
    int st = dtype == XK_F32 ? run_bwd_f32(p, s)
                             : (dtype == XK_BF16 ? run_bwd_bf16(p, s) : run_bwd_f16(p, s));
    if (st != XK_OK) return st;
  }
  if (sums) {
    hipLaunchKernelGGL(sums_kernel, dim3(cdiv(N, kSumCols), 3), dim3(256), 0, s,
                       static_cast<const float*>(workspace), parts, N, dpost_weight, dscale,
                       dpre_weight, wdtype);
    return launch_status();
  }
  return XK_OK;
}
