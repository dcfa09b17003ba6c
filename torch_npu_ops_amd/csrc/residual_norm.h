// Kernels of the step from one block to the next (norm, gate, residual scale,
// residual sum, norm) and of its backward pass, templates over the element
// type T of the block's tensors, RT of the residual stream and WT of the
// weights; residual_norm_*.hip instantiate one T each.
//
//   n = x rstd1 w1', v = n silu(z), h = residual + scale v, y = h rstd2 w2'
//
// HBM-bound: forward reads x, residual, gate and writes h, y once (10 bytes
// per element at 16 bits), backward reads dh, dy, x, residual, gate and writes
// dx, dresidual, dgate (16 bytes).
//  * A team of TPR lanes owns a row and holds it in registers as vectors of
//    VEC elements, NV per lane, so both norms' sums and the outputs take one
//    read.  Vectors are read wherever they start (rows of odd length or
//    offset included): only a row's last, partial vector goes by elements.
//  * Parts that a call leaves out are uniform branches on their pointers.
#pragma once

#include <algorithm>

#include "xk_common.h"

namespace xk {
namespace resnorm {

struct FwdParams {
  const void* x;
  const void* res;
  const void* gate;
  const void* post;
  const void* scale;
  const void* pre;
  void* h;
  void* y;
  float* r1;
  float* r2;
  int64_t sx, sres, sgate, sh, sy;
  int64_t M, N;
  float eps, off;
  xk_dtype dt, rdt, wdt;  // read by the streaming kernels only
};

struct BwdParams {
  const void* dh;
  const void* dy;
  const void* x;
  const void* res;
  const void* gate;
  const void* post;
  const void* scale;
  const void* pre;
  const float* r1;
  const float* r2;
  void* dx;
  void* dres;
  void* dgate;
  float* part;  // [parts][3][N]: sums for post, scale, pre
  int64_t parts;
  int sums;  // bit 0: post, 1: scale, 2: pre
  int64_t sdh, sdy, sx, sres, sgate, sdx, sdres, sdgate;
  int64_t M, N;
  float off;
  xk_dtype dt, rdt, wdt;
};

// Parts that the backward pass's column sums are split into: a row at least
// for each; a team works on one part.
inline int64_t sum_parts(int64_t M, int64_t N) {
  const int64_t cap = N > 8192 ? 256 : (N > 1024 ? 512 : 2048);
  return M < cap ? M : cap;
}

// VEC elements from any address.
template <typename T, int VEC>
struct Row {
  T v[VEC];
};
typedef unsigned int u32;
template <int BYTES, int ALIGN> struct RawAt { using type = void; };
template <> struct RawAt<32, 4> { typedef u32x4 type __attribute__((aligned(4))); };
template <> struct RawAt<16, 4> { typedef u32x4 type __attribute__((aligned(4))); };
template <> struct RawAt<16, 2> { typedef u32x4 type __attribute__((aligned(2))); };

template <typename T, int VEC>
__device__ __forceinline__ Row<T, VEC> ld_at(const T* p) {
  Row<T, VEC> out;
  constexpr int kBytes = VEC * sizeof(T), kChunk = 16, kPer = kChunk / sizeof(T);
  using U = typename RawAt<kChunk, sizeof(T)>::type;
#pragma unroll
  for (int c = 0; c < kBytes / kChunk; ++c) {
    const u32x4 r = __builtin_nontemporal_load(reinterpret_cast<const U*>(p + c * kPer));
    __builtin_memcpy(&out.v[c * kPer], &r, kChunk);
  }
  return out;
}
template <typename T, int VEC>
__device__ __forceinline__ void st_at(T* p, const Row<T, VEC>& in) {
  constexpr int kBytes = VEC * sizeof(T), kChunk = 16, kPer = kChunk / sizeof(T);
  using U = typename RawAt<kChunk, sizeof(T)>::type;
#pragma unroll
  for (int c = 0; c < kBytes / kChunk; ++c) {
    u32x4 r;
    __builtin_memcpy(&r, &in.v[c * kPer], kChunk);
    __builtin_nontemporal_store(r, reinterpret_cast<U*>(p + c * kPer));
  }
}
// The same with `left` elements of the row left (may be <= 0): zeros beyond.
template <typename T, int VEC>
__device__ __forceinline__ Row<T, VEC> ld_row(const T* p, int left) {
  if (left >= VEC) return ld_at<T, VEC>(p);
  Row<T, VEC> out;
#pragma unroll
  for (int u = 0; u < VEC; ++u) out.v[u] = u < left ? p[u] : from_f32<T>(0.f);
  return out;
}
template <typename T, int VEC>
__device__ __forceinline__ void st_row(T* p, const Row<T, VEC>& in, int left) {
  if (left >= VEC) {
    st_at<T, VEC>(p, in);
  } else {
#pragma unroll
    for (int u = 0; u < VEC; ++u)
      if (u < left) p[u] = in.v[u];
  }
}
// Weights are read again by every row and stay in the caches.
template <typename W, int VEC>
__device__ __forceinline__ Row<W, VEC> ld_weight(const void* base, int at, int left) {
  const W* p = static_cast<const W*>(base) + at;
  Row<W, VEC> out;
  if (left >= VEC) {
    constexpr int kPer = 16 / sizeof(W);
    using U = typename RawAt<16, sizeof(W)>::type;
#pragma unroll
    for (int c = 0; c < VEC / kPer; ++c) {
      const u32x4 r = *reinterpret_cast<const U*>(p + c * kPer);
      __builtin_memcpy(&out.v[c * kPer], &r, 16);
    }
  } else {
#pragma unroll
    for (int u = 0; u < VEC; ++u) out.v[u] = u < left ? p[u] : from_f32<W>(0.f);
  }
  return out;
}

// Sum over the TPR lanes of a team.  Teams wider than a wave are the whole
// block and exchange through `red`; `turn` alternates between two halves of
// it, so one barrier a sum is enough.
template <int TPR>
__device__ __forceinline__ float team_sum(float v, float* red, int turn) {
  v = group_sum<kWave>(v);
  if constexpr (TPR > kWave) {
    constexpr int kWaves = TPR / kWave;
    float* at = red + turn * kWaves;
    if (threadIdx.x % kWave == 0) at[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += at[w];
  }
  return v;
}

template <int TPR>
constexpr int block_of() { return TPR > 256 ? TPR : 256; }

template <typename T, typename RT, typename WT, int TPR, int NV>
__global__ void __launch_bounds__(block_of<TPR>()) fwd_kernel(FwdParams p) {
  constexpr int VEC = 16 / sizeof(T), kTeams = block_of<TPR>() / TPR;
  __shared__ float red[2 * (TPR > kWave ? TPR / kWave : 1)];
  const int lane = threadIdx.x % TPR, N = static_cast<int>(p.N);
  const float inv_n = 1.f / static_cast<float>(p.N);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTeams;
  // A team that is a wave runs its own rows; a wider one is the block, whose
  // lanes share the loop's bounds.
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kTeams + threadIdx.x / TPR; row < p.M;
       row += step) {
    const T* xr = static_cast<const T*>(p.x) + row * p.sx;
    const RT* rr = static_cast<const RT*>(p.res) + row * p.sres;
    const T* zr = static_cast<const T*>(p.gate) + row * p.sgate;
    Row<T, VEC> x[NV], z[NV];
    Row<RT, VEC> res[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * TPR + lane) * VEC;
      x[j] = ld_row<T, VEC>(xr + at, N - at);
      res[j] = ld_row<RT, VEC>(rr + at, N - at);
      if (p.gate) z[j] = ld_row<T, VEC>(zr + at, N - at);
    }
    float r1 = 1.f;
    if (p.post) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
          const float f = to_f32(x[j].v[u]);
          ss = fmaf(f, f, ss);
        }
      r1 = 1.f / sqrtf(team_sum<TPR>(ss, red, 0) * inv_n + p.eps);
      if (p.r1 && lane == 0) p.r1[row] = r1;
    }
    float h[NV][VEC], ss = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * TPR + lane) * VEC;
#pragma unroll
      for (int u = 0; u < VEC; ++u) h[j][u] = to_f32(x[j].v[u]);
      if (p.post) {
        const Row<WT, VEC> w = ld_weight<WT, VEC>(p.post, at, N - at);
#pragma unroll
        for (int u = 0; u < VEC; ++u) h[j][u] *= r1 * (to_f32(w.v[u]) + p.off);
      }
      if (p.gate) {
#pragma unroll
        for (int u = 0; u < VEC; ++u) h[j][u] *= silu(to_f32(z[j].v[u]));
      }
      if (p.scale) {
        const Row<WT, VEC> w = ld_weight<WT, VEC>(p.scale, at, N - at);
#pragma unroll
        for (int u = 0; u < VEC; ++u) h[j][u] *= to_f32(w.v[u]);
      }
      Row<RT, VEC> out;
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        h[j][u] += to_f32(res[j].v[u]);
        ss = fmaf(h[j][u], h[j][u], ss);
        out.v[u] = from_f32<RT>(h[j][u]);
      }
      st_row<RT, VEC>(static_cast<RT*>(p.h) + row * p.sh + at, out, N - at);
    }
    if (p.pre) {
      const float r2 = 1.f / sqrtf(team_sum<TPR>(ss, red, 1) * inv_n + p.eps);
      if (p.r2 && lane == 0) p.r2[row] = r2;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int at = (j * TPR + lane) * VEC;
        const Row<WT, VEC> w = ld_weight<WT, VEC>(p.pre, at, N - at);
        Row<T, VEC> out;
#pragma unroll
        for (int u = 0; u < VEC; ++u)
          out.v[u] = from_f32<T>(h[j][u] * r2 * (to_f32(w.v[u]) + p.off));
        st_row<T, VEC>(static_cast<T*>(p.y) + row * p.sy + at, out, N - at);
      }
    }
    // One barrier more where only one of the two sums runs: its half of `red`
    // is the next row's too.
    if constexpr (TPR > kWave) {
      if (!p.post || !p.pre) __syncthreads();
    }
  }
}

template <typename T, typename RT, typename WT, int TPR, int NV>
__global__ void __launch_bounds__(block_of<TPR>()) bwd_kernel(BwdParams p) {
  constexpr int VEC = 16 / sizeof(T), kTeams = block_of<TPR>() / TPR;
  __shared__ float red[2 * (TPR > kWave ? TPR / kWave : 1)];
  const int lane = threadIdx.x % TPR, N = static_cast<int>(p.N);
  const float inv_n = 1.f / static_cast<float>(p.N);
  const int64_t team = static_cast<int64_t>(blockIdx.x) * kTeams + threadIdx.x / TPR;
  float a_post[NV][VEC] = {}, a_scale[NV][VEC] = {}, a_pre[NV][VEC] = {};
  for (int64_t row = team; team < p.parts && row < p.M; row += p.parts) {
    Row<T, VEC> x[NV], z[NV], dy[NV];
    Row<RT, VEC> res[NV], dh[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * TPR + lane) * VEC;
      x[j] = ld_row<T, VEC>(static_cast<const T*>(p.x) + row * p.sx + at, N - at);
      res[j] = ld_row<RT, VEC>(static_cast<const RT*>(p.res) + row * p.sres + at, N - at);
      if (p.gate) z[j] = ld_row<T, VEC>(static_cast<const T*>(p.gate) + row * p.sgate + at, N - at);
      if (p.dy) dy[j] = ld_row<T, VEC>(static_cast<const T*>(p.dy) + row * p.sdy + at, N - at);
      if (p.dh) dh[j] = ld_row<RT, VEC>(static_cast<const RT*>(p.dh) + row * p.sdh + at, N - at);
    }
    const float r1 = p.post ? p.r1[row] : 1.f;
    const float r2 = p.dy ? p.r2[row] : 0.f;
    // h rstd2, and the mean of it with w2' dy.
    float d[NV][VEC], ss = 0.f;  // d: w2' dy, then dH, then w1' dn
    auto branch = [&](int j, int u, const Row<WT, VEC>& w1, float& xh, float& n, float& sg) {
      xh = to_f32(x[j].v[u]) * r1;
      n = p.post ? xh * (to_f32(w1.v[u]) + p.off) : xh;
      sg = p.gate ? sigmoid(to_f32(z[j].v[u])) : 1.f;
      return p.gate ? n * to_f32(z[j].v[u]) * sg : n;
    };
    if (p.dy) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int at = (j * TPR + lane) * VEC;
        Row<WT, VEC> w1, sc;
        if (p.post) w1 = ld_weight<WT, VEC>(p.post, at, N - at);
        if (p.scale) sc = ld_weight<WT, VEC>(p.scale, at, N - at);
        const Row<WT, VEC> w2 = ld_weight<WT, VEC>(p.pre, at, N - at);
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
          float xh, n, sg;
          const float v = branch(j, u, w1, xh, n, sg);
          const float hh = fmaf(p.scale ? to_f32(sc.v[u]) : 1.f, v, to_f32(res[j].v[u])) * r2;
          const float g = to_f32(dy[j].v[u]);
          a_pre[j][u] = fmaf(g, hh, a_pre[j][u]);
          d[j][u] = g * (to_f32(w2.v[u]) + p.off);
          ss = fmaf(d[j][u], hh, ss);
        }
      }
      ss = team_sum<TPR>(ss, red, 0) * inv_n;
    }
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * TPR + lane) * VEC;
      Row<WT, VEC> w1, sc;
      if (p.post) w1 = ld_weight<WT, VEC>(p.post, at, N - at);
      if (p.scale) sc = ld_weight<WT, VEC>(p.scale, at, N - at);
      Row<RT, VEC> o_res;
      Row<T, VEC> o_gate;
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        float xh, n, sg;
        const float v = branch(j, u, w1, xh, n, sg);
        const float s = p.scale ? to_f32(sc.v[u]) : 1.f;
        float g = 0.f;
        if (p.dy) g = r2 * (d[j][u] - fmaf(s, v, to_f32(res[j].v[u])) * r2 * ss);
        if (p.dh) g += to_f32(dh[j].v[u]);
        o_res.v[u] = from_f32<RT>(g);
        a_scale[j][u] = fmaf(g, v, a_scale[j][u]);
        g *= s;
        if (p.gate) {
          const float zf = to_f32(z[j].v[u]);
          o_gate.v[u] = from_f32<T>(g * n * sg * fmaf(zf, 1.f - sg, 1.f));
          g *= zf * sg;
        }
        if (p.post) {
          a_post[j][u] = fmaf(g, xh, a_post[j][u]);
          g *= to_f32(w1.v[u]) + p.off;
          dot = fmaf(g, xh, dot);
        }
        d[j][u] = g;
      }
      if (p.dres) st_row<RT, VEC>(static_cast<RT*>(p.dres) + row * p.sdres + at, o_res, N - at);
      if (p.gate && p.dgate)
        st_row<T, VEC>(static_cast<T*>(p.dgate) + row * p.sdgate + at, o_gate, N - at);
    }
    if (p.post) dot = team_sum<TPR>(dot, red, 1) * inv_n;
    if (p.dx) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int at = (j * TPR + lane) * VEC;
        Row<T, VEC> out;
#pragma unroll
        for (int u = 0; u < VEC; ++u)
          out.v[u] = from_f32<T>(
              p.post ? r1 * (d[j][u] - to_f32(x[j].v[u]) * r1 * dot) : d[j][u]);
        st_row<T, VEC>(static_cast<T*>(p.dx) + row * p.sdx + at, out, N - at);
      }
    }
    if constexpr (TPR > kWave) {
      if (!p.post || !p.dy) __syncthreads();
    }
  }
  if (p.sums && team < p.parts) {
    float* out = p.part + team * 3 * p.N;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        const int at = (j * TPR + lane) * VEC + u;
        if (at < N) {
          if (p.sums & 1) out[at] = a_post[j][u];
          if (p.sums & 2) out[p.N + at] = a_scale[j][u];
          if (p.sums & 4) out[2 * p.N + at] = a_pre[j][u];
        }
      }
  }
}

template <typename T, typename RT, typename WT, int TPR, int NV>
int launch_fwd(const FwdParams& p, hipStream_t s) {
  constexpr int kTeams = block_of<TPR>() / TPR;
  const int64_t most = static_cast<int64_t>(num_cus()) * (2048 / block_of<TPR>());
  const int64_t grid = std::min(cdiv(p.M, kTeams), most);
  hipLaunchKernelGGL((fwd_kernel<T, RT, WT, TPR, NV>), dim3(grid), dim3(block_of<TPR>()), 0, s,
                     p);
  return launch_status();
}

template <typename T, typename RT, typename WT, int TPR, int NV>
int launch_bwd(const BwdParams& p, hipStream_t s) {
  constexpr int kTeams = block_of<TPR>() / TPR;
  hipLaunchKernelGGL((bwd_kernel<T, RT, WT, TPR, NV>), dim3(cdiv(p.parts, kTeams)),
                     dim3(block_of<TPR>()), 0, s, p);
  return launch_status();
}

// Rows of any length, one block each, read as often as needed: only for rows
// longer than a block holds (above 32K elements at 16 bits).
int stream_fwd(const FwdParams& p, hipStream_t s);
int stream_bwd(const BwdParams& p, hipStream_t s);

template <typename T, typename RT, typename WT>
int run_fwd_w(const FwdParams& p, hipStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t nvec = cdiv(p.N, VEC);
  if (nvec <= 64) return launch_fwd<T, RT, WT, 64, 1>(p, s);
  if (nvec <= 128) return launch_fwd<T, RT, WT, 64, 2>(p, s);
  if (nvec <= 256) return launch_fwd<T, RT, WT, 256, 1>(p, s);
  if (nvec <= 512) return launch_fwd<T, RT, WT, 256, 2>(p, s);
  if (nvec <= 1024) return launch_fwd<T, RT, WT, 1024, 1>(p, s);
  if (nvec <= 2048) return launch_fwd<T, RT, WT, 1024, 2>(p, s);
  if (nvec <= 4096) return launch_fwd<T, RT, WT, 1024, 4>(p, s);
  return stream_fwd(p, s);
}

template <typename T, typename RT, typename WT>
int run_bwd_w(const BwdParams& p, hipStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t nvec = cdiv(p.N, VEC);
  if (nvec <= 64) return launch_bwd<T, RT, WT, 64, 1>(p, s);
  if (nvec <= 128) return launch_bwd<T, RT, WT, 64, 2>(p, s);
  if (nvec <= 256) return launch_bwd<T, RT, WT, 256, 1>(p, s);
  if (nvec <= 512) return launch_bwd<T, RT, WT, 256, 2>(p, s);
  if (nvec <= 1024) return launch_bwd<T, RT, WT, 1024, 1>(p, s);
  return stream_bwd(p, s);
}

template <typename T>
int run_fwd(const FwdParams& p, hipStream_t s) {
  const bool r32 = p.rdt != p.dt, w32 = p.wdt != p.dt;
  if constexpr (std::is_same<T, float>::value) {
    return run_fwd_w<T, T, T>(p, s);
  } else {
    if (r32) return w32 ? run_fwd_w<T, float, float>(p, s) : run_fwd_w<T, float, T>(p, s);
    return w32 ? run_fwd_w<T, T, float>(p, s) : run_fwd_w<T, T, T>(p, s);
  }
}
template <typename T>
int run_bwd(const BwdParams& p, hipStream_t s) {
  const bool r32 = p.rdt != p.dt, w32 = p.wdt != p.dt;
  if constexpr (std::is_same<T, float>::value) {
    return run_bwd_w<T, T, T>(p, s);
  } else {
    if (r32) return w32 ? run_bwd_w<T, float, float>(p, s) : run_bwd_w<T, float, T>(p, s);
    return w32 ? run_bwd_w<T, T, float>(p, s) : run_bwd_w<T, T, T>(p, s);
  }
}

int run_fwd_f32(const FwdParams& p, hipStream_t s);
int run_fwd_bf16(const FwdParams& p, hipStream_t s);
int run_fwd_f16(const FwdParams& p, hipStream_t s);
int run_bwd_f32(const BwdParams& p, hipStream_t s);
int run_bwd_bf16(const BwdParams& p, hipStream_t s);
int run_bwd_f16(const BwdParams& p, hipStream_t s);

}  // namespace resnorm
}  // namespace xk
