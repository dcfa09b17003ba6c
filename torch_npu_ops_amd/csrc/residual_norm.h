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
//    offset included); a row's last one overlaps the one before it where the
//    row ends inside a lane.
//  * Parts that a call leaves out are uniform branches on their pointers.
//
// 16,384 x 4,096 bf16 forward 125 us (671 MB, 5.4 TB/s, 87% of a plain copy);
// 8,192 x 4,096 with an fp32 residual 91 us forward, 134 backward and 9.5 for
// the sums over the rows.
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
  float* part;  // [parts][3][part_pitch(N)]: sums for post, scale, pre
  int64_t parts;
  int sums;  // bit 0: post, 1: scale, 2: pre
  int64_t sdh, sdy, sx, sres, sgate, sdx, sdres, sdgate;
  int64_t M, N;
  float off;
  xk_dtype dt, rdt, wdt;
};

// Lanes that hold a row in the backward pass, 16 bytes of x each (0: the row
// is too long for a block).
inline int bwd_lanes(int64_t N, int vec) {
  const int64_t nvec = cdiv(N, vec);
  return nvec <= 64 ? 64 : nvec <= 128 ? 128 : nvec <= 256 ? 256 : nvec <= 512 ? 512
                                                              : nvec <= 1024 ? 1024 : 0;
}
// Parts that the backward pass's column sums are split into: a row at least
// for each, and one for every team that the chip holds (1024 lanes a compute
// unit).  Half as many leave half of the lanes idle: 8,192 x 4,096 180 us and
// 5 for the sums, 1,001 x 2,500 30 and 4.5, against 140 + 9.6 and 24 + 6.5.
inline int64_t sum_parts(int64_t M, int64_t N, int vec) {
  const int lanes = bwd_lanes(N, vec);
  const int64_t cap = 256 * (lanes ? 1024 / lanes : 1);
  return M < cap ? M : cap;
}
// Floats from one row of parts to the next: whole lanes of 16-bit rows.
__host__ __device__ inline int64_t part_pitch(int64_t N) { return (N + 7) / 8 * 8; }

// VEC elements of a row as the words they were loaded in: unpacked where they
// are used, which costs less than holding them in fp32.
template <typename T, int VEC>
struct Row {
  static constexpr int kWords = VEC * sizeof(T) / 4, kPer = 4 / sizeof(T);
  unsigned int w[kWords];
  __device__ __forceinline__ float operator[](int u) const {
    const unsigned int r = w[u / kPer];
    if constexpr (sizeof(T) == 4) {
      return __builtin_bit_cast(float, r);
    } else if constexpr (std::is_same<T, bf16>::value) {
      return __builtin_bit_cast(float, u & 1 ? r & 0xffff0000u : r << 16);
    } else {
      return to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(u & 1 ? r >> 16 : r)));
    }
  }
  // From here on the elements are unpacked again: keeps the compiler from
  // holding an earlier use's fp32 values in registers.
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(w[i]));
  }
};
template <typename T, int VEC>
__device__ __forceinline__ Row<T, VEC> pack(const float (&v)[VEC]) {
  Arr<T, VEC> t;
#pragma unroll
  for (int u = 0; u < VEC; ++u) t.v[u] = from_f32<T>(v[u]);
  return __builtin_bit_cast(Row<T, VEC>, t);
}

// A lane's elements of a row: VEC of them from `at`, or the row's last VEC where
// it ends inside them (TAIL; N >= VEC): the first `twice` of those are the
// lane's before it, which count in no sum and are not written (where h lies over
// the residual they may have changed).  Rows of 3,316 take 28.5 us forward and
// 71 backward, of 3,312 27 and 57 (3,686 rows); with the last elements loaded
// one by one 39 and 81.
// `left`: its own elements if positive and below VEC, nothing if not.
template <int VEC, bool TAIL>
struct Place {
  int at, left, twice;
  __device__ __forceinline__ Place(int first, int N)
      : at(TAIL && first > N - VEC ? N - VEC : first), left(N - first), twice(first - at) {}
  // The sum with element u, or without it.
  __device__ __forceinline__ float own(int u, float with, float without) const {
    return TAIL && u < twice ? without : with;
  }
};

// Moves of a lane's elements, 16 bytes at a time and at any address.  Loads
// give zeros to lanes without elements.  STREAM: read or written once.
typedef u32x4 Word4At2 __attribute__((aligned(2)));
typedef u32x4 Word4At4 __attribute__((aligned(4)));
template <typename T>
using Word4 = typename std::conditional<sizeof(T) == 2, const Word4At2*, const Word4At4*>::type;
template <typename T>
using Word4Out = typename std::conditional<sizeof(T) == 2, Word4At2*, Word4At4*>::type;

template <typename T, int VEC, bool TAIL, bool STREAM = true>
__device__ __forceinline__ Row<T, VEC> ld_row(const T* row, const Place<VEC, TAIL>& l) {
  Row<T, VEC> out{};
  if (l.left > 0) {
#pragma unroll
    for (int c = 0; c < out.kWords / 4; ++c) {
      const Word4<T> q = reinterpret_cast<Word4<T>>(row + l.at + c * (16 / sizeof(T)));
      u32x4 r;
      if constexpr (STREAM)
        r = __builtin_nontemporal_load(q);
      else
        r = *q;
      out.w[4 * c] = r.x;
      out.w[4 * c + 1] = r.y;
      out.w[4 * c + 2] = r.z;
      out.w[4 * c + 3] = r.w;
    }
  }
  return out;
}
template <typename T, int VEC, bool TAIL>
__device__ __forceinline__ void st_row(T* row, const Row<T, VEC>& in, const Place<VEC, TAIL>& l) {
  T* p = row + l.at;
  if (l.left >= VEC) {
#pragma unroll
    for (int c = 0; c < in.kWords / 4; ++c) {
      const u32x4 r = {in.w[4 * c], in.w[4 * c + 1], in.w[4 * c + 2], in.w[4 * c + 3]};
      __builtin_nontemporal_store(r, reinterpret_cast<Word4Out<T>>(p + c * (16 / sizeof(T))));
    }
  } else if constexpr (TAIL) {
    if (l.left > 0) {
      const Arr<T, VEC> t = __builtin_bit_cast(Arr<T, VEC>, in);
#pragma unroll
      for (int u = 1; u < VEC; ++u)
        if (u >= l.twice) p[u] = t.v[u];
    }
  }
}
// Weights are read again by every row and stay in the caches.
template <typename W, int VEC, bool TAIL>
__device__ __forceinline__ Row<W, VEC> ld_weight(const void* base, const Place<VEC, TAIL>& l) {
  return ld_row<W, VEC, TAIL, false>(static_cast<const W*>(base), l);
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

// Teams of a wave share blocks of four; wider ones are a block.
template <int TPR>
constexpr int block_of() { return TPR > kWave ? TPR : 256; }

// FULL: every part is there, with no branches on them.
template <typename T, typename RT, typename WT, int TPR, int NV, bool FULL, bool TAIL>
__global__ void __launch_bounds__(block_of<TPR>()) fwd_kernel(FwdParams p) {
  constexpr int VEC = 16 / sizeof(T), kTeams = block_of<TPR>() / TPR;
  __shared__ float red[2 * (TPR > kWave ? TPR / kWave : 1)];
  const bool post = FULL || p.post, gate = FULL || p.gate, scale = FULL || p.scale,
             pre = FULL || p.pre;
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
    Row<WT, VEC> w1[NV], w2[NV], sc[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Place<VEC, TAIL> l((j * TPR + lane) * VEC, N);
      x[j] = ld_row<T, VEC, TAIL>(xr, l);
      if (gate) z[j] = ld_row<T, VEC, TAIL>(zr, l);
      res[j] = ld_row<RT, VEC, TAIL>(rr, l);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Place<VEC, TAIL> l((j * TPR + lane) * VEC, N);
      if (post) w1[j] = ld_weight<WT, VEC, TAIL>(p.post, l);
      if (scale) sc[j] = ld_weight<WT, VEC, TAIL>(p.scale, l);
      if (pre) w2[j] = ld_weight<WT, VEC, TAIL>(p.pre, l);
    }
    float r1 = 1.f;
    if (post) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const Place<VEC, TAIL> l((j * TPR + lane) * VEC, N);
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
          const float f = x[j][u];
          ss = l.own(u, fmaf(f, f, ss), ss);
        }
      }
      r1 = 1.f / sqrtf(team_sum<TPR>(ss, red, 0) * inv_n + p.eps);
      if (p.r1 && lane == 0) p.r1[row] = r1;
    }
    float h[NV][VEC], ss = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Place<VEC, TAIL> l((j * TPR + lane) * VEC, N);
      float out[VEC];
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        float v = x[j][u];
        if (post) v *= r1 * (w1[j][u] + p.off);
        if (gate) v *= silu(z[j][u]);
        v = scale ? fmaf(v, sc[j][u], res[j][u]) : v + res[j][u];
        h[j][u] = out[u] = v;
        ss = l.own(u, fmaf(v, v, ss), ss);
      }
      st_row<RT, VEC, TAIL>(static_cast<RT*>(p.h) + row * p.sh, pack<RT, VEC>(out), l);
    }
    if (pre) {
      const float r2 = 1.f / sqrtf(team_sum<TPR>(ss, red, 1) * inv_n + p.eps);
      if (p.r2 && lane == 0) p.r2[row] = r2;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const Place<VEC, TAIL> l((j * TPR + lane) * VEC, N);
        float out[VEC];
#pragma unroll
        for (int u = 0; u < VEC; ++u) out[u] = h[j][u] * r2 * (w2[j][u] + p.off);
        st_row<T, VEC, TAIL>(static_cast<T*>(p.y) + row * p.sy, pack<T, VEC>(out), l);
      }
    }
    // One barrier more where only one of the two sums runs: its half of `red`
    // is the next row's too.
    if constexpr (TPR > kWave) {
      if (!post || !pre) __syncthreads();
    }
  }
}

// Backward: a team walks every parts-th row and keeps the column sums of its
// elements in registers.  Per row: h and rstd2's sum from x, gate, residual;
// then dh's total, the gate's and the branch's gradients and rstd1's sum; then
// dx.  The sigmoid is kept between the passes, the cheap products are formed
// again.  fp32 weights beside 16-bit rows hold 24 more registers over the rows, and
// 7 to 14 are spilled (rows that end inside a vector: 4 to 76, with weights of the
// rows' type 4 to 12): 8,192 x 4,096 bf16 132 us, with bf16 weights 112.  All three
// column sums are formed and written where one is asked for.
template <typename T, typename RT, typename WT, int TPR, bool TAIL>
__global__ void __launch_bounds__(block_of<TPR>(), 4) bwd_kernel(BwdParams p) {
  constexpr int VEC = 16 / sizeof(T), kTeams = block_of<TPR>() / TPR;
  __shared__ float red[2 * (TPR > kWave ? TPR / kWave : 1)];
  const bool post = p.post, gate = p.gate, scale = p.scale, has_dy = p.dy, has_dh = p.dh;
  const int lane = threadIdx.x % TPR, N = static_cast<int>(p.N);
  const Place<VEC, TAIL> l(lane * VEC, N);
  const float inv_n = 1.f / static_cast<float>(p.N);
  const int64_t team = static_cast<int64_t>(blockIdx.x) * kTeams + threadIdx.x / TPR;
  float a_post[VEC] = {}, a_scale[VEC] = {}, a_pre[VEC] = {};
  Row<WT, VEC> w1{}, w2{}, sc{};
  if (post) w1 = ld_weight<WT, VEC, TAIL>(p.post, l);
  if (has_dy) w2 = ld_weight<WT, VEC, TAIL>(p.pre, l);
  if (scale) sc = ld_weight<WT, VEC, TAIL>(p.scale, l);
  for (int64_t row = team; team < p.parts && row < p.M; row += p.parts) {
    Row<T, VEC> x, z{}, dy{};
    Row<RT, VEC> res{}, dh{};
    w1.again();
    w2.again();
    sc.again();
    x = ld_row<T, VEC, TAIL>(static_cast<const T*>(p.x) + row * p.sx, l);
    if (gate) z = ld_row<T, VEC, TAIL>(static_cast<const T*>(p.gate) + row * p.sgate, l);
    if (has_dy) {
      dy = ld_row<T, VEC, TAIL>(static_cast<const T*>(p.dy) + row * p.sdy, l);
      res = ld_row<RT, VEC, TAIL>(static_cast<const RT*>(p.res) + row * p.sres, l);
    }
    if (has_dh) dh = ld_row<RT, VEC, TAIL>(static_cast<const RT*>(p.dh) + row * p.sdh, l);
    const float r1 = post ? p.r1[row] : 1.f;
    const float r2 = has_dy ? p.r2[row] : 0.f;
    float sg[VEC], hh[VEC], ss = 0.f;  // hh: h rstd2, then w1' dn
    // n = x rstd1 w1' and v = n z sigmoid(z) of an element.
    auto norm_of = [&](int u) {
      const float f = x[u] * r1;
      return post ? f * (w1[u] + p.off) : f;
    };
#pragma unroll
    for (int u = 0; u < VEC; ++u) {
      if (gate) sg[u] = sigmoid(z[u]);
      if (has_dy) {
        float v = norm_of(u);
        if (gate) v *= z[u] * sg[u];
        hh[u] = (scale ? fmaf(v, sc[u], res[u]) : v + res[u]) * r2;
        const float g = dy[u];
        a_pre[u] = fmaf(g, hh[u], a_pre[u]);
        ss = l.own(u, fmaf(g * (w2[u] + p.off), hh[u], ss), ss);
      }
    }
    if (has_dy) ss = team_sum<TPR>(ss, red, 0) * inv_n;
    float dot = 0.f;
    x.again();
    z.again();
    dy.again();
    w1.again();
    w2.again();
    sc.again();
    float o_res[VEC], o_gate[VEC];
#pragma unroll
    for (int u = 0; u < VEC; ++u) {
      const float xh = x[u] * r1, n = norm_of(u);
      float g = has_dh ? dh[u] : 0.f;
      if (has_dy)
        g = fmaf(r2, fmaf(dy[u], w2[u] + p.off, -hh[u] * ss), g);
      o_res[u] = g;
      const float silu_z = gate ? z[u] * sg[u] : 1.f;
      a_scale[u] = fmaf(g, n * silu_z, a_scale[u]);
      if (scale) g *= sc[u];
      if (gate) {
        o_gate[u] = g * n * fmaf(silu_z, 1.f - sg[u], sg[u]);
        g *= silu_z;
      }
      if (post) {
        a_post[u] = fmaf(g, xh, a_post[u]);
        g *= w1[u] + p.off;
        dot = l.own(u, fmaf(g, xh, dot), dot);
      }
      hh[u] = g;
    }
    if (p.dres)
      st_row<RT, VEC, TAIL>(static_cast<RT*>(p.dres) + row * p.sdres, pack<RT, VEC>(o_res), l);
    if (gate && p.dgate)
      st_row<T, VEC, TAIL>(static_cast<T*>(p.dgate) + row * p.sdgate, pack<T, VEC>(o_gate), l);
    if (post) dot = team_sum<TPR>(dot, red, 1) * inv_n;
    if (p.dx) {
      x.again();
      float out[VEC];
#pragma unroll
      for (int u = 0; u < VEC; ++u) out[u] = post ? r1 * fmaf(x[u] * -r1, dot, hh[u]) : hh[u];
      st_row<T, VEC, TAIL>(static_cast<T*>(p.dx) + row * p.sdx, pack<T, VEC>(out), l);
    }
    if constexpr (TPR > kWave) {
      if (!post || !has_dy) __syncthreads();
    }
  }
  if (p.sums && team < p.parts && l.left > 0) {
    const int64_t pitch = part_pitch(p.N);
    float* out = p.part + team * 3 * pitch + l.at;
    auto put = [&](const float (&v)[VEC]) {
      if (TAIL && l.twice) {
#pragma unroll
        for (int u = 1; u < VEC; ++u)
          if (u >= l.twice) out[u] = v[u];
        out += pitch;
        return;
      }
#pragma unroll
      for (int u = 0; u < VEC; u += 4)
        *reinterpret_cast<Vec<float, 4>*>(out + u) = {{v[u], v[u + 1], v[u + 2], v[u + 3]}};
      out += pitch;
    };
    put(a_post);
    put(a_scale);
    put(a_pre);
  }
}

template <typename T, typename RT, typename WT, int TPR, int NV>
int launch_fwd(const FwdParams& p, hipStream_t s) {
  constexpr int kTeams = block_of<TPR>() / TPR;
  const int64_t most = static_cast<int64_t>(num_cus()) * (2048 / block_of<TPR>());
  const dim3 grid(std::min(cdiv(p.M, kTeams), most)), block(block_of<TPR>());
  if (p.N % (16 / static_cast<int>(sizeof(T))))
    hipLaunchKernelGGL((fwd_kernel<T, RT, WT, TPR, NV, false, true>), grid, block, 0, s, p);
  else if (p.post && p.gate && p.scale && p.pre)
    hipLaunchKernelGGL((fwd_kernel<T, RT, WT, TPR, NV, true, false>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((fwd_kernel<T, RT, WT, TPR, NV, false, false>), grid, block, 0, s, p);
  return launch_status();
}

template <typename T, typename RT, typename WT, int TPR>
int launch_bwd(const BwdParams& p, hipStream_t s) {
  constexpr int kTeams = block_of<TPR>() / TPR;
  const dim3 grid(cdiv(p.parts, kTeams)), block(block_of<TPR>());
  if (p.N % (16 / static_cast<int>(sizeof(T))))
    hipLaunchKernelGGL((bwd_kernel<T, RT, WT, TPR, true>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((bwd_kernel<T, RT, WT, TPR, false>), grid, block, 0, s, p);
  return launch_status();
}

// Rows of any length, one block each, read as often as needed: for rows of less
// than a lane's elements, and for those longer than a block holds: forward above
// 32,768 elements at 16 bits and 16,384 in fp32, backward, with one vector a lane,
// above 8,192 and 4,096.  The backward one reads single elements three times and
// keeps the column sums in memory: 4,096 x 8,192 fp32 1,028 us (8,192 x 4,096 195),
// 2,048 x 16,384 bf16 1,437 (4,096 x 8,192 126).
int stream_fwd(const FwdParams& p, hipStream_t s);
int stream_bwd(const BwdParams& p, hipStream_t s);

// 1,024 lanes of four vectors (above 16,384 elements at 16 bits, 8,192 in fp32)
// spill 28 to 255 registers by the types and parts (fp32: 14 to 22): 1,024 x 32,768
// bf16 103 us, 2,048 x 16,384 73.
//
// Few idle lanes, and teams of which a compute unit holds two: 8,192 rows of
// 2,560 bf16 take 44.8 us with 384 lanes, 49.2 with 256 and two vectors each; of
// 5,120 90 with 768 lanes, 122 with 1,024 (one team fits), 100 with 640 and 98
// with 384 and two; 4,096 of 8,192 64 with 512 and two, 80 with 1,024; 8,192 of
// 12,288 211 with 768 and two, 229 with 1,024 and two.
template <typename T, typename RT, typename WT>
int run_fwd_w(const FwdParams& p, hipStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t nvec = cdiv(p.N, VEC);
  if (p.N < VEC) return stream_fwd(p, s);
  if (nvec <= 64) return launch_fwd<T, RT, WT, 64, 1>(p, s);
  if (nvec <= 128) return launch_fwd<T, RT, WT, 64, 2>(p, s);
  if (nvec <= 256) return launch_fwd<T, RT, WT, 256, 1>(p, s);
  if (nvec <= 384) return launch_fwd<T, RT, WT, 384, 1>(p, s);
  // A wider residual has the registers of a second vector.
  if (nvec <= 512)
    return sizeof(RT) > sizeof(T) ? launch_fwd<T, RT, WT, 512, 1>(p, s)
                                  : launch_fwd<T, RT, WT, 256, 2>(p, s);
  if (nvec <= 768) return launch_fwd<T, RT, WT, 768, 1>(p, s);
  if (nvec <= 1024) return launch_fwd<T, RT, WT, 512, 2>(p, s);
  if (nvec <= 1536) return launch_fwd<T, RT, WT, 768, 2>(p, s);
  if (nvec <= 2048) return launch_fwd<T, RT, WT, 1024, 2>(p, s);
  if (nvec <= 4096) return launch_fwd<T, RT, WT, 1024, 4>(p, s);
  return stream_fwd(p, s);
}

template <typename T, typename RT, typename WT>
int run_bwd_w(const BwdParams& p, hipStream_t s) {
  if (p.N < 16 / static_cast<int>(sizeof(T))) return stream_bwd(p, s);
  switch (bwd_lanes(p.N, 16 / sizeof(T))) {
    case 64: return launch_bwd<T, RT, WT, 64>(p, s);
    case 128: return launch_bwd<T, RT, WT, 128>(p, s);
    case 256: return launch_bwd<T, RT, WT, 256>(p, s);
    case 512: return launch_bwd<T, RT, WT, 512>(p, s);
    case 1024: return launch_bwd<T, RT, WT, 1024>(p, s);
    default: return stream_bwd(p, s);
  }
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
