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

#include <algorithm>

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
  unsigned long long* words;  // [tiles][blocks * channels of a block]
  unsigned int* ticket;
  int blocks;
};

// First token of sequence n (N: the end); without cu_seqlens, N equal runs.
__device__ __forceinline__ int64_t cu_at(const void* cu, int cu64, int64_t n, int64_t run,
                                         int64_t total) {
  if (!cu) return n * run;
  const int64_t v = cu64 ? static_cast<const int64_t*>(cu)[n]
                         : static_cast<int64_t>(static_cast<const int32_t*>(cu)[n]);
  return v < 0 ? 0 : (v > total ? total : v);
}

// ---------------------------------------------------------------------------
// Tiles.  The token axis of the whole batch is cut into windows of kTok tokens,
// one per wave, and tiles of up to kMaxWaves windows, one per block; a lane
// has VEC channels (4 bytes of a row), so a block covers 64 VEC channels.  A
// window's tokens are read once and stay in registers as (alpha - 1, input).
//
// Any span of tokens maps the state before it to the state after it by
// h -> A h + B, and a span in which a sequence starts maps every state to the
// same one (the sequence's own start is part of its B): it is "final", marked
// by A = -1.  A block joins its waves' spans in LDS.  Between tiles each block
// publishes its span per channel as one 64-bit word (A, B), waits for the words
// of the tiles before it, back to a final one, and once it knows the state
// that enters it, replaces its own word by the final (-1, state).  The state
// between tiles is always the chain H_k = fma(A_k, H_{k-1}, B_k), whoever
// computes it and whichever final word it starts from, so the bits do not
// depend on timing.
//
// A block takes its tile from a counter: a tile is waited for only by tiles
// that were taken after it, so the one taken first of those that still run
// never waits for a block that has not started, and every wait ends.  Words
// and counter are cleared by a kernel before.  A word is one atomic access
// and carries its own validity (kUnset is no pair that is published), so no
// fences are needed.
// ---------------------------------------------------------------------------
constexpr int kTok = kWin;
constexpr int kMaxWaves = 8;
constexpr int kBack = 16;  // tiles before its own that a block looks at together
constexpr unsigned long long kUnset = ~0ull;

struct Span {
  float A, B;
};

__device__ __forceinline__ unsigned long long pack(Span s) {
  // A NaN of all ones must not read as kUnset.
  const float A = s.A != s.A ? __builtin_nanf("") : s.A;
  return static_cast<unsigned long long>(__builtin_bit_cast(unsigned int, A)) |
         static_cast<unsigned long long>(__builtin_bit_cast(unsigned int, s.B)) << 32;
}
__device__ __forceinline__ Span unpack(unsigned long long w) {
  return {__builtin_bit_cast(float, static_cast<unsigned int>(w)),
          __builtin_bit_cast(float, static_cast<unsigned int>(w >> 32))};
}
__device__ __forceinline__ void publish(unsigned long long* p, Span s) {
  __hip_atomic_store(p, pack(s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long peek(const unsigned long long* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The state after span s from the state h before it.
__device__ __forceinline__ float apply(Span s, float h) {
  return s.A < 0.f ? s.B : fmaf(s.A, h, s.B);
}
// Span p, then span s.
__device__ __forceinline__ Span join(Span p, Span s) {
  if (s.A < 0.f) return s;
  return {p.A < 0.f ? -1.f : p.A * s.A, fmaf(s.A, p.B, s.B)};
}

__global__ void __launch_bounds__(256)
    glr_clear_kernel(unsigned long long* words, int64_t n, unsigned int* ticket) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) words[i] = kUnset;
  if (i == 0) *ticket = 0;
}

template <int ALIGN> struct LaneWord;
template <> struct LaneWord<2> { typedef unsigned int type __attribute__((aligned(2))); };
template <> struct LaneWord<4> { typedef unsigned int type; };

// A lane's 4 bytes of a row: VEC elements at any address, of which the first
// `nv` exist.
template <typename T, int VEC>
__device__ __forceinline__ unsigned int ld_lane(const T* p, int nv) {
  static_assert(VEC * sizeof(T) == 4, "4 bytes");
  using W = typename LaneWord<sizeof(T)>::type;
  if (nv == VEC) return __builtin_nontemporal_load(reinterpret_cast<const W*>(p));
  if constexpr (VEC == 2) {
    if (nv == 1) return __builtin_bit_cast(unsigned short, p[0]);
  }
  return 0;
}
template <typename T>
__device__ __forceinline__ float lane_f32(unsigned int r, int u) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(float, r);
  } else if constexpr (std::is_same<T, bf16>::value) {
    return __builtin_bit_cast(float, u ? r & 0xffff0000u : r << 16);
  } else {
    return to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(u ? r >> 16 : r)));
  }
}
// What is computed from v later is computed then: keeps the compiler from
// holding a second pass's values in registers from the first one on.
template <typename V>
__device__ __forceinline__ void later(V& v) {
  asm volatile("" : "+v"(v));
}

template <typename T, int VEC>
__device__ __forceinline__ void st_lane(T* p, const float (&v)[VEC], int nv) {
  Arr<T, VEC> t;
#pragma unroll
  for (int u = 0; u < VEC; ++u) t.v[u] = from_f32<T>(v[u]);
  using W = typename LaneWord<sizeof(T)>::type;
  if (nv == VEC) {
    unsigned int r;
    __builtin_memcpy(&r, &t, 4);
    __builtin_nontemporal_store(r, reinterpret_cast<W*>(p));
  } else if (VEC == 2 && nv == 1) {
    p[0] = t.v[0];
  }
}
// fp32 rows of the same channels.
template <int VEC>
__device__ __forceinline__ void ld_f32(const float* p, int nv, float (&v)[VEC]) {
#pragma unroll
  for (int u = 0; u < VEC; ++u) v[u] = u < nv ? p[u] : 0.f;
}
template <int VEC>
__device__ __forceinline__ void st_f32(float* p, int nv, const float (&v)[VEC]) {
#pragma unroll
  for (int u = 0; u < VEC; ++u)
    if (u < nv) p[u] = v[u];
}

// Where sequences start and end in a window: bit j of a mask and entry j of a
// table (the sequence) for token w0 + j.  `lo`, `hi`: the tokens that belong to
// sequences.
struct Marks {
  unsigned int starts, ends;
  int64_t lo, hi;
};

// Called by a whole wave; seqs: 2 * kTok entries of LDS of its own.  empty(n) is
// called, by the wave together, for every empty sequence that the window
// answers for: the ones that stand before one of its tokens, and behind the
// last token those of the last window.
template <typename Empty>
__device__ __forceinline__ Marks find_marks(const void* cu, int cu64, int64_t N, int64_t run,
                                            int64_t total, int64_t w0, bool last, int* seqs,
                                            Empty empty) {
  const int lane = threadIdx.x % kWave;
  auto at = [&](int64_t n) { return cu_at(cu, cu64, n, run, total); };
  Marks m;
  m.lo = at(0);
  m.hi = at(N);
  if (lane < 2 * kTok) seqs[lane] = -1;
  // The first sequence that does not end before the window.
  int64_t base = 0, len = N;
  while (len > kWave) {
    const int64_t step = cdiv(len, kWave);
    const int64_t q = lane * step + step - 1;
    const uint64_t hit = __ballot(q >= len - 1 || at(base + q + 1) >= w0);
    const int64_t f = static_cast<int64_t>(__builtin_ctzll(hit)) * step;
    base += f;
    len = len - f < step ? len - f : step;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  for (; base < N; base += kWave) {
    const int64_t n = base + lane;
    int64_t t0 = total, t1 = total;
    if (n < N) {
      t0 = at(n);
      t1 = at(n + 1);
    }
    if (t0 < t1) {
      if (t0 >= w0 && t0 < w0 + kTok) seqs[t0 - w0] = static_cast<int>(n);
      if (t1 > w0 && t1 <= w0 + kTok) seqs[kTok + t1 - 1 - w0] = static_cast<int>(n);
    }
    const bool mine = n < N && t0 >= t1 && t0 >= w0 && (t0 < w0 + kTok || last);
    for (uint64_t left = __ballot(mine); left; left &= left - 1)
      empty(base + __builtin_ctzll(left));
    if (!last && __any(t0 >= w0 + kTok)) break;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  m.starts = static_cast<unsigned int>(__ballot(lane < kTok && seqs[lane & (kTok - 1)] >= 0));
  m.ends = static_cast<unsigned int>(
      __ballot(lane < kTok && seqs[kTok + (lane & (kTok - 1))] >= 0));
  return m;
}

// The state that enters a tile: the words of up to kBack tiles before it
// (`step` from one to the one before), shared through `look`, until there is
// a final one among them for every channel.  Called by all waves of a block.
template <int VEC>
__device__ __forceinline__ void enter(const unsigned long long* words, int64_t step, int64_t before,
                                      int lane, int wave, int waves, Span (*look)[kWave * VEC],
                                      float (&H)[VEC]) {
  const int reach = static_cast<int>(before < kBack ? before : kBack);
  for (;;) {
    for (int d = wave; d < reach; d += waves) {
      unsigned long long w[VEC];
      for (;;) {
        bool unset = false;
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
          w[u] = peek(words - (d + 1) * step + lane * VEC + u);
          unset |= w[u] == kUnset;
        }
        if (!__any(unset)) break;
        __builtin_amdgcn_s_sleep(1);
      }
#pragma unroll
      for (int u = 0; u < VEC; ++u) look[d][lane * VEC + u] = unpack(w[u]);
    }
    __syncthreads();
    bool known[VEC];
#pragma unroll
    for (int u = 0; u < VEC; ++u) {
      known[u] = false;
      H[u] = 0.f;
    }
    for (int d = reach - 1; d >= 0; --d) {
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        const Span s = look[d][lane * VEC + u];
        known[u] |= s.A < 0.f;
        H[u] = apply(s, H[u]);
      }
    }
    bool all = true;
#pragma unroll
    for (int u = 0; u < VEC; ++u) all &= known[u];
    // Every wave read the same words, so all waves leave together.
    if (__all(all)) return;
    __syncthreads();
    __builtin_amdgcn_s_sleep(1);
  }
}

template <typename T, bool LOOK>
__global__ void __launch_bounds__(kMaxWaves * kWave) glr_fwd_kernel(FwdParams p) {
  constexpr int VEC = 4 / sizeof(T);
  __shared__ unsigned int taken;
  __shared__ int seqs[kMaxWaves][2 * kTok];
  __shared__ Span spans[kMaxWaves][kWave * VEC];
  __shared__ Span look[LOOK ? kBack : 1][kWave * VEC];
  __shared__ int open;  // the tile needs the state before it

  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int waves = blockDim.x / kWave;
  unsigned int id = blockIdx.x;
  if constexpr (LOOK) {
    if (threadIdx.x == 0)
      taken = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    id = __builtin_amdgcn_readfirstlane(taken);
  }
  const int64_t tile = id / p.blocks;
  const int blk = id % p.blocks;
  const int64_t w0 = (tile * waves + wave) * kTok;
  const int64_t ch = (static_cast<int64_t>(blk) * kWave + lane) * VEC;
  const int nv = p.D - ch < VEC ? (p.D > ch ? static_cast<int>(p.D - ch) : 0) : VEC;

  // All of the window's loads, before anything else.
  unsigned int x[kTok], a[kTok], b[kTok];
  const T* xp = static_cast<const T*>(p.x) + w0 * p.sx + ch;
  const T* ap = static_cast<const T*>(p.a) + w0 * p.sa + ch;
  const T* bp = static_cast<const T*>(p.b) + w0 * p.sb + ch;
  if (w0 + kTok <= p.total && (blk + 1) * static_cast<int64_t>(kWave * VEC) <= p.D) {
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      x[j] = ld_lane<T, VEC>(xp + j * p.sx, VEC);
      a[j] = ld_lane<T, VEC>(ap + j * p.sa, VEC);
      b[j] = ld_lane<T, VEC>(bp + j * p.sb, VEC);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      const int have = w0 + j < p.total ? nv : 0;
      x[j] = ld_lane<T, VEC>(xp + j * p.sx, have);
      a[j] = ld_lane<T, VEC>(ap + j * p.sa, have);
      b[j] = ld_lane<T, VEC>(bp + j * p.sb, have);
    }
  }
  float k[VEC];
  ld_f32<VEC>(p.lam + ch, nv, k);
#pragma unroll
  for (int u = 0; u < VEC; ++u) k[u] = -p.c * softplus_f32(k[u]);

  const Marks m = find_marks(p.cu, p.cu64, p.N, p.T, p.total, w0,
                             w0 < p.total + kTok && w0 + kTok >= p.total, seqs[wave],
                             [&](int64_t n) {
                               if (!p.fin) return;
                               float h[VEC] = {};
                               if (p.h0) ld_f32<VEC>(p.h0 + n * p.D + ch, nv, h);
                               st_f32<VEC>(p.fin + n * p.D + ch, nv, h);
                             });

  // The window's gates, and its span.
  float em1[kTok][VEC], add[kTok][VEC];
  Span span[VEC];
#pragma unroll
  for (int u = 0; u < VEC; ++u) span[u] = {1.f, 0.f};
#pragma unroll
  for (int j = 0; j < kTok; ++j) {
#pragma unroll
    for (int u = 0; u < VEC; ++u) {
      const Gate g = gate_of(k[u], sigmoid(lane_f32<T>(a[j], u)));
      em1[j][u] = g.em1;
      add[j][u] = g.s * (sigmoid(lane_f32<T>(b[j], u)) * lane_f32<T>(x[j], u));
    }
    if (m.starts >> j & 1) {
      float h[VEC] = {};
      if (p.h0) ld_f32<VEC>(p.h0 + static_cast<int64_t>(seqs[wave][j]) * p.D + ch, nv, h);
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        add[j][u] += decayed(em1[j][u], h[u]);
        span[u].B = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < VEC; ++u) {
      span[u].A = decayed(em1[j][u], span[u].A);
      span[u].B = decayed(em1[j][u], span[u].B) + add[j][u];
    }
  }
#pragma unroll
  for (int u = 0; u < VEC; ++u) {
    if (m.starts) span[u].A = -1.f;
    spans[wave][lane * VEC + u] = span[u];
  }
  if (wave == 0 && lane == 0) open = !(m.starts & 1);
  __syncthreads();

  // From the tile's start to this window's.
  Span head[VEC];
#pragma unroll
  for (int u = 0; u < VEC; ++u) head[u] = {1.f, 0.f};
  for (int w = 0; w < wave; ++w) {
#pragma unroll
    for (int u = 0; u < VEC; ++u) head[u] = join(head[u], spans[w][lane * VEC + u]);
  }
  float H[VEC] = {};
  if constexpr (LOOK) {
    const int64_t width = static_cast<int64_t>(p.blocks) * kWave * VEC;
    unsigned long long* words = p.words + tile * width + static_cast<int64_t>(blk) * kWave * VEC;
    Span whole[VEC];
    const bool closing = wave == waves - 1;
    if (closing) {
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        whole[u] = join(head[u], span[u]);
        if (tile == 0) whole[u].A = -1.f;
        publish(words + lane * VEC + u, whole[u]);
      }
    }
    if (tile > 0 && open) {
      enter<VEC>(words, width, tile, lane, wave, waves, look, H);
      if (closing) {
#pragma unroll
        for (int u = 0; u < VEC; ++u)
          if (!(whole[u].A < 0.f))
            publish(words + lane * VEC + u, {-1.f, apply(whole[u], H[u])});
      }
    }
  }

  float h[VEC];
#pragma unroll
  for (int u = 0; u < VEC; ++u) h[u] = apply(head[u], H[u]);
  if (p.states && w0 < p.total) st_f32<VEC>(p.states + w0 / kWin * p.D + ch, nv, h);
  T* yp = static_cast<T*>(p.y) + w0 * p.sy + ch;
  const bool whole_window = w0 >= m.lo && w0 + kTok <= m.hi;
#pragma unroll
  for (int j = 0; j < kTok; ++j) {
    if (m.starts >> j & 1) {
#pragma unroll
      for (int u = 0; u < VEC; ++u) h[u] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < VEC; ++u) h[u] = decayed(em1[j][u], h[u]) + add[j][u];
    if (whole_window || (w0 + j >= m.lo && w0 + j < m.hi))
      st_lane<T, VEC>(yp + j * p.sy, h, nv);
    if ((m.ends >> j & 1) && p.fin)
      st_f32<VEC>(p.fin + static_cast<int64_t>(seqs[wave][kTok + j]) * p.D + ch, nv, h);
  }
}

// Tiles, channel blocks and waves of a block for a problem.
struct Cut {
  int64_t tiles;
  int blocks, waves;
  int64_t width;  // words of a tile
};
inline Cut cut_of(int64_t total, int64_t D, int vec, int max_waves) {
  Cut c;
  const int64_t windows = std::max<int64_t>(cdiv(total, kTok), 1);
  c.waves = static_cast<int>(std::min<int64_t>(windows, max_waves));
  c.tiles = cdiv(windows, c.waves);
  c.blocks = static_cast<int>(cdiv(D, kWave * vec));
  c.width = static_cast<int64_t>(c.blocks) * kWave * vec;
  return c;
}
// Bytes of a pass's counter (its own cache line) and words; none for one tile.
inline int64_t words_bytes(const Cut& c) { return c.tiles > 1 ? 256 + c.tiles * c.width * 8 : 0; }

inline void clear_words(const Cut& c, void* workspace, hipStream_t s) {
  const int64_t n = c.tiles * c.width;
  hipLaunchKernelGGL(glr_clear_kernel, dim3(cdiv(n, 256)), dim3(256), 0, s,
                     reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + 256), n,
                     static_cast<unsigned int*>(workspace));
}

template <typename T>
int launch_fwd(FwdParams p, void* workspace, hipStream_t s) {
  const Cut c = cut_of(p.total, p.D, 4 / sizeof(T), kMaxWaves);
  p.blocks = c.blocks;
  const dim3 grid(c.tiles * c.blocks), block(c.waves * kWave);
  if (c.tiles > 1) {
    p.ticket = static_cast<unsigned int*>(workspace);
    p.words = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + 256);
    clear_words(c, workspace, s);
    hipLaunchKernelGGL((glr_fwd_kernel<T, true>), grid, block, 0, s, p);
  } else {
    hipLaunchKernelGGL((glr_fwd_kernel<T, false>), grid, block, 0, s, p);
  }
  return launch_status();
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
  float* part;  // dlam's parts, [tiles][D]; NULL: not asked for
  const void* cu;
  int cu64;
  int64_t N, T, total, D;
  unsigned long long* words;
  unsigned int* ticket;
  int64_t tiles;
  int blocks;
};

// sigmoid(lam) / softplus(lam), 1 in the limit lam -> -inf.
__device__ __forceinline__ float slope_ratio(float lam) {
  if (lam < -17.f) return 1.f;  // 1 - e^lam / 2 rounds to 1
  return 1.f / ((1.f + expf(-lam)) * softplus_f32(lam));
}

// exp(-v) for a sigmoid's value r = 1 / (1 + e) and its complement 1 - r = e r;
// capped at 2^100, so that e r is 1 and not inf * 0 for a closed gate.
__device__ __forceinline__ float exp_neg(float v) {
  return __builtin_amdgcn_exp2f(fminf(v * -1.44269504f, 100.f));
}

// ---------------------------------------------------------------------------
// Backward.  The gradient q that enters a token from behind (of its state)
// leaves it in front as alpha (dy + q): a span of tokens maps q -> A q + B, and
// a sequence's last token makes a span final, its q being d_final_state.  So
// the tiles of the forward kernel run here from the end, in the same way, with
// the sequences' ends in the place of their starts.
//  * h_{t-1} comes from the window's saved state, in the same pass that forms
//    the window's span (in token order: A is the running product of alpha and
//    B the sum of A_t dy_t, so nothing but h_{t-1} is kept for a token).
//  * The second pass, in reverse order, forms the gates again from exp(-a) and
//    exp(-b), which stay in registers.
//  * E = (dL/dl) l = G alpha (h_{t-1} l - i x alpha l / s) gives da = E (1 - r)
//    and dlam = sum E sigmoid(lam) / softplus(lam), with no division by what
//    vanishes as a gate closes: l / s -> 0 with s.
// ---------------------------------------------------------------------------
constexpr int kBwdWaves = 4;

template <typename T, bool LOOK>
__global__ void __launch_bounds__(kBwdWaves * kWave) glr_bwd_kernel(BwdParams p) {
  constexpr int VEC = 4 / sizeof(T);
  __shared__ unsigned int taken;
  __shared__ int seqs[kBwdWaves][2 * kTok];
  __shared__ Span spans[kBwdWaves][kWave * VEC];
  __shared__ Span look[LOOK ? kBack : 1][kWave * VEC];
  __shared__ float sums[kBwdWaves][kWave * VEC];
  __shared__ int open;  // the tile needs the gradient from behind it

  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int waves = blockDim.x / kWave;
  unsigned int id = blockIdx.x;
  if constexpr (LOOK) {
    if (threadIdx.x == 0)
      taken = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    id = __builtin_amdgcn_readfirstlane(taken);
  }
  const int64_t after = id / p.blocks;  // tiles behind this one
  const int64_t tile = p.tiles - 1 - after;
  const int blk = id % p.blocks;
  const int64_t w0 = (tile * waves + wave) * kTok;
  const int64_t ch = (static_cast<int64_t>(blk) * kWave + lane) * VEC;
  const int nv = p.D - ch < VEC ? (p.D > ch ? static_cast<int>(p.D - ch) : 0) : VEC;

  unsigned int x[kTok], dy[kTok], a[kTok], b[kTok];
  const T* xp = static_cast<const T*>(p.x) + w0 * p.sx + ch;
  const T* ap = static_cast<const T*>(p.a) + w0 * p.sa + ch;
  const T* bp = static_cast<const T*>(p.b) + w0 * p.sb + ch;
  const T* gp = static_cast<const T*>(p.dy) + w0 * p.sdy + ch;
  if (w0 + kTok <= p.total && (blk + 1) * static_cast<int64_t>(kWave * VEC) <= p.D) {
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      a[j] = ld_lane<T, VEC>(ap + j * p.sa, VEC);
      b[j] = ld_lane<T, VEC>(bp + j * p.sb, VEC);
      x[j] = ld_lane<T, VEC>(xp + j * p.sx, VEC);
      dy[j] = ld_lane<T, VEC>(gp + j * p.sdy, VEC);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      const int have = w0 + j < p.total ? nv : 0;
      a[j] = ld_lane<T, VEC>(ap + j * p.sa, have);
      b[j] = ld_lane<T, VEC>(bp + j * p.sb, have);
      x[j] = ld_lane<T, VEC>(xp + j * p.sx, have);
      dy[j] = ld_lane<T, VEC>(gp + j * p.sdy, have);
    }
  }
  float k[VEC], h[VEC] = {};
  ld_f32<VEC>(p.lam + ch, nv, k);
  if (w0 < p.total) ld_f32<VEC>(p.states + w0 / kWin * p.D + ch, nv, h);
#pragma unroll
  for (int u = 0; u < VEC; ++u) k[u] = -p.c * softplus_f32(k[u]);

  const Marks m = find_marks(p.cu, p.cu64, p.N, p.T, p.total, w0,
                             w0 < p.total + kTok && w0 + kTok >= p.total, seqs[wave],
                             [&](int64_t n) {
                               if (!p.dh0) return;
                               float q[VEC] = {};
                               if (p.dfin) ld_f32<VEC>(p.dfin + n * p.D + ch, nv, q);
                               st_f32<VEC>(p.dh0 + n * p.D + ch, nv, q);
                             });

  float before[kTok][VEC], ea[kTok][VEC], eb[kTok][VEC];
  Span span[VEC];
#pragma unroll
  for (int u = 0; u < VEC; ++u) span[u] = {1.f, 0.f};
#pragma unroll
  for (int j = 0; j < kTok; ++j) {
    if (m.starts >> j & 1) {
#pragma unroll
      for (int u = 0; u < VEC; ++u) h[u] = 0.f;
      if (p.h0) ld_f32<VEC>(p.h0 + static_cast<int64_t>(seqs[wave][j]) * p.D + ch, nv, h);
    }
#pragma unroll
    for (int u = 0; u < VEC; ++u) {
      ea[j][u] = exp_neg(lane_f32<T>(a[j], u));
      eb[j][u] = exp_neg(lane_f32<T>(b[j], u));
      const Gate g = gate_of(k[u], fast_rcp(1.f + ea[j][u]));
      before[j][u] = h[u];
      h[u] = decayed(g.em1, h[u]) + g.s * (fast_rcp(1.f + eb[j][u]) * lane_f32<T>(x[j], u));
      if (!(m.ends & ((1u << j) - 1))) {  // no sequence ended before: q comes this far
        span[u].A = decayed(g.em1, span[u].A);
        span[u].B = fmaf(span[u].A, lane_f32<T>(dy[j], u), span[u].B);
      }
    }
    if ((m.ends >> j & 1) && !(m.ends & ((1u << j) - 1)) && p.dfin) {
      float q[VEC];
      ld_f32<VEC>(p.dfin + static_cast<int64_t>(seqs[wave][kTok + j]) * p.D + ch, nv, q);
#pragma unroll
      for (int u = 0; u < VEC; ++u) span[u].B = fmaf(span[u].A, q[u], span[u].B);
    }
  }
#pragma unroll
  for (int u = 0; u < VEC; ++u) {
    if (m.ends) span[u].A = -1.f;
    spans[wave][lane * VEC + u] = span[u];
  }
  if (wave == waves - 1 && lane == 0) open = !(m.ends >> (kTok - 1) & 1);
  __syncthreads();

  // From the tile's end to this window's.
  Span head[VEC];
#pragma unroll
  for (int u = 0; u < VEC; ++u) head[u] = {1.f, 0.f};
  for (int w = waves - 1; w > wave; --w) {
#pragma unroll
    for (int u = 0; u < VEC; ++u) head[u] = join(head[u], spans[w][lane * VEC + u]);
  }
  float Q[VEC] = {};
  if constexpr (LOOK) {
    const int64_t width = static_cast<int64_t>(p.blocks) * kWave * VEC;
    unsigned long long* words = p.words + after * width + static_cast<int64_t>(blk) * kWave * VEC;
    Span whole[VEC];
    if (wave == 0) {
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        whole[u] = join(head[u], span[u]);
        if (after == 0) whole[u].A = -1.f;
        publish(words + lane * VEC + u, whole[u]);
      }
    }
    if (after > 0 && open) {
      enter<VEC>(words, width, after, lane, wave, waves, look, Q);
      if (wave == 0) {
#pragma unroll
        for (int u = 0; u < VEC; ++u)
          if (!(whole[u].A < 0.f))
            publish(words + lane * VEC + u, {-1.f, apply(whole[u], Q[u])});
      }
    }
  }

#pragma unroll
  for (int j = 0; j < kTok; ++j) {
    later(x[j]);
    later(dy[j]);
#pragma unroll
    for (int u = 0; u < VEC; ++u) {
      later(ea[j][u]);
      later(eb[j][u]);
    }
  }
  float q[VEC], sum[VEC] = {};
#pragma unroll
  for (int u = 0; u < VEC; ++u) q[u] = apply(head[u], Q[u]);
  T* dxp = static_cast<T*>(p.dx) + w0 * p.sdx + ch;
  T* dap = static_cast<T*>(p.da) + w0 * p.sda + ch;
  T* dbp = static_cast<T*>(p.db) + w0 * p.sdb + ch;
  const bool whole_window = w0 >= m.lo && w0 + kTok <= m.hi;
#pragma unroll
  for (int j = kTok - 1; j >= 0; --j) {
    if (m.ends >> j & 1) {
#pragma unroll
      for (int u = 0; u < VEC; ++u) q[u] = 0.f;
      if (p.dfin)
        ld_f32<VEC>(p.dfin + static_cast<int64_t>(seqs[wave][kTok + j]) * p.D + ch, nv, q);
    }
    const bool live = whole_window || (w0 + j >= m.lo && w0 + j < m.hi);
    float dx[VEC], da[VEC], db[VEC];
#pragma unroll
    for (int u = 0; u < VEC; ++u) {
      const float r = fast_rcp(1.f + ea[j][u]), i = fast_rcp(1.f + eb[j][u]);
      const float xf = lane_f32<T>(x[j], u), l = k[u] * r;
      const Decay d = decay_of(l);
      const float w = -d.em1 * (1.f + d.alpha);  // s^2
      // The instruction takes a denormal w for 0.
      const float inv = w >= 1.17549435e-38f ? __builtin_amdgcn_rsqf(w) : 0.f;
      const float G = lane_f32<T>(dy[j], u) + q[u];
      dx[u] = G * (w * inv) * i;
      db[u] = dx[u] * xf * (eb[j][u] * i);
      const float e = G * d.alpha * (before[j][u] * l - i * xf * d.alpha * (l * inv));
      da[u] = e * (ea[j][u] * r);
      if (live) sum[u] += e;
      q[u] = decayed(d.em1, G);
    }
    if (live) {
      st_lane<T, VEC>(dxp + j * p.sdx, dx, nv);
      st_lane<T, VEC>(dap + j * p.sda, da, nv);
      st_lane<T, VEC>(dbp + j * p.sdb, db, nv);
    }
    if ((m.starts >> j & 1) && p.dh0)
      st_f32<VEC>(p.dh0 + static_cast<int64_t>(seqs[wave][j]) * p.D + ch, nv, q);
  }
  if (p.part) {
#pragma unroll
    for (int u = 0; u < VEC; ++u) sums[wave][lane * VEC + u] = sum[u];
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < waves; ++w) {
#pragma unroll
        for (int u = 0; u < VEC; ++u) sum[u] += sums[w][lane * VEC + u];
      }
      st_f32<VEC>(p.part + tile * p.D + ch, nv, sum);
    }
  }
}

// dlam = sum over tiles of (sum E) sigmoid(lam) / softplus(lam): a block takes
// 64 channels, each of its 16 waves every 16th tile.
__global__ void __launch_bounds__(1024) glr_dlam_kernel(const float* part, int64_t tiles,
                                                        const float* lam, float* dlam, int64_t D) {
  __shared__ float red[16][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t ch = static_cast<int64_t>(blockIdx.x) * kWave + lane;
  float s = 0.f;
  if (ch < D)
    for (int64_t j = wave; j < tiles; j += 16) s += part[j * D + ch];
  red[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && ch < D) {
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += red[w][lane];
    dlam[ch] = s * slope_ratio(lam[ch]);
  }
}

template <typename T>
int launch_bwd(BwdParams p, bool sums, void* workspace, hipStream_t s) {
  const Cut c = cut_of(p.total, p.D, 4 / sizeof(T), kBwdWaves);
  p.blocks = c.blocks;
  p.tiles = c.tiles;
  // The workspace: counter and words, then dlam's parts.
  if (sums) p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + words_bytes(c));
  const dim3 grid(c.tiles * c.blocks), block(c.waves * kWave);
  if (c.tiles > 1) {
    p.ticket = static_cast<unsigned int*>(workspace);
    p.words = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + 256);
    clear_words(c, workspace, s);
    hipLaunchKernelGGL((glr_bwd_kernel<T, true>), grid, block, 0, s, p);
  } else {
    hipLaunchKernelGGL((glr_bwd_kernel<T, false>), grid, block, 0, s, p);
  }
  return launch_status();
}

// Tokens, sequences and tiles are counted in 31 bits, a batch's elements in 62.
bool bad_sizes(int64_t N, int64_t total, int64_t D) {
  constexpr int64_t kMost = int64_t{1} << 31;
  return N < 0 || N >= kMost || total < 0 || total >= kMost || D <= 0 || D >= kMost ||
         cdiv(std::max<int64_t>(total, 1), kTok) * cdiv(D, kWave) >= kMost;
}

bool pitch_ok(int64_t pitch, int64_t D) { return pitch >= D; }

// cu_seqlens of a readable type, or none and N equal runs.
bool seqs_ok(const void* cu, xk_dtype dt, int64_t N, int64_t total) {
  return cu ? dt == XK_I32 || dt == XK_I64 : total % N == 0;
}

}  // namespace
}  // namespace xk

using namespace xk;

extern "C" int64_t xk_gated_linear_recurrence_workspace_bytes(int64_t total_tokens, int64_t D) {
  if (total_tokens <= 0 || D <= 0) return 0;
  // 4-byte elements take more, narrower channel blocks.
  return std::max(words_bytes(cut_of(total_tokens, D, 1, kMaxWaves)),
                  words_bytes(cut_of(total_tokens, D, 2, kMaxWaves)));
}

extern "C" int xk_gated_linear_recurrence(
    const void* x, int64_t stride_x_tok, const void* a, int64_t stride_a_tok, const void* b,
    int64_t stride_b_tok, xk_dtype dtype, const float* lam, float c, void* y,
    int64_t stride_y_tok, const float* initial_state, float* final_state, float* states,
    const void* cu_seqlens, xk_dtype cu_dtype, int64_t N, int64_t total_tokens, int64_t D,
    void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_sizes(N, total_tokens, D) || !(c >= 0.f)) return XK_ERR_INVALID;
  if (!is_float_dtype(dtype)) return XK_ERR_UNSUPPORTED;
  if (N == 0) return XK_OK;
  if (!seqs_ok(cu_seqlens, cu_dtype, N, total_tokens) || !lam) return XK_ERR_INVALID;
  if (total_tokens > 0 &&
      (!x || !a || !b || !y || !pitch_ok(stride_x_tok, D) || !pitch_ok(stride_a_tok, D) ||
       !pitch_ok(stride_b_tok, D) || !pitch_ok(stride_y_tok, D)))
    return XK_ERR_INVALID;
  const int64_t need = xk_gated_linear_recurrence_workspace_bytes(total_tokens, D);
  if (need > 0 && (!workspace || workspace_bytes < static_cast<size_t>(need) ||
                   !aligned(workspace, 256)))
    return XK_ERR_WORKSPACE;
  const FwdParams p{x, a, b, y, stride_x_tok, stride_a_tok, stride_b_tok, stride_y_tok, lam, c,
                    initial_state, final_state, states, cu_seqlens, cu_dtype == XK_I64, N,
                    total_tokens / N, total_tokens, D, nullptr, nullptr, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case XK_F32: return launch_fwd<float>(p, workspace, s);
    case XK_BF16: return launch_fwd<bf16>(p, workspace, s);
    default: return launch_fwd<f16>(p, workspace, s);
  }
}

extern "C" int xk_gated_linear_recurrence_update(
    const void* x, int64_t stride_x_tok, const void* a, int64_t stride_a_tok, const void* b,
    int64_t stride_b_tok, xk_dtype dtype, const float* lam, float c, void* y,
    int64_t stride_y_tok, float* state, int64_t stride_state_slot, int64_t num_slots,
    const int32_t* state_indices, int64_t num_cols, const int32_t* num_accepted_tokens,
    const void* cu_seqlens, xk_dtype cu_dtype, int64_t N, int64_t T, int64_t total_tokens,
    int64_t D, void* stream) {
  if (bad_sizes(N, total_tokens, D) || num_slots < 0 || num_cols < 0 || !(c >= 0.f))
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

extern "C" int64_t xk_gated_linear_recurrence_bwd_workspace_bytes(int64_t total_tokens, int64_t N,
                                                                  int64_t D) {
  if (total_tokens < 0 || N <= 0 || D <= 0) return 0;
  const Cut c1 = cut_of(total_tokens, D, 1, kBwdWaves), c2 = cut_of(total_tokens, D, 2, kBwdWaves);
  return std::max(words_bytes(c1), words_bytes(c2)) + c1.tiles * D * 4;
}

extern "C" int xk_gated_linear_recurrence_bwd(
    const void* dy, int64_t stride_dy_tok, const void* x, int64_t stride_x_tok, const void* a,
    int64_t stride_a_tok, const void* b, int64_t stride_b_tok, xk_dtype dtype, const float* lam,
    float c, const float* states, const float* initial_state, const float* d_final_state,
    void* dx, int64_t stride_dx_tok, void* da, int64_t stride_da_tok, void* db,
    int64_t stride_db_tok, float* dlam, float* d_initial_state, const void* cu_seqlens,
    xk_dtype cu_dtype, int64_t N, int64_t total_tokens, int64_t D, void* workspace,
    size_t workspace_bytes, void* stream) {
  if (bad_sizes(N, total_tokens, D) || !(c >= 0.f)) return XK_ERR_INVALID;
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
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (N > 0) {
    const BwdParams p{dy, x, a, b, dx, da, db, stride_dy_tok, stride_x_tok, stride_a_tok,
                      stride_b_tok, stride_dx_tok, stride_da_tok, stride_db_tok, lam, c, states,
                      initial_state, d_final_state, d_initial_state, nullptr, cu_seqlens,
                      cu_dtype == XK_I64, N, total_tokens / N, total_tokens, D, nullptr, nullptr,
                      0, 0};
    const int st = dtype == XK_F32    ? launch_bwd<float>(p, dlam, workspace, s)
                   : dtype == XK_BF16 ? launch_bwd<bf16>(p, dlam, workspace, s)
                                      : launch_bwd<f16>(p, dlam, workspace, s);
    if (st != XK_OK) return st;
  }
  if (dlam) {
    const Cut cut = cut_of(total_tokens, D, dtype == XK_F32 ? 1 : 2, kBwdWaves);
    const float* part = N > 0 ? reinterpret_cast<const float*>(static_cast<char*>(workspace) +
                                                               words_bytes(cut))
                              : nullptr;
    hipLaunchKernelGGL(glr_dlam_kernel, dim3(cdiv(D, kWave)), dim3(1024), 0, s, part,
                       N > 0 ? cut.tiles : 0, lam, dlam, D);
  }
  return launch_status();
}
