// Gated linear recurrence for gfx950: forward over ragged sequences, the
// decode step on a pool of states, and the backward pass.
//
//   r = sigmoid(a), i = sigmoid(b), l = -c softplus(lam) r, alpha = exp(l),
//   s = sqrt(1 - alpha^2), h_t = alpha h_{t-1} + s i x_t, y_t = h_t
//
// per channel, in fp32.  alpha - 1 is formed as expm1(l) and 1 - alpha^2 as
// -(alpha - 1)(1 + alpha), so neither loses digits where a channel
// keeps nearly all of its state (alpha near 1, the case that matters); where it
// keeps little, alpha itself is what is multiplied by.
#include <math.h>

#include <algorithm>
#include <limits>
#include <type_traits>

#include "xk_common.h"

namespace xk {
namespace {

constexpr int kWin = XK_GLR_WINDOW;

// Per-channel constants: k = -c softplus(lam), so that l = k r.
// softplus(v) = max(v, 0) + log1p(e), e = exp(-|v|) with the argument's
// rounding made good (2^n 2^f, f from the two parts of log2 e), and log1p(e) =
// 2 atanh(e / (2 + e)) by a polynomial (least largest relative error, 4e-9
// before rounding): within 4 units of the last place, in 25 instructions
// where log1pf(expf(v)) takes over 100 and a decode step has one token to
// spread them over.
__device__ __forceinline__ float softplus_f32(float v) {
  const float w = fmaxf(-fabsf(v), -150.f);
  const float n = rintf(w * 1.44269502f);
  const float f = fmaf(w, 1.92596303e-8f, fmaf(w, 1.44269502f, -n));
  const float e = __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(f), static_cast<int>(n));
  const float d = 2.f + e, r = __builtin_amdgcn_rcpf(d);
  float q = e * r;
  q = fmaf(fmaf(-q, d, e), r, q);
  const float z = q * q;
  float p = fmaf(z, 0.14089172f, 0.13980305f);
  p = fmaf(p, z, 0.20012455f);
  p = fmaf(p, z, 0.33333158f);
  p = fmaf(p, z, 1.f);
  return (v < 0.f ? 0.f : v) + 2.f * (q * p);  // NaN stays NaN
}

// The decay of a token for l <= 0: alpha = exp(l) and alpha - 1, each to its
// own last digits.  From -1/4 up a polynomial of (exp(l) - 1) / l (least
// largest relative error, 2.5e-9 before rounding) gives alpha - 1, below it
// the exponential gives alpha.  NEAR: no channel of the wave goes below (k r,
// r < 1); the same bits without the exponential.
//
// From -1/4 up alpha v is v + (alpha - 1) v: one rounding, of the sum, where
// thousands of tokens may lie between a state and its use.  Below it is
// alpha times v: alpha - 1, rounded near -1, has lost alpha's digits (1% of it
// at alpha = 1e-6).  `word` holds either, told apart by the sign bit: alpha - 1
// has it (-0 for a closed gate), alpha has not.  The choice
// costs 2 to 4% where channels go below (16,384 x 4,096 bf16 133 us, with alpha - 1
// throughout 128.5) and up to 7% in windows that are not plain (one tile of
// 100 x 4,096: 10.9 and 10.2).
constexpr float kNear = -0.25f;
struct Decay {
  float alpha, em1, word;
};
template <bool NEAR>
__device__ __forceinline__ Decay decay_of(float l) {
  float p = fmaf(l, 0.007510221f, 0.041488957f);
  p = fmaf(p, l, 0.16665082f);
  p = fmaf(p, l, 0.4999995f);
  const float q = fmaf(p, l, 1.f), series = fmaf(q, l, 1.f);
  p = q * l;
  if constexpr (NEAR) return {series, p, p};
  // The compiler is kept from carrying the comparison along in scalar
  // registers, which it spills: the word's sign says the same.
  float word = l >= kNear ? p : __expf(l);
  asm("" : "+v"(word));
  const bool near = __builtin_bit_cast(int, word) < 0;
  return {near ? series : word, near ? word : word - 1.f, word};
}
// alpha v.
template <bool NEAR>
__device__ __forceinline__ float decayed(float word, float v) {
  if constexpr (NEAR) return fmaf(word, v, v);
  const int near = __builtin_bit_cast(int, word) >> 31;  // all bits, or none
  return fmaf(word, v, __builtin_bit_cast(float, __builtin_bit_cast(int, v) & near));
}

struct Gate {
  float alpha, word;
  float s;  // sqrt(1 - alpha^2)
};
template <bool NEAR>
__device__ __forceinline__ Gate gate_of(float k, float r) {
  const Decay d = decay_of<NEAR>(k * r);
  return {d.alpha, d.word, __builtin_amdgcn_sqrtf(-d.em1 * (1.f + d.alpha))};
}

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
  const float* k;             // [width], where tiles are joined
  const int* plain;           // [windows]
  unsigned long long* words;  // [tiles][width], then [groups][width]
  unsigned int* ticket;
  int64_t tiles, width;  // width: channels of all blocks
  int blocks;
};

// First token of sequence n (N: the end), clamped to the batch; without
// cu_seqlens, N equal runs.  Both types are read as 32-bit words with no
// branch between them, so that several reads are under way together.
__device__ __forceinline__ int cu_at(const void* cu, int cu64, int n, int run, int total) {
  if (!cu) return n * run;
  const int* w = static_cast<const int*>(cu) + (static_cast<int64_t>(n) << cu64);
  const int low = w[0], high = w[cu64];  // int32: the same word
  const int v = cu64 ? (high == 0 && low >= 0 ? low : (high < 0 ? 0 : total)) : low;
  return v < 0 ? 0 : (v > total ? total : v);
}

// ---------------------------------------------------------------------------
// Tiles.  The token axis of the whole batch is cut into windows of kTok tokens,
// one per wave, and tiles of some windows, one per block; a lane has
// VEC channels (4 bytes of a row), so a tile covers 64 VEC channels.  A
// window's tokens are read once and stay in registers as (decay, input).
//
// Any span of tokens maps the state before it to the state after it by
// h -> A h + B, and a span in which a sequence starts maps every state to the
// same one (the sequence's own start is part of its B): it is "final", marked
// by A = -1.  A block joins its waves' spans in LDS.  Between tiles each block
// publishes its span per channel as one 64-bit word (A, B); the last tile of
// a group of kGroup joins the group's words and publishes the group's span,
// and once it knows the state that enters the group, replaces it by the final
// (-1, state behind the group).  A tile needs the words before it in its group
// and the group's word back to a final one.  The state between groups is
// always the chain G_k = fma(A_k, G_{k-1}, B_k), whoever computes it and
// whichever final word it starts from, so the bits do not depend on timing.
// (With the chain from tile to tile, 2.6 us for every 8 of them, 32,768
// tokens x 1,024 channels took 97 us.)
//
// A block takes its tile from a counter: a tile is waited for only by tiles
// that were taken after it, so the one taken first of those that still run
// waits for finished ones only, and every wait ends, whatever blocks are
// resident.  Words and counter are cleared by a kernel before.  A word is one atomic
// access and carries its own validity (kUnset is no pair that is published),
// so no fences are needed.
//
// The forward kernel takes 126 us for 16,384 x 4,096 bf16 (537 MB, 4.3 TB/s):
// with loads and stores alone 92, without the arithmetic (34 instructions a
// channel and token) 104, without the chain 115.  The window's 48 loads are
// issued together, which takes 128 registers (and 4 spilled in bf16, 2 in fp16;
// 93 in fp32): 4 waves a SIMD hide the rest only in part.  Windows of 8 tokens (8 waves) took 150 and more.
// ---------------------------------------------------------------------------
constexpr int kTok = kWin;
// Waves of a block at most: kFew while a pass has no more than kUntil windows
// over all channel blocks, where the chain between tiles is the longest part
// and longer tiles shorten it, else kMany, and where one tile holds the batch
// (no chain, and registers as a tile's waves need them).  Forward, one channel a lane, 16
// against 8 waves: 5,003 x 1,125 29.6 and 32.6 us, 2,048 x 2,048 18.8 and 20.3,
// 16,384 x 1,000 65.6 and 67.9; 8,192 x 4,096 105 and 96.  Two channels: 8
// throughout (16: 2,048 x 2,048 20.4 and 17.4; 4: within 1 to 4%).  Backward, two
// channels, 8 against 4: 2,048 x 2,048 24.7 and 28.4, 16,384 x 1,024 77 and 82;
// 8,192 x 4,096 143 and 132.  One channel: 4 (4,099 x 640, 8: 27.1 and 25.6).
template <int VEC>
struct FwdWaves {
  static constexpr int kFew = VEC == 1 ? 16 : 8, kMany = 8, kUntil = 16384;
  static constexpr int most(bool look) { return look ? kFew : kMany; }
};
template <int VEC>
struct BwdWaves {
  static constexpr int kFew = VEC == 1 ? 4 : 8, kMany = 4, kUntil = 8192;
  static constexpr int most(bool look) { return look ? kFew : kMany; }
};
constexpr int kFwdOcc = 4, kBwdOcc = 2;  // waves a SIMD holds, by their registers
constexpr int kGroup = 4;  // tiles of a group (8, 16: the same times)
constexpr int kBack = 4;   // groups before its own that a tile looks at together
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

// What the tiles of a pass start from, formed by a kernel before them: no
// word is set, no tile is taken; the channels' -c softplus(lam), which every
// window would otherwise form again; and for each window whether all of its
// tokens are inner ones of one sequence, which most windows' are.
struct Begin {
  unsigned long long* words;
  int64_t num_words;
  unsigned int* ticket;
  const float* lam;
  float c;
  float* k;
  int64_t D, width;
  int* plain;
  int64_t windows;
  const void* cu;
  int cu64, N, run, total;
};
__global__ void __launch_bounds__(256) glr_begin_kernel(Begin p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t w = i; w < p.windows; w += step) {
    const int64_t w0 = w * kTok, w1 = w0 + kTok;
    int lo = 0, hi = p.N;  // the first sequence that ends behind token w1
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if (cu_at(p.cu, p.cu64, mid + 1, p.run, p.total) > w1)
        hi = mid;
      else
        lo = mid + 1;
    }
    p.plain[w] = lo < p.N && cu_at(p.cu, p.cu64, lo, p.run, p.total) < w0;
  }
  for (int64_t j = i; j < p.width; j += step) p.k[j] = j < p.D ? -p.c * softplus_f32(p.lam[j]) : 0.f;
  // Pairs of words: a row's are a multiple of 64.
  u32x4* pairs = reinterpret_cast<u32x4*>(p.words);
  for (int64_t j = i; j < p.num_words / 2; j += step) pairs[j] = u32x4{~0u, ~0u, ~0u, ~0u};
  if (i == 0) *p.ticket = 0;
}

// The channels of a lane: VEC of them, 4 bytes of a row (2 where a 16-bit row
// has one channel).  The last lane of an odd D takes the last two channels and
// answers for the second one only.
constexpr unsigned int kRange = 1u << 31;  // more than 16 rows span (checked on the host)
template <int VEC>
struct Lane {
  unsigned int off;  // of its first element in the block's rows, kRange: no channels
  // Its first channel: 32 bits where two channels leave few registers
  // (16,384 x 4,096 bf16 126.6 us, with 64 bits 128.4; fp32 4,099 x 640 forward
  // and backward 47.7 and 47.0).
  typename std::conditional<VEC == 2, unsigned int, int64_t>::type ch;
  bool ok[VEC];
  bool half;  // ok[1] alone
  bool odd;   // the block has such a lane
};
template <typename T, int VEC>
__device__ __forceinline__ Lane<VEC> lane_of(unsigned int lane, int64_t col, int64_t D) {
  const int64_t left = D - col - static_cast<int64_t>(lane) * VEC;
  Lane<VEC> l;
  l.odd = VEC == 2 && (D & 1) && D - col < kWave * VEC;
  l.half = VEC == 2 && left == 1;
  l.ch = static_cast<decltype(l.ch)>(col) + lane * VEC - l.half;
  // Rows of an odd block start one element before its channels.
  l.off = left > 0 ? (lane * VEC + (l.odd && !l.half)) * static_cast<unsigned int>(sizeof(T))
                   : kRange;
#pragma unroll
  for (int u = 0; u < VEC; ++u) l.ok[u] = left > 0 && !(l.half && u == 0);
  return l;
}

// Two 16-bit elements in one word, by one conversion of both (element by
// element the compiler converts twice and joins the halves).
template <typename T>
__device__ __forceinline__ unsigned int pack2(float lo, float hi) {
  typedef T T2 __attribute__((ext_vector_type(2)));
  typedef float F2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned int, __builtin_convertvector((F2{lo, hi}), T2));
}

// A window's rows of one tensor at the block's channels, as a buffer: the row
// of a token is a scalar offset, a lane's word, at any address, a vector
// offset that lanes without channels put out of range, where loads give 0 and
// stores do nothing.
template <typename T, int VEC>
struct Rows {
  __amdgpu_buffer_rsrc_t rsrc;
  unsigned int pitch;  // bytes
  __device__ __forceinline__ Rows(const void* p, int64_t row, int64_t pitch_elems, int64_t col,
                                  bool odd)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(static_cast<const char*>(p)) +
                (row * pitch_elems + col - odd) * static_cast<int64_t>(sizeof(T)),
            0, kRange, 0x00027000)),
        pitch(static_cast<unsigned int>(pitch_elems * sizeof(T))) {}
  __device__ __forceinline__ unsigned int ld(int j, unsigned int off) const {
    if constexpr (kBytes == 2)
      return __builtin_amdgcn_raw_buffer_load_b16(rsrc, off, j * pitch, kStream);
    else
      return __builtin_amdgcn_raw_buffer_load_b32(rsrc, off, j * pitch, kStream);
  }
  // ODD: the block may have a half lane.
  template <bool ODD>
  __device__ __forceinline__ void st(int j, const Lane<VEC>& at, const float (&v)[VEC]) const {
    if constexpr (kBytes == 2) {
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, from_f32<T>(v[0])),
                                            rsrc, at.off, j * pitch, kStream);
    } else {
      unsigned int w;
      if constexpr (VEC == 2)
        w = pack2<T>(v[0], v[1]);
      else
        w = __builtin_bit_cast(unsigned int, v[0]);
      if (ODD && VEC == 2 && at.odd) {
        __builtin_amdgcn_raw_buffer_store_b32(w, rsrc, at.half ? kRange : at.off, j * pitch,
                                              kStream);
        __builtin_amdgcn_raw_buffer_store_b16(static_cast<unsigned short>(w >> 16), rsrc,
                                              at.half ? at.off + 2 : kRange, j * pitch, kStream);
      } else {
        __builtin_amdgcn_raw_buffer_store_b32(w, rsrc, at.off, j * pitch, kStream);
      }
    }
  }

 private:
  static constexpr int kBytes = VEC * sizeof(T);
  static constexpr int kStream = 2;  // nt: read or written once
};

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

// A lane's -c softplus(lam); `ch`: its place in k, which has one for each word.
template <int VEC, bool LOOK, typename P>
__device__ __forceinline__ void ld_k(const P& p, const Lane<VEC>& at, int64_t ch, float (&k)[VEC]) {
#pragma unroll
  for (int u = 0; u < VEC; ++u) {
    if constexpr (LOOK)
      k[u] = p.k[ch + u - at.half];
    else
      k[u] = at.ok[u] ? -p.c * softplus_f32(p.lam[at.ch + u]) : 0.f;
  }
}

// fp32 rows of the same channels; `p`: at channel 0.
template <int VEC>
__device__ __forceinline__ void ld_f32(const float* p, const Lane<VEC>& at, float (&v)[VEC]) {
#pragma unroll
  for (int u = 0; u < VEC; ++u) v[u] = at.ok[u] ? p[at.ch + u] : 0.f;
}
template <int VEC>
__device__ __forceinline__ void st_f32(float* p, const Lane<VEC>& at, const float (&v)[VEC]) {
#pragma unroll
  for (int u = 0; u < VEC; ++u)
    if (at.ok[u]) p[at.ch + u] = v[u];
}

// The sequences' bounds, with the lane's own (of the first 64 sequences)
// requested together.  Windows that are known to be plain need none of them.
struct Seqs {
  const void* cu;
  int cu64, N, run, total;
  int t0, t1, lo, hi;
  __device__ __forceinline__ int operator()(int n) const {
    return cu_at(cu, cu64, n, run, total);
  }
  __device__ __forceinline__ Seqs(const void* c, int c64, int64_t n, int64_t r, int64_t tokens)
      : cu(c), cu64(c64), N(static_cast<int>(n)), run(static_cast<int>(r)),
        total(static_cast<int>(tokens)) {
    const int lane = threadIdx.x % kWave;
    t0 = (*this)(lane < N ? lane : N);
    t1 = (*this)(lane < N ? lane + 1 : N);
    lo = (*this)(0);
    hi = (*this)(N);
  }
};

// Where sequences start and end in a window: bit j of a mask and entry j of a
// table (the sequence) for token w0 + j.  `lo`, `hi`: the tokens that belong to
// sequences.
struct Marks {
  unsigned int starts, ends;
  int lo, hi;
};

// Called by a whole wave; seqs: 2 * kTok entries of LDS of its own.  empty(n) is
// called, by the wave together, for every empty sequence that the window
// answers for: the ones that stand before one of its tokens, and behind the
// last token those of the last window.
template <typename Empty>
__device__ __forceinline__ Marks find_marks(const Seqs& at, int w0, int* seqs, Empty empty) {
  const int lane = threadIdx.x % kWave, N = at.N, total = at.total;
  const bool last = w0 < total + kTok && w0 + kTok >= total;
  Marks m;
  m.lo = __builtin_amdgcn_readfirstlane(at.lo);
  m.hi = __builtin_amdgcn_readfirstlane(at.hi);
  m.starts = m.ends = 0;
  bool any = false;
  // The first sequence that does not end before the window.
  int base = 0, len = N;
  while (len > kWave) {
    const int step = (len - 1) / kWave + 1;
    const int64_t q = static_cast<int64_t>(lane) * step + step - 1;
    const uint64_t hit = __ballot(q >= len - 1 || at(base + static_cast<int>(q) + 1) >= w0);
    const int f = __builtin_ctzll(hit) * step;
    base += f;
    len = len - f < step ? len - f : step;
  }
  for (; base < N; base = base > N - kWave ? N : base + kWave) {
    const int n = base + lane;  // below 2^31 + 64: compared as unsigned
    int t0 = at.t0, t1 = at.t1;
    const bool in = static_cast<unsigned int>(n) < static_cast<unsigned int>(N);
    if (base > 0) {
      t0 = at(in ? n : N);
      t1 = at(in ? n + 1 : N);
    }
    const unsigned int s = t0 - w0, e = t1 - 1 - w0;
    const bool starts = t0 < t1 && s < kTok, ends = t0 < t1 && e < kTok;
    if (__any(starts || ends)) {
      if (!any && lane < 2 * kTok) seqs[lane] = -1;
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      any = true;
      if (starts) seqs[s] = n;
      if (ends) seqs[kTok + e] = n;
    }
    const bool mine = in && t0 >= t1 && t0 >= w0 && (t0 < w0 + kTok || last);
    for (uint64_t left = __ballot(mine); left; left &= left - 1)
      empty(static_cast<int64_t>(base) + __builtin_ctzll(left));
    if (!last && __any(t0 >= w0 + kTok)) break;
  }
  if (any) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint64_t set = __ballot(lane < 2 * kTok && seqs[lane & (2 * kTok - 1)] >= 0);
    m.starts = static_cast<unsigned int>(set) & ((1u << kTok) - 1);
    m.ends = static_cast<unsigned int>(set >> kTok) & ((1u << kTok) - 1);
  }
  return m;
}

// The words of a pass: tiles [tiles][width], groups [groups][width].
struct Words {
  unsigned long long* tile;
  unsigned long long* group;
  int64_t width;
};

// Publishes the span of tile `at` (counted in the order of the pass, `whole`
// in the wave `closer`) and gives the state that enters the tile to all waves
// of the block; `need`: the tile does not begin with a sequence.
template <int VEC>
__device__ __forceinline__ void enter(const Words& words, unsigned int at, unsigned int lane,
                                      int wave, int waves, int closer, bool need,
                                      const Span (&whole)[VEC], Span (*look)[kWave * VEC],
                                      float (*state)[kWave * VEC], float (&H)[VEC]) {
  const bool closing = wave == closer;
  const unsigned int group = at / kGroup;
  const int inside = at % kGroup;
  const bool leads = inside == kGroup - 1;  // answers for the group's word
  unsigned long long* mine = words.tile + at * words.width + lane * VEC;
  if (closing) {
#pragma unroll
    for (int u = 0; u < VEC; ++u)
      publish(mine + u, at == 0 ? Span{-1.f, apply(whole[u], 0.f)} : whole[u]);
  }
  if (at == 0 || !(need || leads)) return;

  // The closing wave asks for the groups' words, the others for those before
  // this tile's in the group: look[d - 1] is d tiles before.
  const int back = group < kBack ? static_cast<int>(group) : kBack;
  unsigned long long* out = words.group + group * words.width + lane * VEC;
  unsigned long long g[kBack][VEC];
  auto ask = [&]() {
#pragma unroll
    for (int d = 0; d < kBack; ++d) {
      // Beyond the first group: the nearest one again.
      const int64_t at_d = d < back ? d + 1 : (back > 0 ? 1 : 0);
#pragma unroll
      for (int u = 0; u < VEC; ++u) g[d][u] = peek(out - at_d * words.width + u);
    }
  };
  const int askers = waves > 1 ? waves - 1 : 1;
  if (closing) ask();
  if (!closing || waves == 1) {
    const int first = waves == 1 || wave < closer ? wave : wave - 1;
    for (int d = first + 1; d <= inside; d += askers) {
      unsigned long long w[VEC];
      for (;;) {
        bool unset = false;
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
          w[u] = peek(mine - d * words.width + u);
          unset |= w[u] == kUnset;
        }
        if (!__any(unset)) break;
        __builtin_amdgcn_s_sleep(1);
      }
#pragma unroll
      for (int u = 0; u < VEC; ++u) look[d - 1][lane * VEC + u] = unpack(w[u]);
    }
  }
  __syncthreads();
  if (closing) {
    // From the group's start to this tile's, and with this tile.
    Span head[VEC], all[VEC];
    bool known = true;
#pragma unroll
    for (int u = 0; u < VEC; ++u) head[u] = {1.f, 0.f};
    for (int d = inside; d > 0; --d) {
#pragma unroll
      for (int u = 0; u < VEC; ++u) head[u] = join(head[u], look[d - 1][lane * VEC + u]);
    }
#pragma unroll
    for (int u = 0; u < VEC; ++u) {
      all[u] = join(head[u], whole[u]);
      if (leads) publish(out + u, all[u]);
      known &= head[u].A < 0.f;
    }
    float G[VEC] = {};  // the state that enters the group
    if (!__all(known)) {
      for (;;) {
        // The nearest word that is final for every channel, if all nearer
        // ones are set.
        int last = -1;
        bool clear = true;
#pragma unroll
        for (int d = 0; d < kBack; ++d) {
          bool unset = d >= back, final = true;
#pragma unroll
          for (int u = 0; u < VEC; ++u) {
            unset |= g[d][u] == kUnset;
            final &= unpack(g[d][u]).A < 0.f;
          }
          if (__any(unset)) clear = false;
          if (clear && last < 0 && __all(final)) last = d;
        }
        if (last >= 0) {
#pragma unroll
          for (int d = kBack - 1; d >= 0; --d) {
            if (d <= last) {
#pragma unroll
              for (int u = 0; u < VEC; ++u) G[u] = apply(unpack(g[d][u]), G[u]);
            }
          }
          break;
        }
        __builtin_amdgcn_s_sleep(1);
        ask();
      }
    }
#pragma unroll
    for (int u = 0; u < VEC; ++u) {
      state[0][lane * VEC + u] = apply(head[u], G[u]);
      if (leads) publish(out + u, {-1.f, apply(all[u], G[u])});
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < VEC; ++u) H[u] = state[0][lane * VEC + u];
}

template <typename T, int VEC, bool LOOK>
__global__ void __launch_bounds__(FwdWaves<VEC>::most(LOOK) * kWave, LOOK ? kFwdOcc : 1)
    glr_fwd_kernel(FwdParams p) {
  constexpr int kWaves = FwdWaves<VEC>::most(LOOK);
  constexpr int kCols = kWave * VEC;
  __shared__ unsigned int taken;
  __shared__ int seqs[kWaves][2 * kTok];
  __shared__ Span spans[kWaves][kCols];
  __shared__ Span look[LOOK ? kGroup - 1 : 1][kCols];
  __shared__ float state[1][kCols];
  __shared__ int open;  // the tile needs the state before it

  const unsigned int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int waves = blockDim.x / kWave;
  const int total = static_cast<int>(p.total);
  unsigned int id = blockIdx.x;
  if constexpr (LOOK) {
    if (threadIdx.x == 0)
      taken = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if constexpr (LOOK) {
    __syncthreads();
    id = __builtin_amdgcn_readfirstlane(taken);
  }
  const unsigned int tile = id / static_cast<unsigned int>(p.blocks);
  const unsigned int blk = id % static_cast<unsigned int>(p.blocks);
  const int64_t row = (static_cast<int64_t>(tile) * waves + wave) * kTok;
  const int64_t col = static_cast<int64_t>(blk) * kCols;
  // Windows behind the last token hold none of them.
  const int w0 = row < total + kTok ? static_cast<int>(row) : total + kTok;
  const Lane<VEC> at = lane_of<T, VEC>(lane, col, p.D);

  float k[VEC];
  const bool plain = LOOK && !at.odd && p.plain[tile * waves + wave];
  ld_k<VEC, LOOK>(p, at, col + lane * VEC, k);
  // All of the window's loads, before anything else.
  unsigned int x[kTok], a[kTok], b[kTok];
  {
    const Rows<T, VEC> xr(p.x, row, p.sx, col, at.odd), ar(p.a, row, p.sa, col, at.odd),
        br(p.b, row, p.sb, col, at.odd);
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      const unsigned int off = w0 + j < total ? at.off : kRange;
      a[j] = ar.ld(j, off);
      b[j] = br.ld(j, off);
      x[j] = xr.ld(j, off);
    }
  }
  auto seq_row = [&](int n) {
    return static_cast<int64_t>(__builtin_amdgcn_readfirstlane(n)) * p.D;
  };
  Marks m{0, 0, 0, 0};
  if (!plain) {
    m = find_marks(Seqs(p.cu, p.cu64, p.N, p.T, p.total), w0, seqs[wave], [&](int64_t n) {
      if (!p.fin) return;
      float h[VEC] = {};
      if (p.h0) ld_f32<VEC>(p.h0 + n * p.D, at, h);
      st_f32<VEC>(p.fin + n * p.D, at, h);
    });
  }

  // The window's gates, and its span; a start folds its state into the input.
  float keep[kTok][VEC], add[kTok][VEC];
  Span span[VEC];
#pragma unroll
  for (int u = 0; u < VEC; ++u) span[u] = {1.f, 0.f};
  auto gates = [&](auto near, auto starts) {
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        const Gate g = gate_of<near>(k[u], sigmoid(lane_f32<T>(a[j], u)));
        keep[j][u] = g.word;
        add[j][u] = g.s * (sigmoid(lane_f32<T>(b[j], u)) * lane_f32<T>(x[j], u));
      }
      if (starts && (m.starts >> j & 1)) {
        float h[VEC] = {};
        if (p.h0) ld_f32<VEC>(p.h0 + seq_row(seqs[wave][j]), at, h);
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
          add[j][u] += decayed<near>(keep[j][u], h[u]);
          span[u].B = 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        span[u].A = decayed<near>(keep[j][u], span[u].A);
        // Not left for the tokens' end, which would hold every token's choice.
        if (!near && j % 2) later(span[u].A);
        span[u].B = decayed<near>(keep[j][u], span[u].B) + add[j][u];
      }
      if (!near) __builtin_amdgcn_sched_barrier(0);
    }
    if (starts && m.starts) {
#pragma unroll
      for (int u = 0; u < VEC; ++u) span[u].A = -1.f;
    }
  };
  bool near = true;
#pragma unroll
  for (int u = 0; u < VEC; ++u) near &= k[u] >= kNear;
  const bool fast = plain && __all(near);
  if (fast)
    gates(std::true_type(), std::false_type());
  else
    gates(std::false_type(), std::true_type());
#pragma unroll
  for (int u = 0; u < VEC; ++u) spans[wave][lane * VEC + u] = span[u];
  if (threadIdx.x == 0) open = !(m.starts & 1);
  __syncthreads();

  // From the tile's start to this window's.
  Span head[VEC];
#pragma unroll
  for (int u = 0; u < VEC; ++u) head[u] = {1.f, 0.f};
  for (int w = 0; w < wave; ++w) {
#pragma unroll
    for (int u = 0; u < VEC; ++u) head[u] = join(head[u], spans[w][lane * VEC + u]);
  }
  float h[VEC] = {};
  if constexpr (LOOK) {
    const Words words{p.words + col, p.words + p.tiles * p.width + col, p.width};
    Span whole[VEC];
#pragma unroll
    for (int u = 0; u < VEC; ++u) whole[u] = join(head[u], span[u]);
    enter<VEC>(words, tile, lane, wave, waves, waves - 1, open, whole, look, state, h);
  }
#pragma unroll
  for (int u = 0; u < VEC; ++u) h[u] = apply(head[u], h[u]);
  if (p.states && w0 < total) st_f32<VEC>(p.states + row / kWin * p.D, at, h);
  const Rows<T, VEC> yr(p.y, row, p.sy, col, at.odd);
  auto outputs = [&](auto near, auto marks) {
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      if (marks && (m.starts >> j & 1)) {
#pragma unroll
        for (int u = 0; u < VEC; ++u) h[u] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        if (!near) later(keep[j][u]);  // nor the first pass's
        h[u] = decayed<near>(keep[j][u], h[u]) + add[j][u];
      }
      if (!marks || (w0 + j >= m.lo && w0 + j < m.hi)) yr.template st<marks>(j, at, h);
      if (marks && (m.ends >> j & 1) && p.fin)
        st_f32<VEC>(p.fin + seq_row(seqs[wave][kTok + j]), at, h);
    }
  };
  if (fast)
    outputs(std::true_type(), std::false_type());
  else if (plain)
    outputs(std::false_type(), std::false_type());
  else
    outputs(std::false_type(), std::true_type());
}

// Tiles, channel blocks and waves of a block for a problem.
struct Cut {
  int64_t tiles;
  int blocks, waves;
  int64_t width;  // words of a tile
};
template <template <int> class Waves, int VEC>
Cut cut_of(int64_t total, int64_t D) {
  using W = Waves<VEC>;
  Cut c;
  const int64_t windows = std::max<int64_t>(cdiv(total, kTok), 1);
  c.blocks = static_cast<int>(cdiv(D, kWave * VEC));
  const bool few = windows > W::kMany && windows * c.blocks <= W::kUntil;
  c.waves = static_cast<int>(std::min<int64_t>(windows, few ? W::kFew : W::kMany));
  if (few && windows <= W::kFew) c.waves = W::kMany;  // two tiles
  c.tiles = cdiv(windows, c.waves);
  c.width = static_cast<int64_t>(c.blocks) * kWave * VEC;
  return c;
}
// The workspace of a pass: its counter (a cache line of its own), its
// channels' k, its windows' flags and the words of its tiles and groups; none
// for one tile.
inline int64_t up256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
inline int64_t words_of(const Cut& c) { return (c.tiles + cdiv(c.tiles, kGroup)) * c.width; }
inline int64_t words_bytes(const Cut& c) {
  if (c.tiles == 1) return 0;
  return 256 + up256(c.width * 4) + up256(c.tiles * c.waves * 4) + words_of(c) * 8;
}

// Lays a pass out in p and starts the kernel that readies its workspace.
template <typename P>
void begin(P& p, const Cut& c, void* workspace, hipStream_t s) {
  p.blocks = c.blocks;
  p.tiles = c.tiles;
  p.width = c.width;
  if (c.tiles == 1) return;
  char* at = static_cast<char*>(workspace);
  p.ticket = reinterpret_cast<unsigned int*>(at);
  float* k = reinterpret_cast<float*>(at += 256);
  int* plain = reinterpret_cast<int*>(at += up256(c.width * 4));
  p.words = reinterpret_cast<unsigned long long*>(at += up256(c.tiles * c.waves * 4));
  p.k = k;
  p.plain = plain;
  const Begin b{p.words, words_of(c), p.ticket, p.lam, p.c, k, p.D, c.width, plain,
                c.tiles * c.waves, p.cu, p.cu64, static_cast<int>(p.N), static_cast<int>(p.T),
                static_cast<int>(p.total)};
  const int64_t grid = std::min<int64_t>(cdiv(b.num_words, 2 * 256), 4 * num_cus());
  hipLaunchKernelGGL(glr_begin_kernel, dim3(grid), dim3(256), 0, s, b);
}

template <typename T, int VEC>
int launch_fwd_vec(FwdParams p, void* workspace, hipStream_t s) {
  const Cut c = cut_of<FwdWaves, VEC>(p.total, p.D);
  begin(p, c, workspace, s);
  const dim3 grid(c.tiles * c.blocks), block(c.waves * kWave);
  if (c.tiles > 1)
    hipLaunchKernelGGL((glr_fwd_kernel<T, VEC, true>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((glr_fwd_kernel<T, VEC, false>), grid, block, 0, s, p);
  return launch_status();
}
template <typename T>
int launch_fwd(const FwdParams& p, void* workspace, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (p.D > 1) return launch_fwd_vec<T, 2>(p, workspace, s);
  }
  return launch_fwd_vec<T, 1>(p, workspace, s);
}

// ---------------------------------------------------------------------------
// Decode: a wave per sequence and 64 VEC channels, its state in registers over
// the window's tokens.  At one token it is all latency: the token's inputs are
// requested before the slot is known, and the tokens of a drafted window
// kUpdTok at a time.
// ---------------------------------------------------------------------------
constexpr int kUpdTok = 4;

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
  unsigned int blocks;  // of a sequence
};

// VEC elements at any address, `left` of which exist.
typedef u32x2 Word2At2 __attribute__((aligned(2)));
typedef u32x4 Word4At4 __attribute__((aligned(4)));
template <int BYTES, int ALIGN> struct UpdWord { using type = void; };
template <> struct UpdWord<8, 2> { using type = Word2At2; using raw = u32x2; };
template <> struct UpdWord<16, 4> { using type = Word4At4; using raw = u32x4; };
template <int VEC, typename T>
__device__ __forceinline__ Arr<T, VEC> ld_some(const T* p, int64_t left) {
  Arr<T, VEC> q;
  if constexpr (VEC == 1) {
    q.v[0] = *p;
  } else if (left >= VEC) {
    using W = UpdWord<VEC * sizeof(T), sizeof(T)>;
    const typename W::raw w = *reinterpret_cast<const typename W::type*>(p);
    __builtin_memcpy(&q, &w, sizeof(q));
  } else {
#pragma unroll
    for (int u = 0; u < VEC; ++u) q.v[u] = p[u < left ? u : 0];
  }
  return q;
}
template <int VEC, typename T>
__device__ __forceinline__ void st_some(T* p, const float (&v)[VEC], int64_t left) {
  Arr<T, VEC> q;
#pragma unroll
  for (int u = 0; u < VEC; ++u) q.v[u] = from_f32<T>(v[u]);
  if constexpr (VEC == 1) {
    *p = q.v[0];
  } else if (left >= VEC) {
    using W = UpdWord<VEC * sizeof(T), sizeof(T)>;
    typename W::raw w;
    __builtin_memcpy(&w, &q, sizeof(q));
    *reinterpret_cast<typename W::type*>(p) = w;
  } else {
#pragma unroll
    for (int u = 0; u < VEC; ++u)
      if (u < left) p[u] = q.v[u];
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kWave) glr_update_kernel(UpdateParams p) {
  const int64_t n = blockIdx.x / p.blocks;
  const int64_t ch =
      (static_cast<int64_t>(blockIdx.x % p.blocks) * kWave + threadIdx.x) * VEC;
  const int64_t left = p.D - ch;
  if (left <= 0) return;
  const int run = static_cast<int>(p.T), total = static_cast<int>(p.total);
  const int64_t t0 = cu_at(p.cu, p.cu64, static_cast<int>(n), run, total);
  const int64_t t1 = cu_at(p.cu, p.cu64, static_cast<int>(n) + 1, run, total);
  Arr<T, VEC> x[kUpdTok], a[kUpdTok], b[kUpdTok];
  auto load = [&](int64_t from) {
#pragma unroll
    for (int j = 0; j < kUpdTok; ++j) {
      const int64_t t = from + j;
      if (t < t1) {
        a[j] = ld_some<VEC>(static_cast<const T*>(p.a) + t * p.sa + ch, left);
        b[j] = ld_some<VEC>(static_cast<const T*>(p.b) + t * p.sb + ch, left);
        x[j] = ld_some<VEC>(static_cast<const T*>(p.x) + t * p.sx + ch, left);
      }
    }
  };
  load(t0);
  const Arr<float, VEC> lam = ld_some<VEC>(p.lam + ch, left);
  const int64_t width = p.cols > 0 ? p.cols : 1;
  int64_t col = p.acc ? static_cast<int64_t>(p.acc[n]) - 1 : 0;
  col = col < 0 ? 0 : (col >= width ? width - 1 : col);
  auto slot_at = [&](int64_t c) -> int64_t { return p.idx ? p.idx[n * width + c] : n; };
  auto inside = [&](int64_t slot) { return slot >= 0 && slot < p.num_slots; };
  const int64_t first = slot_at(col);
  float h[VEC] = {}, k[VEC];
  if (inside(first)) {
    const Arr<float, VEC> q = ld_some<VEC>(p.state + first * p.slot_pitch + ch, left);
#pragma unroll
    for (int u = 0; u < VEC; ++u) h[u] = q.v[u];
  }
#pragma unroll
  for (int u = 0; u < VEC; ++u) k[u] = -p.c * softplus_f32(lam.v[u]);
  auto tokens = [&](int64_t from) {
#pragma unroll
    for (int j = 0; j < kUpdTok; ++j) {
      const int64_t t = from + j;
      if (t < t1) {
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
          const Gate g = gate_of<false>(k[u], sigmoid(to_f32(a[j].v[u])));
          h[u] = decayed<false>(g.word, h[u]) +
                 g.s * (sigmoid(to_f32(b[j].v[u])) * to_f32(x[j].v[u]));
        }
        st_some<VEC>(static_cast<T*>(p.y) + t * p.sy + ch, h, left);
        if (t - t0 < p.cols) {
          const int64_t slot = slot_at(t - t0);
          if (inside(slot)) st_some<VEC>(p.state + slot * p.slot_pitch + ch, h, left);
        }
      }
    }
  };
  tokens(t0);
  for (int64_t from = t0 + kUpdTok; from < t1; from += kUpdTok) {
    load(from);
    tokens(from);
  }
  if (p.cols == 0 && t1 > t0 && inside(first))
    st_some<VEC>(p.state + first * p.slot_pitch + ch, h, left);
}

template <typename T, int VEC>
int launch_update(UpdateParams p, hipStream_t s) {
  const int64_t blocks = cdiv(p.D, kWave * VEC);
  if (p.N * blocks >= int64_t{1} << 26) return XK_ERR_INVALID;  // 2^32 threads
  p.blocks = static_cast<unsigned int>(blocks);
  hipLaunchKernelGGL((glr_update_kernel<T, VEC>), dim3(p.N * blocks), dim3(kWave), 0, s, p);
  return launch_status();
}
// One channel a lane while the chip holds all of these lanes at once (32 waves
// a compute unit), else four (64 sequences x 2,048 channels, 4 drafts: 4.8 us
// with one, 6.4 with four; 256 x 4,096: 8.0 and 6.0).
template <typename T>
int run_update(const UpdateParams& p, hipStream_t s) {
  return p.N * p.D > int64_t{32} * kWave * num_cus() ? launch_update<T, 4>(p, s)
                                                     : launch_update<T, 1>(p, s);
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
  float* part;  // dlam's parts, [tiles][D] (one tile: dlam); NULL: not asked for
  const void* cu;
  int cu64;
  int64_t N, T, total, D;
  const float* k;
  const int* plain;
  unsigned long long* words;
  unsigned int* ticket;
  int64_t tiles, width;
  int blocks;
};

// sigmoid(lam) / softplus(lam), 1 in the limit lam -> -inf.
__device__ __forceinline__ float slope_ratio(float lam) {
  if (lam < -17.f) return 1.f;  // 1 - e^lam / 2 rounds to 1
  return 1.f / ((1.f + expf(-lam)) * softplus_f32(lam));
}

// exp(-v) for a sigmoid's value r = 1 / (1 + e) and its complement 1 - r = e r;
// capped at 2^126, so that e r is 1 and not inf * 0 for a closed gate: the
// largest power whose reciprocal is no denormal, which the instruction gives as
// 0 (at v = -80 a cap of 2^100 left r 4e4 times too large).  The
// minimum is the one that keeps a NaN (fminf gives the cap for it).
__device__ __forceinline__ float exp_neg(float v) {
  return __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(v * -1.44269504f, 126.f));
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
//  * Of the gates exp(-a), exp(-b), r and the decay stay in registers for the
//    second pass, in reverse order; the rest is cheaper formed again.  (With
//    the two exponentials alone 142 us instead of 134 for 8,192 x 4,096 bf16:
//    the arithmetic is as long as the traffic.)  132 us now, 3.6 TB/s, at 2
//    waves a SIMD.
//  * E = (dL/dl) l = G alpha (h_{t-1} l - i x alpha l / s) gives da = E (1 - r)
//    and dlam = sum E sigmoid(lam) / softplus(lam), with no division by what
//    vanishes as a gate closes: l / s -> 0 with s.
// ---------------------------------------------------------------------------
template <typename T, int VEC, bool LOOK>
__global__ void __launch_bounds__(BwdWaves<VEC>::most(LOOK) * kWave, LOOK ? kBwdOcc : 1)
    glr_bwd_kernel(BwdParams p) {
  constexpr int kWaves = BwdWaves<VEC>::most(LOOK);
  constexpr int kCols = kWave * VEC;
  __shared__ unsigned int taken;
  __shared__ int seqs[kWaves][2 * kTok];
  __shared__ Span spans[kWaves][kCols];
  __shared__ Span look[LOOK ? kGroup - 1 : 1][kCols];
  __shared__ float state[1][kCols];
  __shared__ float sums[kWaves][kCols];
  __shared__ int open;  // the tile needs the gradient from behind it

  const unsigned int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int waves = blockDim.x / kWave;
  const int total = static_cast<int>(p.total);
  unsigned int id = blockIdx.x;
  if constexpr (LOOK) {
    if (threadIdx.x == 0)
      taken = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if constexpr (LOOK) {
    __syncthreads();
    id = __builtin_amdgcn_readfirstlane(taken);
  }
  // Tiles are counted from the end here.
  const unsigned int behind = id / static_cast<unsigned int>(p.blocks);
  const unsigned int blk = id % static_cast<unsigned int>(p.blocks);
  const int64_t tile = p.tiles - 1 - behind;
  const int64_t row = (tile * waves + wave) * kTok;
  const int64_t col = static_cast<int64_t>(blk) * kCols;
  const int w0 = row < total + kTok ? static_cast<int>(row) : total + kTok;
  const Lane<VEC> at = lane_of<T, VEC>(lane, col, p.D);

  float k[VEC], h[VEC] = {};
  const bool plain = LOOK && !at.odd && p.plain[tile * waves + wave];
  ld_k<VEC, LOOK>(p, at, col + lane * VEC, k);
  if (w0 < total) ld_f32<VEC>(p.states + row / kWin * p.D, at, h);
  unsigned int x[kTok], dy[kTok], a[kTok], b[kTok];
  {
    const Rows<T, VEC> xr(p.x, row, p.sx, col, at.odd), ar(p.a, row, p.sa, col, at.odd),
        br(p.b, row, p.sb, col, at.odd), gr(p.dy, row, p.sdy, col, at.odd);
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      const unsigned int off = w0 + j < total ? at.off : kRange;
      a[j] = ar.ld(j, off);
      b[j] = br.ld(j, off);
      x[j] = xr.ld(j, off);
      dy[j] = gr.ld(j, off);
    }
  }
  auto seq_row = [&](int n) {
    return static_cast<int64_t>(__builtin_amdgcn_readfirstlane(n)) * p.D;
  };
  Marks m{0, 0, 0, 0};
  if (!plain) {
    m = find_marks(Seqs(p.cu, p.cu64, p.N, p.T, p.total), w0, seqs[wave], [&](int64_t n) {
      if (!p.dh0) return;
      float q[VEC] = {};
      if (p.dfin) ld_f32<VEC>(p.dfin + n * p.D, at, q);
      st_f32<VEC>(p.dh0 + n * p.D, at, q);
    });
  }

  float before[kTok][VEC], ea[kTok][VEC], eb[kTok][VEC], keep[kTok][VEC], rs[kTok][VEC];
  Span span[VEC];
#pragma unroll
  for (int u = 0; u < VEC; ++u) span[u] = {1.f, 0.f};
  auto first = [&](auto near, auto marks) {
#pragma unroll
    for (int j = 0; j < kTok; ++j) {
      if (marks && (m.starts >> j & 1)) {
#pragma unroll
        for (int u = 0; u < VEC; ++u) h[u] = 0.f;
        if (p.h0) ld_f32<VEC>(p.h0 + seq_row(seqs[wave][j]), at, h);
      }
      // No sequence ended before this token: the gradient comes this far.
      const bool reached = !marks || !(m.ends & ((1u << j) - 1));
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        ea[j][u] = exp_neg(lane_f32<T>(a[j], u));
        eb[j][u] = exp_neg(lane_f32<T>(b[j], u));
        rs[j][u] = fast_rcp(1.f + ea[j][u]);
        const Gate g = gate_of<near>(k[u], rs[j][u]);
        before[j][u] = h[u];
        keep[j][u] = g.word;
        // alpha's own rounding is let in: h lives for this window only.
        h[u] = fmaf(g.alpha, h[u], g.s * (fast_rcp(1.f + eb[j][u]) * lane_f32<T>(x[j], u)));
        if (reached) {
          span[u].A = decayed<near>(g.word, span[u].A);
          span[u].B = fmaf(span[u].A, lane_f32<T>(dy[j], u), span[u].B);
        }
      }
      if (marks && reached && (m.ends >> j & 1) && p.dfin) {
        float q[VEC];
        ld_f32<VEC>(p.dfin + seq_row(seqs[wave][kTok + j]), at, q);
#pragma unroll
        for (int u = 0; u < VEC; ++u) span[u].B = fmaf(span[u].A, q[u], span[u].B);
      }
    }
  };
  bool near = true;
#pragma unroll
  for (int u = 0; u < VEC; ++u) near &= k[u] >= kNear;
  const bool fast = plain && __all(near);
  if (fast)
    first(std::true_type(), std::false_type());
  else
    first(std::false_type(), std::true_type());
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
  float q[VEC] = {};
  if constexpr (LOOK) {
    const Words words{p.words + col, p.words + p.tiles * p.width + col, p.width};
    Span whole[VEC];
#pragma unroll
    for (int u = 0; u < VEC; ++u) whole[u] = join(head[u], span[u]);
    enter<VEC>(words, behind, lane, wave, waves, 0, open, whole, look, state, q);
  }
#pragma unroll
  for (int u = 0; u < VEC; ++u) q[u] = apply(head[u], q[u]);
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
  float sum[VEC] = {};
  const Rows<T, VEC> dxr(p.dx, row, p.sdx, col, at.odd), dar(p.da, row, p.sda, col, at.odd),
      dbr(p.db, row, p.sdb, col, at.odd);
  auto second = [&](auto near, auto marks) {
#pragma unroll
    for (int j = kTok - 1; j >= 0; --j) {
      if (marks && (m.ends >> j & 1)) {
#pragma unroll
        for (int u = 0; u < VEC; ++u) q[u] = 0.f;
        if (p.dfin) ld_f32<VEC>(p.dfin + seq_row(seqs[wave][kTok + j]), at, q);
      }
      const bool live = !marks || plain || (w0 + j >= m.lo && w0 + j < m.hi);
      float dx[VEC], da[VEC], db[VEC];
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        const float r = rs[j][u], i = fast_rcp(1.f + eb[j][u]);
        const float xf = lane_f32<T>(x[j], u), l = k[u] * r;
        const Decay d =
            near ? Decay{1.f + keep[j][u], keep[j][u], keep[j][u]} : decay_of<false>(l);
        const float w = -d.em1 * (1.f + d.alpha);  // s^2
        // The instruction takes a denormal w for 0; l and w, both tiny there,
        // keep the products with inv at 0 or below 2^-60.
        const float inv = __builtin_amdgcn_rsqf(fmaxf(w, 1.17549435e-38f));
        const float G = lane_f32<T>(dy[j], u) + q[u];
        dx[u] = G * (w * inv) * i;
        db[u] = dx[u] * xf * (eb[j][u] * i);
        const float e = G * d.alpha * (before[j][u] * l - i * xf * d.alpha * (l * inv));
        da[u] = e * (ea[j][u] * r);
        if (live) sum[u] += e;
        q[u] = decayed<near>(d.word, G);
      }
      if (live) {
        dxr.template st<marks>(j, at, dx);
        dar.template st<marks>(j, at, da);
        dbr.template st<marks>(j, at, db);
      }
      if (marks && (m.starts >> j & 1) && p.dh0)
        st_f32<VEC>(p.dh0 + seq_row(seqs[wave][j]), at, q);
    }
  };
  if (fast)
    second(std::true_type(), std::false_type());
  else
    second(std::false_type(), std::true_type());
  if (p.part) {
#pragma unroll
    for (int u = 0; u < VEC; ++u) sums[wave][lane * VEC + u] = sum[u];
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < waves; ++w) {
#pragma unroll
        for (int u = 0; u < VEC; ++u) sum[u] += sums[w][lane * VEC + u];
      }
      if constexpr (!LOOK) {  // the only tile: dlam itself
#pragma unroll
        for (int u = 0; u < VEC; ++u)
          if (at.ok[u]) sum[u] *= slope_ratio(p.lam[at.ch + u]);
      }
      st_f32<VEC>(p.part + tile * p.D, at, sum);
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

template <typename T, int VEC>
int launch_bwd_vec(BwdParams p, float* dlam, void* workspace, hipStream_t s) {
  const Cut c = cut_of<BwdWaves, VEC>(p.total, p.D);
  // The workspace: counter, k and words, then dlam's parts.
  if (dlam)
    p.part = c.tiles == 1
                 ? dlam
                 : reinterpret_cast<float*>(static_cast<char*>(workspace) + words_bytes(c));
  begin(p, c, workspace, s);
  const dim3 grid(c.tiles * c.blocks), block(c.waves * kWave);
  if (c.tiles > 1)
    hipLaunchKernelGGL((glr_bwd_kernel<T, VEC, true>), grid, block, 0, s, p);
  else
    hipLaunchKernelGGL((glr_bwd_kernel<T, VEC, false>), grid, block, 0, s, p);
  if (dlam && c.tiles > 1)
    hipLaunchKernelGGL(glr_dlam_kernel, dim3(cdiv(p.D, kWave)), dim3(1024), 0, s, p.part, c.tiles,
                       p.lam, dlam, p.D);
  return launch_status();
}
template <typename T>
int launch_bwd(const BwdParams& p, float* dlam, void* workspace, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (p.D > 1) return launch_bwd_vec<T, 2>(p, dlam, workspace, s);
  }
  return launch_bwd_vec<T, 1>(p, dlam, workspace, s);
}

// A window's rows have to lie within kRange bytes: the most elements of a pitch.
constexpr int64_t kMostPitch = kRange / (4 * kTok);
static_assert(kMostPitch == XK_GLR_PITCH);
bool pitch_ok(int64_t pitch, int64_t D) { return pitch >= D && pitch < kMostPitch; }

// A launch has fewer than 2^32 threads (of whole tiles), N is counted in 31 bits.
bool bad_sizes(int64_t N, int64_t total, int64_t D) {
  constexpr int64_t kMost = int64_t{1} << 26, kMostWaves = 16;
  return N < 0 || N >= int64_t{1} << 31 || total < 0 || total >= kMost * kTok || D <= 0 ||
         D >= kMostPitch || (cdiv(total, kTok) + kMostWaves) * cdiv(D, kWave) >= kMost;
}

bool c_ok(float c) { return c >= 0.f && c <= std::numeric_limits<float>::max(); }

// cu_seqlens of a readable type, or none and N equal runs.
bool seqs_ok(const void* cu, xk_dtype dt, int64_t N, int64_t total) {
  return cu ? dt == XK_I32 || dt == XK_I64 : total % N == 0;
}

}  // namespace
}  // namespace xk

using namespace xk;

extern "C" int64_t xk_gated_linear_recurrence_workspace_bytes(int64_t total_tokens, int64_t D) {
  if (bad_sizes(0, total_tokens, D)) return 0;
  // Of the types with one and two channels a lane.
  return std::max(words_bytes(cut_of<FwdWaves, 1>(total_tokens, D)),
                  words_bytes(cut_of<FwdWaves, 2>(total_tokens, D)));
}

extern "C" int xk_gated_linear_recurrence(
    const void* x, int64_t stride_x_tok, const void* a, int64_t stride_a_tok, const void* b,
    int64_t stride_b_tok, xk_dtype dtype, const float* lam, float c, void* y,
    int64_t stride_y_tok, const float* initial_state, float* final_state, float* states,
    const void* cu_seqlens, xk_dtype cu_dtype, int64_t N, int64_t total_tokens, int64_t D,
    void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_sizes(N, total_tokens, D) || !c_ok(c)) return XK_ERR_INVALID;
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
                    total_tokens / N, total_tokens, D, nullptr, nullptr, nullptr, nullptr, 0, 0, 0};
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
  if (bad_sizes(N, total_tokens, D) || num_slots < 0 || num_cols < 0 || !c_ok(c))
    return XK_ERR_INVALID;
  if (!is_float_dtype(dtype)) return XK_ERR_UNSUPPORTED;
  if (N == 0 || total_tokens == 0) return XK_OK;
  if (cu_seqlens ? cu_dtype != XK_I32 && cu_dtype != XK_I64 : T <= 0 || T > total_tokens / N)
    return XK_ERR_INVALID;
  // The inputs' rows may be any way apart: no offset of this kernel is 32 bits.
  if (!x || !a || !b || !y || !lam || (num_slots > 0 && !state) || stride_state_slot < D ||
      (num_cols > 0 && !state_indices) || stride_x_tok < D || stride_a_tok < D ||
      stride_b_tok < D || !pitch_ok(stride_y_tok, D))
    return XK_ERR_INVALID;
  const UpdateParams p{x, a, b, y, stride_x_tok, stride_a_tok, stride_b_tok, stride_y_tok, lam, c,
                       state, stride_state_slot, num_slots, state_indices, num_cols,
                       num_accepted_tokens, cu_seqlens, cu_dtype == XK_I64, N, T, total_tokens, D,
                       0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case XK_F32: return run_update<float>(p, s);
    case XK_BF16: return run_update<bf16>(p, s);
    default: return run_update<f16>(p, s);
  }
}

extern "C" int64_t xk_gated_linear_recurrence_bwd_workspace_bytes(int64_t total_tokens, int64_t N,
                                                                  int64_t D) {
  if (N <= 0 || bad_sizes(N, total_tokens, D)) return 0;
  const Cut c1 = cut_of<BwdWaves, 1>(total_tokens, D), c2 = cut_of<BwdWaves, 2>(total_tokens, D);
  return std::max(words_bytes(c1), words_bytes(c2)) + std::max(c1.tiles, c2.tiles) * D * 4;
}

extern "C" int xk_gated_linear_recurrence_bwd(
    const void* dy, int64_t stride_dy_tok, const void* x, int64_t stride_x_tok, const void* a,
    int64_t stride_a_tok, const void* b, int64_t stride_b_tok, xk_dtype dtype, const float* lam,
    float c, const float* states, const float* initial_state, const float* d_final_state,
    void* dx, int64_t stride_dx_tok, void* da, int64_t stride_da_tok, void* db,
    int64_t stride_db_tok, float* dlam, float* d_initial_state, const void* cu_seqlens,
    xk_dtype cu_dtype, int64_t N, int64_t total_tokens, int64_t D, void* workspace,
    size_t workspace_bytes, void* stream) {
  if (bad_sizes(N, total_tokens, D) || !c_ok(c)) return XK_ERR_INVALID;
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
                      nullptr, nullptr, 0, 0, 0};
    switch (dtype) {
      case XK_F32: return launch_bwd<float>(p, dlam, workspace, s);
      case XK_BF16: return launch_bwd<bf16>(p, dlam, workspace, s);
      default: return launch_bwd<f16>(p, dlam, workspace, s);
    }
  }
  if (dlam)  // no sequences: zeros
    hipLaunchKernelGGL(glr_dlam_kernel, dim3(cdiv(D, kWave)), dim3(1024), 0, s, nullptr, 0, lam,
                       dlam, D);
  return launch_status();
}
