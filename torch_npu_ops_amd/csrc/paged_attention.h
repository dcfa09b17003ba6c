// Attention of a sequence's new tokens over its pages of the key-value cache
// (xk_paged_attention), gfx950: the kernel and its instances' launch; the
// entry points are in paged_attention.hip.
//
// For a new token's query q at position t of a sequence and key-value head h
//     o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m),
// over the positions j <= t (and j > t - window), m the largest score.
//
// What bounds it: HBM.  Every key and value is read once and takes 2 flops a
// byte for each of the M = T * Hq / Hkv query rows that share the head, a
// small part of what the matrix cores do at that rate, so the rows of a
// 16-row MFMA tile that are not used cost nothing.
//
// Work: the positions of all sequences, in tiles of 16 (fp32) or 32, are one line
// that the blocks of a head cut in equal shares, on the device, from the
// lengths that are there (seq_lens never reaches the host); one block for each
// compute unit, two of some kinds.  A block goes through the sequences that its share
// touches, its 4 waves taking tiles in turn, each with statistics and sums of
// its own, and joins them at a sequence's end; the pieces of a sequence that
// lies in several shares are joined by a second launch.
//
// Tile: S^T = K Q^T and O^T = V^T P^T, so that lane l holds query row l % 16
// throughout (C layout: column l % 16, rows 4 (l / 16) + i): statistics and
// rescaling stay in the lane, up to the maximum over the four lane groups.
//   - Both K and V are loaded as they lie (16 lanes of 16 bytes read a row of
//     128 elements): with a row for each lane instead, as K's operand needs it,
//     a copy of the loads alone ran at 5.2 TB/s where whole rows ran at 6.7.
//     K passes through the wave's own part of LDS into the operand's layout.
//   - The order of a product's inner index is free as long as both sides use
//     the same: the scores of tokens 4g + i and 16 + 4g + i that lane group g
//     holds are the slots of group g in P^T, with V's tokens loaded to match,
//     and the lane's 8 tokens x 8 elements of V are turned in registers
//     (v_perm), one product for each of the 8 elements: product e has row
//     l % 16 <-> element 8 (l % 16) + e, so sums come out as 8 neighbours.
//   - The next tile's loads are requested as soon as this one's registers are
//     free, and the loop has no condition on them: with one the compiler waits
//     for the loads at the loop's end, to move their registers.
// For the product with V p is cut in bf16 parts, three that hold all its 24 bits,
// or in two of fp16, 22 bits, scaled by 2^14 so that small weights keep their
// digits.  Scores, statistics and sums are fp32.
//
// Measured (us a call, both launches; TB/s of the keys and values): one sequence
// of 524288, 8 bf16 heads of 128: 329 (6.5; a plain read of such rows 6.6 to 6.7);
// 131072: 91 (5.9); 64 of up to 4096 in pages of 16: 177 (6.1); the same with all
// of 4096 in e4m3: 94 (5.7); one of 900: 10.2.
#pragma once

#include <cmath>

#include "gdn_common.h"
#include "xk_common.h"

namespace xk {
namespace paged {

using gdn::f4_t;
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
struct f8 {  // e4m3, as stored
  unsigned char v;
};

constexpr int kWaves = 4;
constexpr int kBlock = kWaves * kWave;

struct Params {
  const void* q;
  int64_t q_seq, q_tok, q_head;  // elements
  const char* kc;
  int64_t k_head;   // bytes
  uint32_t k_page;  // 8 bytes
  uint32_t k_slot;  // bytes
  const char* vc;
  int64_t v_head;
  uint32_t v_page, v_slot;
  int num_pages, page_size;
  uint32_t page_magic;  // n / page_size = n * magic >> shift for n < 2^28
  int page_shift;
  const int32_t* table;
  int64_t table_row;
  int max_pages;
  const int32_t* lens;
  int most_len;  // positions that a row of the table can name
  float scale2;  // scale * log2(e)
  int window;    // 0: none
  const float* k_scale;
  const float* v_scale;
  void* out;
  int64_t o_seq, o_tok, o_head;
  float* lse;
  int B, T, G, Hkv, D, M, groups;  // M = T * G rows of a head in `groups` groups
  uint32_t g_magic;                // r / G = r * g_magic >> g_shift for r < 2^28
  int g_shift;
  int shares;                      // of a head and group, at the most
  int near;                        // log2 of the heads that share cache lines
  int2* meta;                      // [B]: first piece, pieces
  float2* ml;                      // [2 * shares][Hkv][M]: base, sum
  float* acc;                      // [2 * shares][Hkv][M][D]
};

// The kernel's arguments, loaded again: values that are used once a sequence are
// not kept in scalar registers through the loop, where they are short.
using LateParams = const __attribute__((address_space(4))) Params*;
__device__ __forceinline__ LateParams late_params() {
  auto x = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(x));
  return reinterpret_cast<LateParams>(x);
}
template <typename P>
__device__ __forceinline__ int token_of(P p, int r) {
  return static_cast<int>(static_cast<uint64_t>(r) * p->g_magic >> p->g_shift);
}

// A sequence's tiles: from the first that a row sees to the last; an empty
// sequence has one, so that its rows are written.
struct Span {
  int len, t0, n;
};
template <int TS>
__device__ __forceinline__ Span span_of(const Params& p, int b) {
  const int len = max(0, min(p.lens[b], p.most_len));
  const int lo = p.window ? max(0, len - p.T - p.window + 1) : 0;
  const int t0 = lo / TS, t1 = (len + TS - 1) / TS;
  return {len, t0, max(1, t1 - t0)};
}

// 64 sequences from b0 on, one a lane; `incl`: their tiles up to the lane's.
struct Batch {
  int b0;
  Span own;
  int incl;
};
template <int TS>
__device__ __forceinline__ Batch batch_at(const Params& p, int b0) {
  const int b = b0 + static_cast<int>(threadIdx.x % kWave);
  const Span own = b < p.B ? span_of<TS>(p, b) : Span{0, 0, 0};
  return {b0, own, gdn::wave_incl_scan(own.n)};
}

// (64-bit division takes 150 instructions.)
__device__ __forceinline__ int64_t divide(int64_t a, uint32_t b) {
  return a <= UINT32_MAX ? static_cast<uint32_t>(a) / b : a / b;
}
// Tiles of a share: one for each of the block's waves at the least (fewer, in
// more pieces, took 10.2 us instead of 9.7 for one sequence of 900; two 10.8),
// else as equal as they come (in whole rounds of the waves 7 fp32 sequences of
// 1777 took 23.2 us instead of 22.0, 48 of four new tokens 30.9 instead of 30.1).
__device__ __forceinline__ uint32_t share_size(int64_t total, int shares) {
  const int64_t n = divide(total + shares - 1, shares);
  return static_cast<uint32_t>(max<int64_t>(n, kWaves));
}

// ---------------------------------------------------------------------------
// Types: T of queries and outputs, C of the cache (T or f8).
// ---------------------------------------------------------------------------
template <typename T> struct Op;
template <> struct Op<bf16> { using type = bf8_t; };
template <> struct Op<f16> { using type = h8_t; };
template <> struct Op<float> { using type = f4_t; };

__device__ __forceinline__ f4_t mma(bf8_t a, bf8_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f4_t mma(h8_t a, h8_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// Four products of inner length 4 in place of one of 16.
__device__ __forceinline__ f4_t mma(f4_t a, f4_t b, f4_t c) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

// Two e4m3 values of a word as two of T (exact).
template <typename T>
__device__ __forceinline__ uint32_t widen(uint32_t w, bool high) {
  if constexpr (std::is_same<T, bf16>::value)
    return __builtin_bit_cast(uint32_t, high
        ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true)
        : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
  else
    return __builtin_bit_cast(uint32_t, high
        ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)
        : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
}

// Bytes in device memory; the type says so to the compiler where a pointer came
// from integers.
using GlobalBytes = const __attribute__((address_space(1))) char*;

// N elements of the cache as loaded, and as words of T.
template <typename T, typename C, int N>
struct alignas(N * sizeof(C) < 16 ? N * sizeof(C) : 16) Row {
  static constexpr int kBytes = N * static_cast<int>(sizeof(C));
  static constexpr int kRaw = kBytes / 4, kWords = N * static_cast<int>(sizeof(T)) / 4;
  uint32_t raw[kRaw];
  __device__ __forceinline__ void load(GlobalBytes at) {
    using U = typename RawOf<kBytes>::type;
    const U x = __builtin_nontemporal_load(
        reinterpret_cast<const __attribute__((address_space(1))) U*>(at));
    if constexpr (kRaw == 1) {
      raw[0] = x;
    } else {
#pragma unroll
      for (int i = 0; i < kRaw; ++i) raw[i] = x[i];
    }
  }
  __device__ __forceinline__ void keep(bool yes) {  // or zeros
#pragma unroll
    for (int i = 0; i < kRaw; ++i) raw[i] = yes ? raw[i] : 0;
  }
  __device__ __forceinline__ uint32_t word(int i) const {
    if constexpr (std::is_same<C, f8>::value) return widen<T>(raw[i / 2], i & 1);
    else return raw[i];
  }
  __device__ __forceinline__ bool finite() const {
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const uint32_t w = word(i);
      if constexpr (sizeof(T) == 4) {
        bad |= (w & 0x7f800000u) == 0x7f800000u;
      } else {
        constexpr uint32_t kExp = std::is_same<T, bf16>::value ? 0x7f80u : 0x7c00u;
        bad |= ((w & kExp) == kExp) | ((w >> 16 & kExp) == kExp);
      }
    }
    return bad == 0;
  }
};
// A word of T with NaN in the place of values that are not finite, 0 of others.
template <typename T>
__device__ __forceinline__ uint32_t only_nan(uint32_t w) {
  if constexpr (sizeof(T) == 4) return (w & 0x7f800000u) == 0x7f800000u ? 0x7fffffffu : 0u;
  constexpr uint32_t kExp = std::is_same<T, bf16>::value ? 0x7f80u : 0x7c00u;
  return ((w & kExp) == kExp ? 0x7fffu : 0u) | ((w >> 16 & kExp) == kExp ? 0x7fff0000u : 0u);
}
// 1 for infinity, 2 for minus infinity, 3 for NaN, else 0.
template <typename C>
__device__ __forceinline__ uint32_t not_finite(C x) {
  if constexpr (std::is_same<C, f8>::value) {
    return (x.v & 0x7f) == 0x7f ? 3 : 0;
  } else {
    const float y = to_f32(x);
    return y != y ? 3 : (y == INFINITY ? 1 : (y == -INFINITY ? 2 : 0));
  }
}

// Orders the wave's accesses to LDS: its lanes see what its others wrote
// before, and overwrite nothing that these have yet to read.  A wave's accesses
// run in the order of the program, so this takes no instruction; without it the
// compiler may exchange a lane's store and its load of what another lane stored.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// The larger of the values of lanes that differ in bits 4 and 5, and the sum.
template <typename F>
__device__ __forceinline__ float over_groups(float v, F f) {
  typedef unsigned int u2_t __attribute__((ext_vector_type(2)));
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  u2_t r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  uint32_t x = r[0], y = r[1];
  u = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y)));
  r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  x = r[0];
  y = r[1];
  return f(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}

// A wave-uniform address in scalar registers, to which loads add a lane's 32-bit
// offset: left to itself the compiler adds offsets first and keeps 64 bits for
// each lane and load.
__device__ __forceinline__ GlobalBytes scalar(uint64_t u) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u >> 32));
  return reinterpret_cast<GlobalBytes>(static_cast<uint64_t>(hi) << 32 | lo);
}

// The offset, not to be widened outside the loop: a load takes a scalar address
// and 32 bits a lane only where it sees both.
__device__ __forceinline__ uint32_t lane_offset(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// exp2(a - b) for a <= b, 0 where a is -inf (b then may be -inf too).
__device__ __forceinline__ float weight(float a, float b) {
  return exp2_hw(a - (b == -INFINITY ? 0.f : b));
}

// Two weights as parts of 16 bits, each cut off what the parts before it leave:
// three of bf16 hold all 24 bits of fp32 (in two of them, 16 bits, 3 to 5 of 4096
// outputs of a sequence of 900 were not the nearest bf16 values, 0 or 1 in fp32),
// two of fp16 22 bits, the last one rounded.  No part of a weight is negative, and
// none 0 (fp16's from 2^-38 on, bf16's from 2^-78), so that an infinite value
// times all of them is infinite: of a part 2^-24 is left to the next one in bf16
// (which is off by as much), fp16's second part is the smallest there is at least.
template <typename T> struct Parts {
  static constexpr int kCount = std::is_same<T, bf16>::value ? 3 : 2;
};
template <> struct Parts<float> {
  static constexpr int kCount = 1;
};
__device__ __forceinline__ void split2(float a, float b, uint32_t (&part)[3], bf16) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
    part[i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
    constexpr float kLess = -0x1.fffffep-1f;  // 2^-24 - 1
    a = __builtin_fmaf(__builtin_bit_cast(float, x & 0xffff0000u), kLess, a);
    b = __builtin_fmaf(__builtin_bit_cast(float, y & 0xffff0000u), kLess, b);
  }
}
__device__ __forceinline__ void split2(float a, float b, uint32_t (&part)[2], f16) {
  const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
  float minus = -1.f;  // (a product takes fp16 operands as they are, a difference does not)
  asm("" : "+v"(minus));
  typedef float f2_t __attribute__((ext_vector_type(2)));
  typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
  typedef uint16_t u2_t __attribute__((ext_vector_type(2)));
  const f2_t rest{__builtin_fmaf(static_cast<float>(h[0]), minus, a),
                  __builtin_fmaf(static_cast<float>(h[1]), minus, b)};
  const u2_t hi = __builtin_bit_cast(u2_t, h);
  const u2_t lo = __builtin_bit_cast(u2_t, __builtin_convertvector(rest, h2_t));
  part[0] = __builtin_bit_cast(uint32_t, hi);
  part[1] = __builtin_bit_cast(
      uint32_t, __builtin_elementwise_max(lo, __builtin_elementwise_min(hi, u2_t{1, 1})));
}

// Writes 4 elements of a finished row, and its lse.
template <typename T, typename P>
__device__ __forceinline__ void write_row(P p, int b, int head, int r, int d, f4_t x, float base,
                                          float l) {
  const int tok = token_of(p, r);
  const int64_t hq = static_cast<int64_t>(head) * p->G + (r - tok * p->G);
  // A row that sees nothing has no weights: 0.
  const float inv = l == 0.f ? 0.f : (p->v_scale ? p->v_scale[head] : 1.f) / l;
  float o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = l == 0.f ? 0.f : x[i] * inv;
  store_vec_f32<T, 4>(
      static_cast<T*>(p->out) + b * p->o_seq + tok * p->o_tok + hq * p->o_head + d, o);
  if (p->lse && d == 0)
    p->lse[(static_cast<int64_t>(b) * p->T + tok) * p->Hkv * p->G + hq] =
        l == 0.f ? -INFINITY : (base + __log2f(l)) * 0.69314718056f;
}

// Whether the sums and a tile's keys and values take at most half of 256 registers
// (a third of that is needed beside them).  Where they do, the kernel is held to
// 256: with 512 the sums go to the accumulator registers and are moved to be
// rescaled (48 sequences of 4 tokens, f16 heads of 64: 31.7 us instead of 30.1).
template <typename T, typename C, int DP, int R>
constexpr bool fits_twice() {
  constexpr int kTile = DP * static_cast<int>(sizeof(C)) * 64 / static_cast<int>(sizeof(T)) / 256;
  return DP * R / 4 + 2 * kTile <= 128;
}
// Blocks of a compute unit: two where much is computed for each byte, else one,
// which has fewer pieces to begin, to finish and to join.  us with one and two:
// 48 sequences of 4 tokens, 8 rows a head and token, up to 6000 positions, e4m3
// heads of 128 87.4, 77.8, of 64 61.4, 63.5; bf16 114.0, 121.8 and 61.1, 65.2; one
// token, 64 sequences, bf16 heads of 128 176.4, 179.3; 128 with e4m3 heads of 256
// 72.7, 71.3; one sequence of 8192, bf16 15.0, 17.7.
template <typename T, typename C, int DP, int R>
constexpr int blocks_of() {
  return sizeof(C) == 1 && DP * R >= 256 && fits_twice<T, C, DP, R>() ? 2 : 1;
}

// ---------------------------------------------------------------------------
// The kernel.  DP: the head's length, rounded up to 64, 128 or 256.  R: row
// tiles of a wave.  RUN: positions (16 at least, a tile at most) that pages are
// whole runs of, with one scalar address each; 0 for none, an address for each
// lane and load.
// ---------------------------------------------------------------------------
template <typename T, typename C, int DP, int R, int RUN>
__global__ void __launch_bounds__(kBlock, (fits_twice<T, C, DP, R>() ? 2 : 1)) attention_kernel(Params p) {
  using OpT = typename Op<T>::type;
  constexpr int CB = sizeof(C);
  constexpr int KV = 16 / sizeof(T);  // values of an operand in a lane
  constexpr int TS = 4 * KV, NH = TS / 16;  // positions of a tile: of a product with V
  constexpr int NK = DP / TS;               // products over a head
  constexpr int CH = DP / KV;   // K: chunks of a row, a lane each
  constexpr int RPI = kWave / CH, NL = TS / RPI;   // rows of a load, loads of a tile
  constexpr int KO = RPI < 16 ? 16 / RPI : 1;      // loads of a half tile
  constexpr int VB = KV < DP / 16 ? KV : DP / 16;  // V: elements of a load
  constexpr int NB = DP / (16 * VB);               // and loads of a row
  constexpr uint32_t kAll = ~0u >> (32 - TS);
  // log2 of what p is scaled by (see above).
  constexpr float kShift = std::is_same<T, f16>::value ? 14.f : 0.f;
  using KRow = Row<T, C, KV>;
  using VRow = Row<T, C, VB>;

  constexpr int DJ = DP < 128 ? DP : 128;  // elements that are joined together
  constexpr int kPitch = DJ + 4;           // rows of the join 4 banks apart
  union Shared {
    KRow k[kWaves][TS * CH];
    float acc[kWaves][16][kPitch];
  };
  __shared__ __align__(16) Shared sh;
  __shared__ __align__(16) OpT sq[R * NK][kWave];  // Q, as the operands take it
  __shared__ float2 ml[kWaves][16];
  // Rows of a tile that see infinity (the lower 16 bits), minus infinity, or NaN (both).
  __shared__ uint32_t poison[kWaves][R][DP];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave, l15 = lane % 16, g = lane / 16;
  // Blocks that read the same positions of neighbouring heads start together, a
  // head to each of the 8 XCDs; heads that share cache lines go to one (8 apart).
  const uint32_t turn = blockIdx.x >> 3, near = turn & ((1 << p.near) - 1);
  uint32_t id = (turn >> p.near << 3) + (blockIdx.x & 7);
  const uint32_t of_heads = p.Hkv >> p.near;
  const int head = (id % of_heads << p.near) + near;
  id /= of_heads;
  const int group = id % p.groups, share = id / p.groups;
  if (share >= p.shares) return;  // whole block

  // The block's share of the line, and the sequence that it begins in.
  Batch bt = batch_at<TS>(p, 0);
  int64_t total = __builtin_amdgcn_readlane(bt.incl, kWave - 1);
  for (int b0 = kWave; b0 < p.B; b0 += kWave)
    total += __builtin_amdgcn_readlane(batch_at<TS>(p, b0).incl, kWave - 1);
  const uint32_t size = share_size(total, p.shares);
  const int64_t g0 = static_cast<int64_t>(share) * size, g1 = min<int64_t>(total, g0 + size);
  if (g0 >= total) return;  // whole block
  int64_t at = 0;  // where sequence b begins
  for (int n; at + (n = __builtin_amdgcn_readlane(bt.incl, kWave - 1)) <= g0; at += n)
    bt = batch_at<TS>(p, bt.b0 + kWave);
  int b = __popcll(__ballot(at + bt.incl <= g0));
  at += __builtin_amdgcn_readlane(bt.incl - bt.own.n, b);
  b += bt.b0;

  const uint64_t kc = reinterpret_cast<uint64_t>(p.kc + head * p.k_head);
  const uint64_t vc = reinterpret_cast<uint64_t>(p.vc + head * p.v_head);
  // Scores are scaled by something positive, that leaves a masked one -inf: a
  // sign, NaN and 0 go to Q, where 0 leaves NaN of what is not finite.  (Without
  // branches: with one for each, 48 sequences of 4 tokens took 30.5 us, not 29.8.)
  float scale2 = p.scale2;
  if (p.k_scale) scale2 *= p.k_scale[head];
  const bool some = scale2 > 0.f || scale2 < 0.f;  // neither 0 nor NaN
  const uint32_t q_keep = __builtin_amdgcn_readfirstlane(some ? ~0u : 0u);
  const uint32_t q_flip = __builtin_amdgcn_readfirstlane(
      scale2 < 0.f ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u)
                   : (scale2 >= 0.f ? 0u : 0x7fff7fffu));
  scale2 = some ? fabsf(scale2) : 1.f;
  const int r0 = group * 16 * R;
  const int first_tok = token_of(&p, r0), last_tok = token_of(&p, min(p.M - 1, r0 + 16 * R - 1));
  // K's chunks lie in the wave's part of LDS with a row's chunks permuted, so
  // that the 16 rows of one operand's read fall on different banks.
  KRow* const kt = sh.k[wave];
  auto k_place = [&](int row, int c) {
    return row * CH + (c ^ (CH == 8 ? row / 2 % 8 : row % 16));
  };
  auto page_of = [&](int pos) {
    return static_cast<int>(static_cast<uint64_t>(pos) * p.page_magic >> p.page_shift);
  };

  // The piece of a sequence that lies in the share: its positions, and its
  // tiles without those that no row of the group sees.
  struct Piece {
    int b, len, n;
    int64_t at;
    int begin, end;
    const int32_t* table;
  };
  auto piece_of = [&](int seq, int64_t where) {
    Piece x;
    x.b = seq;
    x.at = where;
    x.len = __builtin_amdgcn_readlane(bt.own.len, seq - bt.b0);
    x.n = __builtin_amdgcn_readlane(bt.own.n, seq - bt.b0);
    const int t0 = __builtin_amdgcn_readlane(bt.own.t0, seq - bt.b0);
    const int first_pos = x.len - p.T + first_tok, last_pos = x.len - p.T + last_tok;
    x.begin = t0 + static_cast<int>(max<int64_t>(g0 - where, 0));
    x.end = t0 + static_cast<int>(min<int64_t>(g1 - where, x.n));
    if (p.window) x.begin = max(x.begin, max(0, first_pos - p.window + 1) / TS);
    x.end = min(x.end, last_pos < 0 ? 0 : last_pos / TS + 1);
    x.table = p.table + seq * p.table_row;
    return x;
  };
  // The wave's share of Q's operands of a sequence, requested and stored.
  constexpr int NQ = (R * NK + kWaves - 1) / kWaves;
  u32x4 qx[NQ];
  auto load_q = [&](int seq) {
    const LateParams late = late_params();
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
      const int u = c * kWaves + wave, j = u / NK, s = u % NK;
      const int r = r0 + 16 * j + l15, t = token_of(late, r), d = (4 * s + g) * KV;
      qx[c] = u32x4{};
      if (u < R * NK && r < late->M && d < late->D)
        qx[c] = *reinterpret_cast<const u32x4*>(
            static_cast<const T*>(late->q) + seq * late->q_seq + t * late->q_tok +
            (static_cast<int64_t>(head) * late->G + (r - t * late->G)) * late->q_head + d);
    }
  };
  auto store_q = [&]() {
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
      const int u = c * kWaves + wave;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qx[c][i] = ((qx[c][i] & q_keep) ^ q_flip) | (only_nan<T>(qx[c][i]) & ~q_keep);
      if (u < R * NK) sq[u][lane] = __builtin_bit_cast(OpT, qx[c]);
    }
  };

  // The table's entries of a tile (one, one for each half, or the lane's
  // position's).  Positions past the sequence's end stand for its last ones.
  constexpr int NE = RUN ? TS / RUN : 1;
  auto pos_of = [&](int len, int tile, int h) {
    return RUN ? min(tile * TS + RUN * h, (len - 1) & -RUN) : min(tile * TS + lane % TS, len - 1);
  };
  int entry[NE];
  auto look_up = [&](const int32_t* table, int len, int tile) {
#pragma unroll
    for (int h = 0; h < NE; ++h) entry[h] = table[page_of(pos_of(len, tile, h))];
  };
  // What the first tile waits for is requested before all else is computed.
  Piece cur = piece_of(b, at);
  if (cur.begin + wave < cur.end) look_up(cur.table, cur.len, cur.begin + wave);
  load_q(b);
  bool first = true;
  bool loaded = false;  // the registers hold the piece's first tile of the wave
  // What holds for every sequence: lane offsets from the start of a half tile;
  // beyond the head the row's last vector again.
  const int chunk = lane % CH, krow = lane / CH;
  const bool k_in = chunk * KV < p.D;
  uint32_t k_off[KO], v_off[4][NB];
#pragma unroll
  for (int i = 0; i < KO; ++i)
    k_off[i] = (i * RPI + krow) * p.k_slot + min(chunk * KV, p.D - KV) * CB;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < NB; ++n)
      v_off[i][n] = (4 * g + i) * p.v_slot + min((n * 16 + l15) * VB, p.D - VB) * CB;
  int tok[R];  // of the lane's rows; beyond them, one that sees nothing
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int r = r0 + 16 * j + l15;
    tok[j] = r < p.M ? token_of(&p, r) : -(1 << 30);
  }
  KRow k[NL];
  VRow v[KV][NB];
  uint32_t ok = 0;  // which positions of the tile there are
  // Where a tile's rows are, and which of them are in a page that there is
  // (a bit each); the others are read from the first page.
  GlobalBytes kh[NH], vh[NH];
  uint64_t ko = 0, vo = 0;
  auto place = [&](int len, int tile) -> uint32_t {
    uint32_t ok = 0;
#pragma unroll
    for (int h = 0; h < NE; ++h) {
      const uint32_t e = RUN ? __builtin_amdgcn_readfirstlane(entry[h]) : entry[h];
      const bool in = e < static_cast<uint32_t>(p.num_pages);
      const uint64_t page = in ? e : 0;
      const int pos = pos_of(len, tile, h);
      const uint32_t row = pos - page_of(pos) * p.page_size;
      ko = kc + (page * p.k_page << 3) + row * p.k_slot;
      vo = vc + (page * p.v_page << 3) + row * p.v_slot;
      if constexpr (RUN == 0) {
        ok = static_cast<uint32_t>(__ballot(in)) & kAll;
      } else {
        constexpr int kPer = RUN / 16;  // half tiles of a run
        kh[h * kPer] = scalar(ko);
        vh[h * kPer] = scalar(vo);
#pragma unroll
        for (int u = 1; u < kPer; ++u) {
          kh[h * kPer + u] = kh[h * kPer] + u * (16 * p.k_slot);
          vh[h * kPer + u] = vh[h * kPer] + u * (16 * p.v_slot);
        }
        ok |= in ? (~0u >> (32 - RUN)) << (RUN * h) : 0;
      }
    }
    return ok;
  };
  // Of a tile that there is not, all lanes of a load take one vector, in a row
  // that there is (where each position has an address, the row's first one).
  uint32_t wanted = ~0u;  // or 0, for the lanes' offsets
  auto load_k = [&]() {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      if constexpr (RUN > 0)
        k[i].load(kh[i * RPI / 16] + lane_offset(k_off[i % KO] & wanted));
      else
        k[i].load(reinterpret_cast<GlobalBytes>(__shfl(ko, i * RPI + krow)) +
                  ((k_off[0] - krow * p.k_slot) & wanted));
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int i = 0; i < KV; ++i) {
      uint64_t at_row = 0;
      if constexpr (RUN == 0) at_row = __shfl(vo, 16 * (i / 4) + 4 * g + i % 4);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if constexpr (RUN > 0)
          v[i][n].load(vh[i / 4] + lane_offset(v_off[i % 4][n] & wanted));
        else
          v[i][n].load(reinterpret_cast<GlobalBytes>(at_row) +
                       ((v_off[0][n] - 4 * g * p.v_slot) & wanted));
      }
    }
  };
  // Chunks beyond the head stay zero in LDS.
  auto clear_k = [&]() {
    if (!k_in) {
#pragma unroll
      for (int i = 0; i < NL; ++i) kt[k_place(i * RPI + krow, chunk)] = KRow{};
    }
  };

  for (;;) {
    const int len = cur.len, end = cur.end;
    // The piece after this one: its first tile of the wave is requested in the
    // last step of this one, its queries now.
    const bool more = cur.at + cur.n < g1;
    Piece next = cur;
    if (more) {
      if (cur.b + 1 == bt.b0 + kWave) bt = batch_at<TS>(p, cur.b + 1);
      next = piece_of(cur.b + 1, cur.at + cur.n);
    }
    // The first piece of a share and the last have places of their own where
    // they are not all of a sequence.
    const bool all = cur.at >= g0 && cur.at + cur.n <= g1;
    const int slot = 2 * share + (cur.at > g0);
    if (cur.at >= g0 && head == 0 && group == 0 && threadIdx.x == 0) {
      const int last = static_cast<int>(divide(cur.at + cur.n - 1, size));
      int2* meta = late_params()->meta;  // NULL where one share holds all
      if (meta) meta[cur.b] = make_int2(slot, last - share + 1);
    }
    // Rows: token r / G of the sequence's new ones, at position len - T + token.
    const int pos_0 = len - p.T;
    const int first_pos = pos_0 + first_tok, last_pos = pos_0 + last_tok;
    const int low_first = p.window ? max(0, first_pos - p.window + 1) : 0;
    const int low_last = p.window ? max(0, last_pos - p.window + 1) : 0;

    f4_t acc[R][NB][VB] = {};
    float base[R], sum[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      base[j] = -INFINITY;
      sum[j] = 0.f;
    }
    int tile = cur.begin + wave;
    const int ahead = next.begin + wave;
    const bool go_on = more && ahead < next.end;
    // A piece with one tile of the wave was entered without the table's entries
    // of what comes after it.
    const bool cross = go_on && tile < end && (!loaded || tile + kWaves < end);
    if (tile < end && !loaded && !first) look_up(cur.table, len, tile);
    first = false;
    store_q();
    clear_k();
    if (tile < end && !loaded) {
      ok = place(len, tile);
      wanted = ~0u;
      load_k();
      // (the loop's order, by which it counts the loads to wait for)
      const bool same = tile + kWaves < end || !cross;
      look_up(same ? cur.table : next.table, same ? len : next.len,
              same ? tile + kWaves : ahead);
      load_v();
    }
    if (more) load_q(next.b);
    __syncthreads();  // Q
    loaded = cross;
    while (tile < end) {
      const int pos0 = tile * TS;
      const bool whole = pos0 >= low_last && pos0 + TS - 1 <= first_pos && ok == kAll;
      if (k_in) {
#pragma unroll
        for (int i = 0; i < NL; ++i) kt[k_place(i * RPI + krow, chunk)] = k[i];
      }
      wave_sync();
      // The wave's next two tiles, in this piece or the next one.
      const bool in_1 = tile + kWaves < end || !cross, in_2 = tile + 2 * kWaves < end || !cross;
      const int tile_1 = in_1 ? tile + kWaves : ahead;
      wanted = tile_1 < (in_1 ? end : next.end) ? ~0u : 0u;
      const uint32_t ok_next = place(in_1 ? len : next.len, tile_1);
      load_k();
      look_up(in_2 ? cur.table : next.table, in_2 ? len : next.len,
              in_2 ? tile + 2 * kWaves : (in_1 ? ahead : ahead + kWaves));
      f4_t sc[R][NH] = {};
#pragma unroll
      for (int s = 0; s < NK; ++s) {
        OpT q[R];
#pragma unroll
        for (int j = 0; j < R; ++j) q[j] = sq[j * NK + s][lane];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const KRow row = kt[k_place(16 * h + l15, 4 * s + g)];
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = row.word(i);
#pragma unroll
          for (int j = 0; j < R; ++j) sc[j][h] = mma(__builtin_bit_cast(OpT, w), q[j], sc[j][h]);
        }
        if (s % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      wave_sync();  // V's rows or the next tile's keys may take their place
      // Positions that a row does not see; values that no row sees are no part
      // of the sums, whatever they are.
      if (!whole) {
        const uint32_t there = ok >> 4 * g;
        // (how far a position lies back, and past the first one seen, as
        // unsigned numbers: one comparison each)
        const uint32_t span = p.window ? p.window : INT32_MAX;
        const uint32_t most = last_pos - low_first;
        const int past = pos0 + 4 * g - low_first;
        bool fine = true;
#pragma unroll
        for (int i = 0; i < KV; ++i) {
          const int t = 16 * (i / 4) + i % 4;
          const bool in = there >> t & 1;
#pragma unroll
          for (int j = 0; j < R; ++j) {
            const uint32_t back = pos_0 + tok[j] - (pos0 + 4 * g) - t;
            const bool seen = in && back < span;
            sc[j][i / 4][i % 4] = seen ? sc[j][i / 4][i % 4] : -INFINITY;
          }
          const bool any = in && static_cast<uint32_t>(past + t) <= most;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            v[i][n].keep(any);
            if (first_tok < last_tok) fine = fine && v[i][n].finite();
          }
        }
        // A value that is not finite where some new tokens see it and others do
        // not: 0 * inf would be NaN for all of them, so it is taken out, and
        // added to the sums of the rows that see it.  Rare, and so in LDS, in
        // loops: unrolled in registers it took 70 more of them.
        if (!__all(fine)) {
          C* const vt = reinterpret_cast<C*>(kt);  // [TS][DP]
          auto v_at = [&](int i, int n) {
            return reinterpret_cast<VRow*>(vt + (16 * (i / 4) + 4 * g + i % 4) * DP +
                                           (n * 16 + l15) * VB);
          };
#pragma unroll
          for (int i = 0; i < KV; ++i)
#pragma unroll
            for (int n = 0; n < NB; ++n) *v_at(i, n) = v[i][n];
          wave_sync();
#pragma unroll 1
          for (int d = lane; d < DP; d += kWave) {
            uint32_t rows[R] = {};  // those that see such a value
#pragma unroll 1
            for (int t = 0; t < TS; ++t) {
              const uint32_t bad = not_finite(vt[t * DP + d]);
              if (bad) vt[t * DP + d] = C{};
#pragma unroll
              for (int j = 0; j < R; ++j) {
                const int back = pos_0 + tok[j] - (pos0 + t);
                const uint64_t see = __ballot(back >= 0 && (!p.window || back < p.window));
                const uint32_t of = static_cast<uint32_t>(see) & 0xffffu;
                rows[j] |= (bad & 1 ? of : 0u) | (bad & 2 ? of << 16 : 0u);
              }
            }
#pragma unroll
            for (int j = 0; j < R; ++j) poison[wave][j][d] = rows[j];
          }
          wave_sync();
#pragma unroll
          for (int i = 0; i < KV; ++i)
#pragma unroll
            for (int n = 0; n < NB; ++n) v[i][n] = *v_at(i, n);
          wave_sync();
          clear_k();
#pragma unroll
          for (int j = 0; j < R; ++j)
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < VB; ++e) {
                  const uint32_t bits = poison[wave][j][(n * 16 + 4 * g + i) * VB + e] >> l15;
                  acc[j][n][e][i] += bits & 1 ? INFINITY : 0.f;
                  acc[j][n][e][i] -= bits >> 16 & 1 ? INFINITY : 0.f;
                }
        }
      }

      constexpr int kParts = Parts<T>::kCount;
      u32x4 pw[R][kParts];
#pragma unroll
      for (int j = 0; j < R; ++j) {
        float x[KV], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < KV; ++i) {
          x[i] = sc[j][i / 4][i % 4];
          top = fmaxf(top, x[i]);
        }
        top = over_groups(top, [](float a, float c) { return fmaxf(a, c); });
        const float now = fmaxf(base[j], top * scale2 - kShift);
        const float from = now == -INFINITY ? 0.f : now;
        const float before = base[j], keep = exp2_hw(before - from);
        base[j] = now;
        float add = 0.f;
#pragma unroll
        for (int i = 0; i < KV; ++i) {
          x[i] = exp2_hw(__builtin_fmaf(x[i], scale2, -from));
          add += x[i];
        }
        sum[j] = sum[j] * keep + add;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t part[kParts];
          if constexpr (sizeof(T) == 4) part[0] = __builtin_bit_cast(uint32_t, x[u]);
          else split2(x[2 * u], x[2 * u + 1], part, T());
#pragma unroll
          for (int i = 0; i < kParts; ++i) pw[j][i][u] = part[i];
        }
        // (nothing to rescale in most tiles; the empty asm keeps the products
        // in the branch: before it, old and scaled sums would both be held)
        if (__any(keep != 1.f)) {
          // (0 before the first score, when a sum may be infinite already)
          float by = before == -INFINITY ? 1.f : keep;
          asm volatile("" : "+v"(by));
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < VB; ++e) acc[j][n][e] *= by;
        }
      }
      // acc += V^T P^T
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < VB; ++e) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4)
              w[i] = v[i][n].word(e);
            else
              w[i] = __builtin_amdgcn_perm(v[2 * i + 1][n].word(e / 2), v[2 * i][n].word(e / 2),
                                           e & 1 ? 0x07060302u : 0x05040100u);
          }
          const OpT a = __builtin_bit_cast(OpT, w);
#pragma unroll
          for (int j = 0; j < R; ++j)
#pragma unroll
            for (int i = 0; i < kParts; ++i)
              acc[j][n][e] = mma(a, __builtin_bit_cast(OpT, pw[j][i]), acc[j][n][e]);
          // (else all operands are turned before the first product, in
          // twice the registers)
          if (e % 2) __builtin_amdgcn_sched_barrier(0);
        }
      load_v();
      ok = ok_next;
      tile += kWaves;
    }

    // The waves join: a row's base is the largest, sums are scaled to it.  Wide
    // heads join in two halves.
    for (int j = 0; j < R; ++j) {
      const int rows = min(16, p.M - r0 - 16 * j);
      if (rows <= 0) break;
      // (a select, so that the arrays stay in registers)
      float my_base = base[0], my_sum = sum[0];
#pragma unroll
      for (int i = 1; i < R; ++i) {
        my_base = j == i ? base[i] : my_base;
        my_sum = j == i ? sum[i] : my_sum;
      }
      my_sum = over_groups(my_sum, [](float a, float c) { return a + c; });
#pragma unroll
      for (int half = 0; half < DP / DJ; ++half) {
        __syncthreads();
        if (half == 0 && g == 0) ml[wave][l15] = make_float2(my_base, my_sum);
        if (l15 < rows) {
#pragma unroll
          for (int n = half * (NB * DJ / DP); n < (half + 1) * (NB * DJ / DP); ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int e = 0; e < VB; e += 4) {
                f4_t x;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                  float y = acc[0][n][e + u][i];
#pragma unroll
                  for (int m = 1; m < R; ++m) y = j == m ? acc[m][n][e + u][i] : y;
                  x[u] = y;
                }
                *reinterpret_cast<f4_t*>(
                    &sh.acc[wave][l15][(n * 16 + 4 * g + i) * VB + e - half * DJ]) = x;
              }
        }
        __syncthreads();
        const LateParams late = late_params();
        for (int u = threadIdx.x; u < rows * (DJ / 4); u += kBlock) {
          const int row = u / (DJ / 4), d = u % (DJ / 4) * 4, r = r0 + 16 * j + row;
          if (half * DJ + d >= late->D) continue;
          float m = ml[0][row].x;
#pragma unroll
          for (int w = 1; w < kWaves; ++w) m = fmaxf(m, ml[w][row].x);
          float l = 0.f;
          f4_t x = {};
#pragma unroll
          for (int w = 0; w < kWaves; ++w) {
            const float by = weight(ml[w][row].x, m);
            l += ml[w][row].y * by;
            x += *reinterpret_cast<const f4_t*>(&sh.acc[w][row][d]) * by;
          }
          if (all) {
            write_row<T>(late, cur.b, head, r, half * DJ + d, x, m, l);
          } else {
            const int64_t to = (static_cast<int64_t>(slot) * late->Hkv + head) * late->M + r;
            *reinterpret_cast<f4_t*>(late->acc + to * late->D + half * DJ + d) = x;
            if (half * DJ + d == 0) late->ml[to] = make_float2(m, l);
          }
        }
      }
    }
    if (!more) break;
    cur = next;
    __syncthreads();  // the join's reads are over
  }
}

// Joins the pieces of sequences that lie in several shares: a block for a
// (sequence, head) and some of its rows.  `team` lanes read a piece's row, 4
// elements each; as many teams as there are pieces (a power of two of them)
// share a row, so that few pieces leave the block to several rows.
template <typename T>
__global__ void __launch_bounds__(kBlock) join_kernel(Params p, int team) {
  __shared__ float2 ml[16];
  __shared__ __align__(16) f4_t sums[kBlock];
  const int b = blockIdx.x / p.Hkv, head = blockIdx.x % p.Hkv;
  const int2 meta = p.meta[b];
  const int pieces = meta.y;
  if (pieces <= 1) return;
  const int teams = kBlock / team, own = threadIdx.x / team, d = threadIdx.x % team * 4;
  int split = 1;  // teams of a row
  while (split < pieces && split < teams) split *= 2;
  const int part = own % split, step = gridDim.y * (teams / split);
  // The first piece, then the first ones of the shares that follow.
  const int64_t apart = 2 * static_cast<int64_t>(p.Hkv) * p.M;
  const int64_t first = (static_cast<int64_t>(meta.x) * p.Hkv + head) * p.M;
  const int64_t even = (static_cast<int64_t>(meta.x & ~1) * p.Hkv + head) * p.M;
  for (int r0 = blockIdx.y * (teams / split); r0 < p.M; r0 += step) {
    const int r = r0 + own / split;
    float base = -INFINITY, sum = 0.f;
    f4_t acc = {};
    // `ahead` pieces that a lane requests together: one where it has no more
    // (with eight for all, the statistics of those that are not there took most
    // of the time).
    auto take = [&](auto ahead) {
      constexpr int kAhead = ahead;
      for (int i0 = part; i0 < pieces && r < p.M; i0 += kAhead * split) {
        float2 x[kAhead];
        f4_t y[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const int i = i0 + a * split;
          x[a] = make_float2(-INFINITY, 0.f);
          y[a] = f4_t{};
          if (i < pieces) {
            const int64_t at = (i ? even + i * apart : first) + r;
            x[a] = p.ml[at];
            if (d < p.D) y[a] = *reinterpret_cast<const f4_t*>(p.acc + at * p.D + d);
          }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          if constexpr (kAhead == 1) {  // (the lane's only one)
            base = x[a].x;
            sum = x[a].y;
            acc = y[a];
          } else {
            const float now = fmaxf(base, x[a].x), c = weight(base, now), e = weight(x[a].x, now);
            sum = sum * c + x[a].y * e;
            acc = acc * c + y[a] * e;
            base = now;
          }
        }
      }
    };
    if (split >= pieces) take(std::integral_constant<int, 1>());
    else take(std::integral_constant<int, 8>());
    if (threadIdx.x % team == 0) ml[own] = make_float2(base, sum);
    sums[threadIdx.x] = acc;
    __syncthreads();
    if (part == 0 && r < p.M && d < p.D) {
      float top = base, l = 0.f;
      for (int i = 1; i < split; ++i) top = fmaxf(top, ml[own + i].x);
      f4_t x = {};
      for (int i = 0; i < split; ++i) {
        const float2 one = ml[own + i];
        const float by = weight(one.x, top);
        l += one.y * by;
        x += sums[threadIdx.x + i * team] * by;
      }
      write_row<T>(&p, b, head, r, d, x, top, l);
    }
    __syncthreads();
  }
}

template <typename T, typename C, int DP, int R>
void launch_pages(Params& p, hipStream_t s) {
  const int64_t lines = static_cast<int64_t>(p.Hkv) * p.groups;
  p.shares = static_cast<int>(std::min<int64_t>(
      p.shares, std::max<int64_t>(1, int64_t{num_cus()} * blocks_of<T, C, DP, R>() / lines)));
  // Heads that share cache lines (rows below 128 bytes, of 64 sequences of 4096
  // with 8 e4m3 heads of 64: 71.6 us together, 94.4 apart, where each XCD reads all
  // lines; for heads that share 512 bytes it is the other way: 185 and 176 with 8
  // bf16 heads of 128).
  p.near = 0;
  while (p.near < 4 && p.k_head * (2 << p.near) <= 128 && p.Hkv % (2 << p.near) == 0) ++p.near;
  const dim3 grid(static_cast<uint32_t>(cdiv(p.shares * lines >> p.near, 8) << (3 + p.near)));
  constexpr int kTile = 64 / static_cast<int>(sizeof(T));
  auto launch = [&](auto run) {
    if constexpr (run <= kTile)
      hipLaunchKernelGGL((attention_kernel<T, C, DP, R, run>), grid, dim3(kBlock), 0, s, p);
  };
  if (kTile >= 32 && p.page_size % 32 == 0) launch(std::integral_constant<int, 32>());
  else if (p.page_size % 16 == 0) launch(std::integral_constant<int, 16>());
  else launch(std::integral_constant<int, 0>());
}

template <typename T, typename C, int DP>
void launch_rows(Params& p, int tiles, hipStream_t s) {
  if constexpr (sizeof(T) == 4 && DP == 256) {  // (two tiles do not fit the registers)
    launch_pages<T, C, DP, 1>(p, s);
  } else {
    if (tiles == 1) launch_pages<T, C, DP, 1>(p, s);
    else launch_pages<T, C, DP, 2>(p, s);
  }
}

// `tiles`: row tiles of a wave, as the entry point counted p.groups by.
template <typename T, typename C>
int run(Params& p, int tiles, hipStream_t s) {
  if (p.D <= 64) launch_rows<T, C, 64>(p, tiles, s);
  else if (p.D <= 128) launch_rows<T, C, 128>(p, tiles, s);
  else launch_rows<T, C, 256>(p, tiles, s);
  int st = launch_status();
  if (st != XK_OK || p.shares == 1) return st;
  const int team = p.D <= 64 ? 16 : (p.D <= 128 ? 32 : 64);
  const int64_t heads = static_cast<int64_t>(p.B) * p.Hkv;
  const dim3 grid(static_cast<uint32_t>(heads),
                  static_cast<uint32_t>(std::min<int64_t>(p.M, cdiv(2048, heads))));
  hipLaunchKernelGGL((join_kernel<T>), grid, dim3(kBlock), 0, s, p, team);
  return launch_status();
}

int run_f32(Params& p, int tiles, hipStream_t s);
int run_bf16(Params& p, int tiles, hipStream_t s);
int run_f16(Params& p, int tiles, hipStream_t s);
int run_bf16_f8(Params& p, int tiles, hipStream_t s);
int run_f16_f8(Params& p, int tiles, hipStream_t s);

}  // namespace paged
}  // namespace xk
