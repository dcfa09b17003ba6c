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
// Work: the tiles of every sequence (32 positions of 16-bit rows, 16 of fp32)
// are cut into parts of equal length on the device, from the lengths that are
// there (seq_lens never reaches the host); a block of 4 waves takes one part
// of one head.  Its waves take tiles in turn, each with statistics and sums of
// its own, and join at the end; parts of one sequence are joined by a second
// launch.
//
// Tile: no LDS and no barrier in the loop.  S^T = K Q^T and O^T = V^T P^T, so
// that lane l holds query row l % 16 throughout (C layout: column l % 16,
// rows 4 (l / 16) + i): statistics and rescaling stay in the lane, up to the
// maximum over the four lane groups.  The order of a product's inner index is
// free as long as both sides use the same:
//   - the scores of tokens 4g + i and 16 + 4g + i that lane group g holds are
//     the slots of group g in P^T, with V's tokens loaded to match;
//   - V's rows are loaded as they lie (16 lanes read one row of 128 elements)
//     and the lane's 8 tokens x 8 elements turned in registers (v_perm), one
//     product for each of the 8 elements: product e has row l % 16 <->
//     element 8 (l % 16) + e, so the sums come out as 8 neighbours.
// p is split in two 16-bit parts (hi + lo, 16 bits of mantissa and more) for
// the product with V; fp16's is scaled by 2^14 so that small weights keep
// their digits.  Scores, statistics and sums are fp32.
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
constexpr int kMinChunk = kWaves;  // tiles of a part, at the least

struct Params {
  const void* q;
  int64_t q_seq, q_tok, q_head;  // elements
  const char* kc;
  int64_t k_page, k_slot, k_head;  // bytes
  const char* vc;
  int64_t v_page, v_slot, v_head;
  int num_pages, page_size, page_shift;  // shift: -1 where no power of two
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
  int want;                        // parts wanted in all, beyond one a sequence
  int slots;                       // parts that the workspace holds
  bool alone;                      // no sequence can have two parts
  int2* meta;                      // [B]: first part, parts
  float2* ml;                      // [slots][Hkv][M]: base, sum
  float* acc;                      // [slots][Hkv][M][D]
};

// A sequence's tiles: from the first that a row sees to the last.
struct Span {
  int len, t0, n;
};
template <int TS>
__device__ __forceinline__ Span span_of(const Params& p, int b) {
  const int len = max(0, min(p.lens[b], p.most_len));
  const int lo = p.window ? max(0, len - p.T - p.window + 1) : 0;
  const int t0 = lo / TS, t1 = (len + TS - 1) / TS;
  return {len, t0, max(0, t1 - t0)};
}

struct Part {
  int b;        // -1: none
  int index, of;  // the part's number in its sequence, and how many there are
  Span span;
};

// Part `slot` of the batch, found by every wave from the lengths: the chunk is
// what gives about p.want parts, never below kMinChunk tiles, in whole rounds
// of the block's waves.  At most p.want + B parts, since a sequence has at
// least one (an empty one, whose rows are written as zeros).
template <int TS>
__device__ __forceinline__ Part locate(const Params& p, int slot) {
  const int lane = threadIdx.x % kWave;
  int64_t total = 0;
  Span own{0, 0, 0};
  for (int b0 = 0; b0 < p.B; b0 += kWave) {
    own = b0 + lane < p.B ? span_of<TS>(p, b0 + lane) : Span{0, 0, 0};
    total += __builtin_amdgcn_readlane(gdn::wave_incl_scan(own.n), kWave - 1);
  }
  int64_t c = (total + p.want - 1) / p.want;
  c = (c + kWaves - 1) / kWaves * kWaves;
  const int chunk = static_cast<int>(max<int64_t>(kMinChunk, min<int64_t>(c, 1 << 30)));
  int first = 0;
  for (int b0 = 0; b0 < p.B; b0 += kWave) {
    if (p.B > kWave) own = b0 + lane < p.B ? span_of<TS>(p, b0 + lane) : Span{0, 0, 0};
    const int parts = b0 + lane < p.B ? max(1, (own.n + chunk - 1) / chunk) : 0;
    const int incl = gdn::wave_incl_scan(parts);
    const int all = __builtin_amdgcn_readlane(incl, kWave - 1);
    if (slot < first + all) {
      const int k = __popcll(__ballot(first + incl <= slot));
      const int of = __builtin_amdgcn_readlane(parts, k);
      const int begin = first + __builtin_amdgcn_readlane(incl, k) - of;
      return {b0 + k, slot - begin, of,
              {__builtin_amdgcn_readlane(own.len, k), __builtin_amdgcn_readlane(own.t0, k),
               __builtin_amdgcn_readlane(own.n, k)}};
    }
    first += all;
  }
  return {-1, 0, 0, {0, 0, 0}};
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

// N elements of the cache as loaded, and as words of T.
template <typename T, typename C, int N>
struct Row {
  static constexpr int kBytes = N * static_cast<int>(sizeof(C));
  static constexpr int kRaw = kBytes / 4, kWords = N * static_cast<int>(sizeof(T)) / 4;
  uint32_t raw[kRaw];
  __device__ __forceinline__ void load(const char* at) {
    using U = typename RawOf<kBytes>::type;
    const U x = __builtin_nontemporal_load(reinterpret_cast<const U*>(at));
    if constexpr (kRaw == 1) {
      raw[0] = x;
    } else {
#pragma unroll
      for (int i = 0; i < kRaw; ++i) raw[i] = x[i];
    }
  }
  __device__ __forceinline__ void keep(bool yes) {
#pragma unroll
    for (int i = 0; i < kRaw; ++i) raw[i] = yes ? raw[i] : 0;
  }
  __device__ __forceinline__ uint32_t word(int i) const {
    if constexpr (std::is_same<C, f8>::value) return widen<T>(raw[i / 2], i & 1);
    else return raw[i];
  }
  __device__ __forceinline__ bool finite() const {
    bool ok = true;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const uint32_t w = word(i);
      if constexpr (sizeof(T) == 4) {
        ok = ok && (w & 0x7f800000u) != 0x7f800000u;
      } else {
        constexpr uint32_t kExp = std::is_same<T, bf16>::value ? 0x7f80u : 0x7c00u;
        ok = ok && (w & kExp) != kExp && (w >> 16 & kExp) != kExp;
      }
    }
    return ok;
  }
};

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

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// exp2(a - b) for a <= b, 0 where a is -inf (b then may be -inf too).
__device__ __forceinline__ float weight(float a, float b) {
  return exp2_hw(a - (b == -INFINITY ? 0.f : b));
}

// ---------------------------------------------------------------------------
// The kernel.  DP: the head's length, rounded up to 64, 128 or 256.  R: row
// tiles of a wave.  P16: pages are whole runs of 16 positions, so that a half
// tile lies in one page and its address is one scalar.
// ---------------------------------------------------------------------------
template <typename T, typename C, int DP, int R, bool P16>
__global__ void __launch_bounds__(kBlock, 2) attention_kernel(Params p) {
  using OpT = typename Op<T>::type;
  constexpr int KV = 16 / sizeof(T);       // values of an operand in a lane
  constexpr int TS = 4 * KV, NH = TS / 16;  // positions of a tile, halves
  constexpr int NK = DP / (4 * KV);        // products over a head
  constexpr int VB = KV < DP / 16 ? KV : DP / 16;  // V: elements of a load
  constexpr int NB = DP / (16 * VB);               // and loads of a row
  constexpr int CB = sizeof(C);
  // log2 of what p is scaled by (see above).
  constexpr float kShift = std::is_same<T, f16>::value ? 14.f : 0.f;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave, l15 = lane % 16, g = lane / 16;
  uint32_t id = blockIdx.x;
  const int head = id % p.Hkv;
  id /= p.Hkv;
  const int group = id % p.groups, slot = id / p.groups;
  const Part part = locate<TS>(p, slot);
  if (part.b < 0) return;  // whole block
  if (!p.alone && part.index == 0 && head == 0 && group == 0 && threadIdx.x == 0)
    p.meta[part.b] = make_int2(slot, part.of);

  // Rows: token r / G of the sequence's new ones, at position len - T + token.
  const int r0 = group * 16 * R, len = part.span.len;
  const int first_tok = r0 / p.G, last_tok = min(p.M - 1, r0 + 16 * R - 1) / p.G;
  const int first_pos = len - p.T + first_tok, last_pos = len - p.T + last_tok;
  const int low_first = p.window ? max(0, first_pos - p.window + 1) : 0;
  const int low_last = p.window ? max(0, last_pos - p.window + 1) : 0;
  int hi[R], lo[R];
  OpT q[R][NK];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int r = r0 + 16 * j + l15, tok = r / p.G;
    hi[j] = r < p.M ? len - p.T + tok : -1;
    lo[j] = p.window ? hi[j] - p.window + 1 : 0;
    const T* src = static_cast<const T*>(p.q) + part.b * p.q_seq + tok * p.q_tok +
                   (static_cast<int64_t>(head) * p.G + (r - tok * p.G)) * p.q_head;
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      const int d = (4 * s + g) * KV;
      OpT x = {};
      if (r < p.M && d < p.D) x = *reinterpret_cast<const OpT*>(src + d);
      q[j][s] = x;
    }
  }

  // The part's tiles, without those that no row of the group sees.
  const int each = (part.span.n + part.of - 1) / part.of;
  int begin = part.span.t0 + part.index * each;
  int end = min(part.span.t0 + part.span.n, begin + each);
  begin = max(begin, low_first / TS);
  end = min(end, last_pos < 0 ? 0 : last_pos / TS + 1);

  float scale2 = p.scale2;
  if (p.k_scale) scale2 *= p.k_scale[head];
  const char* const kc = p.kc + head * p.k_head;
  const char* const vc = p.vc + head * p.v_head;
  const int32_t* const table = p.table + part.b * p.table_row;
  const bool ragged = p.D < DP;
  // Lane offsets inside a row; beyond the head the row's last vector again.
  uint32_t kd[NK], vd[NB];
#pragma unroll
  for (int s = 0; s < NK; ++s) kd[s] = min((4 * s + g) * KV, p.D - KV) * CB;
#pragma unroll
  for (int n = 0; n < NB; ++n) vd[n] = min((n * 16 + l15) * VB, p.D - VB) * CB;
  const uint32_t k_lane = l15 * static_cast<uint32_t>(p.k_slot);
  const uint32_t v_lane = 4 * g * static_cast<uint32_t>(p.v_slot);

  Row<T, C, KV> k[NH][NK];
  Row<T, C, VB> v[KV][NB];
  f4_t acc[R][NB][VB] = {};
  float base[R], sum[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    base[j] = -INFINITY;
    sum[j] = 0.f;
  }

  auto page_of = [&](int pos) { return p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size; };
  // The table's entries of a tile (P16: one for each half; else the lane's
  // position's), -1 where there is no position.
  int entry[P16 ? NH : 1];
  auto look_up = [&](int tile) {
    if constexpr (P16) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const int pos = tile * TS + 16 * h;
        entry[h] = tile < end && pos < len ? table[page_of(pos)] : -1;
      }
    } else {
      const int pos = tile * TS + lane % TS;
      entry[0] = tile < end && pos < len ? table[page_of(pos)] : -1;
    }
  };
  // Where a tile's rows are, and which of its positions there are (a bit
  // each).  Rows that are not there are read from the first page.
  const char *kh[NH], *vh[NH];
  int64_t ko = 0, vo = 0;
  auto place = [&](int tile) -> uint32_t {
    if constexpr (P16) {
      uint32_t ok = 0;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const int pos = tile * TS + 16 * h;
        const int e = __builtin_amdgcn_readfirstlane(entry[h]);
        const bool in = static_cast<uint32_t>(e) < static_cast<uint32_t>(p.num_pages);
        const int at = in ? pos - page_of(pos) * p.page_size : 0;
        const int64_t page = in ? e : 0;
        kh[h] = kc + page * p.k_page + at * p.k_slot;
        vh[h] = vc + page * p.v_page + at * p.v_slot;
        if (in) ok |= 0xffffu << (16 * h);
      }
      return ok;
    } else {
      const int pos = tile * TS + lane % TS;
      const bool in = static_cast<uint32_t>(entry[0]) < static_cast<uint32_t>(p.num_pages);
      const int at = in ? pos - page_of(pos) * p.page_size : 0;
      const int64_t page = in ? entry[0] : 0;
      ko = page * p.k_page + at * p.k_slot;
      vo = page * p.v_page + at * p.v_slot;
      return static_cast<uint32_t>(__ballot(in)) & static_cast<uint32_t>((uint64_t{1} << TS) - 1);
    }
  };
  auto load_k = [&]() {
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      int64_t off = 0;
      if constexpr (!P16) off = __shfl(ko, 16 * h + l15);
#pragma unroll
      for (int s = 0; s < NK; ++s) {
        if constexpr (P16) k[h][s].load(kh[h] + (k_lane + kd[s]));
        else k[h][s].load(kc + off + kd[s]);
      }
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int i = 0; i < KV; ++i) {
      int64_t off = 0;
      if constexpr (!P16) off = __shfl(vo, 16 * (i / 4) + 4 * g + i % 4);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if constexpr (P16) v[i][n].load(vh[i / 4] + (i % 4) * p.v_slot + (v_lane + vd[n]));
        else v[i][n].load(vc + off + vd[n]);
      }
    }
  };
  // acc[j] += V^T P^T[j], for the rows that `take` names, without the values
  // that `cut` takes out of word i of an operand.
  auto add_values = [&](const OpT (&ph)[R], const OpT (&pl)[R], auto cut, auto take) {
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
          w[i] = cut(i, w[i]);
        }
        const OpT a = __builtin_bit_cast(OpT, w);
#pragma unroll
        for (int j = 0; j < R; ++j) {
          f4_t x = mma(a, ph[j], acc[j][n][e]);
          if constexpr (sizeof(T) == 2) x = mma(a, pl[j], x);
          acc[j][n][e] = take(j) ? x : acc[j][n][e];
        }
      }
  };
  const auto nothing = [](int, uint32_t w) { return w; };
  const auto all_rows = [](int) { return true; };

  int tile = begin + wave;
  look_up(tile);
  uint32_t ok = place(tile);
  if (tile < end) {
    load_k();
    load_v();
  }
  look_up(tile + kWaves);
  while (tile < end) {
    const int pos0 = tile * TS;
    const bool whole = pos0 >= low_last && pos0 + TS - 1 <= first_pos && ok == ((uint64_t{1} << TS) - 1);
    if (ragged) {
#pragma unroll
      for (int s = 0; s < NK; ++s)
#pragma unroll
        for (int h = 0; h < NH; ++h) k[h][s].keep((4 * s + g) * KV < p.D);
    }
    f4_t sc[R][NH] = {};
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int s = 0; s < NK; ++s) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = k[h][s].word(i);
#pragma unroll
        for (int j = 0; j < R; ++j) sc[j][h] = mma(__builtin_bit_cast(OpT, w), q[j][s], sc[j][h]);
      }
    const int next = tile + kWaves;
    const uint32_t ok_next = place(next);
    if (next < end) load_k();
    look_up(next + kWaves);

    OpT ph[R], pl[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      float x[KV], top = -INFINITY;
#pragma unroll
      for (int i = 0; i < KV; ++i) {
        x[i] = sc[j][i / 4][i % 4] * scale2;
        if (!whole) {
          const int t = 16 * (i / 4) + 4 * g + i % 4, pos = pos0 + t;
          x[i] = pos <= hi[j] && pos >= lo[j] && (ok >> t & 1) ? x[i] : -INFINITY;
        }
        top = fmaxf(top, x[i]);
      }
      top = over_groups(top, [](float a, float b) { return fmaxf(a, b); });
      const float now = fmaxf(base[j], top - kShift);
      const float from = now == -INFINITY ? 0.f : now;
      const float keep = exp2_hw(base[j] - from);
      base[j] = now;
      float add = 0.f;
#pragma unroll
      for (int i = 0; i < KV; ++i) {
        x[i] = exp2_hw(x[i] - from);
        add += x[i];
      }
      sum[j] = sum[j] * keep + add;
#pragma unroll
      for (int i = 0; i < KV; ++i) {
        if constexpr (sizeof(T) == 4) {
          ph[j][i] = x[i];
        } else {
          const T h = static_cast<T>(x[i]);
          ph[j][i] = h;
          pl[j][i] = static_cast<T>(x[i] - static_cast<float>(h));
        }
      }
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < VB; ++e) acc[j][n][e] *= keep;
    }
    if (whole) {
      add_values(ph, pl, nothing, all_rows);
    } else {
      // Values at positions that no row sees are no part of the sums, whatever
      // they are; those that some new tokens see and others do not are taken
      // for each token apart where one is not finite (0 * inf is NaN).
      bool fine = true;
#pragma unroll
      for (int i = 0; i < KV; ++i) {
        const int t = 16 * (i / 4) + 4 * g + i % 4, pos = pos0 + t;
        const bool in = pos <= last_pos && pos >= low_first && (ok >> t & 1);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          v[i][n].keep(in);
          fine = fine && v[i][n].finite();
        }
      }
      if (first_tok == last_tok || __all(fine)) {
        add_values(ph, pl, nothing, all_rows);
      } else {
        for (int pos_t = first_pos; pos_t <= last_pos; ++pos_t) {
          const auto seen = [&](int i) {
            const int pos = pos0 + 16 * (i / 4) + 4 * g + i % 4;
            return pos <= pos_t && (!p.window || pos > pos_t - p.window);
          };
          add_values(
              ph, pl,
              [&](int i, uint32_t w) {
                if constexpr (sizeof(T) == 4) return seen(i) ? w : 0;
                else return w & ((seen(2 * i) ? 0xffffu : 0) | (seen(2 * i + 1) ? 0xffff0000u : 0));
              },
              [&](int j) { return hi[j] == pos_t; });
        }
      }
    }
    if (next < end) load_v();
    ok = ok_next;
    tile = next;
  }

  // The block's waves join: a row's base is the largest, sums are scaled to it.
  constexpr int kPitch = DP + 4;  // rows 4 banks apart
  __shared__ float2 ml[kWaves][16];
  __shared__ __align__(16) float part_acc[kWaves][16][kPitch];
  const float v_scale = p.v_scale ? p.v_scale[head] : 1.f;
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
    my_sum = over_groups(my_sum, [](float a, float b) { return a + b; });
    if (j) __syncthreads();
    if (g == 0) ml[wave][l15] = make_float2(my_base, my_sum);
    __syncthreads();
    float top = ml[0][l15].x;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, ml[w][l15].x);
    const float mine = weight(my_base, top);
    if (l15 < rows) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
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
              x[u] = y * mine;
            }
            *reinterpret_cast<f4_t*>(&part_acc[wave][l15][(n * 16 + 4 * g + i) * VB + e]) = x;
          }
    }
    __syncthreads();
    const int quads = p.D / 4;
    for (int u = threadIdx.x; u < rows * quads; u += kBlock) {
      const int row = u / quads, d = (u - row * quads) * 4, r = r0 + 16 * j + row;
      float b = ml[0][row].x;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) b = fmaxf(b, ml[w][row].x);
      float l = 0.f;
      f4_t x = {};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        l += ml[w][row].y * weight(ml[w][row].x, b);
        x += *reinterpret_cast<const f4_t*>(&part_acc[w][row][d]);
      }
      if (part.of > 1) {
        const int64_t at = (static_cast<int64_t>(slot) * p.Hkv + head) * p.M + r;
        *reinterpret_cast<f4_t*>(p.acc + at * p.D + d) = x;
        if (d == 0) p.ml[at] = make_float2(b, l);
        continue;
      }
      const int tok = r / p.G;
      const int64_t hq = static_cast<int64_t>(head) * p.G + (r - tok * p.G);
      const float inv = l == 0.f ? 0.f : v_scale / l;
      float o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = l == 0.f ? 0.f : x[i] * inv;
      store_vec_f32<T, 4>(static_cast<T*>(p.out) + part.b * p.o_seq + tok * p.o_tok +
                              hq * p.o_head + d, o);
      if (p.lse && d == 0)
        p.lse[(static_cast<int64_t>(part.b) * p.T + tok) * p.Hkv * p.G + hq] =
            l == 0.f ? -INFINITY : (b + __log2f(l)) * 0.69314718056f;
    }
  }
}

// Joins the parts of sequences that have several: a block for a (sequence,
// head) and every gridDim.y-th of its rows; D / 4 lanes (a power of two of
// them) read a part's row, the block's teams take parts in turn.
template <typename T>
__global__ void __launch_bounds__(kBlock) join_kernel(Params p, int team) {
  __shared__ float2 ml[16];
  __shared__ __align__(16) float sums[kBlock * 4];
  const int b = blockIdx.x / p.Hkv, head = blockIdx.x % p.Hkv;
  const int2 meta = p.meta[b];
  if (meta.y <= 1) return;
  const int teams = kBlock / team, own = threadIdx.x / team, d = threadIdx.x % team * 4;
  const float v_scale = p.v_scale ? p.v_scale[head] : 1.f;
  for (int r = blockIdx.y; r < p.M; r += gridDim.y) {
    float base = -INFINITY, sum = 0.f;
    f4_t acc = {};
#pragma unroll 4
    for (int i = own; i < meta.y; i += teams) {
      const int64_t at = (static_cast<int64_t>(meta.x + i) * p.Hkv + head) * p.M + r;
      const float2 x = p.ml[at];
      f4_t y = {};
      if (d < p.D) y = *reinterpret_cast<const f4_t*>(p.acc + at * p.D + d);
      const float now = fmaxf(base, x.x), a = weight(base, now), c = weight(x.x, now);
      sum = sum * a + x.y * c;
      acc = acc * a + y * c;
      base = now;
    }
    if (threadIdx.x % team == 0) ml[own] = make_float2(base, sum);
    __syncthreads();
    float top = ml[0].x;
    for (int i = 1; i < teams; ++i) top = fmaxf(top, ml[i].x);
    acc *= weight(base, top);
    *reinterpret_cast<f4_t*>(&sums[threadIdx.x * 4]) = acc;
    __syncthreads();
    if (own == 0 && d < p.D) {
      float l = 0.f;
      f4_t x = {};
      for (int i = 0; i < teams; ++i) {
        l += ml[i].y * weight(ml[i].x, top);
        x += *reinterpret_cast<const f4_t*>(&sums[(i * team + threadIdx.x) * 4]);
      }
      const int tok = r / p.G;
      const int64_t hq = static_cast<int64_t>(head) * p.G + (r - tok * p.G);
      const float inv = l == 0.f ? 0.f : v_scale / l;
      float o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = l == 0.f ? 0.f : x[i] * inv;
      store_vec_f32<T, 4>(static_cast<T*>(p.out) + b * p.o_seq + tok * p.o_tok + hq * p.o_head +
                              d, o);
      if (p.lse && d == 0)
        p.lse[(static_cast<int64_t>(b) * p.T + tok) * p.Hkv * p.G + hq] =
            l == 0.f ? -INFINITY : (top + __log2f(l)) * 0.69314718056f;
    }
    __syncthreads();
  }
}

template <typename T, typename C, int DP, int R>
void launch_pages(const Params& p, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(p.slots) * p.groups * p.Hkv);
  if (p.page_size % 16 == 0)
    hipLaunchKernelGGL((attention_kernel<T, C, DP, R, true>), grid, dim3(kBlock), 0, s, p);
  else
    hipLaunchKernelGGL((attention_kernel<T, C, DP, R, false>), grid, dim3(kBlock), 0, s, p);
}

template <typename T, typename C, int DP>
void launch_rows(const Params& p, int tiles, hipStream_t s) {
  if constexpr (DP <= 128) {
    if (tiles == 2) return launch_pages<T, C, DP, 2>(p, s);
  }
  launch_pages<T, C, DP, 1>(p, s);
}

// `tiles`: row tiles of a wave, as the entry point counted p.groups by.
template <typename T, typename C>
int run(const Params& p, int tiles, hipStream_t s) {
  if (p.D <= 64) launch_rows<T, C, 64>(p, tiles, s);
  else if (p.D <= 128) launch_rows<T, C, 128>(p, tiles, s);
  else launch_rows<T, C, 256>(p, tiles, s);
  int st = launch_status();
  if (st != XK_OK || p.alone) return st;
  const int team = p.D <= 64 ? 16 : (p.D <= 128 ? 32 : 64);
  const int64_t heads = static_cast<int64_t>(p.B) * p.Hkv;
  const dim3 grid(static_cast<uint32_t>(heads),
                  static_cast<uint32_t>(std::min<int64_t>(p.M, cdiv(1024, heads))));
  hipLaunchKernelGGL((join_kernel<T>), grid, dim3(kBlock), 0, s, p, team);
  return launch_status();
}

int run_f32(const Params& p, int tiles, hipStream_t s);
int run_bf16(const Params& p, int tiles, hipStream_t s);
int run_f16(const Params& p, int tiles, hipStream_t s);
int run_bf16_f8(const Params& p, int tiles, hipStream_t s);
int run_f16_f8(const Params& p, int tiles, hipStream_t s);

}  // namespace paged
}  // namespace xk
