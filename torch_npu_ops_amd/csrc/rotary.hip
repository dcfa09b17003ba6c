// Rotary positions for gfx950: xk_rotary_embedding (q and k turned, or the
// gradients turned back) and xk_rotary_cache_append (the same, with k and v
// stored in their slots of a paged cache).
//
// A pair (u, v) of a head at position t becomes L (u cos - v sin, v cos +
// u sin) with the angle t f; pairs are (i, i + r/2) or (2i, 2i + 1) of the
// first r elements, the others are copied.  The backward pass is the same
// with the angle's sign changed, since the turn is orthogonal up to L.
//
// The angle is formed in 64 bits (t f is exact to 53 bits there; in fp32 it
// would be off by half a radian at t = 10^7) and reduced to [-pi/4, pi/4]
// before it is rounded to fp32.
//
// What bounds it: HBM for many tokens, one wave's chain (position -> angle ->
// LDS -> rotation -> store) for few.  So a block's four waves take four tokens,
// or parts of two, of one or of a part of one: they form cos and sin of its
// tokens' pairs once, into LDS, and then lanes take units of two vectors, the two
// that a rotation by halves pairs or any two.  A lane reads what it overwrites
// itself, so outputs may be the inputs.  The first units' loads are requested
// before the angle is formed.  What is read and written passes once, so both ask
// for no room in the caches (75.2 us without, 66.5 with, for the 335 MB of 16384
// tokens of 32 + 8 bf16 heads of 128: 5.2 TB/s, what a copy reaches over as much).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "xk_common.h"

namespace xk {
namespace {

using f8 = unsigned char;  // e4m3, as stored
constexpr float kF8Max = 448.f;
constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr int kMaxDim = 512;
constexpr int kMaxHeads = 4096;
// Units that a lane requests together, and takes in all where tokens fill the
// card.  16384 tokens of 32 + 8 bf16 heads of 128, us: 2 and 3 64.1, 2 and 5
// 67.3, 2 and 2 75.0, 3 and 3 63.9, 5 and 5 66.2; 8192 in fp32 59.9, 61.6, 65.9,
// 60.6, 63.3; heads of 256 with 64 turned in fp32 31.6, 30.3, 31.2, 30.5, 29.9.
constexpr int kAhead = 2;
constexpr int kUnits = 3;

struct Rows {  // [tokens, heads, D]
  const void* src;
  int64_t st, sh;
  void* dst;
  int64_t dt, dh;
};

struct RotaryParams {
  Rows q, k;
  // The cache (append only): v's rows come in `v`, k's and v's places are
  // dst + page * page pitch + place * place pitch + head * dh.
  Rows v;
  int64_t k_page, k_place, v_page, v_place;
  const void* slots;
  int slots_i64;
  int64_t num_slots, page_size;
  int flat;  // a slot's row is at slot * place pitch in both caches
  const float* k_scale;
  const float* v_scale;
  const void* pos;  // NULL: nothing is turned
  int pos_i64;
  const float* freq;
  int half;  // pairs turned
  float len;
  float sign;
  int64_t T;
  int D, hq, hkv;
  int units;       // of a head
  uint32_t magic;  // ceil(2^32 / units); 0 for one unit
  int of_wave;     // log2 of a block's waves that take one token
  int slices;      // blocks that take the same tokens
};

// cos and sin of t f.  n quarter turns are taken off in 64 bits (the second
// fma adds what pi/2's first 53 bits leave out), so that the rest r, at most
// pi/4, is right to 2^-25 when it is rounded.  There the Taylor series end at
// r^9 and r^10: what follows is below r^11/11! < 2^-28 and r^12/12! < 2^-32.
// With their roundings both are off by at most 2.8 * 2^-25 (measured: 2.35; the
// nearest fp32 values: 1).
__device__ __forceinline__ void turn_of(double t, float f, float& c, float& s) {
  const double a = t * static_cast<double>(f);
  const double n = __builtin_rint(a * 0.63661977236758134308);
  const double d = __builtin_fma(n, -6.12323399573676603587e-17,
                                 __builtin_fma(n, -1.57079632679489655800, a));
  const float r = static_cast<float>(d), z = r * r;
  float sr = __builtin_fmaf(z, 1.f / 362880, -1.f / 5040);
  sr = __builtin_fmaf(z, sr, 1.f / 120);
  sr = __builtin_fmaf(z, sr, -1.f / 6);
  sr = __builtin_fmaf(z * r, sr, r);
  float cr = __builtin_fmaf(z, -1.f / 3628800, 1.f / 40320);
  cr = __builtin_fmaf(z, cr, -1.f / 720);
  cr = __builtin_fmaf(z, cr, 1.f / 24);
  cr = __builtin_fmaf(z, cr, -0.5f);
  cr = __builtin_fmaf(z, cr, 1.f);
  // n modulo 4, exact for every n.
  const int q = static_cast<int>(__builtin_fma(__builtin_floor(n * 0.25), -4.0, n));
  const float x = q & 1 ? sr : cr, y = q & 1 ? cr : sr;
  c = (q == 1 || q == 2) ? -x : x;
  s = q >= 2 ? -y : y;
}

__device__ __forceinline__ int64_t load_int(const void* p, int is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// One value in e4m3, to nearest even; beyond 448 it stays there, NaN is NaN.
__device__ __forceinline__ float f8_range(float x) {
  const float c = __builtin_fminf(__builtin_fmaxf(x, -kF8Max), kF8Max);
  return x != x ? x : c;
}

template <int V>
__device__ __forceinline__ Vec<f8, V> to_f8(const float (&x)[V], float scale) {
  Vec<f8, V> o;
  if constexpr (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(f8_range(x[i] / scale), f8_range(x[i + 1] / scale),
                                              0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(f8_range(x[i + 2] / scale),
                                          f8_range(x[i + 3] / scale), w, true);
#pragma unroll
      for (int j = 0; j < 4; ++j) o.v[i + j] = static_cast<f8>(w >> (8 * j));
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      o.v[i] = static_cast<f8>(
          __builtin_amdgcn_cvt_pk_fp8_f32(f8_range(x[i] / scale), 0.f, 0, false));
  }
  return o;
}

template <typename T, int V>
__device__ __forceinline__ void put(T* d, const float (&x)[V]) {
  Vec<T, V> o;
#pragma unroll
  for (int i = 0; i < V; ++i) o.v[i] = from_f32<T>(x[i]);
  st_stream(reinterpret_cast<Vec<T, V>*>(d), o);
}

// T: the tokens' type.  C: the cache's (f8 or T), void without a cache.
// V: elements of a vector; NEXT: pairs are neighbours.
template <typename T, typename C, int V, bool NEXT>
__global__ void __launch_bounds__(kBlock) rotary_kernel(RotaryParams p) {
  constexpr bool kCache = !std::is_void<C>::value;
  using VT = Vec<T, V>;
  extern __shared__ __align__(16) float2 tab_all[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  // The block's tokens, the wave's one and its part of that.
  const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x;
  const uint32_t group = p.slices == 1 ? id : id / p.slices;
  const int in_block = wave >> p.of_wave, part = wave & ((1 << p.of_wave) - 1);
  const int slice = ((id - group * p.slices) << p.of_wave) + part;
  int64_t tok = static_cast<int64_t>(group) * (kWaves >> p.of_wave) + in_block;
  const bool none = tok >= p.T;  // the last block's
  if (none) tok = p.T - 1;
  float2* tab = tab_all + in_block * p.half;

  const int heads = p.hq + p.hkv * (kCache ? 2 : 1);
  const int total = none ? 0 : heads * p.units;
  const int step = (p.slices << p.of_wave) * kWave;
  // Half pairs: units below `pairs` hold two vectors half a turn apart.
  const int pairs = NEXT ? 0 : p.half / V;

  struct Unit {
    VT a, b;
    int head, at, bt;  // at, bt: first elements
  };
  auto src_of = [&](int head) -> const T* {
    if (head < p.hq) return static_cast<const T*>(p.q.src) + tok * p.q.st + head * p.q.sh;
    head -= p.hq;
    if (!kCache || head < p.hkv)
      return static_cast<const T*>(p.k.src) + tok * p.k.st + head * p.k.sh;
    return static_cast<const T*>(p.v.src) + tok * p.v.st + (head - p.hkv) * p.v.sh;
  };
  auto request = [&](int u, Unit& w) {
    w.head = p.magic ? static_cast<int>(__umulhi(static_cast<uint32_t>(u), p.magic)) : u;
    const int i = u - w.head * p.units;
    // (The two vectors of a unit without such pairs are far from each other too,
    // so that neighbouring lanes take neighbouring vectors; a pair of neighbours
    // is one unit where a vector is one element.)
    const bool apart = i < pairs;
    if constexpr (NEXT && V == 1) {
      w.at = 2 * i;
      w.bt = w.at + 1;
    } else {
      w.at = (apart || NEXT ? 0 : p.half) + i * V;
      w.bt = w.at + (apart ? p.half : (p.units - pairs) * V);
    }
    const T* s = src_of(w.head);
    w.a = ld_stream(reinterpret_cast<const VT*>(s + w.at));
    w.b = ld_stream(reinterpret_cast<const VT*>(s + (w.bt < p.D ? w.bt : w.at)));
  };

  int u0 = slice * kWave + lane;
  Unit w[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (u0 + i * step < total) request(u0 + i * step, w[i]);

  // The row of the cache, known by now or not at all (a slot outside it).
  int64_t k_row = 0, v_row = 0;
  bool stored = false;
  if constexpr (kCache) {
    const int64_t slot = load_int(p.slots, p.slots_i64, tok);
    stored = slot >= 0 && slot < p.num_slots;
    if (stored) {
      int64_t page = 0, place = slot;
      if (!p.flat) {
        page = p.num_slots <= UINT32_MAX ? static_cast<uint32_t>(slot) /
                                               static_cast<uint32_t>(p.page_size)
                                         : slot / p.page_size;
        place = slot - page * p.page_size;
      }
      k_row = page * p.k_page + place * p.k_place;
      v_row = page * p.v_page + place * p.v_place;
    }
  }
  if (p.pos) {
    const double t = static_cast<double>(load_int(p.pos, p.pos_i64, tok));
    for (int i = part * kWave + lane; i < p.half; i += kWave << p.of_wave) {
      float c, s;
      turn_of(t, p.freq[i], c, s);
      tab[i] = make_float2(c * p.len, s * p.len * p.sign);
    }
    __syncthreads();
  }

  auto finish = [&](Unit& w) {
    float a[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      a[i] = to_f32(w.a.v[i]);
      b[i] = to_f32(w.b.v[i]);
    }
    const bool is_v = kCache && w.head >= p.hq + p.hkv;
    if (p.pos && !is_v) {
      if constexpr (NEXT && V >= 2) {
        const int turned = 2 * p.half;
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          if (w.at < turned) {
            const float2 t = tab[(w.at + i) / 2];
            const float x = a[i], y = a[i + 1];
            a[i] = x * t.x - y * t.y;
            a[i + 1] = y * t.x + x * t.y;
          }
          if (w.bt < turned) {
            const float2 t = tab[(w.bt + i) / 2];
            const float x = b[i], y = b[i + 1];
            b[i] = x * t.x - y * t.y;
            b[i + 1] = y * t.x + x * t.y;
          }
        }
      } else if (w.at < (NEXT ? 2 * p.half : p.half)) {
        const int first = NEXT ? w.at / 2 : w.at;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float2 t = tab[first + i];
          const float x = a[i], y = b[i];
          a[i] = x * t.x - y * t.y;
          b[i] = y * t.x + x * t.y;
        }
      }
    }
    const bool two = w.bt < p.D;
    if (w.head < p.hq || !kCache) {
      const bool is_q = w.head < p.hq;
      T* d = is_q ? static_cast<T*>(p.q.dst) + tok * p.q.dt + w.head * p.q.dh
                  : static_cast<T*>(p.k.dst) + tok * p.k.dt + (w.head - p.hq) * p.k.dh;
      put<T, V>(d + w.at, a);
      if (two) put<T, V>(d + w.bt, b);
      return;
    }
    if constexpr (kCache) {
      if (!stored) return;
      const int h = w.head - p.hq - (is_v ? p.hkv : 0);
      C* d = is_v ? static_cast<C*>(p.v.dst) + v_row + h * p.v.dh
                  : static_cast<C*>(p.k.dst) + k_row + h * p.k.dh;
      if constexpr (std::is_same<C, f8>::value) {
        const float* sc = is_v ? p.v_scale : p.k_scale;
        const float scale = sc ? sc[h] : 1.f;
        *reinterpret_cast<Vec<f8, V>*>(d + w.at) = to_f8<V>(a, scale);
        if (two) *reinterpret_cast<Vec<f8, V>*>(d + w.bt) = to_f8<V>(b, scale);
      } else {
        put<C, V>(d + w.at, a);
        if (two) put<C, V>(d + w.bt, b);
      }
    }
  };
  while (true) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (u0 + i * step < total) finish(w[i]);
    u0 += kAhead * step;
    if (u0 - lane >= total) break;  // the wave's first lane
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (u0 + i * step < total) request(u0 + i * step, w[i]);
  }
}

template <typename T, typename C, int V>
int launch_v(RotaryParams& p, bool next, hipStream_t s) {
  // Units of a head: two vectors each, the last perhaps one.
  const int turned = 2 * p.half;
  p.units = next ? static_cast<int>(cdiv(p.D, 2 * V))
                 : p.half / V + static_cast<int>(cdiv(p.D - turned, 2 * V));
  p.magic = p.units == 1 ? 0 : static_cast<uint32_t>((0x100000000ull + p.units - 1) / p.units);
  const int64_t heads = p.hq + static_cast<int64_t>(p.hkv) * (std::is_void<C>::value ? 1 : 2);
  const int64_t total = heads * p.units;
  // (u * units < 2^32 keeps the multiplication by `magic` exact: u is below
  // 3 * kMaxHeads * units, units at most kMaxDim / 2.)
  // Waves of a token: as many as leave a lane kUnits units, more where tokens
  // alone do not give a compute unit 16 waves, but none without a unit.
  const int64_t full = cdiv(total, kWave);
  const int64_t room = std::max<int64_t>(1, 16 * num_cus() / p.T);
  const int64_t want = std::max(std::min(room, full), cdiv(full, kUnits));
  p.of_wave = want >= 4 ? 2 : want >= 2 ? 1 : 0;
  p.slices = static_cast<int>(cdiv(want, 1 << p.of_wave));
  const int64_t blocks = cdiv(p.T, kWaves >> p.of_wave) * p.slices;
  if (blocks > INT32_MAX) return XK_ERR_UNSUPPORTED;
  const size_t lds = sizeof(float2) * (p.pos ? p.half : 0) * (kWaves >> p.of_wave);
  // (2^32 threads at the most in a dimension; blocks past the last token have none.)
  const int64_t wide = std::min<int64_t>(blocks, 1 << 23);
  const dim3 grid(static_cast<uint32_t>(wide), static_cast<uint32_t>(cdiv(blocks, wide)));
  if (next)
    hipLaunchKernelGGL((rotary_kernel<T, C, V, true>), grid, dim3(kBlock), lds, s, p);
  else
    hipLaunchKernelGGL((rotary_kernel<T, C, V, false>), grid, dim3(kBlock), lds, s, p);
  return launch_status();
}

// The widest vector that every row, place and part of a head starts and ends
// on (16 bytes of the tokens' type at the most).
template <typename T>
int vector_of(const RotaryParams& p, bool next, int cache_bytes) {
  for (int v = 16 / sizeof(T); v > 1; v /= 2) {
    bool ok = p.D % v == 0 && (next ? 2 * p.half : p.half) % v == 0;
    auto rows = [&](const Rows& r, bool dst_is_cache) {
      const int db = dst_is_cache ? cache_bytes : static_cast<int>(sizeof(T));
      ok = ok && r.st % v == 0 && r.sh % v == 0 && aligned(r.src, v * sizeof(T)) &&
           r.dt % v == 0 && r.dh % v == 0 && aligned(r.dst, v * db);
    };
    if (p.hq) rows(p.q, false);
    if (p.hkv) rows(p.k, cache_bytes > 0);
    if (cache_bytes) {
      rows(p.v, true);
      ok = ok && p.k_page % v == 0 && p.k_place % v == 0 && p.v_page % v == 0 &&
           p.v_place % v == 0;
    }
    if (ok) return v;
  }
  return 1;
}

template <typename T, typename C>
int launch(RotaryParams& p, bool next, hipStream_t s) {
  int cache_bytes = 0;
  if constexpr (!std::is_void<C>::value) cache_bytes = sizeof(C);
  switch (vector_of<T>(p, next, cache_bytes)) {
    case 8:
      if constexpr (sizeof(T) == 2) return launch_v<T, C, 8>(p, next, s);
      return XK_ERR_UNSUPPORTED;
    case 4: return launch_v<T, C, 4>(p, next, s);
    case 2: return launch_v<T, C, 2>(p, next, s);
    default: return launch_v<T, C, 1>(p, next, s);
  }
}

// What both entry points check of the positions and the turned part.
int check_turn(const void* positions, xk_dtype pos_dtype, const float* inv_freq,
               int64_t rotary_dim, float scale, int64_t num_tokens, int64_t head_dim,
               xk_dtype dtype) {
  if (num_tokens < 0 || head_dim <= 0 || head_dim > kMaxDim || rotary_dim < 0 ||
      rotary_dim % 2 || rotary_dim > head_dim || !(scale > 0.f && scale < INFINITY))
    return XK_ERR_INVALID;
  if (!is_float_dtype(dtype)) return XK_ERR_UNSUPPORTED;
  if (positions && pos_dtype != XK_I32 && pos_dtype != XK_I64) return XK_ERR_UNSUPPORTED;
  if (positions && (rotary_dim == 0 || !inv_freq)) return XK_ERR_INVALID;
  return XK_OK;
}

}  // namespace
}  // namespace xk

using namespace xk;

extern "C" int xk_rotary_embedding(
    const void* q, int64_t stride_q_tok, int64_t stride_q_head, void* q_out,
    int64_t stride_qo_tok, int64_t stride_qo_head, int64_t Hq, const void* k,
    int64_t stride_k_tok, int64_t stride_k_head, void* k_out, int64_t stride_ko_tok,
    int64_t stride_ko_head, int64_t Hk, const void* positions, xk_dtype pos_dtype,
    const float* inv_freq, int64_t rotary_dim, int interleaved, float scale, int inverse,
    int64_t num_tokens, int64_t head_dim, xk_dtype dtype, void* stream) {
  const int st = check_turn(positions, pos_dtype, inv_freq, rotary_dim, scale, num_tokens,
                            head_dim, dtype);
  if (st != XK_OK) return st;
  if (Hq < 0 || Hk < 0 || Hq > kMaxHeads || Hk > kMaxHeads) return XK_ERR_INVALID;
  if (num_tokens == 0 || Hq + Hk == 0) return XK_OK;
  if (!positions || (Hq && (!q || !q_out)) || (Hk && (!k || !k_out))) return XK_ERR_INVALID;
  RotaryParams p{};
  p.q = {q, stride_q_tok, stride_q_head, q_out, stride_qo_tok, stride_qo_head};
  p.k = {k, stride_k_tok, stride_k_head, k_out, stride_ko_tok, stride_ko_head};
  p.pos = positions;
  p.pos_i64 = pos_dtype == XK_I64;
  p.freq = inv_freq;
  p.half = static_cast<int>(rotary_dim / 2);
  p.len = scale;
  p.sign = inverse ? -1.f : 1.f;
  p.T = num_tokens;
  p.D = static_cast<int>(head_dim);
  p.hq = static_cast<int>(Hq);
  p.hkv = static_cast<int>(Hk);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case XK_F32: return launch<float, void>(p, interleaved, s);
    case XK_BF16: return launch<bf16, void>(p, interleaved, s);
    default: return launch<f16, void>(p, interleaved, s);
  }
}

extern "C" int xk_rotary_cache_append(
    const void* q, int64_t stride_q_tok, int64_t stride_q_head, void* q_out,
    int64_t stride_qo_tok, int64_t stride_qo_head, int64_t Hq, const void* k,
    int64_t stride_k_tok, int64_t stride_k_head, const void* v, int64_t stride_v_tok,
    int64_t stride_v_head, int64_t Hkv, void* k_cache, int64_t stride_kc_page,
    int64_t stride_kc_slot, int64_t stride_kc_head, void* v_cache, int64_t stride_vc_page,
    int64_t stride_vc_slot, int64_t stride_vc_head, xk_dtype cache_dtype, int64_t num_pages,
    int64_t page_size, const void* slots, xk_dtype slot_dtype, const void* positions,
    xk_dtype pos_dtype, const float* inv_freq, int64_t rotary_dim, int interleaved, float scale,
    const float* k_scale, const float* v_scale, int64_t num_tokens, int64_t head_dim,
    xk_dtype dtype, void* stream) {
  const int st = check_turn(positions, pos_dtype, inv_freq, rotary_dim, scale, num_tokens,
                            head_dim, dtype);
  if (st != XK_OK) return st;
  if (Hq < 0 || Hkv <= 0 || Hq > kMaxHeads || Hkv > kMaxHeads || num_pages < 0 ||
      page_size <= 0 || num_pages > INT64_MAX / page_size)
    return XK_ERR_INVALID;
  const bool eight = cache_dtype == XK_F8E4M3;
  if (eight ? dtype == XK_F32 : cache_dtype != dtype) return XK_ERR_UNSUPPORTED;
  if (!eight && (k_scale || v_scale)) return XK_ERR_INVALID;
  if (slot_dtype != XK_I32 && slot_dtype != XK_I64) return XK_ERR_UNSUPPORTED;
  if (num_tokens == 0) return XK_OK;
  if ((Hq && (!q || !q_out)) || !k || !v || !slots) return XK_ERR_INVALID;
  if (num_pages > 0 && (!k_cache || !v_cache)) return XK_ERR_INVALID;
  RotaryParams p{};
  p.q = {q, stride_q_tok, stride_q_head, q_out, stride_qo_tok, stride_qo_head};
  p.k = {k, stride_k_tok, stride_k_head, k_cache, 0, stride_kc_head};
  p.v = {v, stride_v_tok, stride_v_head, v_cache, 0, stride_vc_head};
  p.k_page = stride_kc_page;
  p.k_place = stride_kc_slot;
  p.v_page = stride_vc_page;
  p.v_place = stride_vc_slot;
  p.slots = slots;
  p.slots_i64 = slot_dtype == XK_I64;
  p.num_slots = num_pages * page_size;
  p.page_size = page_size;
  p.flat = num_pages <= 1 || (stride_kc_page == page_size * stride_kc_slot &&
                              stride_vc_page == page_size * stride_vc_slot);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.pos = positions;
  p.pos_i64 = pos_dtype == XK_I64;
  p.freq = inv_freq;
  p.half = positions ? static_cast<int>(rotary_dim / 2) : 0;
  p.len = scale;
  p.sign = 1.f;
  p.T = num_tokens;
  p.D = static_cast<int>(head_dim);
  p.hq = static_cast<int>(Hq);
  p.hkv = static_cast<int>(Hkv);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool next = interleaved && positions;
  switch (dtype) {
    case XK_F32: return launch<float, float>(p, next, s);
    case XK_BF16:
      return eight ? launch<bf16, f8>(p, next, s) : launch<bf16, bf16>(p, next, s);
    default: return eight ? launch<f16, f8>(p, next, s) : launch<f16, f16>(p, next, s);
  }
}
