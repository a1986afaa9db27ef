// Key/value cache held in 4 bits: append (with the decode step's rotation),
// read-back, and attention over it.
//
// Groups of 32 values of one head share a zero point z = fp16(min) and a scale
// s = fp16((max - z) / 15); a value x is held as the code rint((x - z) / s),
// 0..15, and stands for z + s code. Magnitudes above 57344 are held as that.
// That is 5 bits a value. z and s are taken in 64 bits and codes are decided
// exactly, ties to even, so that the same key has the same codes everywhere.
// A token's key or value with a NaN makes the token's key scales NaN (in that
// head): each query that sees it becomes NaN, and no other query does.
//
// Memory, for batch b, key head n, L tokens rounded up to 64, G = h / 32,
// Q = max(1, h / 64):
//   k_codes [b, n, L, h / 2]: the dword of values 8w..8w+7 holds value
//       2j + p in bits 4j + 16p, so that a mask and a shift give the pair
//       (2j, 2j + 1) in two halves of a register
//   k_meta  [b, n, L, G, 2] fp16: s, z
//   v_codes [b, n, L / 4, 16, 2 pairs, Q, 2 tokens] 16 bits: chunk c has
//       the values c h/16 .. of four tokens, and two tokens that meet in one
//       register are neighbours already: the matrix instruction contracts
//       over tokens
//   v_meta  [b, n, G, L / 4, 2, 4] fp16: four tokens' s, then their z

#include "common.h"

#include <torch/extension.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>

namespace {

constexpr int kGroup = 32;
constexpr float kHeldMax = 57344.f;

struct CacheView {
  unsigned char* k_codes;
  __half* k_meta;
  unsigned char* v_codes;
  __half* v_meta;
  int b, heads, h;
  long room;      // tokens, a multiple of 64
  long capacity;  // tokens that may be used
};

struct Start {
  const long* at;  // [b] or [1], or null: the scalar counts
  long stride, scalar;
  // held where a token's number can be added to it or a place taken from it
  __device__ __forceinline__ long of(int ib) const {
    const long t = at ? at[ib * stride] : scalar;
    return min(max(t, -(1l << 60)), 1l << 60);
  }
};

__host__ __device__ __forceinline__ int v_quarters(int h) {
  return h >= 64 ? h / 64 : 1;
}

// Places within a head's memory, for a token t counted from a block of four
// on: the 16-bit piece of v_codes with 4 values (2 where h = 32) from value d
// on, and a group's scale in v_meta, four before its zero point.
template <int H>
struct Pieces {
  static constexpr unsigned kQuarters = H >= 64 ? H / 64 : 1;
  static constexpr unsigned kBlock = 64 * kQuarters;  // of four tokens

  static __device__ __forceinline__ unsigned at(unsigned t, unsigned d) {
    constexpr unsigned per = H / 16;
    const unsigned chunk = d / per, quarter = (d % per) / 4;
    return (t >> 2) * kBlock + chunk * 4 * kQuarters +
           (((t >> 1) & 1) * kQuarters + quarter) * 2 + (t & 1);
  }
  static __device__ __forceinline__ long scale_at(const CacheView& c,
                                                  unsigned t, int group) {
    return (long)group * (c.room * 2) + (t >> 2) * 8 + (t & 3);
  }
};

// A sequence's head from the block of four tokens that holds token t on.
template <int H>
struct HeadView {
  unsigned* k_codes;  // these two from token t itself on
  __half2* k_meta;
  unsigned short* v_codes;
  __half* v_meta;
  unsigned first;  // token t's number in its block

  __device__ __forceinline__ HeadView(const CacheView& c, long bh, long t)
      : k_codes((unsigned*)c.k_codes + (bh * c.room + t) * (H / 8)),
        k_meta((__half2*)c.k_meta + (bh * c.room + t) * (H / kGroup)),
        v_codes((unsigned short*)c.v_codes +
                (bh * (c.room >> 2) + (t >> 2)) * Pieces<H>::kBlock),
        v_meta(c.v_meta + bh * (c.room * 2) * (H / kGroup) + (t >> 2) * 8),
        first(t & 3) {}
};

// code of x: the nearest whole number of s above z, ties to even, by products
// in 64 bits; inv is about 1 / s.
__device__ __forceinline__ float code_between(float x, float z, float s,
                                              float inv) {
  const double above = (double)x - (double)z;
  float n = floorf((float)above * inv);
  n = fminf(fmaxf(n, 0.f), 15.f);
  // n may be one off: bring it to the floor, then round by twice the rest
  double rest = above - (double)n * (double)s;
  if (rest < 0.0 && n > 0.f) {
    n -= 1.f;
    rest += s;
  } else if (rest >= (double)s && n < 15.f) {
    n += 1.f;
    rest -= s;
  }
  const double twice = 2.0 * rest;
  const bool up =
      twice > (double)s || (twice == (double)s && ((unsigned)n & 1));
  return up && n < 15.f ? n + 1.f : n;
}

// 64 bits to 32, kept as a step of its own: the compiler would join it with a
// rounding to fp16 that follows, and differ from the plain form where the two
// roundings do.
__device__ __forceinline__ float to_32(double x) {
  float f = (float)x;
  asm volatile("" : "+v"(f));
  return f;
}

struct AppendSource {
  const void* x;
  long ss, bs, ns;
};

// Rotated value d of a row, rounded to T. In 64 bits: the codes of a rotated
// key hang on this rounding.
template <typename T>
__device__ __forceinline__ float rotated(const T* x, const float* cos_row,
                                         const float* sin_row, int d, int r,
                                         bool interleaved) {
  if (d >= 2 * r) return DTypeTraits<T>::to_float(x[d]);
  const int j = interleaved ? d >> 1 : (d < r ? d : d - r);
  const bool second = interleaved ? d & 1 : d >= r;
  const int i1 = interleaved ? 2 * j : j;
  const int i2 = interleaved ? 2 * j + 1 : j + r;
  const double x1 = DTypeTraits<T>::to_float(x[i1]);
  const double x2 = DTypeTraits<T>::to_float(x[i2]);
  const double c = cos_row[j], s = sin_row[j];
  const double y = second ? x2 * c + x1 * s : x1 * c - x2 * s;
  return DTypeTraits<T>::to_float(DTypeTraits<T>::from_float(to_32(y)));
}

template <typename T>
union Eight {
  uint4 u;
  T t[8];
};

// WIDE: all rows lie at multiples of 16 bytes
template <bool WIDE, typename T>
__device__ __forceinline__ void load_eight(Eight<T>& v, const T* x) {
  if constexpr (WIDE) {
    v.u = *(const uint4*)x;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v.t[i] = x[i];
  }
}

// All loads are on their way before any is waited for: left to itself the
// compiler takes the first one apart before it asks for the next.
template <typename T>
__device__ __forceinline__ void hold_all(Eight<T>& a, Eight<T>& b, long& t) {
  asm volatile(""
               : "+v"(a.u.x), "+v"(a.u.y), "+v"(a.u.z), "+v"(a.u.w),
                 "+v"(b.u.x), "+v"(b.u.y), "+v"(b.u.z), "+v"(b.u.w),
                 "+v"(t));
}

template <typename T>
__device__ __forceinline__ void to_floats(float (&y)[8], const Eight<T>& v) {
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = DTypeTraits<T>::to_float(v.t[i]);
}

// Four lanes hold a group's 32 values: codes in the order of the values, and
// its scale and zero point. A NaN counts as 0.
struct Held {
  float code[8];
  __half scale, zero;
  bool nan;  // in the group
};

// v of the lane's neighbour in its group of four, 1 or 2 lanes off
template <int OFF>
__device__ __forceinline__ float beside(float v) {
  constexpr int kOrder = OFF == 1 ? 0xb1 : 0x4e;  // 1 0 3 2 and 2 3 0 1
  const int i = __float_as_int(v);
  return __int_as_float(
      __builtin_amdgcn_update_dpp(i, i, kOrder, 0xf, 0xf, true));
}

// of three values without a NaN, as they are: fminf would settle signalling
// ones first
__device__ __forceinline__ float least(float a, float b, float c) {
  float y;
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(y) : "v"(a), "v"(b), "v"(c));
  return y;
}

__device__ __forceinline__ float most(float a, float b, float c) {
  float y;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(y) : "v"(a), "v"(b), "v"(c));
  return y;
}

__device__ __forceinline__ Held hold_eight(const float (&x)[8]) {
  Held y;
  float v[8];
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = x[i];
    odd |= !(fabsf(x[i]) <= kHeldMax);
  }
  y.nan = false;
  if (__any(odd)) {
    int nan = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      nan |= x[i] != x[i];
      v[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -kHeldMax), kHeldMax);
    }
    nan |= __shfl_xor(nan, 1, WAVE_SIZE);
    nan |= __shfl_xor(nan, 2, WAVE_SIZE);
    y.nan = nan;
  }
  float low = least(v[0], v[1], v[2]), high = most(v[0], v[1], v[2]);
  low = least(least(low, v[3], v[4]), v[5], v[6]);
  high = most(most(high, v[3], v[4]), v[5], v[6]);
  low = least(low, v[7], v[7]), high = most(high, v[7], v[7]);
  float other = beside<1>(low);
  low = least(low, other, other);
  other = beside<2>(low);
  low = least(low, other, other);
  other = beside<1>(high);
  high = most(high, other, other);
  other = beside<2>(high);
  high = most(high, other, other);
  y.zero = __float2half(low);
  const float z = __half2float(y.zero);
  // 32 bits settle the scale where what they may be off by, 3 * 2^-24 of it,
  // crosses no border of 16 bits
  const float about = (high - z) * (1.f / 15.f);
  y.scale = __float2half(about * (1.f - 0x1p-22f));
  const __half above = __float2half(about * (1.f + 0x1p-22f));
  if (__any(__half_as_ushort(y.scale) != __half_as_ushort(above)))
    y.scale = __float2half(to_32(((double)high - (double)z) / 15.0));
  const float s = __half2float(y.scale);
  const float inv = s > 0.f ? __builtin_amdgcn_rcpf(s) : 0.f;
  // In 32 bits a quotient is off by 16 * 4 * 2^-24 where it is up to 16 (the
  // difference, the reciprocal's two and the product's rounding); nearer to a
  // border than twice that, products in 64 bits decide.
  constexpr float kNear = 0.5f - 1e-5f;
  float off[8], far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = (v[i] - z) * inv;
    const float whole = rintf(q);
    off[i] = q - whole;
    y.code[i] = __builtin_amdgcn_fmed3f(whole, 0.f, 15.f);
  }
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    asm("v_max3_f32 %0, %0, |%1|, |%2|"
        : "+v"(far)
        : "v"(off[i]), "v"(off[i + 1]));
  if (__any(far > kNear)) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (fabsf(off[i]) > kNear && s > 0.f)
        y.code[i] = code_between(v[i], z, s, inv);
  }
  return y;
}

// Four codes in 16 bits, the first one lowest.
__device__ __forceinline__ unsigned four_codes(float a, float b, float c,
                                               float d) {
  return (unsigned)fmaf(fmaf(fmaf(d, 16.f, c), 16.f, b), 16.f, a);
}

// Codes of a key's word and of a value's, in the cache's order.
__device__ __forceinline__ unsigned key_word(const Held& y) {
  const float* c = y.code;
  return four_codes(c[0], c[2], c[4], c[6]) |
         four_codes(c[1], c[3], c[5], c[7]) << 16;
}

__device__ __forceinline__ unsigned value_word(const Held& y) {
  const float* c = y.code;
  return four_codes(c[0], c[1], c[2], c[3]) |
         four_codes(c[4], c[5], c[6], c[7]) << 16;
}

// v of any of the row's lanes
template <int LANES>
__device__ __forceinline__ bool row_any(bool v) {
  if (!__any(v)) return false;
  int y = v;
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) y |= __shfl_xor(y, o, WAVE_SIZE);
  return y;
}

// The scales and zero points of a row's groups, by the first lane of each; the
// row is `token` tokens from the view's first.
template <int H>
__device__ __forceinline__ void store_scales(const CacheView& cache,
                                             const HeadView<H>& to,
                                             unsigned token, int part,
                                             const Held& k, const Held& v,
                                             bool nan_row) {
  if (part & 3) return;
  const __half nan = __ushort_as_half(0x7e00);
  const int group = part / 4;
  const __half2 m = {nan_row ? nan : k.scale, k.zero};
  to.k_meta[token * (H / kGroup) + group] = m;
  __half* w =
      to.v_meta + Pieces<H>::scale_at(cache, to.first + token, group);
  w[0] = v.nan ? nan : v.scale;
  w[4] = v.zero;
}

// A prompt: a wave takes 512 / h neighbouring positions of one head, aligned
// to as many, h / 8 lanes and 8 values a lane for each, so that the pairs of
// tokens that share words of v_codes meet in a wave and all stores are whole
// words next to each other. 4 x 2047 tokens of 8 heads of 128 take 14 to 15 us
// (21 with the head size known at run time only, the borders of codes looked
// at one by one and the value's load behind the key's; 41 with a row's lanes
// anywhere and pieces of 16 bits). 44 MB are read and written, 9 us at a
// copy's rate, and 355 instructions a wave, mostly the choice of codes, issue
// for about as long. Both would fit side by side; but a wave loads, computes
// and stores once and waits half of its cycles.
template <typename T, int H, bool WIDE>
__global__ __launch_bounds__(256) void append_kernel(CacheView cache,
                                                     AppendSource k,
                                                     AppendSource v,
                                                     Start start, long s,
                                                     unsigned tiles) {
  constexpr int lanes = H / 8, per = 64 / lanes;
  const int lane = threadIdx.x & 63;
  const int part = lane & (lanes - 1), d0 = part * 8;
  const unsigned wave =
      blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned row = wave / tiles;
  if (row >= (unsigned)cache.b * cache.heads) return;
  const long bh = row;
  const int ib = row / (unsigned)cache.heads;
  const int head = row - ib * cache.heads;
  const long t = start.of(ib);
  if (t < 0) return;  // idle
  // positions from the begin's tile on
  const long base = (t & -per) + (long)(wave - row * tiles) * per;
  if (base >= cache.capacity) return;
  const int token = lane / lanes;
  const long is0 = base - t, is = is0 + token;
  const bool real = is >= 0 && is < s && base + token < cache.capacity;
  Eight<T> k_raw, v_raw;
  k_raw.u = v_raw.u = make_uint4(0, 0, 0, 0);
  if (real) {
    const T* kp = (const T*)k.x + is0 * k.ss + ib * k.bs + head * k.ns;
    const T* vp = (const T*)v.x + is0 * v.ss + ib * v.bs + head * v.ns;
    load_eight<WIDE>(k_raw, kp + (token * k.ss + d0));
    load_eight<WIDE>(v_raw, vp + (token * v.ss + d0));
  }
  long unused = 0;
  hold_all(k_raw, v_raw, unused);
  float kx[8], vx[8];
  to_floats(kx, k_raw);
  to_floats(vx, v_raw);
  const Held hk = hold_eight(kx), hv = hold_eight(vx);
  const bool nan_row = row_any<lanes>(hk.nan || hv.nan);

  const HeadView<H> to(cache, bh, base);
  const unsigned place = to.first + token;  // from a block of four on
  if (real) {
    to.k_codes[lane] = key_word(hk);
    store_scales<H>(cache, to, token, part, hk, hv, nan_row);
  }
  const unsigned own = value_word(hv);
  const unsigned other = __shfl_xor(own, lanes, WAVE_SIZE);
  const int other_real = __shfl_xor((int)real, lanes, WAVE_SIZE);
  const bool both = real && other_real;
  if (H < 64) {  // a piece has two values
    if (real)
      for (int i = 0; i < 4; ++i)
        to.v_codes[Pieces<H>::at(place, d0 + 2 * i)] = (own >> (8 * i)) & 255;
  } else if (both) {  // one word of two pieces for either token's lane
    const bool odd = place & 1;
    const unsigned word = odd ? (other >> 16) | (own & 0xffff0000u)
                              : (own & 0xffffu) | (other << 16);
    *(unsigned*)(to.v_codes +
                 Pieces<H>::at(place & ~1u, d0 + (odd ? 4 : 0))) = word;
  } else if (real) {
    to.v_codes[Pieces<H>::at(place, d0)] = (unsigned short)own;
    to.v_codes[Pieces<H>::at(place, d0 + 4)] = (unsigned short)(own >> 16);
  }
}

// A decode step: a row (token, sequence, head) takes h / 8 lanes with 8 values
// each. Rows of q come behind those of k and v and are only rotated. 16 tokens
// of 32 query and 8 key heads take 5.0 us, one way to memory after another
// (position, table) and the rotation's 64-bit steps; 6.2 where loads wait for
// each other and arguments come by the lane, 10 with values one by one.
template <typename T, int H, bool WIDE>
__global__ __launch_bounds__(256) void append_rotated_kernel(
    CacheView cache, AppendSource k, AppendSource v, AppendSource q,
    T* __restrict__ q_out, int n, const float* __restrict__ cos_t,
    const float* __restrict__ sin_t, int r, long table_rows, bool interleaved,
    Start start, long s) {
  constexpr int lanes = H / 8;
  const unsigned index = blockIdx.x * 256 + threadIdx.x;
  const unsigned row = index / (unsigned)lanes;
  const int part = index & (lanes - 1), d0 = part * 8;
  const unsigned kv_rows = (unsigned)s * cache.b * cache.heads;
  const unsigned rows = kv_rows + (unsigned)s * cache.b * n;
  if (row >= rows) return;
  const bool is_q = row >= kv_rows;
  const unsigned heads = is_q ? n : cache.heads;
  const unsigned local = is_q ? row - kv_rows : row;
  const unsigned token = local / heads;
  const int head = local - token * heads;
  const int is = token / (unsigned)cache.b;
  const int ib = token - is * cache.b;
  const T* x = (const T*)(is_q ? q.x : k.x) + is * (is_q ? q.ss : k.ss) +
               ib * (is_q ? q.bs : k.bs) + head * (is_q ? q.ns : k.ns);
  float own[8], vx[8], pair[8], c[8], sn[8];
  Eight<T> raw, v_raw;
  // a row of q loads itself again, so that no branch parts the loads
  const T* vx_row = is_q ? x
                         : (const T*)v.x + is * v.ss + ib * v.bs + head * v.ns;
  long t = start.of(ib);
  load_eight<WIDE>(raw, x + d0);
  load_eight<WIDE>(v_raw, vx_row + d0);
  hold_all(raw, v_raw, t);
  const bool idle = t < 0;
  to_floats(own, raw);
  to_floats(vx, v_raw);
  const long pos = t + is;
  const bool known = !idle && pos < table_rows;

  // Rotation in 64 bits, rounded to T: the codes of a rotated key hang on it.
  // A lane's values lie before or behind their partners, or are a pair's both.
  const bool turns = d0 < 2 * r;
  if (turns && known) {
    const float* cos_row = cos_t + pos * r;
    const float* sin_row = sin_t + pos * r;
    if (interleaved || r % 8 == 0) {
      const bool behind = !interleaved && d0 >= r;
      const int j0 = interleaved ? d0 / 2 : behind ? d0 - r : d0;
      const int turned = interleaved ? 4 : 8;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < turned && j0 + i < r) {
          c[i] = cos_row[j0 + i];
          sn[i] = sin_row[j0 + i];
        }
      if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (j0 + i >= r) break;
          const double x1 = own[2 * i], x2 = own[2 * i + 1];
          const double y1 = x1 * c[i] - x2 * sn[i];
          const double y2 = x2 * c[i] + x1 * sn[i];
          own[2 * i] = to_32(y1);
          own[2 * i + 1] = to_32(y2);
        }
      } else {
        load_eight<WIDE>(raw, x + (behind ? d0 - r : d0 + r));
        to_floats(pair, raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double a = (double)own[i] * c[i];
          const double b = (double)pair[i] * sn[i];
          own[i] = to_32(behind ? a + b : a - b);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        own[i] = DTypeTraits<T>::to_float(DTypeTraits<T>::from_float(own[i]));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        own[i] = rotated<T>(x, cos_row, sin_row, d0 + i, r, interleaved);
    }
  } else if (turns) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d0 + i < 2 * r) own[i] = NAN;
  }

  if (is_q) {
    Eight<T> y;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y.t[i] = DTypeTraits<T>::from_float(idle ? 0.f : own[i]);
    *(uint4*)(q_out + (long)local * H + d0) = y.u;
    return;
  }
  const bool real = !idle && pos < cache.capacity;  // of the whole row
  const Held hk = hold_eight(own), hv = hold_eight(vx);
  const bool nan_row = row_any<lanes>(hk.nan || hv.nan);
  if (!real) return;
  const HeadView<H> to(cache, (long)ib * cache.heads + head, pos);
  to.k_codes[part] = key_word(hk);
  store_scales<H>(cache, to, 0, part, hk, hv, nan_row);
  const unsigned word = value_word(hv);
  if (H >= 64) {
    to.v_codes[Pieces<H>::at(to.first, d0)] = (unsigned short)word;
    to.v_codes[Pieces<H>::at(to.first, d0 + 4)] =
        (unsigned short)(word >> 16);
  } else {  // a piece has two values
    for (int i = 0; i < 4; ++i)
      to.v_codes[Pieces<H>::at(to.first, d0 + 2 * i)] =
          (word >> (8 * i)) & 255;
  }
}

// Reads back with the same lanes as append_kernel; positions outside the cache
// read as NaN. 4 x 2047 tokens of 8 heads of 128 take 8.3 us, 5.3 TB/s (11.4
// with the head size known at run time only, 48 with a thread for a value).
template <typename T, int H>
__global__ __launch_bounds__(256) void dequantize_kernel(
    CacheView cache, Start start, long length, unsigned tiles,
    T* __restrict__ k_out, T* __restrict__ v_out) {
  constexpr int lanes = H / 8, per = 64 / lanes;
  const int lane = threadIdx.x & 63;
  const int part = lane & (lanes - 1), d0 = part * 8;
  const unsigned wave =
      blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned row = wave / tiles;
  if (row >= (unsigned)cache.b * cache.heads) return;
  const long bh = row;
  const int ib = row / (unsigned)cache.heads;
  const int head = row - ib * cache.heads;
  const long t = start.of(ib);
  // positions from the begin's tile on, rounded down also where it is negative
  const long base = (t & -per) + (long)(wave - row * tiles) * per;
  const int token = lane / lanes;
  const long is0 = base - t, is = is0 + token, pos = base + token;
  if (is < 0 || is >= length) return;
  Eight<T> ky, vy;
  if (pos >= 0 && pos < cache.capacity) {
    const HeadView<H> from(cache, bh, base);
    const unsigned place = from.first + token;
    const int group = part / 4;
    const unsigned kw = from.k_codes[lane];
    const __half2 km = from.k_meta[token * (H / kGroup) + group];
    unsigned vw = 0;
    if (H >= 64) {
      vw = from.v_codes[Pieces<H>::at(place, d0)] |
           (unsigned)from.v_codes[Pieces<H>::at(place, d0 + 4)] << 16;
    } else {
      for (int i = 0; i < 4; ++i)
        vw |= (from.v_codes[Pieces<H>::at(place, d0 + 2 * i)] & 255u)
              << (8 * i);
    }
    const __half* vm =
        from.v_meta + Pieces<H>::scale_at(cache, place, group);
    const float ks = __half2float(km.x), kz = __half2float(km.y);
    const float vs = __half2float(vm[0]), vz = __half2float(vm[4]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ky.t[i] = DTypeTraits<T>::from_float(
          fmaf(ks, (float)((kw >> ((i >> 1) * 4 + (i & 1) * 16)) & 15), kz));
      vy.t[i] = DTypeTraits<T>::from_float(
          fmaf(vs, (float)((vw >> (i * 4)) & 15), vz));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      ky.t[i] = vy.t[i] = DTypeTraits<T>::from_float(NAN);
  }
  const long at0 = ((is0 * cache.b + ib) * cache.heads + head) * H;
  const long at = token * ((long)cache.b * cache.heads * H) + d0;
  *(uint4*)(k_out + at0 + at) = ky.u;
  *(uint4*)(v_out + at0 + at) = vy.u;
}

// ---------------------------------------------------------------------------
// Attention. A workgroup of four waves takes up to 16 MT query rows (heads of
// one key head x new tokens) and a share of the tokens; each wave takes every
// fourth tile of 32 tokens and keeps a running maximum, sum and output of its
// own, joined through LDS at the end, and across workgroups by a second
// kernel. Per tile, with g = lane / 16 and r = lane % 16:
//
//   S^T = K Q^T: the codes of token r and the head's quarter g come as one
//       load, become fp16 in registers and are the A operand; S^T leaves the
//       matrix core with query row r and tokens 4g + i in each lane.
//   O^T += V^T P^T: that is just the layout of the B operand P^T, if the
//       contraction runs over tokens in the order 4g + i of the tile's first
//       half, then of its second; the cache holds values in that order. No
//       value crosses lanes but in the rare update of the maximum.
//
// Codes become fp16 by or-ing them into 1024 + code, which is exact, and one
// rounded multiply-add by the group's scale and zero point. Query rows are
// brought to a maximum in [1, 2) by a power of two first, so that bf16 values
// are exact in fp16 too. Sums and statistics are held in 32 bits.
//
// For a bf16 output held keys, held values and weights are operands in fp16,
// each rounded by a relative 2^-11 at most, under the output's own 2^-8: three
// bits more than keys and values have in a cache of the model's type. Against
// 64 bits the output is off by 0.0017 of its norm, the plain form by 0.0016 to
// 0.0017; the fp16 path's three products bring the latter and take 54 us for 44
// (32 streams of up to 8192 tokens) and 33 for 26.5 (4 of up to 32768). A
// weight under 2^-21 of the wave's largest is held to 2^-32 of that one
// (kLift), so that n tokens are off by n 2^-32 of the largest value at most.
//
// The rounding of an fp16 output is 2^-11 too, so there (EXACT) what the
// roundings left out is multiplied as well, and the middle of each group,
// z + 8 s, goes through products of its own in two parts: the output is as far
// off as the plain form's (2.1e-4) against 4.4e-4 without.

// What bounds it: turning codes into fp16 takes 208 of the 265 instructions
// that a wave spends on a tile of 5 KB (h = 128). Alone they would take half
// the time that the tiles take to come from memory; with three waves a SIMD
// each hides most of the other. Measured (h = 128, bf16): 32 streams of up to
// 8192 tokens, 8 key heads, 174 MB: 41 to 48 us, 3.6 to 4.2 TB/s; 4 streams of
// up to 32768, 105 MB: 26 to 31 us. Loads alone take 29 and 22 of those.

using h2 = __attribute__((ext_vector_type(2))) _Float16;
using h8 = __attribute__((ext_vector_type(8))) _Float16;
using f4 = __attribute__((ext_vector_type(4))) float;

constexpr int kTile = 32;       // tokens of a wave's step
constexpr int kLeast = 128;     // tokens of a workgroup at least
constexpr float kUnset = -3e38f;  // maximum before the first score
// Weights are 2^(score - m) with m = the running maximum - kLift, and m stays
// until a score passes it by kLift + kSlack: they reach 2^15, just under fp16's
// largest, so that small ones keep what fp16 has under the largest.
constexpr float kLift = 7.f, kSlack = 8.f;

struct AttentionArgs {
  CacheView cache;
  const void* q;
  long q_ss, q_bs, q_ns;
  void* out;
  float* part_o;   // [b * heads, chunks, rows, H], unless chunks == 1
  float* part_ml;  // [b * heads, chunks, rows, 2]
  int n, rep, rows, q_blocks, chunks, groups;
  int* part_per;  // tiles of a chunk
  float scale_log2e;
  long window, sinks;
  Start start;
  bool q_wide;  // rows of q lie at multiples of 16 bytes
};

// The tiles that some row of [first, last] of a sequence sees: those of the
// sinks, then those from the window's begin to the last row's position.
struct Tiles {
  int sink, low, count;
  __device__ __forceinline__ int at(int i) const {
    return i < sink ? i : low + i - sink;
  }
};

__device__ __forceinline__ Tiles tiles_of(const AttentionArgs& a, long t0,
                                          int first_row, int last_row) {
  Tiles t{0, 0, 0};
  if (t0 < 0 || t0 >= a.cache.capacity) return t;
  const int last = (int)min(t0 + (unsigned)last_row / (unsigned)a.rep,
                            a.cache.capacity - 1);
  if (a.window > 0) {
    const long low =
        max(0l, t0 + (unsigned)first_row / (unsigned)a.rep - a.window + 1);
    t.low = (int)(low / kTile);
    t.sink = (int)min((a.sinks + kTile - 1) / kTile, (long)t.low);
  }
  t.count = t.sink + max(0, last / kTile + 1 - t.low);
  return t;
}

// Sums over the wave by row shifts and broadcasts: lane i gets that of the
// lanes up to i.
__device__ __forceinline__ int wave_scan(int v) {
#define SCAN_STEP(CTRL, ROWS) \
  v += __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false)
  SCAN_STEP(0x111, 0xf);  // from 1, 2, 4, 8 lanes below, within 16
  SCAN_STEP(0x112, 0xf);
  SCAN_STEP(0x114, 0xf);
  SCAN_STEP(0x118, 0xf);
  SCAN_STEP(0x142, 0xa);  // from the last lane of the 16 below
  SCAN_STEP(0x143, 0xc);  // from lane 31
#undef SCAN_STEP
  return v;
}

__device__ __forceinline__ int wave_total(int v) {
  return __builtin_amdgcn_readlane(wave_scan(v), 63);
}

// The largest of the wave's numbers, none of them negative.
__device__ __forceinline__ int wave_most(int v) {
#define MOST_STEP(CTRL, ROWS) \
  v = max(v, __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false))
  MOST_STEP(0x111, 0xf);
  MOST_STEP(0x112, 0xf);
  MOST_STEP(0x114, 0xf);
  MOST_STEP(0x118, 0xf);
  MOST_STEP(0x142, 0xa);
  MOST_STEP(0x143, 0xc);
#undef MOST_STEP
  return __builtin_amdgcn_readlane(v, 63);
}

// A workgroup's share of the tokens, settled from where the sequences end:
// each share has `per` tiles, a multiple of what four waves take at once, and
// `per` is about the least with which the shares of all sequences are no more
// than `groups`. They are numbered without gaps: workgroups that end at once
// between others would leave some of the card's engines with more than they
// hold and others idle, since they are dealt out in turn.
struct Share {
  int per, ib, chunk;  // ib < 0: none
};

__device__ __forceinline__ Share share_of(const AttentionArgs& a, int index) {
  const int lane = threadIdx.x & 63;
  auto tiles_in = [&](int ib) {
    return ib < a.cache.b ? tiles_of(a, a.start.of(ib), 0, a.rows - 1).count
                          : 0;
  };
  const int first = tiles_in(lane);
  auto total_of = [&](auto f) {
    int t = f(first);
    for (int ib = lane + 64; ib < a.cache.b; ib += 64) t += f(tiles_in(ib));
    return wave_total(t);
  };
  int longest = first;
  for (int ib = lane + 64; ib < a.cache.b; ib += 64)
    longest = max(longest, tiles_in(ib));
  longest = wave_most(longest);
  const int total = total_of([](int n) { return n; });
  int per = max(kLeast / kTile, max((total + a.groups - 1) / a.groups,
                                    (longest + a.chunks - 1) / a.chunks));
  per = (per + 3) & ~3;
  auto shares = [&](int n) {
    return (int)(((unsigned)n + per - 1) / (unsigned)per);
  };
  // there are at least twice as many groups as sequences, so this ends
  while (total_of(shares) > a.groups) per += max(4, per / 8 & ~3);
  Share s{per, -1, 0};
  int before = 0;
  for (int low = 0; low < a.cache.b; low += 64) {
    const int own = shares(low ? tiles_in(low + lane) : first);
    const int upto = before + wave_scan(own);
    const unsigned long after = __ballot(upto > index);
    if (after) {
      const int at = __builtin_ctzl(after);
      s.ib = low + at;
      s.chunk = index - __builtin_amdgcn_readlane(upto - own, at);
      break;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return s;
}

template <int WORDS>
__device__ __forceinline__ void load_words(unsigned (&w)[WORDS],
                                           const void* p) {
  if constexpr (WORDS == 1) {
    w[0] = *(const unsigned*)p;
  } else if constexpr (WORDS == 2) {
    const uint2 v = *(const uint2*)p;
    w[0] = v.x, w[1] = v.y;
  } else {
    for (int i = 0; i < WORDS; i += 4) {
      const uint4 v = ((const uint4*)p)[i / 4];
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  }
}

__device__ __forceinline__ h2 as_h2(unsigned u) {
  return __builtin_bit_cast(h2, u);
}

// The four pairs of codes in a word as values scale * code + zero; with EXACT
// as scale * (code - 8), which takes 15 bits: rounded, and what that left out.
template <bool EXACT>
__device__ __forceinline__ void pairs_of(h2 (&y)[4], h2 (&left)[4],
                                         unsigned word, h2 scale, h2 zero,
                                         unsigned exponent) {
  const unsigned up = word >> 8, e = exponent;
  constexpr float kOff = EXACT ? 8.f : 0.f;
  const h2 big = {(_Float16)(1024 + kOff), (_Float16)(1024 + kOff)};
  const h2 part = {(_Float16)0.0625, (_Float16)0.0625};
  const h2 less = {(_Float16)(-64 - kOff), (_Float16)(-64 - kOff)};
  const h2 x[4] = {
      as_h2((word & 0x000f000fu) | e) - big,
      __builtin_elementwise_fma(as_h2((word & 0x00f000f0u) | e),
                                part, less),
      as_h2((up & 0x000f000fu) | e) - big,
      __builtin_elementwise_fma(as_h2((up & 0x00f000f0u) | e), part,
                                less)};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (EXACT) {
      y[j] = x[j] * scale;
      left[j] = __builtin_elementwise_fma(x[j], scale, -y[j]);
    } else {
      y[j] = __builtin_elementwise_fma(x[j], scale, zero);
    }
  }
}

__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) {
  return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

template <int H>
struct HeadShape {
  static constexpr int kWords = H / 32;     // dwords of keys in a lane
  static constexpr int kKeyGroups = H >= 256 ? H / 128 : 1;
  static constexpr int kQuarters = H >= 64 ? H / 64 : 1;
  static constexpr int kValueWords = 2 * kQuarters;  // for four tokens
  static constexpr int kBlocks = H / 16;    // of 16 output values
  static constexpr int kGroups = H / kGroup;
};

// what a lane holds of a tile: two halves of 16 tokens
template <int H>
struct TileRegs {
  using S = HeadShape<H>;
  unsigned k[2][S::kWords], km[2][S::kKeyGroups];
  unsigned v[2][S::kValueWords], vm[2][4];
};

// A tile in LDS: its keys' codes, its values' codes, its keys' scales, its
// values' scales, each as in memory. It comes straight from memory, so that
// tiles in flight take no registers.
template <int H>
struct TileLds {
  using S = HeadShape<H>;
  static constexpr int kV = kTile * H / 2;
  static constexpr int kKm = kV + 1024 * S::kQuarters;
  static constexpr int kVm = kKm + 128 * S::kGroups;
  static constexpr int kBytes = kVm + 128 * S::kGroups;
  static constexpr int kLoads = (kTile * H / 2 + 1023) / 1024 +
                                S::kQuarters + (S::kGroups > 4 ? 2 : 1);
};

// 16 bytes a lane from memory to LDS at `to` + 16 lane. Not known to the
// compiler as a load: wait_loads() is what orders it. The second form reads
// at a uniform address + `offset` of the lane; STEP counts for both sides. (A
// scalar address that a vector instruction wrote may be read by a load after
// five cycles, m0 after one: the waits are here, since the compiler does not
// look into the block.)
__device__ __forceinline__ void load_to_lds(unsigned to, const void* from) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off"
      :
      : "s"(to), "v"(from)
      : "memory", "m0");
}

template <int STEP>
__device__ __forceinline__ void load_to_lds(unsigned to, const void* from,
                                            unsigned offset) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 4\n\t"
      "global_load_lds_dwordx4 %1, %2 offset:%3"
      :
      : "s"(to), "v"(offset), "s"(from), "n"(STEP)
      : "memory", "m0");
}

template <int STEPS>
__device__ __forceinline__ void load_steps(unsigned to, const void* from,
                                           unsigned offset) {
  if constexpr (STEPS >= 1) load_to_lds<0>(to, from, offset);
  if constexpr (STEPS >= 2) load_to_lds<1 * 1024>(to, from, offset);
  if constexpr (STEPS >= 3) load_to_lds<2 * 1024>(to, from, offset);
  if constexpr (STEPS >= 4) load_to_lds<3 * 1024>(to, from, offset);
}

template <int LEFT>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LEFT) : "memory");
}

struct HeadMemory {
  const unsigned char *k_codes, *v_codes;
  const __half *k_meta, *v_meta;  // v_meta: of group 0
  long meta_stride;               // from group to group of v_meta
};

template <int H>
__device__ __forceinline__ void fetch_tile(unsigned to, const HeadMemory& m,
                                           long tile, int lane) {
  using S = HeadShape<H>;
  using L = TileLds<H>;
  const unsigned char* k = m.k_codes + tile * kTile * (H / 2);
  const unsigned char* v = m.v_codes + tile * (kTile / 4) * 128 * S::kQuarters;
  const __half* km = m.k_meta + tile * kTile * S::kGroups * 2;
  const __half* vm = m.v_meta + tile * (kTile / 4) * 8;
  if (H >= 64 || lane < 32)
    load_steps<(kTile * H / 2 + 1023) / 1024>(to, k, lane * 16);
  load_steps<S::kQuarters>(to + L::kV, v, lane * 16);
  constexpr int kLanes = 8 * S::kGroups;  // 16 bytes each
  const int j = lane - (kLanes < 64 ? kLanes : 0);
  const __half* vm_lane = vm + (j >> 3) * m.meta_stride + (j & 7) * 8;
  if constexpr (kLanes < 64) {  // both kinds of scales in one load
    if (lane < 2 * kLanes)
      load_to_lds(to + L::kKm, lane < kLanes ? km + lane * 8 : vm_lane);
  } else {
    load_to_lds(to + L::kKm, km + lane * 8);
    load_to_lds(to + L::kVm, vm_lane);
  }
}

template <int H>
__device__ __forceinline__ void read_tile(TileRegs<H>& t,
                                          const unsigned char* from,
                                          int lane) {
  using S = HeadShape<H>;
  using L = TileLds<H>;
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    load_words(t.k[half], from + (half * 16 + r) * (H / 2) + g * (H / 8));
    load_words(t.km[half],
               from + L::kKm + ((half * 16 + r) * S::kGroups +
                                g * (H / 4) / kGroup) * 4);
    load_words(t.v[half], from + L::kV +
                              ((half * 4 + g) * 16 + r) * 8 * S::kQuarters);
    load_words(t.vm[half], from + L::kVm +
                               ((r * S::kBlocks / kGroup) * 8 + half * 4 + g) *
                                   16);
  }
}

template <typename T, int H, int MT>
__global__ __launch_bounds__(256, MT * H <= 128 ? 3 : MT * H <= 256 ? 2 : 1)
void attention_kernel(AttentionArgs a) {
  using S = HeadShape<H>;
  using L = TileLds<H>;
  constexpr int kAhead = 2;  // tiles in flight or in use, per wave
  constexpr bool kExact = std::is_same_v<T, __half>;
  __shared__ h8 q_lds[MT][S::kWords][64];
  __shared__ h8 sum_lds[kExact ? MT : 1][64];  // of q, in two parts
  __shared__ float c_lds[MT][16];
  __shared__ float ml_lds[MT][4][16][2], row_lds[MT][16][2];
  // the waves' tiles, and once those are used up their outputs
  constexpr int kTogether = MT * H <= 256 ? MT : 1;
  constexpr int kRing = 4 * kAhead * L::kBytes;
  constexpr int kOut = kTogether * 4 * 16 * (H + 1) * 4;
  __shared__ __align__(16) unsigned char ring[kRing > kOut ? kRing : kOut];
  float(*o_lds)[16][H + 1] = (float(*)[16][H + 1])ring;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;

  // workgroups that share tokens are 8 apart: they run on the same die, whose
  // second level cache holds the tokens between them
  const unsigned x = blockIdx.x & 7, rest = blockIdx.x >> 3;
  const int block = rest % (unsigned)a.q_blocks;
  const unsigned work = rest / (unsigned)a.q_blocks * 8 + x;
  const unsigned index = work / (unsigned)a.cache.heads;
  const int kv_head = work % (unsigned)a.cache.heads;
  Share share{0, (int)index, 0};
  if (a.chunks > 1) {
    share = share_of(a, index);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.part_per = share.per;
    if (share.ib < 0) return;
  } else if (index >= (unsigned)a.cache.b) {
    return;
  }
  const int ib = share.ib, chunk = share.chunk;
  const long bh = (long)ib * a.cache.heads + kv_head;
  const int row0 = block * 16 * MT;
  const int row1 = min(a.rows, row0 + 16 * MT) - 1;
  const long t0 = a.start.of(ib);
  const Tiles tiles = tiles_of(a, t0, row0, row1);
  const int i_low = chunk * share.per;
  const int i_high =
      a.chunks > 1 ? min(tiles.count, i_low + share.per) : tiles.count;
  if (i_low >= i_high && a.chunks > 1) return;  // the join leaves it out

  const HeadMemory memory{
      a.cache.k_codes + bh * a.cache.room * (H / 2),
      a.cache.v_codes + bh * (a.cache.room / 4) * 128 * S::kQuarters,
      a.cache.k_meta + bh * a.cache.room * S::kGroups * 2,
      a.cache.v_meta + bh * a.cache.room * S::kGroups * 2,
      a.cache.room * 2};
  const unsigned char* mine = ring + wave * kAhead * L::kBytes;
  const unsigned mine_at =
      (unsigned)(unsigned long)(__attribute__((address_space(3)))
                                const unsigned char*)mine;
  int i = i_low + wave;
#pragma unroll
  for (int ahead = 0; ahead < kAhead; ++ahead)
    if (i + 4 * ahead < i_high)
      fetch_tile<H>(mine_at + ahead * L::kBytes, memory,
                    tiles.at(i + 4 * ahead), lane);

  // a negative scale goes to the query, so that the largest product of a row
  // is its largest score
  const float sign = a.scale_log2e < 0.f ? -1.f : 1.f;
  for (int mt = wave; mt < MT; mt += 4) {
    // behind the last row that one again (it is not put out): no branch parts
    // the loads
    const int row = min(row0 + mt * 16 + r, a.rows - 1);
    float v[H / 4], peak = 0.f;
    const unsigned token = (unsigned)row / (unsigned)a.rep;
    const T* q = (const T*)a.q + (long)token * a.q_ss + ib * a.q_bs +
                 (long)(kv_head * a.rep + row - token * a.rep) * a.q_ns +
                 g * (H / 4);
    if (a.q_wide) {
#pragma unroll
      for (int i = 0; i < H / 4; i += 8) {
        union {
          uint4 u;
          T t[8];
        } y;
        y.u = *(const uint4*)(q + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i + e] = DTypeTraits<T>::to_float(y.t[e]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < H / 4; ++i)
        v[i] = DTypeTraits<T>::to_float(q[i]);
    }
#pragma unroll
    for (int i = 0; i < H / 4; ++i) peak = fmaxf(peak, fabsf(v[i]));
    peak = fmaxf(peak, __shfl_xor(peak, 16, WAVE_SIZE));
    peak = fmaxf(peak, __shfl_xor(peak, 32, WAVE_SIZE));
    const int e =
        peak > 0.f && peak < INFINITY ? __builtin_amdgcn_frexp_expf(peak) - 1
                                      : 0;
    float sum[S::kKeyGroups] = {};
#pragma unroll
    for (int w = 0; w < S::kWords; ++w) {
      h8 y;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = (_Float16)__builtin_amdgcn_ldexpf(v[w * 8 + i] * sign, -e);
        sum[w * S::kKeyGroups / S::kWords] += (float)y[i];
      }
      q_lds[mt][w][lane] = y;
    }
    if constexpr (kExact) {
      h8 y = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < S::kKeyGroups; ++i) {
        const _Float16 high = (_Float16)sum[i];
        y[3 * i] = y[3 * i + 1] = high;
        y[3 * i + 2] = (_Float16)(sum[i] - (float)high);
      }
      sum_lds[mt][lane] = y;
    }
    if (g == 0)
      c_lds[mt][r] = fmaxf(
          __builtin_amdgcn_ldexpf(fabsf(a.scale_log2e), e), 1e-37f);
  }
  __syncthreads();

  float c[MT], m[MT], l[MT];
  long pos[MT];
  f4 o[MT][S::kBlocks], mid[MT];  // mid: the groups' middles' part
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    c[mt] = c_lds[mt][r];
    m[mt] = kUnset;
    l[mt] = 0.f;
    mid[mt] = f4{0.f, 0.f, 0.f, 0.f};
    pos[mt] = t0 + (row0 + mt * 16 + r) / a.rep;
#pragma unroll
    for (int j = 0; j < S::kBlocks; ++j) o[mt][j] = f4{0.f, 0.f, 0.f, 0.f};
  }
  // whole tiles from here on need a look at each token's place
  const long pos_first = t0 + row0 / a.rep, pos_last = t0 + row1 / a.rep;

  unsigned exponent = 0x64006400u;  // in a register: and + or in one step
  asm("" : "+v"(exponent));
  h8 q_reg[S::kWords];
  if constexpr (MT == 1)
#pragma unroll
    for (int w = 0; w < S::kWords; ++w) q_reg[w] = q_lds[0][w][lane];
  auto q_of = [&](int mt, int w) {
    return MT == 1 ? q_reg[w] : q_lds[mt][w][lane];
  };

  auto step = [&](auto slot_number) {
    constexpr int kSlot = decltype(slot_number)::value;
    const int tile = tiles.at(i);
    if (i + 4 * (kAhead - 1) < i_high)
      wait_loads<(kAhead - 1) * L::kLoads>();
    else
      wait_loads<0>();
    TileRegs<H> now;
    read_tile<H>(now, mine + kSlot * L::kBytes, lane);
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    if (i + 4 * kAhead < i_high)
      fetch_tile<H>(mine_at + kSlot * L::kBytes, memory,
                    tiles.at(i + 4 * kAhead), lane);

    f4 st[MT][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) st[mt][half] = f4{0.f, 0.f, 0.f, 0.f};
      if constexpr (kExact) {
        h8 c8 = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < S::kKeyGroups; ++i) {
          const h2 sz = as_h2(now.km[half][i]);
          const float middle = fmaf(8.f, (float)sz.x, (float)sz.y);
          c8[3 * i] = c8[3 * i + 2] = (_Float16)middle;
          c8[3 * i + 1] = (_Float16)(middle - (float)c8[3 * i]);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          st[mt][half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              c8, sum_lds[mt][lane], st[mt][half], 0, 0, 0);
      }
#pragma unroll
      for (int w = 0; w < S::kWords; ++w) {
        const h2 sz =
            as_h2(now.km[half][w * S::kKeyGroups / S::kWords]);
        h2 y[4], z[4];
        pairs_of<kExact>(y, z, now.k[half][w], h2{sz.x, sz.x},
                         h2{sz.y, sz.y}, exponent);
        const h8 k8 = join(y[0], y[1], y[2], y[3]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          st[mt][half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              k8, q_of(mt, w), st[mt][half], 0, 0, 0);
        if constexpr (kExact) {
          const h8 l8 = join(z[0], z[1], z[2], z[3]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            st[mt][half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                l8, q_of(mt, w), st[mt][half], 0, 0, 0);
        }
      }
    }

    const long t_tile = (long)tile * kTile;
    const bool partly =
        t_tile + kTile - 1 > pos_first ||
        (a.window > 0 && t_tile <= pos_last - a.window);
    h8 p8[MT], p_left[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float sc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) sc[e] = st[mt][e >> 2][e & 3];
      if (partly) {
        // places in the tile, as 32-bit numbers: all fits where it matters
        const int last = (int)min(pos[mt] - t_tile, (long)kTile);
        const int low = a.window > 0
                            ? (int)max(pos[mt] - a.window - t_tile, -1l)
                            : -1;
        const int sink =
            (int)min(max(a.sinks - t_tile, 0l), (long)kTile);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = (e >> 2) * 16 + g * 4 + (e & 3);
          const bool seen = (t <= last) & ((t > low) | (t < sink));
          sc[e] = seen ? sc[e] : -INFINITY;
        }
      }
      float peak = sc[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) peak = fmaxf(peak, sc[e]);
      peak *= c[mt];
      if (__any(peak > m[mt] + (kLift + kSlack))) {
        peak = fmaxf(peak, __shfl_xor(peak, 16, WAVE_SIZE));
        peak = fmaxf(peak, __shfl_xor(peak, 32, WAVE_SIZE));
        const float up = fmaxf(m[mt], peak - kLift);
        const float alpha = __builtin_amdgcn_exp2f(m[mt] - up);
        m[mt] = up;
        l[mt] *= alpha;
#pragma unroll
        for (int j = 0; j < S::kBlocks; ++j) o[mt][j] *= alpha;
        if constexpr (kExact) mid[mt] *= alpha;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w =
            __builtin_amdgcn_exp2f(fmaf(sc[e], c[mt], -m[mt]));
        l[mt] += w;
        p8[mt][e] = (_Float16)w;
        if constexpr (kExact)
          p_left[mt][e] = (_Float16)(w - (float)p8[mt][e]);
      }
    }

    // a NaN group's scale is taken as 0: what sees the token is NaN already
    h2 vs[2][2], vz[2][2];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        vs[half][p] = __builtin_elementwise_max(as_h2(now.vm[half][p]),
                                                h2{0, 0});
        vz[half][p] = as_h2(now.vm[half][2 + p]);
      }
    if constexpr (kExact) {
      h8 high, low;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float middle =
            fmaf(8.f, (float)vs[e >> 2][(e >> 1) & 1][e & 1],
                 (float)vz[e >> 2][(e >> 1) & 1][e & 1]);
        high[e] = (_Float16)middle;
        low[e] = (_Float16)(middle - (float)high[e]);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mid[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(high, p8[mt],
                                                         mid[mt], 0, 0, 0);
        mid[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(high, p_left[mt],
                                                         mid[mt], 0, 0, 0);
        mid[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(low, p8[mt],
                                                         mid[mt], 0, 0, 0);
      }
    }
#pragma unroll
    for (int quarter = 0; quarter < S::kQuarters; ++quarter) {
      h2 y[2][2][4], z[2][2][4];
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          pairs_of<kExact>(y[half][p], z[half][p],
                           now.v[half][p * S::kQuarters + quarter],
                           vs[half][p], vz[half][p], exponent);
#pragma unroll
      for (int j = 0; j < (H >= 64 ? 4 : 2); ++j) {
        const h8 v8 = join(y[0][0][j], y[0][1][j], y[1][0][j], y[1][1][j]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          o[mt][quarter * 4 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              v8, p8[mt], o[mt][quarter * 4 + j], 0, 0, 0);
        if constexpr (kExact) {
          const h8 l8 =
              join(z[0][0][j], z[0][1][j], z[1][0][j], z[1][1][j]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            o[mt][quarter * 4 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                v8, p_left[mt], o[mt][quarter * 4 + j], 0, 0, 0);
            o[mt][quarter * 4 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                l8, p8[mt], o[mt][quarter * 4 + j], 0, 0, 0);
          }
        }
      }
    }
    };
  static_assert(kAhead == 2, "two slots take turns");
  for (; i < i_high; i += 4) {
    step(std::integral_constant<int, 0>());
    i += 4;
    if (i >= i_high) break;
    step(std::integral_constant<int, 1>());
  }

  // join the four waves, as many tiles of rows at a time as LDS has room for
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    float sum = l[mt] + __shfl_xor(l[mt], 16, WAVE_SIZE);
    sum += __shfl_xor(sum, 32, WAVE_SIZE);
    if (g == 0) {
      ml_lds[mt][wave][r][0] = m[mt];
      ml_lds[mt][wave][r][1] = sum;
    }
  }
#pragma unroll
  for (int base = 0; base < MT; base += kTogether) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      const int mt = base + k;
      float top = kUnset, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, ml_lds[mt][w][r][0]);
#pragma unroll
      for (int w = 0; w < 4; ++w)
        sum += ml_lds[mt][w][r][1] *
               __builtin_amdgcn_exp2f(ml_lds[mt][w][r][0] - top);
      if (wave == 0 && g == 0) {
        row_lds[mt][r][0] = top;
        row_lds[mt][r][1] = sum;
      }
      const float f = __builtin_amdgcn_exp2f(m[mt] - top);
#pragma unroll
      for (int j = 0; j < S::kBlocks; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o_lds[k * 4 + wave][r][(4 * g + e) * S::kBlocks + j] =
              (o[mt][j][e] + mid[mt][e]) * f;
    }
    __syncthreads();
    const int rows = min(a.rows - row0 - base * 16, kTogether * 16);
    for (int idx = threadIdx.x; idx < rows * H; idx += 256) {
      const int k = idx / (16 * H), rr = idx / H % 16, d = idx % H;
      const int row = row0 + base * 16 + idx / H;
      float y = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) y += o_lds[k * 4 + w][rr][d];
      const float* ml = row_lds[base + k][rr];
      if (a.chunks > 1) {
        const long at = (bh * a.chunks + chunk) * a.rows + row;
        a.part_o[at * H + d] = y;
        if (d < 2) a.part_ml[at * 2 + d] = ml[d];
      } else {
        const unsigned i = (unsigned)row / (unsigned)a.rep;
        const int head = kv_head * a.rep + row - i * a.rep;
        float z = y / ml[1];
        if (t0 < 0) z = 0.f;
        else if (t0 + i >= a.cache.capacity) z = NAN;
        T* out =
            (T*)a.out + (((long)i * a.cache.b + ib) * a.n + head) * H + d;
        *out = DTypeTraits<T>::from_float(z);
      }
    }
  }
}

// Joins the chunks of a row. WAVES waves share a row, each with every
// WAVES-th chunk, of which lane i holds the i-th one's maximum and sum; each
// lane has H / 64 values. What a chunk left is read before it is known to be
// used: one way to memory less. Chunks come eight at a time: one by one, as
// the compiler leaves a loop with lane reads, 256 rows of 21 took 5.1 us.
template <typename T, int H, int MT, int WAVES>
__global__ __launch_bounds__(256) void join_kernel(AttentionArgs a) {
  constexpr int kEach = H >= 64 ? H / 64 : 1;
  __shared__ float o_lds[WAVES > 1 ? WAVES : 1][H], ml_lds[4][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = WAVES > 1 ? wave : 0;
  const unsigned number = WAVES > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
  const unsigned bh = number / (unsigned)a.rows;
  if (bh >= (unsigned)a.cache.b * a.cache.heads) return;
  const unsigned row = number - bh * a.rows;
  const unsigned ib = bh / (unsigned)a.cache.heads;
  const unsigned kv_head = bh - ib * a.cache.heads;
  const int d = lane * kEach;
  // from chunk to chunk of a (sequence, key head, row)
  const long step = a.rows;
  const long at = (long)bh * a.chunks * step + row;
  const int mine = lane * WAVES + part;
  float2 ml = {kUnset, 0.f};
  if (mine < a.chunks)
    ml = *(const float2*)(a.part_ml + (at + mine * step) * 2);
  const unsigned per = *a.part_per;
  const long t0 = a.start.of(ib);

  const unsigned i = row / (unsigned)a.rep;
  const int head = kv_head * a.rep + row - i * a.rep;
  T* out = (T*)a.out + (((long)i * a.cache.b + ib) * a.n + head) * H;
  if (t0 < 0 || t0 + i >= a.cache.capacity) {
    if (part == 0 && d < H)
      for (int e = 0; e < kEach; ++e)
        out[d + e] = DTypeTraits<T>::from_float(t0 < 0 ? 0.f : NAN);
    return;
  }
  const int row0 = row / (16 * MT) * 16 * MT;
  const int row1 = min(a.rows, row0 + 16 * MT) - 1;
  const Tiles tiles = tiles_of(a, t0, row0, row1);
  const int used = (tiles.count + per - 1) / per;
  if (mine >= used) ml = {kUnset, 0.f};
  const float top = wave_reduce_max(ml.x);
  const float f = __builtin_amdgcn_exp2f(ml.x - top);
  float sum = wave_reduce_sum(ml.y * f);
  float y[kEach] = {};
  const float* po = a.part_o + at * H + d;
  constexpr int kBatch = 8;  // chunks on their way together
  for (int base = part; base < used; base += kBatch * WAVES) {
    float v[kBatch][kEach];
    // behind the last chunk that one again: no branch parts the loads
    const int last = base + (used - 1 - base) / WAVES * WAVES;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int c = min(base + k * WAVES, last);
      // (with h = 32 half of the lanes have no values: they take the others')
      for (int e = 0; e < kEach; ++e)
        v[k][e] = po[c * step * H + e - (d < H ? 0 : H)];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int c = base + k * WAVES;
      const float fc = __uint_as_float(__builtin_amdgcn_readlane(
          (int)__float_as_uint(f), min(c, last) / WAVES));
      for (int e = 0; e < kEach; ++e)
        y[e] = c <= last ? fmaf(v[k][e], fc, y[e]) : y[e];
    }
  }
  if constexpr (WAVES == 1) {
    if (d < H)
      for (int e = 0; e < kEach; ++e)
        out[d + e] = DTypeTraits<T>::from_float(y[e] / sum);
  } else {
    if (d < H)
      for (int e = 0; e < kEach; ++e) o_lds[wave][d + e] = y[e];
    if (lane == 0) {
      ml_lds[wave][0] = top;
      ml_lds[wave][1] = sum;
    }
    __syncthreads();
    if (threadIdx.x < H) {
      const int t = threadIdx.x;
      float high = kUnset, o = 0.f;
      for (int w = 0; w < WAVES; ++w) high = fmaxf(high, ml_lds[w][0]);
      sum = 0.f;
      for (int w = 0; w < WAVES; ++w) {
        const float g = __builtin_amdgcn_exp2f(ml_lds[w][0] - high);
        o += o_lds[w][t] * g;
        sum += ml_lds[w][1] * g;
      }
      out[t] = DTypeTraits<T>::from_float(o / sum);
    }
  }
}

template <typename T, int H, int MT>
void launch_attention(AttentionArgs a, hipStream_t stream) {
  const long work =
      (long)(a.chunks > 1 ? a.groups : a.cache.b) * a.cache.heads;
  const long grid = (work + 7) / 8 * 8 * a.q_blocks;
  const long joins = (long)a.cache.b * a.cache.heads * a.rows;
  TORCH_CHECK(grid < (1l << 31) && joins < (1l << 31),
              "quant_kv: too many queries at once");
  hipLaunchKernelGGL((attention_kernel<T, H, MT>), dim3(grid), dim3(256), 0,
                     stream, a);
  // few chunks: a wave for a row (2840 rows of 6 chunks: 3.8 us; four waves
  // took half as long again); many: four (256 rows of 21: 4.2 us)
  if (a.chunks > 1 && a.chunks <= 32)
    hipLaunchKernelGGL((join_kernel<T, H, MT, 1>), dim3((joins + 3) / 4),
                       dim3(256), 0, stream, a);
  else if (a.chunks > 1)
    hipLaunchKernelGGL((join_kernel<T, H, MT, 4>), dim3(joins), dim3(256), 0,
                       stream, a);
}

CacheView view_of(const std::vector<torch::Tensor>& c, int64_t capacity) {
  TORCH_CHECK(c.size() == 4, "quant_kv: four buffers make a cache");
  for (const auto& t : c)
    TORCH_CHECK(t.is_cuda() && t.is_contiguous() &&
                    t.device() == c[0].device(),
                "quant_kv: buffers must be contiguous on one GPU");
  TORCH_CHECK(c[0].dim() == 4 && c[0].scalar_type() == torch::kUInt8);
  CacheView v;
  v.b = c[0].size(0);
  v.heads = c[0].size(1);
  v.room = c[0].size(2);
  v.h = c[0].size(3) * 2;
  v.capacity = capacity;
  const long rows = (long)v.b * v.heads * v.room, groups = v.h / kGroup;
  TORCH_CHECK(v.h == 32 || v.h == 64 || v.h == 128 || v.h == 256,
              "quant_kv: head_dim must be 32, 64, 128 or 256");
  TORCH_CHECK(v.room % 64 == 0 && capacity >= 1 && capacity <= v.room);
  TORCH_CHECK(c[1].scalar_type() == torch::kHalf &&
                  c[1].numel() == rows * groups * 2 &&
                  c[2].scalar_type() == torch::kUInt8 &&
                  c[2].numel() == rows * 32 * v_quarters(v.h) &&
                  c[3].scalar_type() == torch::kHalf &&
                  c[3].numel() == rows * groups * 2,
              "quant_kv: buffers do not belong together");
  v.k_codes = c[0].data_ptr<uint8_t>();
  v.k_meta = (__half*)c[1].data_ptr();
  v.v_codes = c[2].data_ptr<uint8_t>();
  v.v_meta = (__half*)c[3].data_ptr();
  return v;
}

Start start_of(const c10::optional<torch::Tensor>& t, int64_t scalar,
               const CacheView& c, const torch::Tensor& like) {
  if (!t.has_value()) return Start{nullptr, 0, scalar};
  TORCH_CHECK(t->device() == like.device() &&
                  t->scalar_type() == torch::kLong && t->dim() == 1 &&
                  (t->size(0) == 1 || t->size(0) == c.b),
              "quant_kv: start must be int64 with 1 or b elements");
  return Start{t->data_ptr<long>(), t->size(0) == 1 ? 0 : t->stride(0), 0};
}

void check_rows(const torch::Tensor& x, const torch::Tensor& like,
                const CacheView& c, const char* what) {
  TORCH_CHECK(x.device() == like.device() && x.dim() == 4 &&
                  x.stride(3) == 1 && x.size(1) == c.b && x.size(3) == c.h,
              "quant_kv: ", what, " must be [s, b, heads, h] on the cache's "
              "device with dense head_dim");
  TORCH_CHECK(x.scalar_type() == torch::kBFloat16 ||
                  x.scalar_type() == torch::kHalf,
              "quant_kv: bf16 or fp16 only");
}

AppendSource source_of(const torch::Tensor& x) {
  return AppendSource{x.data_ptr(), x.stride(0), x.stride(1), x.stride(2)};
}

#define DISPATCH_HEAD(H, FN, T)                                              \
  do {                                                                       \
    switch (H) {                                                             \
      case 32: FN(T, 32); break;                                             \
      case 64: FN(T, 64); break;                                             \
      case 128: FN(T, 128); break;                                           \
      default: FN(T, 256);                                                   \
    }                                                                        \
  } while (0)

#define DISPATCH_HALF(TENSOR, FN)                                            \
  do {                                                                       \
    if ((TENSOR).scalar_type() == torch::kBFloat16) {                        \
      FN(__hip_bfloat16);                                                    \
    } else {                                                                 \
      FN(__half);                                                            \
    }                                                                        \
  } while (0)

}  // namespace

c10::optional<torch::Tensor> quant_kv_append(
    std::vector<torch::Tensor> buffers, int64_t capacity, torch::Tensor key,
    torch::Tensor value, c10::optional<torch::Tensor> start, int64_t start_s,
    c10::optional<torch::Tensor> query, c10::optional<torch::Tensor> cos,
    c10::optional<torch::Tensor> sin, bool interleaved) {
  const CacheView cache = view_of(buffers, capacity);
  const c10::hip::HIPGuard guard(buffers[0].get_device());
  check_rows(key, buffers[0], cache, "key");
  check_rows(value, buffers[0], cache, "value");
  TORCH_CHECK(key.sizes() == value.sizes() && key.size(2) == cache.heads &&
                  key.scalar_type() == value.scalar_type(),
              "quant_kv: key and value must match the cache");
  const Start at = start_of(start, start_s, cache, buffers[0]);
  const long s = key.size(0);
  AppendSource q{nullptr, 0, 0, 0};
  torch::Tensor q_out;
  int n = 0, r = 0;
  long table_rows = 0;
  const float *cos_p = nullptr, *sin_p = nullptr;
  if (cos.has_value()) {
    TORCH_CHECK(query.has_value() && sin.has_value(),
                "quant_kv: query, cos and sin come together");
    check_rows(*query, buffers[0], cache, "query");
    TORCH_CHECK(query->size(0) == s &&
                    query->scalar_type() == key.scalar_type(),
                "quant_kv: query must match the key");
    TORCH_CHECK(cos->device() == key.device() &&
                    sin->device() == key.device() && cos->dim() == 2 &&
                    cos->sizes() == sin->sizes() && cos->is_contiguous() &&
                    sin->is_contiguous() &&
                    cos->scalar_type() == torch::kFloat32 &&
                    sin->scalar_type() == torch::kFloat32 &&
                    cos->size(1) >= 1 && 2 * cos->size(1) <= cache.h,
                "quant_kv: cos and sin must be contiguous fp32 tables alike");
    n = query->size(2);
    r = cos->size(1);
    table_rows = cos->size(0);
    cos_p = cos->data_ptr<float>();
    sin_p = sin->data_ptr<float>();
    q = source_of(*query);
    q_out = torch::empty({s, cache.b, n, cache.h}, query->options());
  } else {
    TORCH_CHECK(!query.has_value() && !sin.has_value(),
                "quant_kv: query, cos and sin come together");
  }
  auto wide = [](const torch::Tensor& x) {
    return (unsigned long)x.data_ptr() % 16 == 0 && x.stride(0) % 8 == 0 &&
           x.stride(1) % 8 == 0 && x.stride(2) % 8 == 0;
  };
  bool all_wide = wide(key) && wide(value);
  auto stream = c10::hip::getCurrentHIPStream();
  if (s > 0 && q.x) {
    all_wide = all_wide && wide(*query);
    const long grid =
        (s * cache.b * (cache.heads + (long)n) * (cache.h / 8) + 255) / 256;
    TORCH_CHECK(grid < (1l << 24), "quant_kv: too many tokens at once");
#define LAUNCH_ROWS(T, H, W)                                                 \
  hipLaunchKernelGGL((append_rotated_kernel<T, H, W>), dim3(grid),           \
                     dim3(256), 0, stream, cache, source_of(key),            \
                     source_of(value), q, (T*)q_out.data_ptr(), n, cos_p,    \
                     sin_p, r, table_rows, interleaved, at, s)
#define LAUNCH_HEAD(T, H)                                                    \
  do {                                                                       \
    if (all_wide) LAUNCH_ROWS(T, H, true);                                   \
    else LAUNCH_ROWS(T, H, false);                                           \
  } while (0)
#define LAUNCH_APPEND(T) DISPATCH_HEAD(cache.h, LAUNCH_HEAD, T)
    DISPATCH_HALF(key, LAUNCH_APPEND);
#undef LAUNCH_APPEND
#undef LAUNCH_HEAD
#undef LAUNCH_ROWS
    HIP_CHECK(hipGetLastError());
  } else if (s > 0) {
    // the begin may lie anywhere in a wave's tile
    const long per = 512 / cache.h, tiles = (s + per - 2) / per + 1;
    const long grid = ((long)cache.b * cache.heads * tiles + 3) / 4;
    TORCH_CHECK(grid < (1l << 30), "quant_kv: too many tokens at once");
#define LAUNCH_TILES(T, H, W)                                                \
  hipLaunchKernelGGL((append_kernel<T, H, W>), dim3(grid), dim3(256), 0,     \
                     stream, cache, source_of(key), source_of(value), at, s, \
                     (unsigned)tiles)
#define LAUNCH_HEAD(T, H)                                                    \
  do {                                                                       \
    if (all_wide) LAUNCH_TILES(T, H, true);                                  \
    else LAUNCH_TILES(T, H, false);                                          \
  } while (0)
#define LAUNCH_APPEND(T) DISPATCH_HEAD(cache.h, LAUNCH_HEAD, T)
    DISPATCH_HALF(key, LAUNCH_APPEND);
#undef LAUNCH_APPEND
#undef LAUNCH_HEAD
#undef LAUNCH_TILES
    HIP_CHECK(hipGetLastError());
  }
  if (!query.has_value()) return c10::nullopt;
  return q_out;
}

std::vector<torch::Tensor> quant_kv_dequantize(
    std::vector<torch::Tensor> buffers, int64_t capacity,
    c10::optional<torch::Tensor> start, int64_t start_s, int64_t length,
    bool bf16) {
  const CacheView cache = view_of(buffers, capacity);
  const c10::hip::HIPGuard guard(buffers[0].get_device());
  const Start at = start_of(start, start_s, cache, buffers[0]);
  auto options =
      buffers[1].options().dtype(bf16 ? torch::kBFloat16 : torch::kHalf);
  auto k = torch::empty({length, cache.b, cache.heads, cache.h}, options);
  auto v = torch::empty_like(k);
  if (k.numel() == 0) return {k, v};
  const long per = 512 / cache.h, tiles = (length + per - 2) / per + 1;
  const long grid = ((long)cache.b * cache.heads * tiles + 3) / 4;
  TORCH_CHECK(grid < (1l << 30), "quant_kv: too many tokens at once");
  auto stream = c10::hip::getCurrentHIPStream();
#define LAUNCH_TILES(T, H)                                                   \
  hipLaunchKernelGGL((dequantize_kernel<T, H>), dim3(grid), dim3(256), 0,    \
                     stream, cache, at, (long)length, (unsigned)tiles,       \
                     (T*)k.data_ptr(), (T*)v.data_ptr())
#define LAUNCH_DEQUANTIZE(T) DISPATCH_HEAD(cache.h, LAUNCH_TILES, T)
  DISPATCH_HALF(k, LAUNCH_DEQUANTIZE);
#undef LAUNCH_DEQUANTIZE
#undef LAUNCH_TILES
  HIP_CHECK(hipGetLastError());
  return {k, v};
}

torch::Tensor quant_kv_attention(std::vector<torch::Tensor> buffers,
                                 int64_t capacity, torch::Tensor query,
                                 c10::optional<torch::Tensor> start,
                                 int64_t start_s, double scale,
                                 int64_t window, int64_t sinks) {
  const CacheView cache = view_of(buffers, capacity);
  const c10::hip::HIPGuard guard(buffers[0].get_device());
  check_rows(query, buffers[0], cache, "query");
  const long s = query.size(0);
  const int n = query.size(2);
  TORCH_CHECK(n >= 1 && n % cache.heads == 0,
              "quant_kv: query heads must be a multiple of key heads");
  const Start at = start_of(start, start_s, cache, buffers[0]);
  auto out = torch::empty({s, cache.b, (long)n * cache.h}, query.options());
  if (out.numel() == 0) return out;
  AttentionArgs a;
  a.cache = cache;
  a.q = query.data_ptr();
  a.q_ss = query.stride(0);
  a.q_bs = query.stride(1);
  a.q_ns = query.stride(2);
  a.out = out.data_ptr();
  a.n = n;
  a.rep = n / cache.heads;
  TORCH_CHECK(s * a.rep < (1l << 30), "quant_kv: too many queries at once");
  a.rows = (int)s * a.rep;
  a.scale_log2e = (float)(scale * 1.4426950408889634);
  a.window = window;
  a.sinks = sinks;
  a.start = at;

  // query tiles of a workgroup: one decodes, more share the work on the codes
  const int tiles = (a.rows + 15) / 16;
  const int mt = tiles == 1 ? 1 : tiles == 2 || cache.h == 256 ? 2 : 4;
  a.q_blocks = (tiles + mt - 1) / mt;
  a.q_wide = (unsigned long)a.q % 16 == 0 &&
             a.q_ss % 8 == 0 && a.q_bs % 8 == 0 && a.q_ns % 8 == 0;
  // Workgroups that the card holds at once share the tokens, or, where there
  // are about as many key heads and query blocks, one more for each of those.
  // A sequence may be several times the mean in length.
  const long span =
      window > 0 ? std::min<long>(cache.capacity, window + sinks + s + 64)
                 : cache.capacity;
  const long each = (long)cache.heads * a.q_blocks, base = cache.b * each;
  const int resident = mt * cache.h <= 128 ? 3 : mt * cache.h <= 256 ? 2 : 1;
  a.groups = (int)std::max<long>(2l * cache.b, 256 * resident / each);
  const long most = (span + kLeast - 1) / kLeast;
  // and what they leave for the join stays under 128 MB: with that many query
  // rows the card is full without shares
  const long room = (1l << 25) / ((long)cache.b * cache.heads * a.rows *
                                  (cache.h + 2));
  a.chunks = (int)std::max<long>(
      1, std::min<long>(std::min<long>(most, std::min<long>(room, 256)),
                        4 * (a.groups * each + base - 1) / base));
  TORCH_CHECK(cache.capacity < (1l << 31) && base * a.chunks < (1l << 31) &&
                  a.groups * each < (1l << 31),
              "quant_kv: too many tokens or queries at once");
  torch::Tensor part;
  a.part_o = a.part_ml = nullptr;
  a.part_per = nullptr;
  if (a.chunks > 1) {
    const long parts = (long)cache.b * cache.heads * a.chunks * a.rows;
    part = torch::empty({parts * (cache.h + 2) + 1},
                        query.options().dtype(torch::kFloat32));
    a.part_o = part.data_ptr<float>();
    a.part_ml = a.part_o + parts * cache.h;
    a.part_per = (int*)(a.part_ml + parts * 2);
  }
  auto stream = c10::hip::getCurrentHIPStream();
#define LAUNCH_ATTENTION(T)                                                  \
  switch (cache.h * 8 + mt) {                                                \
    case 32 * 8 + 1: launch_attention<T, 32, 1>(a, stream); break;           \
    case 32 * 8 + 2: launch_attention<T, 32, 2>(a, stream); break;           \
    case 32 * 8 + 4: launch_attention<T, 32, 4>(a, stream); break;           \
    case 64 * 8 + 1: launch_attention<T, 64, 1>(a, stream); break;           \
    case 64 * 8 + 2: launch_attention<T, 64, 2>(a, stream); break;           \
    case 64 * 8 + 4: launch_attention<T, 64, 4>(a, stream); break;           \
    case 128 * 8 + 1: launch_attention<T, 128, 1>(a, stream); break;         \
    case 128 * 8 + 2: launch_attention<T, 128, 2>(a, stream); break;         \
    case 128 * 8 + 4: launch_attention<T, 128, 4>(a, stream); break;         \
    case 256 * 8 + 1: launch_attention<T, 256, 1>(a, stream); break;         \
    case 256 * 8 + 2: launch_attention<T, 256, 2>(a, stream); break;         \
    default: TORCH_CHECK(false, "quant_kv: head_dim");                       \
  }
  DISPATCH_HALF(query, LAUNCH_ATTENTION);
#undef LAUNCH_ATTENTION
  HIP_CHECK(hipGetLastError());
  return out;
}
