// Next tokens from logits and given uniform numbers: temperature, top-k,
// top-p and min-p in one kernel, one workgroup per row.
//
// With m the row's largest logit a token weighs w = exp((x - m) / T). Tokens
// are ordered by logit, equal ones by index. top-k keeps the first k; top-p
// keeps, of those, each whose predecessors weigh at most top_p of them all;
// min-p keeps the tokens with w >= min_p. The drawn token is the first index
// whose kept weights up to and with it exceed u times all kept weights.
//
// Weights are whole numbers of 2^-shift (64 bits, shift = 62 - log2 of the
// vocabulary, 51 at most): their sums are exact in any order, so that filters
// and draw agree with each other and from run to run. Exponentials are taken
// in 64 bits, since a draw hangs on sums that lie next to a border.
//
// A row with a NaN, or with no logit above -inf, gives -1.
//
// One compute unit does a row, whatever the number of rows, and its passes bound
// it: 32000 logits in 32 bits with top-k 40 take 11 us (1.5 of them the first
// pass over the row), 64 rows of 65024 in 16 bits with all filters 27 on a
// quarter of the card, 256 rows of 50257 in 32 bits without filters 32, of which
// the first pass takes 7.5 at 7 TB/s and the sum of the weights 15; more than
// half of the waves' cycles there go by waiting. Sums bit by bit took 190, 700
// and 219.

#include "common.h"

#include <torch/extension.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / WAVE_SIZE;
using u64 = unsigned long long;

struct SampleArgs {
  const void* logits;
  long row_stride;
  const float* uniform;
  long* out;
  int vocab;
  int shift;
  // per-row settings; the scalar counts where the pointer is null
  const float* temperature;
  const long* top_k;
  const float* top_p;
  const float* min_p;
  double temperature_s, top_p_s, min_p_s;
  long top_k_s;
};

// larger floats have larger keys; both zeros have the same one
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float key_value(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

constexpr int kBins = 2048;
constexpr int kList = 256;  // tokens that are ranked one against another

__constant__ const double kPower[64] = {  // 2^(j / 64)
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951};
__constant__ const double kFine[4] = {  // 2^(j / 256)
    1.0, 1.0027112750502025,
    1.0054299011128027, 1.0081558981184175};

struct Token {
  float v;
  int index;
  u64 weight;
};

struct Lds {
  u64 mass[kBins];
  unsigned count[kBins];
  Token list[kList];
  double power[256];
  u64 wave[2][kWaves];
  u64 answer[4];
  float extreme[2][kWaves];
  u64 found_above;
  float found;
  unsigned listed, low, high;
};

// Joins a wave's values by row shifts and broadcasts: lane i gets those of the
// lanes up to i, `none` standing for lanes that are not there. With ROW within
// 16 lanes only.
template <bool ROW = false, typename F>
__device__ __forceinline__ unsigned wave_join(unsigned v, unsigned none,
                                              F join) {
#define JOIN_STEP(CTRL, ROWS)                                                \
  v = join(v, (unsigned)__builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, \
                                                    ROWS, 0xf, false))
  JOIN_STEP(0x111, 0xf);  // from 1, 2, 4, 8 lanes below, within 16
  JOIN_STEP(0x112, 0xf);
  JOIN_STEP(0x114, 0xf);
  JOIN_STEP(0x118, 0xf);
  if (!ROW) {
    JOIN_STEP(0x142, 0xa);  // from the last lane of the 16 below
    JOIN_STEP(0x143, 0xc);  // from lane 31
  }
#undef JOIN_STEP
  return v;
}

template <bool ROW = false>
__device__ __forceinline__ u64 wave_scan(u64 v) {
#define SCAN_STEP(CTRL, ROWS)                                               \
  v += (u64)(unsigned)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL,  \
                                                  ROWS, 0xf, false)         \
           << 32 |                                                          \
       (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf,    \
                                             false)
  SCAN_STEP(0x111, 0xf);
  SCAN_STEP(0x112, 0xf);
  SCAN_STEP(0x114, 0xf);
  SCAN_STEP(0x118, 0xf);
  if (!ROW) {
    SCAN_STEP(0x142, 0xa);
    SCAN_STEP(0x143, 0xc);
  }
#undef SCAN_STEP
  return v;
}

__device__ __forceinline__ u64 lane_value(u64 v, int lane) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane)
             << 32 |
         (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}

__device__ __forceinline__ u64 wave_sum(u64 v) {
  return lane_value(wave_scan(v), 63);
}

__device__ __forceinline__ float wave_max(float v) {
  return __uint_as_float(__builtin_amdgcn_readlane(
      (int)wave_join(__float_as_uint(v), __float_as_uint(-INFINITY),
                     [](unsigned x, unsigned y) {
                       return __float_as_uint(
                           fmaxf(__uint_as_float(x), __uint_as_float(y)));
                     }),
      63));
}

__device__ __forceinline__ u64 block_sum(u64 v, u64* lds) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return lane_value(wave_scan<true>(lds[threadIdx.x & (kWaves - 1)]),
                    kWaves - 1);
}

// sum of the values of all threads before this one
__device__ __forceinline__ u64 block_scan(u64 v, u64* lds) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const u64 up = wave_scan(v);
  __syncthreads();
  if (lane == 63) lds[wave] = up;
  __syncthreads();
  const u64 waves = wave_scan<true>(lds[lane & (kWaves - 1)]);
  return up - v + (wave ? lane_value(waves, wave - 1) : 0);
}

__device__ __forceinline__ u64 floor_u64(double x, u64 most) {
  if (!(x > 0.0)) return 0;
  return x >= (double)most ? most : (u64)x;
}

// A row, read 16 bytes at a time where they lie within it. Each wave has a
// run of indices of its own, so that sums by wave are sums in order.
template <typename T>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  static constexpr int kBatch = 4;  // loads in flight
  const T* x;
  int vocab, shift;  // x - shift is a multiple of 16 bytes
  int first, last;   // this wave's run

  __device__ Row(const T* x, int vocab) : x(x), vocab(vocab) {
    shift = (int)((unsigned long)x & 15) / (int)sizeof(T);
    const int step = WAVE_SIZE * kVec;
    const int run = ((vocab + shift + kWaves - 1) / kWaves + step - 1) /
                    step * step;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    first = min(vocab, max(0, wave * run - shift));
    last = min(vocab, (wave + 1) * run - shift);
  }

  __device__ __forceinline__ float at(int i) const {
    return DTypeTraits<T>::to_float(x[i]);
  }

  // f(value, index) for every value of the wave's run
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int lane = threadIdx.x & 63;
    union Vec {
      uint4 u;
      T t[kVec];
    };
    // the run's begin lies on 16 bytes, but for the row's own
    int base = first == 0 ? -shift : first;
    constexpr int kStep = WAVE_SIZE * kVec;
    if (base < 0 && base + kStep <= last) {  // the row's begin
      const int i = base + lane * kVec;
      for (int e = 0; e < kVec; ++e)
        if (i + e >= 0) f(at(i + e), i + e);
      base += kStep;
    }
    if (base >= 0) {
      for (; base + kBatch * kStep <= last; base += kBatch * kStep) {
        Vec v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          v[k].u = *(const uint4*)(x + base + (k * WAVE_SIZE + lane) * kVec);
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            f(DTypeTraits<T>::to_float(v[k].t[e]),
              base + (k * WAVE_SIZE + lane) * kVec + e);
      }
    }
    for (; base < last; base += kStep) {
      const int i = base + lane * kVec;
      if (i >= 0 && i + kVec <= last) {
        Vec v;
        v.u = *(const uint4*)(x + i);
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          f(DTypeTraits<T>::to_float(v.t[e]), i + e);
      } else {
        for (int e = 0; e < kVec; ++e)
          if (i + e >= 0 && i + e < last) f(at(i + e), i + e);
      }
    }
  }
};

// Weights of a row: 2^(y / 256) with y = 256 (x - top) / T log2 e <= 0, from a
// table of 2^(j / 256) and a polynomial of the third degree on the rest, which
// is at most ln 2 / 512 (relative error under 2^-42). As a whole number of
// 2^-shift a weight is read off the low bits of its sum with 2^(52-shift).
using LdsDouble = const __attribute__((address_space(3))) double;

struct Weights {
  double top, per;  // 256 log2 e / T
  double unit;      // 2^(52 - shift)
  double big, c1, c2, c3;
  LdsDouble* power;

  __device__ Weights(float top_, double temperature, int shift, Lds& lds)
      : top(top_),
        per(256.0 * 1.4426950408889634 / temperature),
        unit(__longlong_as_double((long long)(1023 + 52 - shift) << 52)),
        power((LdsDouble*)lds.power) {
    constexpr double c = 0.6931471805599453 / 256;
    big = 6755399441055744.0;  // 1.5 * 2^52
    c1 = c, c2 = c * c / 2, c3 = c * c * c / 6;
    // held in registers: fewer moves than from constants
    asm("" : "+v"(big), "+v"(c1), "+v"(c2), "+v"(c3));
  }

  __device__ __forceinline__ double of(float v) const {
    const double y = fmax(((double)v - top) * per, -256000.0);
    const double k = y + big;
    const double r = y - (k - big);
    const double p = fma(r, fma(r, fma(r, c3, c2), c1), 1.0);
    const int n = __double2loint(k);
    const double q = power[n & 255];
    return p * __hiloint2double(__double2hiint(q) + ((n & ~255) << 12),
                                __double2loint(q));
  }
  __device__ __forceinline__ u64 whole(double w) const {
    return (u64)(__double_as_longlong(w + unit) - __double_as_longlong(unit));
  }
  // of a value that may be infinite, as the largest then is
  __device__ __forceinline__ u64 whole_of(float v) const {
    return whole((double)v == top ? 1.0 : of(v));
  }
};

// Tokens with a larger logit are kept, and the first `ties` of those with
// this one; or the list holds all that can be kept.
struct Cut {
  float v;
  u64 ties;
  int listed;
};

// Down from the largest logit, where `limit` is passed: by count (MASS false)
// the limit-th token, by mass the least logit whose larger ones weigh at most
// `limit`. low and high are the extremes of the tokens that count, finite;
// more than `limit` of them there are.
//
// Each step shares the range out over bins, finds the bin in which the limit
// is passed and goes on within it, until it holds one logit or few tokens; or,
// with few tokens from there up, lists those.
template <bool MASS, typename T>
__device__ Cut find_cut(Lds& lds, const Row<T>& row, const Weights& weights,
                        float low, float high, u64 limit) {
  const int tid = threadIdx.x;
  u64 above = 0;     // count or mass of the tokens over `high`
  unsigned over = 0;  // count of them
  for (int step = 0; low < high; ++step) {
    if (step == 8) {  // a range that bins cannot tell apart: bit by bit
      unsigned l = order_key(low), h = order_key(high);
      auto part_over = [&](unsigned t) {
        u64 part = 0;
        row.each([&](float v, int) {
          if (order_key(v) > t)
            part += MASS ? weights.whole(weights.of(v)) : 1;
        });
        return block_sum(part, lds.wave[0]);
      };
      while (l < h) {
        const unsigned t = l + (h - l) / 2;
        const u64 part = part_over(t);
        if (MASS ? part <= limit : part < limit)
          h = t;
        else
          l = t + 1;
      }
      above = part_over(l);
      low = key_value(l);
      break;
    }
    const float scale = fminf((kBins - 0.5f) / (high - low), 3e38f);
    const float shift = -low * scale;
    auto bin_of = [&](float v) {  // rises with v, rounding and all
      return min(kBins - 1, max(0, (int)fmaf(v, scale, shift)));
    };
    for (int i = tid; i < kBins; i += kThreads) {
      lds.count[i] = 0;
      if (MASS) lds.mass[i] = 0;
    }
    if (tid == 0) {
      lds.listed = 0;
      lds.low = ~0u;
      lds.high = 0;
    }
    __syncthreads();
    row.each([&](float v, int) {
      if (v >= low && v <= high) {
        const int bin = bin_of(v);
        atomicAdd(&lds.count[bin], 1u);
        if (MASS) atomicAdd(&lds.mass[bin], weights.whole(weights.of(v)));
      }
    });
    __syncthreads();
    // thread t has two bins, from the top
    constexpr int kEach = kBins / kThreads;
    u64 own[kEach], sum = 0, tokens = 0;
    for (int e = 0; e < kEach; ++e) {
      const int bin = kBins - 1 - (tid * kEach + e);
      own[e] = MASS ? lds.mass[bin] : lds.count[bin];
      sum += own[e];
      tokens += lds.count[bin];
    }
    u64 upto = above + block_scan(sum, lds.wave[0]);
    u64 tokens_upto = over;
    if (MASS) tokens_upto += block_scan(tokens, lds.wave[1]);
    for (int e = 0; e < kEach; ++e) {
      const int bin = kBins - 1 - (tid * kEach + e);
      if (!MASS) tokens_upto = upto;
      const bool here = MASS ? upto <= limit && upto + own[e] > limit
                             : upto < limit && upto + own[e] >= limit;
      if (here) {
        lds.answer[0] = bin;
        lds.answer[1] = upto;
        lds.answer[2] = tokens_upto;
        lds.answer[3] = tokens_upto + lds.count[bin];
      }
      upto += own[e];
      tokens_upto += lds.count[bin];
    }
    __syncthreads();
    const int bin = (int)lds.answer[0];
    above = lds.answer[1];
    over = (unsigned)lds.answer[2];
    if (lds.answer[3] <= kList) {  // all from this bin up
      row.each([&](float v, int i) {
        if (v > high || (v >= low && bin_of(v) >= bin)) {
          const unsigned at = atomicAdd(&lds.listed, 1u);
          lds.list[at] = Token{v, i, 0};
        }
      });
      __syncthreads();
      return Cut{0.f, 0, (int)lds.listed};
    }
    unsigned least = ~0u, most = 0;
    row.each([&](float v, int i) {
      if (v >= low && v <= high && bin_of(v) == bin) {
        const unsigned key = order_key(v);
        least = min(least, key);
        most = max(most, key);
        const unsigned at = atomicAdd(&lds.listed, 1u);
        if (at < kList)
          lds.list[at] = Token{v, i, MASS ? weights.whole_of(v) : 1};
      }
    });
    if (most) {
      atomicMin(&lds.low, least);
      atomicMax(&lds.high, most);
    }
    __syncthreads();
    low = key_value(lds.low);
    high = key_value(lds.high);
    const int listed = (int)lds.listed;
    // the ranking's answer has a word of its own: a wave that comes late still
    // reads the bin's extremes above, so that all waves take the same way
    if (low < high && listed <= kList) {
      const int at = tid >> 2;  // four threads rank a token
      if (at < listed) {
        const float own_v = lds.list[at].v;
        u64 larger = 0, equal = 0;
        for (int j = tid & 3; j < listed; j += 4) {
          const Token other = lds.list[j];
          if (other.v > own_v) larger += other.weight;
          if (other.v == own_v) equal += other.weight;
        }
        for (int o = 1; o < 4; o <<= 1) {
          larger += __shfl_xor(larger, o, WAVE_SIZE);
          equal += __shfl_xor(equal, o, WAVE_SIZE);
        }
        larger += above;
        if (MASS ? larger <= limit && larger + equal > limit
                 : larger < limit && larger + equal >= limit) {
          lds.found = own_v;
          lds.found_above = larger;
        }
      }
      __syncthreads();
      low = high = lds.found;
      above = lds.found_above;
    }
    __syncthreads();
  }
  if (!MASS) return Cut{low, limit - above, -1};
  const u64 w = weights.whole_of(low);
  return Cut{low, w ? (limit - above) / w + 1 : (u64)row.vocab, -1};
}

// Lists the tokens that can be among the first top_k, if they are few: those
// from about the top_k-th largest of the threads' own maxima up. That many
// tokens lie there at least; in a row in no particular order not many more.
template <typename T>
__device__ Cut list_largest(Lds& lds, const Row<T>& row, float own_high,
                            float top, unsigned top_k) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  for (int i = tid; i < kBins; i += kThreads) lds.count[i] = 0;
  if (tid == 0) {
    lds.listed = 0;
    lds.low = ~0u;
    lds.answer[0] = kBins;
  }
  const bool some = own_high > -INFINITY;
  float low = -wave_max(some ? -own_high : -INFINITY);
  if (lane == 0) lds.extreme[1][wave] = low;
  __syncthreads();
  low = -wave_max(-lds.extreme[1][lane & (kWaves - 1)]);
  const float scale = fminf((kBins - 0.5f) / (top - low), 3e38f);
  const int bin = min(kBins - 1, max(0, (int)((own_high - low) * scale)));
  if (some) atomicAdd(&lds.count[bin], 1u);
  __syncthreads();
  constexpr int kEach = kBins / kThreads;
  u64 sum = 0;
  for (int e = 0; e < kEach; ++e)
    sum += lds.count[kBins - 1 - (tid * kEach + e)];
  u64 upto = block_scan(sum, lds.wave[0]);
  for (int e = 0; e < kEach; ++e) {
    const int b = kBins - 1 - (tid * kEach + e);
    const u64 own = lds.count[b];
    if (upto < top_k && upto + own >= top_k) lds.answer[0] = b;
    upto += own;
  }
  __syncthreads();
  const int from = (int)lds.answer[0];
  if (from == kBins) return Cut{-INFINITY, (u64)row.vocab, -1};
  if (some && bin >= from) atomicMin(&lds.low, order_key(own_high));
  __syncthreads();
  const float least = key_value(lds.low);
  row.each([&](float v, int i) {
    if (v >= least) {
      const unsigned at = atomicAdd(&lds.listed, 1u);
      if (at < kList) lds.list[at] = Token{v, i, 0};
    }
  });
  __syncthreads();
  const int listed = (int)lds.listed;
  __syncthreads();
  return Cut{-INFINITY, (u64)row.vocab, listed <= kList ? listed : -1};
}

// Draws from the listed tokens: ranks them, filters, and sums the kept ones in
// the order of their indices. PARTS threads work for a token.
template <int PARTS>
__device__ __forceinline__ void draw_listed(
    Lds& lds, const Weights& weights, int listed, u64 top_k, bool by_mass,
    bool known, u64 most, double top_p, double min_p, float uniform,
    long* out) {
  const int tid = threadIdx.x, at = tid / PARTS, part = tid % PARTS;
  const bool mine = at < listed;
  Token own{0.f, 0, 0};
  double w = 0.0;
  if (mine) {
    own = lds.list[at];
    w = weights.of(own.v);
    own.weight = weights.whole(w);
    if (part == 0) lds.list[at].weight = own.weight;
  }
  __syncthreads();
  auto over_parts = [](u64 sum) {
    for (int o = 1; o < PARTS; o <<= 1) sum += __shfl_xor(sum, o, WAVE_SIZE);
    return sum;
  };
  u64 mass = 0;
  unsigned rank = 0;
  if (mine) {
#pragma unroll 4
    for (int j = part; j < listed; j += PARTS) {
      const Token t = lds.list[j];
      const bool before =
          t.v > own.v || (t.v == own.v && t.index < own.index);
      rank += before;
      mass += before ? t.weight : 0;
    }
  }
  for (int o = 1; o < PARTS; o <<= 1)
    rank += __shfl_xor((int)rank, o, WAVE_SIZE);
  bool keep = mine && rank < top_k;
  if (by_mass) {
    mass = over_parts(mass);
    if (!known) {
      const u64 all =
          block_sum(keep && part == 0 ? own.weight : 0, lds.wave[0]);
      most = floor_u64(top_p * (double)all, all);
    }
    keep &= mass <= most;
  }
  keep &= !(w < min_p);
  __syncthreads();
  if (mine && part == 0 && !keep) lds.list[at].weight = 0;
  const u64 total =
      block_sum(keep && part == 0 ? own.weight : 0, lds.wave[0]);
  const u64 target = floor_u64((double)uniform * (double)total, total - 1);
  u64 upto = 0;
  if (mine) {
#pragma unroll 4
    for (int j = part; j < listed; j += PARTS) {
      const Token t = lds.list[j];
      upto += t.index < own.index ? t.weight : 0;
    }
  }
  upto = over_parts(upto);
  if (keep && part == 0 && upto <= target && target < upto + own.weight)
    *out = own.index;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ Lds lds;
  const long number = blockIdx.x;
  const int tid = threadIdx.x, V = a.vocab, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Row<T> row((const T*)a.logits + number * a.row_stride, V);

  double temperature =
      a.temperature ? a.temperature[number] : a.temperature_s;
  long top_k = a.top_k ? a.top_k[number] : a.top_k_s;
  const double top_p = a.top_p ? a.top_p[number] : a.top_p_s;
  double min_p = a.min_p ? a.min_p[number] : a.min_p_s;
  const float uniform = a.uniform[number];
  if (!(temperature > 0.0)) {  // greedy
    temperature = 1.0;
    top_k = 1;
  }
  temperature = fmin(fmax(temperature, 1e-300), 1e30);
  if (top_k <= 0 || top_k > V) top_k = V;
  if (min_p > 1.0) min_p = 1.0;
  const bool by_mass = top_p > 0.0 && top_p < 1.0 && top_k > 1;
  const bool by_count = top_k > 1 && top_k < V;

  if (tid < 256) lds.power[tid] = kPower[tid >> 2] * kFine[tid & 3];
  float own_high = -INFINITY;
  bool bad = false;
  row.each([&](float v, int) {
    bad |= v != v;
    own_high = fmaxf(own_high, v);
  });
  // a wave with a NaN says so by one
  float high = wave_max(__any(bad) ? NAN : own_high);
  if (__any(bad)) high = NAN;
  if (lane == 0) lds.extreme[0][wave] = high;
  __syncthreads();
  const float wave_high = lds.extreme[0][lane & (kWaves - 1)];
  high = wave_max(wave_high);
  if (__any(wave_high != wave_high) || high == -INFINITY) {
    if (tid == 0) a.out[number] = -1;
    return;
  }
  const float top = high;

  if (top_k == 1) {  // the first of the largest
    if (tid == 0) lds.low = ~0u;
    __syncthreads();
    unsigned at = ~0u;
    row.each([&](float v, int i) {
      if (v == top) at = min(at, (unsigned)i);
    });
    if (at != ~0u) atomicMin(&lds.low, at);
    __syncthreads();
    if (tid == 0) a.out[number] = lds.low;
    return;
  }

  const Weights weights(top, temperature, a.shift, lds);
  Cut cut{-INFINITY, (u64)V, -1};
  if (top == INFINITY) {  // the others weigh nothing
    cut = Cut{top, (u64)top_k, -1};
  } else {
    if (by_count && top_k <= kList)
      cut = list_largest(lds, row, own_high, top, (unsigned)top_k);
    if (cut.listed < 0 && (by_count || by_mass)) {
      // the least logit above -inf, and how many those are
      float low = INFINITY;
      u64 some = 0;
      row.each([&](float v, int) {
        if (v > -INFINITY) {
          low = fminf(low, v);
          ++some;
        }
      });
      some = block_sum(some, lds.wave[0]);
      low = -wave_max(-low);
      if (lane == 0) lds.extreme[1][wave] = low;
      __syncthreads();
      low = -wave_max(-lds.extreme[1][lane & (kWaves - 1)]);
      cut.v = low;  // below come those that weigh nothing
      if ((u64)top_k < some)
        cut = find_cut<false>(lds, row, weights, low, high, (u64)top_k);
    }
  }
  bool known = false;
  u64 most = 0;
  if (by_mass && cut.listed < 0) {
    u64 mass = 0, equal = 0;
    float next = INFINITY;  // the least logit over the cut
    row.each([&](float v, int) {
      if (v > cut.v) {
        mass += weights.whole(weights.of(v));
        next = fminf(next, v);
      }
      equal += v == cut.v;
    });
    mass = block_sum(mass, lds.wave[0]);
    equal = min(block_sum(equal, lds.wave[1]), cut.ties);
    const u64 each = weights.whole_of(cut.v);
    const u64 all = mass + equal * each;
    most = floor_u64(top_p * (double)all, all);
    known = true;
    if (mass <= most) {
      if (each) cut.ties = min(cut.ties, (most - mass) / each + 1);
    } else {
      next = -wave_max(-next);
      __syncthreads();
      if (lane == 0) lds.extreme[1][wave] = next;
      __syncthreads();
      next = -wave_max(-lds.extreme[1][lane & (kWaves - 1)]);
      cut = find_cut<true>(lds, row, weights, next, high, most);
    }
  }
  if (cut.listed >= 0) {
    if (cut.listed <= kThreads / 16)
      draw_listed<16>(lds, weights, cut.listed, (u64)top_k, by_mass, known,
                      most, top_p, min_p, uniform, a.out + number);
    else
      draw_listed<4>(lds, weights, cut.listed, (u64)top_k, by_mass, known,
                     most, top_p, min_p, uniform, a.out + number);
    return;
  }

  auto weigh = [&](float v) -> u64 {
    const double w = weights.of(v);
    return w < min_p ? 0 : weights.whole(w);
  };
  const u64 tie_weight =
      cut.v == top ? weights.whole(1.0) : weigh(cut.v);
  // how the kept weights lie over the waves' runs
  u64 sum = 0, equal = 0;
  if (cut.v == -INFINITY && !(min_p > 0.0)) {
    row.each(
        [&](float v, int) { sum += weights.whole(weights.of(v)); });
  } else {
    row.each([&](float v, int) {
      if (v > cut.v) sum += weigh(v);
      equal += v == cut.v;
    });
  }
  sum = wave_sum(sum);
  equal = wave_sum(equal);
  __syncthreads();
  if (lane == 0) {
    lds.wave[0][wave] = sum;
    lds.wave[1][wave] = equal;
  }
  __syncthreads();
  auto kept_ties = [&](u64 before, u64 n) {
    return before >= cut.ties ? 0 : min(n, cut.ties - before);
  };
  // every wave finds the run with the target, a lane for each run (the lanes
  // behind the first 16 repeat them)
  const int run = lane & (kWaves - 1);
  const u64 run_ties = lds.wave[1][run];
  const u64 ties_before = wave_scan<true>(run_ties) - run_ties;
  const u64 own =
      lds.wave[0][run] + kept_ties(ties_before, run_ties) * tie_weight;
  const u64 run_upto = wave_scan<true>(own);
  const u64 total = lane_value(run_upto, kWaves - 1);
  const u64 target =
      floor_u64((double)uniform * (double)total, total - 1);
  const int owner = __builtin_ctzl(__ballot(target < run_upto));
  u64 upto = lane_value(run_upto - own, owner);
  const u64 ties = lane_value(ties_before, owner);
  // all threads share that run, each a few neighbours
  if (tid == owner * 64) {
    lds.answer[0] = row.first;
    lds.answer[1] = row.last;
  }
  __syncthreads();
  const int run_low = (int)lds.answer[0], run_high = (int)lds.answer[1];
  const int each = (run_high - run_low + kThreads - 1) / kThreads;
  const int first = min(run_high, run_low + tid * each);
  const int last = min(run_high, first + each);
  sum = equal = 0;
  for (int i = first; i < last; ++i) {
    const float v = row.at(i);
    if (v > cut.v) sum += weigh(v);
    equal += v == cut.v;
  }
  u64 rank = ties + block_scan(equal, lds.wave[1]);
  sum += kept_ties(rank, equal) * tie_weight;
  upto += block_scan(sum, lds.wave[0]);
  if (upto <= target && target < upto + sum) {
    for (int i = first; i < last; ++i) {
      const float v = row.at(i);
      if (v > cut.v)
        upto += weigh(v);
      else if (v == cut.v && rank++ < cut.ties)
        upto += tie_weight;
      if (upto > target) {
        a.out[number] = i;
        break;
      }
    }
  }
}

}  // namespace

torch::Tensor sample_tokens(torch::Tensor logits, torch::Tensor uniform,
                            c10::optional<torch::Tensor> temperature,
                            c10::optional<torch::Tensor> top_k,
                            c10::optional<torch::Tensor> top_p,
                            c10::optional<torch::Tensor> min_p,
                            double temperature_s, int64_t top_k_s,
                            double top_p_s, double min_p_s) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1,
              "sample: logits must be a 2-D GPU tensor with dense rows");
  const c10::hip::HIPGuard guard(logits.get_device());
  const long b = logits.size(0), v = logits.size(1);
  TORCH_CHECK(v >= 1 && v <= (1 << 20), "sample: 1 to 2^20 tokens");
  auto row_of = [&](const torch::Tensor& t, torch::ScalarType type) {
    TORCH_CHECK(t.device() == logits.device() && t.dim() == 1 &&
                    t.size(0) == b && t.is_contiguous() &&
                    t.scalar_type() == type,
                "sample: settings per row must be contiguous [b] tensors");
  };
  row_of(uniform, torch::kFloat32);
  for (auto* t : {&temperature, &top_p, &min_p})
    if (t->has_value()) row_of(**t, torch::kFloat32);
  if (top_k.has_value()) row_of(*top_k, torch::kLong);
  auto out = torch::empty({b}, logits.options().dtype(torch::kLong));
  if (b == 0) return out;

  SampleArgs a;
  a.logits = logits.data_ptr();
  a.row_stride = logits.stride(0);
  a.uniform = uniform.data_ptr<float>();
  a.out = out.data_ptr<long>();
  a.vocab = (int)v;
  a.shift = 51;
  while (v > (1l << (62 - a.shift))) --a.shift;
  auto f = [](const c10::optional<torch::Tensor>& t) {
    return t.has_value() ? t->data_ptr<float>() : nullptr;
  };
  a.temperature = f(temperature);
  a.top_p = f(top_p);
  a.min_p = f(min_p);
  a.top_k = top_k.has_value() ? top_k->data_ptr<long>() : nullptr;
  a.temperature_s = temperature_s;
  a.top_p_s = top_p_s;
  a.min_p_s = min_p_s;
  a.top_k_s = top_k_s;
  auto stream = c10::hip::getCurrentHIPStream();
#define LAUNCH_SAMPLE(T)                                                     \
  hipLaunchKernelGGL((sample_kernel<T>), dim3(b), dim3(kThreads), 0, stream, \
                     a)
  switch (logits.scalar_type()) {
    case torch::kFloat32: LAUNCH_SAMPLE(float); break;
    case torch::kBFloat16: LAUNCH_SAMPLE(__hip_bfloat16); break;
    case torch::kFloat16: LAUNCH_SAMPLE(__half); break;
    default: TORCH_CHECK(false, "sample: fp32, bf16 or fp16 logits only");
  }
#undef LAUNCH_SAMPLE
  HIP_CHECK(hipGetLastError());
  return out;
}
