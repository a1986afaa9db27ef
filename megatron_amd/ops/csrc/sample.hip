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
// vocabulary): their sums are exact in any order, so that filters and draw
// agree with each other and from run to run. Exponentials are taken in 64
// bits, since a draw hangs on sums that lie next to a border.
//
// A row with a NaN, or with no logit above -inf, gives -1.

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
constexpr int kList = 256;  // candidates that are ranked one against another

struct Lds {
  u64 mass[kBins];
  unsigned count[kBins];
  u64 list_weight[kList];
  unsigned list_key[kList];
  u64 wave[2][kWaves];
  double power[64];  // 2^(j / 64)
  u64 answer[4];
  unsigned listed, low, high;
};

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, u64* lds, F join) {
  for (int o = 32; o > 0; o >>= 1) v = join(v, __shfl_xor(v, o, WAVE_SIZE));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  V all = (V)lds[0];
  for (int w = 1; w < kWaves; ++w) all = join(all, (V)lds[w]);
  return all;
}

template <typename V>
__device__ __forceinline__ V block_sum(V v, u64* lds) {
  return block_reduce(v, lds, [](V a, V b) { return a + b; });
}

// sum of the values of all threads before this one
__device__ __forceinline__ u64 block_scan(u64 v, u64* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 up = v;
  for (int o = 1; o < 64; o <<= 1) {
    const u64 other = __shfl_up(up, o, WAVE_SIZE);
    if (lane >= o) up += other;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = up;
  __syncthreads();
  for (int w = 0; w < wave; ++w) up += lds[w];
  return up - v;
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
    const int wave = threadIdx.x >> 6;
    first = min(vocab, max(0, wave * run - shift));
    last = min(vocab, (wave + 1) * run - shift);
  }

  __device__ __forceinline__ float at(int i) const {
    return DTypeTraits<T>::to_float(x[i]);
  }

  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int lane = threadIdx.x & 63;
    // the run's begin lies on 16 bytes, but for the row's own
    const int begin = first == 0 ? -shift : first;
    for (int base = begin; base < last; base += kBatch * WAVE_SIZE * kVec) {
      union {
        uint4 u;
        T t[kVec];
      } v[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int i = base + (k * WAVE_SIZE + lane) * kVec;
        if (i >= 0 && i + kVec <= last) {
          v[k].u = *(const uint4*)(x + i);
        } else {
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            if (i + e >= 0 && i + e < last) v[k].t[e] = x[i + e];
        }
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int i = base + (k * WAVE_SIZE + lane) * kVec;
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (i + e >= 0 && i + e < last)
            f(DTypeTraits<T>::to_float(v[k].t[e]));
      }
    }
  }
};

// Weights of a row: 2^y with y = (x - top) / T log2 e <= 0, from a table of
// 2^(j / 64) and a polynomial of the fourth degree on the rest, which is at
// most ln 2 / 128 (relative error under 2^-44).
struct Weights {
  float top;
  double per;  // log2 e / T, 64 times
  int shift;
  const double* power;

  __device__ __forceinline__ double of(float v) const {
    if (v == top) return 1.0;
    const double y = fmax(((double)v - (double)top) * per, -64.0 * 1000.0);
    const double k = rint(y);
    const double r = (y - k) * (0.6931471805599453 / 64);
    double p = fma(r, 1.0 / 24, 1.0 / 6);
    p = fma(r, p, 0.5);
    p = fma(r, p, 1.0);
    p = fma(r, p, 1.0);
    const int n = (int)k;
    return ldexp(p * power[n & 63], n >> 6);
  }
  __device__ __forceinline__ u64 whole(double w) const {
    const double high = trunc(ldexp(w, shift - 32));
    const unsigned h = (unsigned)high;
    return (u64)h << 32 | (unsigned)ldexp(ldexp(w, shift - 32) - high, 32);
  }
  __device__ __forceinline__ u64 whole_of(float v) const {
    return whole(of(v));
  }
};

// Tokens with a larger key are kept, and the first `ties` of those with this.
struct Cut {
  unsigned key;
  u64 ties;
};

// Down from the largest key, where `limit` is passed: by count (MASS false)
// the key of the limit-th token, by mass the least key whose larger ones weigh
// at most `limit`. Tokens above `floor` count, which more than `limit` have;
// low..high are their extreme keys, both finite.
//
// Each step shares the keys' range out over bins, finds the bin in which the
// limit is passed and goes on within it, until it is one key or few tokens.
template <bool MASS, typename T>
__device__ Cut find_cut(Lds& lds, const Row<T>& row, const Weights& weights,
                        unsigned low, unsigned high, u64 limit) {
  const int tid = threadIdx.x;
  u64 above = 0;  // count or mass of the keys over `high`
  for (int step = 0; low < high; ++step) {
    if (step == 8) {  // ranges that bins cannot tell apart: bit by bit
      while (low < high) {
        const unsigned t = low + (high - low) / 2;
        u64 part = 0;
        row.each([&](float v) {
          if (order_key(v) > t) part += MASS ? weights.whole_of(v) : 1;
        });
        part = block_sum(part, lds.wave[0]);
        if (MASS ? part <= limit : part < limit)
          high = t;
        else
          low = t + 1;
      }
      u64 part = 0;
      row.each([&](float v) {
        if (order_key(v) > low) part += MASS ? weights.whole_of(v) : 1;
      });
      above = block_sum(part, lds.wave[0]);
      break;
    }
    const float base = 0.5f * key_value(low);
    const float scale =
        fminf(kBins / (0.5f * key_value(high) - base), 3e38f);
    auto bin_of = [&](float v) {
      return min(kBins - 1, (int)((0.5f * v - base) * scale));
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
    row.each([&](float v) {
      const unsigned key = order_key(v);
      if (key < low || key > high) return;
      const int bin = bin_of(v);
      if (MASS)
        atomicAdd(&lds.mass[bin], weights.whole_of(v));
      else
        atomicAdd(&lds.count[bin], 1u);
    });
    __syncthreads();
    // thread t has the bins from the top: 2t and 2t + 1
    constexpr int kEach = kBins / kThreads;
    u64 own[kEach], sum = 0;
    for (int e = 0; e < kEach; ++e) {
      const int bin = kBins - 1 - (tid * kEach + e);
      own[e] = MASS ? lds.mass[bin] : lds.count[bin];
      sum += own[e];
    }
    u64 upto = above + block_scan(sum, lds.wave[0]);
    for (int e = 0; e < kEach; ++e) {
      const bool here = MASS ? upto <= limit && upto + own[e] > limit
                             : upto < limit && upto + own[e] >= limit;
      if (here) {
        lds.answer[0] = kBins - 1 - (tid * kEach + e);
        lds.answer[1] = upto;
      }
      upto += own[e];
    }
    __syncthreads();
    const int bin = (int)lds.answer[0];
    above = lds.answer[1];
    unsigned least = ~0u, most = 0;
    row.each([&](float v) {
      const unsigned key = order_key(v);
      if (key < low || key > high || bin_of(v) != bin) return;
      least = min(least, key);
      most = max(most, key);
      const unsigned at = atomicAdd(&lds.listed, 1u);
      if (at < kList) {
        lds.list_key[at] = key;
        if (MASS) lds.list_weight[at] = weights.whole_of(v);
      }
    });
    if (most) {
      atomicMin(&lds.low, least);
      atomicMax(&lds.high, most);
    }
    __syncthreads();
    low = lds.low;
    high = lds.high;
    const int listed = (int)lds.listed;
    if (low < high && listed <= kList) {
      if (tid < listed) {
        const unsigned key = lds.list_key[tid];
        u64 over = above, equal = 0;
        for (int j = 0; j < listed; ++j) {
          const unsigned other = lds.list_key[j];
          const u64 w = MASS ? lds.list_weight[j] : 1;
          if (other > key) over += w;
          if (other == key) equal += w;
        }
        if (MASS ? over <= limit && over + equal > limit
                 : over < limit && over + equal >= limit) {
          lds.answer[2] = key;
          lds.answer[3] = over;
        }
      }
      __syncthreads();
      low = high = (unsigned)lds.answer[2];
      above = lds.answer[3];
    }
    __syncthreads();
  }
  if (!MASS) return Cut{low, limit - above};
  const u64 w = weights.whole_of(key_value(low));
  return Cut{low, w ? (limit - above) / w + 1 : (u64)row.vocab};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ Lds lds;
  const long number = blockIdx.x;
  const int tid = threadIdx.x, V = a.vocab;
  const Row<T> row((const T*)a.logits + number * a.row_stride, V);

  double temperature =
      a.temperature ? a.temperature[number] : a.temperature_s;
  long top_k = a.top_k ? a.top_k[number] : a.top_k_s;
  const double top_p = a.top_p ? a.top_p[number] : a.top_p_s;
  double min_p = a.min_p ? a.min_p[number] : a.min_p_s;
  if (!(temperature > 0.0)) {  // greedy
    temperature = 1.0;
    top_k = 1;
  }
  temperature = fmin(temperature, 1e30);
  if (top_k <= 0) top_k = V;
  if (min_p > 1.0) min_p = 1.0;

  if (tid < 64) lds.power[tid] = exp2(tid / 64.0);
  // extreme keys of the logits above -inf, and how many those are
  unsigned high = 0, low = ~0u, some = 0, bad = 0;
  row.each([&](float v) {
    bad |= v != v;
    const unsigned key = order_key(v);
    high = max(high, key);
    if (v > -INFINITY) {
      low = min(low, key);
      ++some;
    }
  });
  auto larger = [](unsigned x, unsigned y) { return max(x, y); };
  high = block_reduce(bad ? ~0u : high, lds.wave[0], larger);
  if (high == ~0u || high == order_key(-INFINITY)) {
    if (tid == 0) a.out[number] = -1;
    return;
  }
  const float top = key_value(high);
  const Weights weights{top, 64.0 * 1.4426950408889634 / temperature, a.shift,
                        lds.power};

  const bool by_mass = top_p > 0.0 && top_p < 1.0;
  Cut cut{0, (u64)V};
  if (top == INFINITY) {  // the others weigh nothing
    cut = Cut{high, (u64)top_k};
  } else if (top_k == 1) {
    cut = Cut{high, 1};
  } else if (top_k < V || by_mass) {
    low = block_reduce(low, lds.wave[1],
                       [](unsigned x, unsigned y) { return min(x, y); });
    const u64 above = block_sum((u64)some, lds.wave[0]);
    cut.key = low;  // below come those that weigh nothing
    if ((u64)top_k < above)
      cut = find_cut<false>(lds, row, weights, low, high, (u64)top_k);
  }
  if (by_mass) {
    u64 mass = 0, equal = 0;
    unsigned next = ~0u;  // the least key over the cut
    row.each([&](float v) {
      const unsigned key = order_key(v);
      if (key > cut.key) {
        mass += weights.whole_of(v);
        next = min(next, key);
      }
      equal += key == cut.key;
    });
    mass = block_sum(mass, lds.wave[0]);
    equal = min(block_sum(equal, lds.wave[1]), cut.ties);
    const u64 each = weights.whole_of(key_value(cut.key));
    const u64 all = mass + equal * each;
    const u64 most = floor_u64(top_p * (double)all, all);
    if (mass <= most) {
      if (each) cut.ties = min(cut.ties, (most - mass) / each + 1);
    } else {
      next = block_reduce(next, lds.wave[0], [](unsigned x, unsigned y) {
        return min(x, y);
      });
      cut = find_cut<true>(lds, row, weights, next, high, most);
    }
  }

  auto weigh = [&](float v) -> u64 {
    const double w = weights.of(v);
    return w < min_p ? 0 : weights.whole(w);
  };
  const u64 tie_weight = weigh(key_value(cut.key));
  // how the kept weights lie over the waves' runs
  u64 sum = 0, equal = 0;
  row.each([&](float v) {
    const unsigned key = order_key(v);
    if (key > cut.key) sum += weigh(v);
    equal += key == cut.key;
  });
  for (int o = 32; o > 0; o >>= 1) {
    sum += __shfl_xor(sum, o, WAVE_SIZE);
    equal += __shfl_xor(equal, o, WAVE_SIZE);
  }
  __syncthreads();
  if ((tid & 63) == 0) {
    lds.wave[0][tid >> 6] = sum;
    lds.wave[1][tid >> 6] = equal;
  }
  __syncthreads();
  auto kept_ties = [&](u64 before, u64 n) {
    return before >= cut.ties ? 0 : min(n, cut.ties - before);
  };
  u64 total = 0, ties = 0;
  for (int w = 0; w < kWaves; ++w) {
    total += lds.wave[0][w] + kept_ties(ties, lds.wave[1][w]) * tie_weight;
    ties += lds.wave[1][w];
  }
  const u64 target =
      floor_u64((double)a.uniform[number] * (double)total, total - 1);
  u64 upto = 0;
  ties = 0;
  int owner = 0;
  for (; owner < kWaves; ++owner) {
    const u64 here = lds.wave[0][owner] +
                     kept_ties(ties, lds.wave[1][owner]) * tie_weight;
    if (target < upto + here) break;
    upto += here;
    ties += lds.wave[1][owner];
  }
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
    const unsigned key = order_key(v);
    if (key > cut.key) sum += weigh(v);
    equal += key == cut.key;
  }
  u64 rank = ties + block_scan(equal, lds.wave[1]);
  sum += kept_ties(rank, equal) * tie_weight;
  upto += block_scan(sum, lds.wave[0]);
  if (upto <= target && target < upto + sum) {
    for (int i = first; i < last; ++i) {
      const float v = row.at(i);
      const unsigned key = order_key(v);
      if (key > cut.key)
        upto += weigh(v);
      else if (key == cut.key && rank++ < cut.ties)
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
  a.shift = 62;
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
