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

template <typename V>
__device__ __forceinline__ V block_sum(V v, V* lds) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE_SIZE);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  V total = 0;
  for (int w = 0; w < kWaves; ++w) total += lds[w];
  return total;
}

// sum of the values of all threads before this one
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  V up = v;
  for (int o = 1; o < 64; o <<= 1) {
    const V other = __shfl_up(up, o, WAVE_SIZE);
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

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ u64 lds[kWaves];
  const long row = blockIdx.x;
  const T* x = (const T*)a.logits + row * a.row_stride;
  const int tid = threadIdx.x, V = a.vocab;

  double temperature = a.temperature ? a.temperature[row] : a.temperature_s;
  long top_k = a.top_k ? a.top_k[row] : a.top_k_s;
  double top_p = a.top_p ? a.top_p[row] : a.top_p_s;
  double min_p = a.min_p ? a.min_p[row] : a.min_p_s;
  if (!(temperature > 0.0)) {  // greedy
    temperature = 1.0;
    top_k = 1;
  }
  temperature = fmin(temperature, 1e30);
  if (top_k <= 0 || top_k > V) top_k = V;
  if (min_p > 1.0) min_p = 1.0;

  unsigned key_max = 0;
  u64 bad = 0;
  for (int i = tid; i < V; i += kThreads) {
    const float v = DTypeTraits<T>::to_float(x[i]);
    bad += v != v;
    key_max = max(key_max, order_key(v));
  }
  bad = block_sum(bad, lds);
  for (int o = 32; o > 0; o >>= 1)
    key_max = max(key_max, (unsigned)__shfl_xor((int)key_max, o, WAVE_SIZE));
  __syncthreads();
  if ((tid & 63) == 0) lds[tid >> 6] = key_max;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) key_max = max(key_max, (unsigned)lds[w]);
  if (bad || key_max == order_key(-INFINITY)) {
    if (tid == 0) a.out[row] = -1;
    return;
  }
  const float top = __uint_as_float(
      key_max & 0x80000000u ? key_max & 0x7fffffffu : ~key_max);
  const double inv = 1.0 / temperature;
  const double unit = (double)(1ull << a.shift);
  auto weight = [&](float v) {
    return v == top ? 1.0 : exp(((double)v - (double)top) * inv);
  };
  auto whole = [&](double w) { return (u64)rint(w * unit); };

  // tokens with a larger key than cut are kept, and the first `ties` of those
  // with this key
  unsigned cut = 0;
  u64 ties = V;
  if (top_k < V) {
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned t = cut | (1u << bit);
      u64 n = 0;
      for (int i = tid; i < V; i += kThreads)
        n += order_key(DTypeTraits<T>::to_float(x[i])) >= t;
      if (block_sum(n, lds) >= (u64)top_k) cut = t;
    }
    u64 n = 0;
    for (int i = tid; i < V; i += kThreads)
      n += order_key(DTypeTraits<T>::to_float(x[i])) > cut;
    ties = top_k - block_sum(n, lds);
  }
  if (top_p > 0.0 && top_p < 1.0) {
    u64 mass = 0, at_cut = 0;
    for (int i = tid; i < V; i += kThreads) {
      const float v = DTypeTraits<T>::to_float(x[i]);
      const unsigned key = order_key(v);
      if (key > cut) mass += whole(weight(v));
      at_cut += key == cut;
    }
    mass = block_sum(mass, lds);
    at_cut = block_sum(at_cut, lds);
    const float cut_value = __uint_as_float(
        cut & 0x80000000u ? cut & 0x7fffffffu : ~cut);
    if (at_cut) mass += min(ties, at_cut) * whole(weight(cut_value));
    const u64 most = floor_u64(top_p * (double)mass, mass);
    // the least key t whose larger tokens weigh at most `most`
    unsigned low = cut, high = key_max;
    while (low < high) {
      const unsigned t = low + (high - low) / 2;
      u64 m = 0;
      for (int i = tid; i < V; i += kThreads) {
        const float v = DTypeTraits<T>::to_float(x[i]);
        if (order_key(v) > t) m += whole(weight(v));
      }
      if (block_sum(m, lds) <= most) high = t; else low = t + 1;
    }
    u64 m = 0;
    for (int i = tid; i < V; i += kThreads) {
      const float v = DTypeTraits<T>::to_float(x[i]);
      if (order_key(v) > low) m += whole(weight(v));
    }
    m = block_sum(m, lds);
    const float value = __uint_as_float(
        low & 0x80000000u ? low & 0x7fffffffu : ~low);
    const u64 w = value == value ? whole(weight(value)) : 0;
    const u64 kept = w ? (most - m) / w + 1 : (u64)V;
    ties = low > cut ? kept : min(ties, kept);
    cut = low;
  }

  // each thread owns a run of indices, so that ties are counted in order
  const int each = (V + kThreads - 1) / kThreads;
  const int first = min(V, tid * each), last = min(V, first + each);
  u64 equal = 0;
  for (int i = first; i < last; ++i)
    equal += order_key(DTypeTraits<T>::to_float(x[i])) == cut;
  u64 rank = block_scan(equal, lds);
  u64 sum = 0, rank0 = rank;
  auto kept = [&](float v, u64& rank) -> u64 {
    const unsigned key = order_key(v);
    if (key < cut) return 0;
    if (key == cut && rank++ >= ties) return 0;
    const double w = weight(v);
    return w < min_p ? 0 : whole(w);
  };
  for (int i = first; i < last; ++i)
    sum += kept(DTypeTraits<T>::to_float(x[i]), rank);
  const u64 total = block_sum(sum, lds);
  u64 upto = block_scan(sum, lds);
  u64 target = floor_u64((double)a.uniform[row] * (double)total, total - 1);
  if (upto <= target && target < upto + sum) {
    for (int i = first; i < last; ++i) {
      upto += kept(DTypeTraits<T>::to_float(x[i]), rank0);
      if (upto > target) {
        a.out[row] = i;
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
