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
  __device__ __forceinline__ long of(int ib) const {
    return at ? at[ib * stride] : scalar;
  }
};

__host__ __device__ __forceinline__ int v_quarters(int h) {
  return h >= 64 ? h / 64 : 1;
}

// 16-bit piece of v_codes with 4 values (2 where h = 32) from value d on
__device__ __forceinline__ long v_piece(const CacheView& c, long bh, long t,
                                        int d) {
  const int per = c.h / 16, q = v_quarters(c.h);
  const int chunk = d / per, quarter = (d % per) / 4;
  const long block = (bh * (c.room / 4) + t / 4) * 16 + chunk;
  return (block * 2 * q + ((t >> 1) & 1) * q + quarter) * 2 + (t & 1);
}

__device__ __forceinline__ long v_meta_at(const CacheView& c, long bh, long t,
                                          int group) {
  return ((bh * (c.h / kGroup) + group) * (c.room / 4) + t / 4) * 8 + (t & 3);
}

// code of x: the nearest whole number of s above z, ties to even. The quotient
// in 32 bits is off by less than one code; 64-bit products decide.
__device__ __forceinline__ unsigned code_of(float x, float z, float s,
                                            float inv) {
  if (!(s > 0.f)) return 0;
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
  const unsigned code = (unsigned)n;
  const double twice = 2.0 * rest;
  const bool up = twice > (double)s || (twice == (double)s && (code & 1));
  return up && code < 15 ? code + 1 : code;
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

// A row (token, sequence, head) takes h / 8 lanes with 8 values each; four
// lanes share a group. Rows of q, if any, come behind those of k and v and
// are only rotated.
template <typename T>
__global__ __launch_bounds__(256) void append_kernel(
    CacheView cache, AppendSource k, AppendSource v, AppendSource q,
    T* __restrict__ q_out, int n, const float* __restrict__ cos_t,
    const float* __restrict__ sin_t, int r, long table_rows, bool interleaved,
    Start start, long s) {
  const int lanes = cache.h / 8;
  const long index = (long)blockIdx.x * 256 + threadIdx.x;
  const long row = index / lanes;
  const int part = index % lanes, d0 = part * 8;
  const long kv_rows = s * cache.b * cache.heads;
  const long rows = kv_rows + (q.x ? s * cache.b * n : 0);
  if (row >= rows) return;
  const bool is_q = row >= kv_rows;
  const int heads = is_q ? n : cache.heads;
  const long local = is_q ? row - kv_rows : row;
  const int head = local % heads;
  const int ib = (local / heads) % cache.b;
  const long is = local / heads / cache.b;
  const long t = start.of(ib);
  const bool idle = t < 0;
  const long pos = t + is;

  const float *cos_row = nullptr, *sin_row = nullptr;
  const bool turn = r > 0;
  const bool known = pos >= 0 && pos < table_rows;
  if (turn && known) {
    cos_row = cos_t + pos * r;
    sin_row = sin_t + pos * r;
  }
  auto value = [&](const T* x, int d) -> float {
    if (!turn) return DTypeTraits<T>::to_float(x[d]);
    if (!known && d < 2 * r) return NAN;
    return rotated<T>(x, cos_row, sin_row, d, r, interleaved);
  };

  if (is_q) {
    const T* x = (const T*)q.x + is * q.ss + ib * q.bs + head * q.ns;
    T* y = q_out + local * cache.h + d0;
    for (int i = 0; i < 8; ++i)
      y[i] = DTypeTraits<T>::from_float(idle ? 0.f : value(x, d0 + i));
    return;
  }
  if (idle || pos >= cache.capacity) return;  // a whole row returns together

  const T* kx = (const T*)k.x + is * k.ss + ib * k.bs + head * k.ns;
  const T* vx = (const T*)v.x + is * v.ss + ib * v.bs + head * v.ns;
  float kv[8], vv[8];
  bool nan_k = false, nan_v = false;
  float k_low = INFINITY, k_high = -INFINITY;
  float v_low = INFINITY, v_high = -INFINITY;
  for (int i = 0; i < 8; ++i) {
    const float a = value(kx, d0 + i);
    const float b = DTypeTraits<T>::to_float(vx[d0 + i]);
    nan_k |= a != a;
    nan_v |= b != b;
    kv[i] = a != a ? 0.f : fminf(fmaxf(a, -kHeldMax), kHeldMax);
    vv[i] = b != b ? 0.f : fminf(fmaxf(b, -kHeldMax), kHeldMax);
    k_low = fminf(k_low, kv[i]);
    k_high = fmaxf(k_high, kv[i]);
    v_low = fminf(v_low, vv[i]);
    v_high = fmaxf(v_high, vv[i]);
  }
  // lanes of a row share a wave: 64 is a multiple of h / 8
  for (int o = 1; o < 4; o <<= 1) {
    k_low = fminf(k_low, __shfl_xor(k_low, o, WAVE_SIZE));
    k_high = fmaxf(k_high, __shfl_xor(k_high, o, WAVE_SIZE));
    v_low = fminf(v_low, __shfl_xor(v_low, o, WAVE_SIZE));
    v_high = fmaxf(v_high, __shfl_xor(v_high, o, WAVE_SIZE));
  }
  int nan_group = nan_v, nan_row = nan_k || nan_v;
  for (int o = 1; o < 4; o <<= 1)
    nan_group |= __shfl_xor(nan_group, o, WAVE_SIZE);
  for (int o = 1; o < lanes; o <<= 1)
    nan_row |= __shfl_xor(nan_row, o, WAVE_SIZE);

  const __half k_z = __float2half(k_low), v_z = __float2half(v_low);
  const float kz = __half2float(k_z), vz = __half2float(v_z);
  __half k_s = __float2half(to_32(((double)k_high - (double)kz) / 15.0));
  __half v_s = __float2half(to_32(((double)v_high - (double)vz) / 15.0));
  const float ks = __half2float(k_s), vs = __half2float(v_s);
  const float k_inv = 1.f / ks, v_inv = 1.f / vs;
  unsigned k_word = 0, v_word = 0;
  for (int i = 0; i < 8; ++i) {
    k_word |= code_of(kv[i], kz, ks, k_inv) << ((i >> 1) * 4 + (i & 1) * 16);
    v_word |= code_of(vv[i], vz, vs, v_inv) << (i * 4);
  }
  const __half nan = __ushort_as_half(0x7e00);
  if (nan_row) k_s = nan;
  if (nan_group) v_s = nan;

  const long bh = (long)ib * cache.heads + head;
  const long tok = bh * cache.room + pos;
  *(unsigned*)(cache.k_codes + tok * (cache.h / 2) + part * 4) = k_word;
  unsigned short* pieces = (unsigned short*)cache.v_codes;
  if (cache.h >= 64) {
    pieces[v_piece(cache, bh, pos, d0)] = (unsigned short)v_word;
    pieces[v_piece(cache, bh, pos, d0 + 4)] = (unsigned short)(v_word >> 16);
  } else {  // a piece has two values
    for (int i = 0; i < 4; ++i)
      pieces[v_piece(cache, bh, pos, d0 + 2 * i)] = (v_word >> (8 * i)) & 255;
  }
  if ((part & 3) == 0) {
    const int group = part / 4;
    __half* m = cache.k_meta + (tok * (cache.h / kGroup) + group) * 2;
    m[0] = k_s;
    m[1] = k_z;
    __half* w = cache.v_meta + v_meta_at(cache, bh, pos, group);
    w[0] = v_s;
    w[4] = v_z;
  }
}

__device__ __forceinline__ float held_k(const CacheView& c, long bh, long t,
                                        int d) {
  const long tok = bh * c.room + t;
  const unsigned word =
      *(const unsigned*)(c.k_codes + tok * (c.h / 2) + d / 8 * 4);
  const int i = d & 7;
  const float code = (word >> ((i >> 1) * 4 + (i & 1) * 16)) & 15;
  const __half* m = c.k_meta + (tok * (c.h / kGroup) + d / kGroup) * 2;
  return __half2float(m[1]) + __half2float(m[0]) * code;
}

__device__ __forceinline__ float held_v(const CacheView& c, long bh, long t,
                                        int d) {
  const unsigned piece =
      ((const unsigned short*)c.v_codes)[v_piece(c, bh, t, d)];
  const int within = c.h >= 64 ? d % 4 : d % 2;
  const float code = (piece >> (within * 4)) & 15;
  const __half* m = c.v_meta + v_meta_at(c, bh, t, d / kGroup);
  return __half2float(m[4]) + __half2float(m[0]) * code;
}

// One thread per value; positions outside the cache read as NaN.
template <typename T>
__global__ __launch_bounds__(256) void dequantize_kernel(
    CacheView cache, Start start, long length, T* __restrict__ k_out,
    T* __restrict__ v_out) {
  const long total = length * cache.b * cache.heads * cache.h;
  for (long idx = (long)blockIdx.x * 256 + threadIdx.x; idx < total;
       idx += (long)gridDim.x * 256) {
    const int d = idx % cache.h;
    const long row = idx / cache.h;
    const int head = row % cache.heads;
    const int ib = (row / cache.heads) % cache.b;
    const long pos = start.of(ib) + row / cache.heads / cache.b;
    float k = NAN, v = NAN;
    if (pos >= 0 && pos < cache.capacity) {
      const long bh = (long)ib * cache.heads + head;
      k = held_k(cache, bh, pos, d);
      v = held_v(cache, bh, pos, d);
    }
    k_out[idx] = DTypeTraits<T>::from_float(k);
    v_out[idx] = DTypeTraits<T>::from_float(v);
  }
}

// One wave per query row: lanes share the tokens for the scores, then the
// values of a token for the output.
template <typename T>
__global__ __launch_bounds__(64) void attention_kernel(
    CacheView cache, const T* __restrict__ q, long q_ss, long q_bs, long q_ns,
    T* __restrict__ out, int n, Start start, float scale, long window,
    long sinks) {
  __shared__ float q_row[256];
  const int lane = threadIdx.x, h = cache.h;
  const int head = blockIdx.x, ib = blockIdx.y;
  const long is = blockIdx.z;
  const long bh = (long)ib * cache.heads + head / (n / cache.heads);
  T* o = out + ((is * cache.b + ib) * n + head) * h;
  const long t0 = start.of(ib), pos = t0 + is;
  if (t0 < 0 || pos >= cache.capacity) {
    for (int d = lane; d < h; d += 64)
      o[d] = DTypeTraits<T>::from_float(t0 < 0 ? 0.f : NAN);
    return;
  }
  const T* qx = q + is * q_ss + ib * q_bs + head * q_ns;
  for (int d = lane; d < h; d += 64)
    q_row[d] = DTypeTraits<T>::to_float(qx[d]) * scale;
  __syncthreads();
  float m = -INFINITY, sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (long base = 0; base <= pos; base += 64) {
    const long t = base + lane;
    const bool seen = t <= pos &&
                      (window <= 0 || t > pos - window || t < sinks);
    float score = -INFINITY;
    if (seen) {
      score = 0.f;
      for (int d = 0; d < h; ++d) score += q_row[d] * held_k(cache, bh, t, d);
    }
    if (!__any(seen)) continue;
    const bool broken = __any(score != score);
    const float peak = broken ? NAN : fmaxf(m, wave_reduce_max(score));
    const float alpha = m == -INFINITY ? 0.f : __expf(m - peak);
    const float p = seen ? __expf(score - peak) : 0.f;
    m = peak;
    sum = sum * alpha + wave_reduce_sum(p);
    for (int i = 0; i < 4; ++i) acc[i] *= alpha;
    for (int j = 0; j < 64; ++j) {
      const float pj = __shfl(p, j, WAVE_SIZE);
      if (!__shfl((int)seen, j, WAVE_SIZE)) continue;
      for (int i = 0; i < 4 && lane + 64 * i < h; ++i)
        acc[i] += pj * held_v(cache, bh, base + j, lane + 64 * i);
    }
  }
  for (int i = 0; i < 4 && lane + 64 * i < h; ++i)
    o[lane + 64 * i] = DTypeTraits<T>::from_float(acc[i] / sum);
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
  const long rows = s * cache.b * (cache.heads + (long)n);
  if (rows > 0) {
    const long grid = (rows * (cache.h / 8) + 255) / 256;
    TORCH_CHECK(grid < (1l << 31), "quant_kv: too many tokens at once");
    auto stream = c10::hip::getCurrentHIPStream();
#define LAUNCH_APPEND(T)                                                     \
  hipLaunchKernelGGL((append_kernel<T>), dim3(grid), dim3(256), 0, stream,   \
                     cache, source_of(key), source_of(value), q,             \
                     q.x ? (T*)q_out.data_ptr() : nullptr, n, cos_p, sin_p,  \
                     r, table_rows, interleaved, at, s)
    DISPATCH_HALF(key, LAUNCH_APPEND);
#undef LAUNCH_APPEND
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
  const int grid = (int)std::min<long>((k.numel() + 255) / 256, 32768);
  auto stream = c10::hip::getCurrentHIPStream();
#define LAUNCH_DEQUANTIZE(T)                                                 \
  hipLaunchKernelGGL((dequantize_kernel<T>), dim3(grid), dim3(256), 0,       \
                     stream, cache, at, (long)length, (T*)k.data_ptr(),      \
                     (T*)v.data_ptr())
  DISPATCH_HALF(k, LAUNCH_DEQUANTIZE);
#undef LAUNCH_DEQUANTIZE
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
  auto stream = c10::hip::getCurrentHIPStream();
  TORCH_CHECK(s < 65536 && cache.b < 65536);
  dim3 grid(n, cache.b, s);
#define LAUNCH_ATTENTION(T)                                                  \
  hipLaunchKernelGGL((attention_kernel<T>), grid, dim3(64), 0, stream,       \
                     cache, (const T*)query.data_ptr(), query.stride(0),     \
                     query.stride(1), query.stride(2), (T*)out.data_ptr(),   \
                     n, at, (float)scale, (long)window, (long)sinks)
  DISPATCH_HALF(query, LAUNCH_ATTENTION);
#undef LAUNCH_ATTENTION
  HIP_CHECK(hipGetLastError());
  return out;
}
