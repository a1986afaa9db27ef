// Rotary positions for query and key in one launch: interleaved or half
// layout, part of the head, a position per token.
//
//   q, k:      [s, b, n | nkv, h] strided, head_dim dense (fp32/bf16/fp16)
//   cos, sin:  [S, r] fp32, r <= h / 2; any frequency scaling is in the tables
//   positions: [b, s] int64 strided, or none: token i of a sequence is at i
//
// A pair (x1, x2) of position p and frequency j becomes
//   (x1 c - x2 s, x2 c + x1 s),  c = cos[p, j], s = sin[p, j]
// with the pair at (2j, 2j + 1) (interleaved) or (j, j + r) (half); values
// past 2r are copied. The backward pass is the transpose: the same with -s.
// A position outside the tables gives NaN; the tables are never read there.
//
// Memory bounds it: each value is read and written once, at three operations.
// 4096 x 4 tokens of 64 heads of 128 values in bf16 take 100 us a direction,
// 5.4 TB/s, a little over what a copy of 2 GB reaches here (4.9); 107 with the
// loads parted by branches, 350 with a pair a thread, which is what widths,
// strides and addresses that do not fill 16 bytes get.

#include "common.h"

#include <torch/extension.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>

namespace {

struct RotaryTensor {
  const void* x;
  void* y;             // [s, b, heads, h] contiguous
  long ss, bs, ns;     // strides of x in elements
  int heads;
};

// One thread per pair or, past the pairs, per copied value: any strides and
// widths.
template <typename T>
__global__ __launch_bounds__(256) void rotary_kernel(
    RotaryTensor q, RotaryTensor k, const float* __restrict__ cos_t,
    const float* __restrict__ sin_t, const long* __restrict__ positions,
    long p_bs, long p_ss, long tokens, int b, int h, int r, long table_rows,
    bool interleaved, float sign) {
  const int units = h - r;  // r pairs and h - 2r copied values
  const int heads = q.heads + k.heads;
  const long total = tokens * heads * units;
  for (long idx = (long)blockIdx.x * 256 + threadIdx.x; idx < total;
       idx += (long)gridDim.x * 256) {
    const int u = idx % units;
    const long rest = idx / units;
    int head = rest % heads;
    const long token = rest / heads;
    const int ib = token % b;
    const long is = token / b;
    const RotaryTensor& t = head < q.heads ? q : k;
    if (head >= q.heads) head -= q.heads;
    const T* x = (const T*)t.x + is * t.ss + ib * t.bs + head * t.ns;
    T* y = (T*)t.y + (token * t.heads + head) * h;
    if (u >= r) {
      y[r + u] = x[r + u];
      continue;
    }
    const long p = positions ? positions[ib * p_bs + is * p_ss] : is;
    const bool inside = p >= 0 && p < table_rows;
    const float c = inside ? cos_t[p * r + u] : NAN;
    const float s = inside ? sin_t[p * r + u] * sign : NAN;
    const int i1 = interleaved ? 2 * u : u;
    const int i2 = interleaved ? 2 * u + 1 : u + r;
    const float x1 = DTypeTraits<T>::to_float(x[i1]);
    const float x2 = DTypeTraits<T>::to_float(x[i2]);
    y[i1] = DTypeTraits<T>::from_float(x1 * c - x2 * s);
    y[i2] = DTypeTraits<T>::from_float(x2 * c + x1 * s);
  }
}

// 16 bytes a lane. A workgroup takes one token and a run of heads: each thread
// keeps its place in the head, so that the tables' values stay in registers
// while it goes from head to head, four of them in flight.
//
// A unit is a vector of a head (interleaved: its pairs are in it; past the
// pairs: copied) or, in the half layout, a vector and its partners r further.
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_vec_kernel(
    RotaryTensor q, RotaryTensor k, const float* __restrict__ cos_t,
    const float* __restrict__ sin_t, const long* __restrict__ positions,
    long p_bs, long p_ss, int b, int h, int r, long table_rows, float sign,
    int heads_each) {
  constexpr int kVec = 16 / sizeof(T);
  constexpr int kTurns = INTERLEAVED ? kVec / 2 : kVec;  // table values
  constexpr int kFlight = 4;
  using Vec = union {
    uint4 u;
    T t[kVec];
  };
  const int units = (INTERLEAVED ? h : h - r) / kVec;
  const int side = 256 / units;  // heads side by side
  const int unit = threadIdx.x % units;
  const int line = threadIdx.x / units;
  if (line >= side) return;
  const long token = blockIdx.x;
  const int is = (unsigned)token / (unsigned)b;
  const int ib = token - (long)is * b;
  const int heads = q.heads + k.heads;
  const int first = blockIdx.y * heads_each + line;
  const int last = min(heads, (int)(blockIdx.y + 1) * heads_each);
  // where the unit lies, and whether it turns
  const bool turns = INTERLEAVED ? unit * kVec < 2 * r : unit * kVec < r;
  const int at = INTERLEAVED || turns ? unit * kVec : unit * kVec + r;

  float c[kTurns], s[kTurns];
  if (turns) {
    const long p = positions ? positions[ib * p_bs + is * p_ss] : is;
    const bool inside = p >= 0 && p < table_rows;
    const int j = INTERLEAVED ? at / 2 : at;
    if (inside) {  // once for all, so that the values come together
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        c[i] = cos_t[p * r + j + i];
        s[i] = sin_t[p * r + j + i] * sign;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kTurns; ++i) c[i] = s[i] = NAN;
    }
  }
  for (int base = first; base < last; base += kFlight * side) {
    Vec x[kFlight], z[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      // behind the last head that one again: no branch parts the loads
      const int head = min(base + f * side, last - 1);
      const bool is_q = head < q.heads;
      const T* from =
          is_q ? (const T*)q.x + is * q.ss + ib * q.bs + head * q.ns
               : (const T*)k.x + is * k.ss + ib * k.bs +
                     (head - q.heads) * k.ns;
      x[f].u = *(const uint4*)(from + at);
      if (!INTERLEAVED) z[f].u = *(const uint4*)(from + (turns ? at + r : at));
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int head = base + f * side;
      if (head < last) {
        const bool is_q = head < q.heads;
        T* to = is_q ? (T*)q.y + (token * q.heads + head) * h
                     : (T*)k.y + (token * k.heads + head - q.heads) * h;
        if (turns) {
#pragma unroll
          for (int i = 0; i < kTurns; ++i) {
            T& t1 = INTERLEAVED ? x[f].t[2 * i] : x[f].t[i];
            T& t2 = INTERLEAVED ? x[f].t[2 * i + 1] : z[f].t[i];
            const float x1 = DTypeTraits<T>::to_float(t1);
            const float x2 = DTypeTraits<T>::to_float(t2);
            t1 = DTypeTraits<T>::from_float(x1 * c[i] - x2 * s[i]);
            t2 = DTypeTraits<T>::from_float(x2 * c[i] + x1 * s[i]);
          }
          if (!INTERLEAVED) *(uint4*)(to + at + r) = z[f].u;
        }
        *(uint4*)(to + at) = x[f].u;
      }
    }
  }
}

}  // namespace

std::vector<torch::Tensor> rotary_apply(
    torch::Tensor q, c10::optional<torch::Tensor> k, torch::Tensor cos,
    torch::Tensor sin, c10::optional<torch::Tensor> positions,
    bool interleaved, bool inverse) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 4 && q.stride(3) == 1,
              "rotary: query must be a 4-D GPU tensor with dense head_dim");
  const c10::hip::HIPGuard guard(q.get_device());
  const long s = q.size(0), b = q.size(1);
  const int h = q.size(3);
  TORCH_CHECK(cos.device() == q.device() && sin.device() == q.device() &&
                  cos.scalar_type() == torch::kFloat32 &&
                  sin.scalar_type() == torch::kFloat32 && cos.dim() == 2 &&
                  cos.sizes() == sin.sizes() && cos.is_contiguous() &&
                  sin.is_contiguous(),
              "rotary: cos and sin must be contiguous fp32 tables alike");
  const long rows = cos.size(0);
  const int r = cos.size(1);
  TORCH_CHECK(r >= 1 && 2 * r <= h, "rotary: tables wider than the head");
  const long* pos = nullptr;
  long p_bs = 0, p_ss = 0;
  if (positions.has_value()) {
    TORCH_CHECK(positions->device() == q.device() &&
                    positions->scalar_type() == torch::kLong &&
                    positions->dim() == 2 && positions->size(0) == b &&
                    positions->size(1) == s,
                "rotary: positions must be int64 [b, s]");
    pos = positions->data_ptr<long>();
    p_bs = positions->stride(0);
    p_ss = positions->stride(1);
  } else {
    TORCH_CHECK(rows >= s, "rotary: tables shorter than the sequence");
  }
  auto yq = torch::empty({s, b, q.size(2), h}, q.options());
  std::vector<torch::Tensor> out = {yq};
  RotaryTensor tq{q.data_ptr(), yq.data_ptr(), q.stride(0), q.stride(1),
                  q.stride(2), (int)q.size(2)};
  RotaryTensor tk{nullptr, nullptr, 0, 0, 0, 0};
  if (k.has_value()) {
    TORCH_CHECK(k->device() == q.device() && k->dim() == 4 &&
                    k->stride(3) == 1 && k->size(0) == s && k->size(1) == b &&
                    k->size(3) == h && k->scalar_type() == q.scalar_type(),
                "rotary: key must match the query");
    auto yk = torch::empty({s, b, k->size(2), h}, q.options());
    tk = RotaryTensor{k->data_ptr(), yk.data_ptr(), k->stride(0),
                      k->stride(1), k->stride(2), (int)k->size(2)};
    out.push_back(yk);
  }
  const long total = s * b * (tq.heads + tk.heads) * (long)(h - r);
  if (total == 0) return out;
  auto stream = c10::hip::getCurrentHIPStream();

  // vectors: all rows on 16 bytes, and pairs that fill whole vectors
  const int vec = 16 / (int)q.element_size();
  auto wide = [&](const RotaryTensor& t) {
    return (unsigned long)t.x % 16 == 0 && t.ss % vec == 0 &&
           t.bs % vec == 0 && t.ns % vec == 0;
  };
  const int units = (interleaved ? h : h - r) / vec;
  if (wide(tq) && wide(tk) && h % vec == 0 &&
      (interleaved ? 2 * r : r) % vec == 0 && units <= 256 &&
      s * b < (1l << 31)) {
    // a workgroup goes over all heads of a token, unless there are so few
    // tokens that their heads have to fill the card (at 16 tokens of 40 heads
    // one round each takes 3.0 us, all rounds 3.3)
    const int heads = tq.heads + tk.heads, side = 256 / units;
    const int rounds = (heads + side - 1) / side;
    const int split =
        (int)std::max<long>(1, std::min<long>(rounds, 2048 / (s * b)));
    const int heads_each = (rounds + split - 1) / split * side;
    const dim3 grid((unsigned)(s * b), (heads + heads_each - 1) / heads_each);
#define LAUNCH_ROTARY_VEC(T, I)                                              \
  hipLaunchKernelGGL((rotary_vec_kernel<T, I>), grid, dim3(256), 0, stream,  \
                     tq, tk, cos.data_ptr<float>(), sin.data_ptr<float>(),   \
                     pos, p_bs, p_ss, (int)b, h, r, rows,                    \
                     inverse ? -1.f : 1.f, heads_each)
#define LAUNCH_ROTARY_LAYOUT(T)                                              \
  do {                                                                       \
    if (interleaved) LAUNCH_ROTARY_VEC(T, true);                             \
    else LAUNCH_ROTARY_VEC(T, false);                                        \
  } while (0)
    switch (q.scalar_type()) {
      case torch::kFloat32: LAUNCH_ROTARY_LAYOUT(float); break;
      case torch::kBFloat16: LAUNCH_ROTARY_LAYOUT(__hip_bfloat16); break;
      case torch::kFloat16: LAUNCH_ROTARY_LAYOUT(__half); break;
      default: TORCH_CHECK(false, "rotary: fp32, bf16 or fp16 only");
    }
#undef LAUNCH_ROTARY_LAYOUT
#undef LAUNCH_ROTARY_VEC
    HIP_CHECK(hipGetLastError());
    return out;
  }
  const int grid = (int)std::min<long>((total + 255) / 256, 32768);
#define LAUNCH_ROTARY(T)                                                     \
  hipLaunchKernelGGL((rotary_kernel<T>), dim3(grid), dim3(256), 0, stream,   \
                     tq, tk, cos.data_ptr<float>(), sin.data_ptr<float>(),   \
                     pos, p_bs, p_ss, s * b, (int)b, h, r, rows,             \
                     interleaved, inverse ? -1.f : 1.f)
  switch (q.scalar_type()) {
    case torch::kFloat32: LAUNCH_ROTARY(float); break;
    case torch::kBFloat16: LAUNCH_ROTARY(__hip_bfloat16); break;
    case torch::kFloat16: LAUNCH_ROTARY(__half); break;
    default: TORCH_CHECK(false, "rotary: fp32, bf16 or fp16 only");
  }
#undef LAUNCH_ROTARY
  HIP_CHECK(hipGetLastError());
  return out;
}
