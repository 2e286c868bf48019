// Rotary positions of many tokens: queries and keys of a step in one launch, either pair layout, part
// of a head, any positions, and the gradient (the rotation by the negative angle).
#include "kv_layout.cuh"
#include "launchers.h"

namespace tcrv {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeTensors = 4;
constexpr uint32_t kRopeSmemPairs = 4096;  // angles of a CTA's tokens: 32 KB of (cos, sin)

struct RopeTensor {
  const void *x;
  void *y;
  size_t x_token, x_head, y_token, y_head;
  uint32_t first_head;  // of this tensor among all tensors' heads
};

struct RopeParams {
  RopeTensor tensor[kRopeTensors];
  uint32_t count, heads, dim, n_rot, cta_tokens, cta_heads;
  size_t tokens;
  const void *positions;
  const double *freqs;
  float magnitude;
  bool wide_positions;
  Divisor by_access, by_head;  // a head's accesses, a CTA's heads
};

// (cos, sin) of position * freq.  The product and its reduction to one turn are done in 64 bits: a
// float angle of a far position has lost the digits that the rotation depends on (at 2^20 radians its
// step is 1/16).  What is left, within half a turn either way, is rounded to f32: 2^-23 at most, below
// the rounding of the f32 cosine's own result.
__device__ __forceinline__ float2 rope_angle(double position, double freq, float magnitude, float sign) {
  const double turns = position * freq * 0.15915494309189535;  // 1 / (2 pi)
  // (the reduction goes by the angle itself: turns only says how many whole ones to take off)
  const double whole = rint(turns);
  const double rest = fma(-whole, 2.4492935982947064e-16, fma(-whole, 6.283185307179586, position * freq));
  float s, c;
  sincosf(static_cast<float>(rest), &s, &c);
  return make_float2(c * magnitude, s * magnitude * sign);
}

// The pair's rotation, the left product of each result fused as in rope_apply_kernel, so that a
// value's bits do not depend on the kernel that a call takes.
__device__ __forceinline__ float turn_lo(float u, float v, float2 r) { return __fmaf_rn(u, r.x, -__fmul_rn(v, r.y)); }
__device__ __forceinline__ float turn_hi(float u, float v, float2 r) { return __fmaf_rn(u, r.y, __fmul_rn(v, r.x)); }

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// A CTA takes cta_tokens tokens and cta_heads of the heads of all tensors: it works out the tokens'
// angles once (shared memory), then streams over the heads.  kN elements to an access (16 bytes, or
// one): with adjacent pairs an access holds kN / 2 pairs, in the halves layout two accesses hold kN.
// Bound by bytes: each element is read and written once; the angles cost one sincosf for each pair of
// a token, a fortieth of the elements at 40 heads.
template <typename T, bool kHalves, int kN, bool kInverse>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
  extern __shared__ float2 rope_cs[];
  pdl_enter();
  const uint32_t pairs = p.n_rot / 2;
  const size_t token0 = static_cast<size_t>(blockIdx.x) * p.cta_tokens;
  const uint32_t ntok = static_cast<uint32_t>(p.tokens - token0 < p.cta_tokens ? p.tokens - token0 : p.cta_tokens);
  for (uint32_t i = threadIdx.x; i < ntok * pairs; i += kRopeThreads) {
    const uint32_t t = i / pairs, pair = i - t * pairs;
    const double position = p.wide_positions ? static_cast<double>(static_cast<const int64_t *>(p.positions)[token0 + t])
                                             : static_cast<double>(static_cast<const int32_t *>(p.positions)[token0 + t]);
    rope_cs[i] = rope_angle(position, p.freqs[pair], p.magnitude, kInverse ? -1.0f : 1.0f);
  }
  __syncthreads();
  const uint32_t head0 = blockIdx.y * p.cta_heads;
  const uint32_t nheads = p.heads - head0 < p.cta_heads ? p.heads - head0 : p.cta_heads;
  using P = Pack<T, kN>;
  // accesses of a head: those that rotate, then those that copy
  constexpr uint32_t kStep = kHalves ? 1 : (kN > 1 ? 1 : 2);  // (single elements: a pair is two of them)
  const uint32_t turning = kHalves ? pairs / kN : p.n_rot / (kN * kStep);
  const uint32_t per_head = turning + (p.dim - p.n_rot) / kN;
  const uint32_t items = ntok * nheads * per_head;
  // Two 16-byte loads to a thread before the first store, for 64 warps of one each do not cover the memory's latency
  // (2047 tokens, half of each head of 128, f32: 43 us with one, 28 with two).  An item of the halves layout is two by itself
  // and goes alone: two items cost the registers of a CTA (8192 tokens, bf16: 32 us with one, 44 with two).
  if constexpr (kHalves) {
    for (uint32_t i = threadIdx.x; i < items; i += kRopeThreads) {
      const uint32_t row = p.by_access.of(i), a = i - row * per_head;
      const uint32_t t = nheads == p.cta_heads ? p.by_head.of(row) : row / nheads, head = head0 + (row - t * nheads);
      uint32_t w = 0;
#pragma unroll
      for (int j = 1; j < kRopeTensors; ++j)
        w += j < p.count && head >= p.tensor[j].first_head;
      const RopeTensor &tensor = p.tensor[w];
      const size_t token = token0 + t, h = head - tensor.first_head;
      const T *x = static_cast<const T *>(tensor.x) + token * tensor.x_token + h * tensor.x_head;
      T *y = static_cast<T *>(tensor.y) + token * tensor.y_token + h * tensor.y_head;
      const float2 *cs = rope_cs + t * pairs;
      if (a >= turning) {
        const uint32_t at = p.n_rot + (a - turning) * kN;
        if (tensor.x != tensor.y)
          *reinterpret_cast<P *>(y + at) = *reinterpret_cast<const P *>(x + at);
      } else {
        const P lo = *reinterpret_cast<const P *>(x + a * kN), hi = *reinterpret_cast<const P *>(x + pairs + a * kN);
        P ylo, yhi;
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          const float2 r = cs[a * kN + e];
          const float u = to_float(lo.v[e]), v = to_float(hi.v[e]);
          ylo.v[e] = from_float<T>(turn_lo(u, v, r));
          yhi.v[e] = from_float<T>(turn_hi(u, v, r));
        }
        *reinterpret_cast<P *>(y + a * kN) = ylo;
        *reinterpret_cast<P *>(y + pairs + a * kN) = yhi;
      }
    }
    return;
  }
  constexpr int kAtOnce = 2;
  for (uint32_t i0 = threadIdx.x; i0 < items; i0 += kAtOnce * kRopeThreads) {
    P lo[kAtOnce], hi[kAtOnce];
    T *to[kAtOnce];
    const float2 *angle[kAtOnce];
    bool turns[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const uint32_t i = i0 + k * kRopeThreads;
      to[k] = nullptr;
      if (i >= items)
        continue;
      const uint32_t row = p.by_access.of(i), a = i - row * per_head;
      const uint32_t t = nheads == p.cta_heads ? p.by_head.of(row) : row / nheads, head = head0 + (row - t * nheads);
      uint32_t w = 0;
#pragma unroll
      for (int j = 1; j < kRopeTensors; ++j)
        w += j < p.count && head >= p.tensor[j].first_head;
      const RopeTensor &tensor = p.tensor[w];
      const size_t token = token0 + t, h = head - tensor.first_head;
      turns[k] = a < turning;
      const uint32_t at = turns[k] ? a * (kN * kStep) : p.n_rot + (a - turning) * kN;
      const T *x = static_cast<const T *>(tensor.x) + token * tensor.x_token + h * tensor.x_head + at;
      if (!turns[k] && tensor.x == tensor.y)
        continue;
      to[k] = static_cast<T *>(tensor.y) + token * tensor.y_token + h * tensor.y_head + at;
      angle[k] = rope_cs + t * pairs + at / 2;
      lo[k] = *reinterpret_cast<const P *>(x);
      if (turns[k] && kN == 1)
        hi[k] = *reinterpret_cast<const P *>(x + 1);
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (to[k] == nullptr)
        continue;
      if (turns[k]) {
        if constexpr (kN == 1) {
#pragma unroll
          for (int e = 0; e < kN; ++e) {
            const float2 r = angle[k][e];
            const float u = to_float(lo[k].v[e]), v = to_float(hi[k].v[e]);
            lo[k].v[e] = from_float<T>(turn_lo(u, v, r));
            hi[k].v[e] = from_float<T>(turn_hi(u, v, r));
          }
          *reinterpret_cast<P *>(to[k] + 1) = hi[k];
        } else {
#pragma unroll
          for (int e = 0; e < kN; e += 2) {
            const float2 r = angle[k][e / 2];
            const float u = to_float(lo[k].v[e]), v = to_float(lo[k].v[e + 1]);
            lo[k].v[e] = from_float<T>(turn_lo(u, v, r));
            lo[k].v[e + 1] = from_float<T>(turn_hi(u, v, r));
          }
        }
      }
      *reinterpret_cast<P *>(to[k]) = lo[k];
    }
  }
}

__global__ void rope_frequencies_kernel(uint32_t pairs, double base, int scaling, double factor, double original, double low,
                                        double high, double *freqs) {
  const uint32_t p = blockIdx.x * blockDim.x + threadIdx.x;
  if (p >= pairs)
    return;
  const double two_pi = 6.283185307179586, n_rot = 2.0 * pairs;
  const double f = pow(base, -2.0 * p / n_rot);
  double keep = 1.0;
  if (scaling == TCRV_CUDA_ROPE_SCALING_LINEAR) {
    keep = 0.0;
  } else if (scaling == TCRV_CUDA_ROPE_SCALING_YARN) {
    // the (fractional) pair that turns r times within `original` positions: base^(-2p/n) = 2 pi r / original
    const double from = fmax(0.0, floor(n_rot * log(original / (high * two_pi)) / (2.0 * log(base))));
    const double to = fmin(n_rot - 1.0, ceil(n_rot * log(original / (low * two_pi)) / (2.0 * log(base))));
    keep = 1.0 - fmin(1.0, fmax(0.0, (p - from) / fmax(to - from, 0.001)));
  } else if (scaling == TCRV_CUDA_ROPE_SCALING_BANDS) {
    keep = fmin(1.0, fmax(0.0, (original * f / two_pi - low) / (high - low)));
  }
  freqs[p] = f * keep + f / factor * (1.0 - keep);
}

template <typename T, bool kHalves, int kN>
auto rope_kernel_of(bool inverse) -> void (*)(const RopeParams) {
  return inverse ? rope_kernel<T, kHalves, kN, true> : rope_kernel<T, kHalves, kN, false>;
}

template <typename T>
int rope_launch(RopeParams &p, bool halves, bool inverse, cudaStream_t stream) {
  constexpr int kN = 16 / sizeof(T);
  const uint32_t pairs = p.n_rot / 2;
  bool wide = (halves ? pairs : p.n_rot) % kN == 0 && p.dim % kN == 0 && p.n_rot % kN == 0;
  for (uint32_t j = 0; j < p.count; ++j) {
    const RopeTensor &t = p.tensor[j];
    wide = wide && reinterpret_cast<uintptr_t>(t.x) % 16 == 0 && reinterpret_cast<uintptr_t>(t.y) % 16 == 0 &&
           (t.x_token | t.x_head | t.y_token | t.y_head) % kN == 0;
  }
  // as many tokens to a CTA as leave four CTAs for each SM, and their angles room; then heads are split
  // until the SMs have two each (or a CTA has less than one access to a thread)
  const size_t sms = static_cast<size_t>(sm_count());
  size_t tokens = p.tokens / (4 * sms);
  const size_t room = pairs ? kRopeSmemPairs / pairs : 64;
  tokens = tokens < 1 ? 1 : tokens > 4 ? 4 : tokens;
  tokens = tokens > room && room >= 1 ? room : tokens;
  const size_t per_head = p.dim / (wide ? kN : 1);
  size_t ctas = (p.tokens + tokens - 1) / tokens, split = 1;
  while (ctas * split < 2 * sms && split < p.heads && tokens * ((p.heads + split - 1) / split) * per_head > kRopeThreads)
    split *= 2;
  p.cta_tokens = static_cast<uint32_t>(tokens);
  p.cta_heads = static_cast<uint32_t>((p.heads + split - 1) / split);
  const dim3 grid(static_cast<unsigned>(ctas), (p.heads + p.cta_heads - 1) / p.cta_heads);
  const uint32_t n = wide ? kN : 1, step = halves ? 1 : wide ? 1 : 2;
  const uint32_t accesses = (halves ? pairs / n : p.n_rot / (n * step)) + (p.dim - p.n_rot) / n;
  const uint64_t rows = static_cast<uint64_t>(p.cta_tokens) * p.cta_heads;
  p.by_access = Divisor(accesses, rows * accesses);
  p.by_head = Divisor(p.cta_heads, rows);
  const size_t smem = tokens * pairs * sizeof(float2);
  auto *kernel = halves ? (wide ? rope_kernel_of<T, true, kN>(inverse) : rope_kernel_of<T, true, 1>(inverse))
                        : (wide ? rope_kernel_of<T, false, kN>(inverse) : rope_kernel_of<T, false, 1>(inverse));
  TCRV_CUDA_TRY(launch_pdl(kernel, grid, kRopeThreads, smem, stream, p));
  return TCRV_CUDA_OK;
}

}  // namespace

int launch_rope_rows(int type, size_t tokens, size_t dim, size_t n_rot, const tcrv_cuda_rope_tensor *tensors, size_t count,
                     const void *positions, const double *freqs, float magnitude, unsigned flags, cudaStream_t stream) {
  RopeParams p = {};
  for (size_t j = 0; j < count; ++j) {
    if (tensors[j].heads == 0)
      continue;
    p.tensor[p.count++] = {tensors[j].x,           tensors[j].y,           tensors[j].x_token_stride, tensors[j].x_head_stride,
                           tensors[j].y_token_stride, tensors[j].y_head_stride, p.heads};
    p.heads += static_cast<uint32_t>(tensors[j].heads);
  }
  if (tokens == 0 || p.heads == 0)
    return TCRV_CUDA_OK;
  p.dim = static_cast<uint32_t>(dim);
  p.n_rot = static_cast<uint32_t>(n_rot);
  p.tokens = tokens;
  p.positions = positions;
  p.freqs = freqs;
  p.magnitude = magnitude;
  p.wide_positions = flags & TCRV_CUDA_ROPE_POSITIONS_I64;
  const bool halves = flags & TCRV_CUDA_ROPE_HALVES, inverse = flags & TCRV_CUDA_ROPE_INVERSE;
  if (type == TCRV_CUDA_TYPE_F32)
    return rope_launch<float>(p, halves, inverse, stream);
  if (type == TCRV_CUDA_TYPE_F16)
    return rope_launch<__half>(p, halves, inverse, stream);
  return rope_launch<__nv_bfloat16>(p, halves, inverse, stream);
}

int launch_rope_frequencies_f64(size_t n_rot, double theta_base, int scaling, double factor, double original, double low,
                                double high, double *freqs, cudaStream_t stream) {
  const uint32_t pairs = static_cast<uint32_t>(n_rot / 2);
  if (pairs == 0)
    return TCRV_CUDA_OK;
  rope_frequencies_kernel<<<(pairs + 63) / 64, 64, 0, stream>>>(pairs, theta_base, scaling, factor, original, low, high, freqs);
  TCRV_CUDA_TRY(cudaGetLastError());
  return TCRV_CUDA_OK;
}

}  // namespace tcrv
