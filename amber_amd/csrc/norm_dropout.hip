// activation -> LayerNorm -> dropout on rows, forward and backward, and the counter-based generator behind the dropout
// (include/amber_mpn.h: amber_mpn_tail_forward / _backward, amber_mpn_keep_mask, amber_mpn_generator_take).
// reference: the layers of the decoder MLP in train() mode (src/algorithm/architecture/mlp.py:58-96,128-130) and the edge
// dropout (src/mpn/common/edge_dropout.py:24-25).
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "mpn_internal.h"

#define DEVINL __device__ __forceinline__

namespace amber {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxBlocks = 2048;  // 256 CUs x 8 resident blocks of 4 waves

// ---------------------------------------------------------------------------------------------------
// element types: 32 bits inside, one rounding (to nearest even) at a store
// ---------------------------------------------------------------------------------------------------
using bf16 = __hip_bfloat16;
using f16 = _Float16;
template <class T>
DEVINL float to_f(T v) { return static_cast<float>(v); }
template <>
DEVINL float to_f<bf16>(bf16 v) { return __bfloat162float(v); }
template <class T>
DEVINL T from_f(float v) { return static_cast<T>(v); }
template <>
DEVINL bf16 from_f<bf16>(float v) { return __float2bfloat16(v); }

// weight / bias [width] in fp32 or in the element type
template <class T>
DEVINL float load_weight(const void* w, int fp32, int64_t i, float missing) {
  if (!w) return missing;
  return fp32 ? static_cast<const float*>(w)[i] : to_f(static_cast<const T*>(w)[i]);
}
template <class T>
DEVINL void store_weight(void* w, int fp32, int64_t i, float v) {
  if (!w) return;
  if (fp32) static_cast<float*>(w)[i] = v;
  else static_cast<T*>(w)[i] = from_f<T>(v);
}

// ---------------------------------------------------------------------------------------------------
// activations from the pre-activation x, torch's formulas and default arguments
// ---------------------------------------------------------------------------------------------------
DEVINL float act_of(float x, int act) {
  switch (act) {
    case AMBER_ACT_RELU: return x < 0.f ? 0.f : x;  // NaN stays NaN
    case AMBER_ACT_LEAKYRELU: return x > 0.f ? x : 0.01f * x;
    case AMBER_ACT_TANH: return tanhf(x);
    case AMBER_ACT_ELU: return x > 0.f ? x : expm1f(x);
    case AMBER_ACT_SILU: return x / (1.f + expf(-x));
    case AMBER_ACT_MISH: return x * tanhf(x > 20.f ? x : log1pf(expf(x)));
    case AMBER_ACT_GELU: return 0.5f * x * (1.f + erff(x * 0.70710678118654752440f));
    default: return x;
  }
}
// act(x) and act'(x) (at the kink of relu / leakyrelu / elu: the value from the left, as torch)
DEVINL float act_grad(float x, int act) {
  switch (act) {
    case AMBER_ACT_RELU: return x > 0.f ? 1.f : 0.f;
    case AMBER_ACT_LEAKYRELU: return x > 0.f ? 1.f : 0.01f;
    case AMBER_ACT_TANH: {
      const float t = tanhf(x);
      return 1.f - t * t;
    }
    case AMBER_ACT_ELU: return x > 0.f ? 1.f : expf(x);
    case AMBER_ACT_SILU: {
      const float s = 1.f / (1.f + expf(-x));
      return s * (1.f + x * (1.f - s));
    }
    case AMBER_ACT_MISH: {
      const float t = tanhf(x > 20.f ? x : log1pf(expf(x)));
      const float s = 1.f / (1.f + expf(-x));
      return t + x * (1.f - t * t) * s;
    }
    case AMBER_ACT_GELU:
      return 0.5f * (1.f + erff(x * 0.70710678118654752440f)) + x * 0.39894228040143267794f * expf(-0.5f * x * x);
    default: return 1.f;
  }
}

// ---------------------------------------------------------------------------------------------------
// Philox-4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011): ten rounds of two 32 x 32 -> 64 products
// ---------------------------------------------------------------------------------------------------
struct Words {
  uint32_t w[4];
};
struct Stream {
  uint32_t k0, k1, c2, c3;
};
DEVINL Stream stream_of(const int64_t* state, int64_t sequence) {
  const uint64_t seed = static_cast<uint64_t>(state[0]);
  const uint64_t offset = static_cast<uint64_t>(state[1]) + static_cast<uint64_t>(sequence);
  return {static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32), static_cast<uint32_t>(offset),
          static_cast<uint32_t>(offset >> 32)};
}
DEVINL Words philox(const Stream& s, uint64_t group) {
  uint32_t c0 = static_cast<uint32_t>(group), c1 = static_cast<uint32_t>(group >> 32), c2 = s.c2, c3 = s.c3;
  uint32_t k0 = s.k0, k1 = s.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u;
    const uint64_t p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(p1);
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}
DEVINL bool kept(const TailArgs& a, const Stream& s, int64_t i) {
  return philox(s, static_cast<uint64_t>(i) >> 2).w[i & 3] > a.last_dropped;
}

__global__ void generator_take_kernel(int64_t* state, int64_t count, int64_t* taken) {
  taken[0] = state[0];
  taken[1] = static_cast<int64_t>(atomicAdd(reinterpret_cast<unsigned long long*>(state + 1), static_cast<unsigned long long>(count)));
}

__global__ __launch_bounds__(kBlock) void keep_mask_kernel(TailArgs a, uint8_t* out) {
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < a.rows; i += static_cast<int64_t>(gridDim.x) * kBlock)
    out[i] = !a.drop || kept(a, s, i) ? 1 : 0;
}

// ---------------------------------------------------------------------------------------------------
// without the norm: elementwise
// ---------------------------------------------------------------------------------------------------
template <class T, bool BWD>
__global__ __launch_bounds__(kBlock) void elementwise_kernel(TailArgs a) {
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  const int64_t n = a.rows * a.width;
  const T* x = static_cast<const T*>(a.x);
  const T* g = static_cast<const T*>(a.g);
  T* y = static_cast<T*>(a.y);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kBlock) {
    float v = BWD ? to_f(g[i]) : act_of(to_f(x[i]), a.act);
    if (a.drop) v = kept(a, s, i) ? v * a.scale : 0.f;
    if (BWD && a.act != AMBER_ACT_NONE) v = v * act_grad(to_f(x[i]), a.act);
    y[i] = from_f<T>(v);
  }
}

// ---------------------------------------------------------------------------------------------------
// with the norm: a block per row
// ---------------------------------------------------------------------------------------------------
DEVINL float wave_sum(float v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}
// sum over the block in a fixed order; `box` may be used again after the next barrier
DEVINL float block_sum(float v, float* box) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < kBlock / 64; ++w) t += box[w];
  return t;
}

template <class T>
__global__ __launch_bounds__(kBlock) void norm_forward_kernel(TailArgs a) {
  __shared__ float box[kBlock / 64];
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  const float inv = 1.f / static_cast<float>(a.width);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    T* y = static_cast<T*>(a.y) + row * a.width;
    float sum = 0.f;
    for (int64_t c = threadIdx.x; c < a.width; c += kBlock) sum += act_of(to_f(x[c]), a.act);
    const float mean = block_sum(sum, box) * inv;
    float sq = 0.f;
    for (int64_t c = threadIdx.x; c < a.width; c += kBlock) {
      const float d = act_of(to_f(x[c]), a.act) - mean;
      sq += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum(sq, box) * inv + a.eps);
    for (int64_t c = threadIdx.x; c < a.width; c += kBlock) {
      float v = (act_of(to_f(x[c]), a.act) - mean) * rstd;
      v = v * load_weight<T>(a.weight, a.weight_dtype == AMBER_DTYPE_F32, c, 1.f) +
          load_weight<T>(a.bias, a.weight_dtype == AMBER_DTYPE_F32, c, 0.f);
      if (a.drop) v = kept(a, s, row * a.width + c) ? v * a.scale : 0.f;
      y[c] = from_f<T>(v);
    }
    if (a.stats && threadIdx.x == 0) {
      a.stats[2 * row] = mean;
      a.stats[2 * row + 1] = rstd;
    }
  }
}

template <class T>
__global__ __launch_bounds__(kBlock) void norm_backward_kernel(TailArgs a) {
  __shared__ float box[kBlock / 64];
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  const float inv = 1.f / static_cast<float>(a.width);
  float* pw = a.partial ? a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.width : nullptr;
  if (pw)
    for (int64_t c = threadIdx.x; c < 2 * a.width; c += kBlock) pw[c] = 0.f;
  __syncthreads();  // the loop below updates partial sums that other threads have cleared
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* g = static_cast<const T*>(a.g) + row * a.ldg;
    const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
    float s0 = 0.f, s1 = 0.f;
    for (int64_t c = threadIdx.x; c < a.width; c += kBlock) {
      float v = to_f(g[c]);
      if (a.drop) v = kept(a, s, row * a.width + c) ? v * a.scale : 0.f;
      const float n = (act_of(to_f(x[c]), a.act) - mean) * rstd;
      const float h = v * load_weight<T>(a.weight, a.weight_dtype == AMBER_DTYPE_F32, c, 1.f);
      s0 += h;
      s1 += h * n;
      if (pw) {
        pw[c] += v * n;
        pw[a.width + c] += v;
      }
    }
    s0 = block_sum(s0, box) * inv;
    s1 = block_sum(s1, box) * inv;
    if (a.y) {
      T* y = static_cast<T*>(a.y) + row * a.width;
      for (int64_t c = threadIdx.x; c < a.width; c += kBlock) {
        float v = to_f(g[c]);
        if (a.drop) v = kept(a, s, row * a.width + c) ? v * a.scale : 0.f;
        const float xv = to_f(x[c]);
        const float n = (act_of(xv, a.act) - mean) * rstd;
        const float h = v * load_weight<T>(a.weight, a.weight_dtype == AMBER_DTYPE_F32, c, 1.f);
        y[c] = from_f<T>(rstd * (h - s0 - n * s1) * act_grad(xv, a.act));
      }
    }
  }
}

// gradients of weight and bias: the blocks' partial sums, added in the blocks' order
template <class T>
__global__ __launch_bounds__(kBlock) void weight_gradient_kernel(TailArgs a, int64_t blocks) {
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; c < 2 * a.width; c += static_cast<int64_t>(gridDim.x) * kBlock) {
    float sum = 0.f;
    for (int64_t b = 0; b < blocks; ++b) sum += a.partial[b * 2 * a.width + c];
    const int fp32 = a.weight_dtype == AMBER_DTYPE_F32;
    if (c < a.width) store_weight<T>(a.grad_weight, fp32, c, sum);
    else store_weight<T>(a.grad_bias, fp32, c - a.width, sum);
  }
}

unsigned blocks_for(int64_t work, int64_t limit) { return static_cast<unsigned>(work < 1 ? 1 : work < limit ? work : limit); }

template <class T>
hipError_t forward_t(const TailArgs& a, bool normalize, hipStream_t s) {
  if (normalize)
    hipLaunchKernelGGL((norm_forward_kernel<T>), dim3(blocks_for(a.rows, kMaxBlocks)), dim3(kBlock), 0, s, a);
  else
    hipLaunchKernelGGL((elementwise_kernel<T, false>), dim3(blocks_for((a.rows * a.width + kBlock - 1) / kBlock, kMaxBlocks)), dim3(kBlock),
                       0, s, a);
  return hipGetLastError();
}
template <class T>
hipError_t backward_t(const TailArgs& a, bool normalize, hipStream_t s) {
  if (!normalize) {
    hipLaunchKernelGGL((elementwise_kernel<T, true>), dim3(blocks_for((a.rows * a.width + kBlock - 1) / kBlock, kMaxBlocks)), dim3(kBlock),
                       0, s, a);
    return hipGetLastError();
  }
  const int64_t blocks = a.rows > 0 ? tail_partial_blocks(a) : 0;
  if (a.rows > 0) hipLaunchKernelGGL((norm_backward_kernel<T>), dim3(static_cast<unsigned>(blocks)), dim3(kBlock), 0, s, a);
  if (a.grad_weight || a.grad_bias)  // no rows: zeros
    hipLaunchKernelGGL((weight_gradient_kernel<T>), dim3(blocks_for((2 * a.width + kBlock - 1) / kBlock, kMaxBlocks)), dim3(kBlock), 0, s, a,
                       blocks);
  return hipGetLastError();
}

}  // namespace

int64_t tail_partial_blocks(const TailArgs& a) { return blocks_for(a.rows, 1024); }

hipError_t launch_tail_forward(const TailArgs& a, bool normalize, hipStream_t s) {
  switch (a.dtype) {
    case AMBER_DTYPE_F32: return forward_t<float>(a, normalize, s);
    case AMBER_DTYPE_BF16: return forward_t<bf16>(a, normalize, s);
    default: return forward_t<f16>(a, normalize, s);
  }
}
hipError_t launch_tail_backward(const TailArgs& a, bool normalize, hipStream_t s) {
  switch (a.dtype) {
    case AMBER_DTYPE_F32: return backward_t<float>(a, normalize, s);
    case AMBER_DTYPE_BF16: return backward_t<bf16>(a, normalize, s);
    default: return backward_t<f16>(a, normalize, s);
  }
}
hipError_t launch_keep_mask(const TailArgs& a, uint8_t* out, hipStream_t s) {
  hipLaunchKernelGGL(keep_mask_kernel, dim3(blocks_for((a.rows + kBlock - 1) / kBlock, kMaxBlocks)), dim3(kBlock), 0, s, a, out);
  return hipGetLastError();
}
hipError_t launch_generator_take(int64_t* state, int64_t count, int64_t* taken, hipStream_t s) {
  hipLaunchKernelGGL(generator_take_kernel, dim3(1), dim3(1), 0, s, state, count, taken);
  return hipGetLastError();
}

}  // namespace amber
