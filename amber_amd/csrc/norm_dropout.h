// activation -> LayerNorm -> dropout on rows, forward and backward, and the counter-based generator behind the dropout
// (include/amber_mpn.h: amber_mpn_tail_forward / _backward, amber_mpn_keep_mask, amber_mpn_generator_take).
// reference: the layers of the decoder MLP in train() mode (src/algorithm/architecture/mlp.py:58-96,128-130) and the edge
// dropout (src/mpn/common/edge_dropout.py:24-25).
#pragma once
#include "mpn_internal.h"

#define DEVINL __device__ __forceinline__

namespace amber {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxBlocks = 2048;  // 256 CUs x 8 resident blocks of 4 waves

// ---------------------------------------------------------------------------------------------------
// element types: 32 bits inside, one rounding (to nearest even) at a store
// ---------------------------------------------------------------------------------------------------
using bf16 = __bf16;
using f16 = _Float16;
template <class T>
DEVINL float to_f(T v) { return static_cast<float>(v); }
template <class T>
DEVINL T from_f(float v) { return static_cast<T>(v); }

// V elements = 16 bytes; the types' own alignment is enough for one 16-byte access, so rows may start anywhere
template <class T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));
template <class T>
using Pack = T __attribute__((ext_vector_type(kVec<T>)));
template <class T>
using LoosePack = Pack<T> __attribute__((aligned(sizeof(T))));

// the first `count` of V elements (count >= V: all of them); the rest are 0
template <class T, int V = kVec<T>>
DEVINL void load_pack(const T* p, int count, float (&v)[V]) {
  if (count >= V) {
    const Pack<T> q = *reinterpret_cast<const LoosePack<T>*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_f(q[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = j < count ? to_f(p[j]) : 0.f;
  }
}
template <class T, int V = kVec<T>>
DEVINL void store_pack(T* p, int count, const float (&v)[V]) {
  if (count >= V) {
    Pack<T> q;
#pragma unroll
    for (int j = 0; j < V; ++j) q[j] = from_f<T>(v[j]);
    *reinterpret_cast<LoosePack<T>*>(p) = q;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < count) p[j] = from_f<T>(v[j]);
  }
}

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
// activations and their derivatives from the pre-activation x (torch's definitions and default arguments; at the kink of
// relu / leakyrelu / elu the derivative from the left).  fp32 on the hardware's 2^x and reciprocal (1 unit in the last place):
//   exp(x) = 2^(x log2 e): relative error (1.5 |x| + 1) 2^-24, which in every use below multiplies a value that falls like exp(-|x|)
//   tanh: x P(x^2) below 1/2 (relative error 1.3e-8), 1 - 2 / (1 + e^2|x|) above
//   expm1: x P(x) above -1/2 (1.4e-9), exp(x) - 1 below
//   mish: tanh(log(1 + w)) = n / (n + 2) with w = e^x, n = w (w + 2): no cancellation; beyond x = 20 it is 1 in fp32
//   gelu: Phi(-a) = e^(-a^2/2) t Q(t), t = 1 / (1 + 0.3 a), a = |x| (relative error 5e-8 up to a = 9): the tail itself is
//         approximated, so x Phi(x) keeps its relative accuracy for negative x, and the derivative shares the exponential
// The polynomials are least-maximum fits of these functions.
// ---------------------------------------------------------------------------------------------------
DEVINL float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
DEVINL float rcp_of(float x) { return __builtin_amdgcn_rcpf(x); }
DEVINL float tanh_of(float x) {
  const float a = fabsf(x), z = x * x;
  float p = 0.01715129399739507f;
  p = fmaf(p, z, -0.05299422865708484f);
  p = fmaf(p, z, 0.13324906927244848f);
  p = fmaf(p, z, -0.3333307579068465f);
  p = fmaf(p, z, 0.99999998737373f);
  const float far = 1.f - 2.f * rcp_of(1.f + exp_of(2.f * a));
  return a < 0.5f ? x * p : copysignf(far, x);
}
DEVINL float expm1_of(float x) {  // x <= 0
  float p = 0.0011216346774701612f;
  p = fmaf(p, x, 0.008187385691190183f);
  p = fmaf(p, x, 0.04162908900354672f);
  p = fmaf(p, x, 0.16666224080228778f);
  p = fmaf(p, x, 0.4999998074594835f);
  p = fmaf(p, x, 0.9999999986263833f);
  return x > -0.5f ? x * p : exp_of(x) - 1.f;
}
struct Gelu {
  float tail, density;  // Phi(-|x|), e^(-x^2 / 2)
};
DEVINL Gelu gelu_parts(float a) {
  const float t = rcp_of(fmaf(0.3f, a, 1.f));
  float q = 0.03753587207292055f;
  q = fmaf(q, t, -0.16502039737444713f);
  q = fmaf(q, t, 0.21997266723558018f);
  q = fmaf(q, t, -0.0664040520700526f);
  q = fmaf(q, t, 0.13542105016317393f);
  q = fmaf(q, t, 0.09778364147982758f);
  q = fmaf(q, t, 0.12110575544066968f);
  q = fmaf(q, t, 0.1196054879202132f);
  const float e = __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f);
  return {t * q * e, e};
}
DEVINL float act_of(float x, int act) {
  switch (act) {
    case AMBER_ACT_RELU: return x < 0.f ? 0.f : x;  // NaN stays NaN
    case AMBER_ACT_LEAKYRELU: return x > 0.f ? x : 0.01f * x;
    case AMBER_ACT_TANH: return tanh_of(x);
    case AMBER_ACT_ELU: return x > 0.f ? x : expm1_of(x);
    case AMBER_ACT_SILU: return x * rcp_of(1.f + exp_of(-x));
    case AMBER_ACT_MISH: {
      const float w = exp_of(fminf(x, 20.f)), n = w * (w + 2.f);
      return x * (n * rcp_of(n + 2.f));
    }
    case AMBER_ACT_GELU: {
      const float a = fabsf(x);
      return fmaxf(x, 0.f) - fminf(a, 16.f) * gelu_parts(a).tail;
    }
    default: return x;
  }
}
struct ActGrad {
  float a, d;  // act(x), act'(x)
};
DEVINL ActGrad act_grad(float x, int act) {
  switch (act) {
    case AMBER_ACT_RELU: return {x < 0.f ? 0.f : x, x > 0.f ? 1.f : 0.f};
    case AMBER_ACT_LEAKYRELU: return x > 0.f ? ActGrad{x, 1.f} : ActGrad{0.01f * x, 0.01f};
    case AMBER_ACT_TANH: {
      const float t = tanh_of(x);
      return {t, fmaf(-t, t, 1.f)};
    }
    case AMBER_ACT_ELU: return x > 0.f ? ActGrad{x, 1.f} : ActGrad{expm1_of(x), exp_of(x)};
    case AMBER_ACT_SILU: {
      const float s = rcp_of(1.f + exp_of(-x));
      return {x * s, s * fmaf(x, 1.f - s, 1.f)};
    }
    case AMBER_ACT_MISH: {
      const float w = exp_of(fminf(x, 20.f)), n = w * (w + 2.f), r = rcp_of(n + 2.f), t = n * r;
      return {x * t, fmaf(x * r, 4.f * w * (w + 1.f) * r, t)};
    }
    case AMBER_ACT_GELU: {
      const float a = fabsf(x), ac = fminf(a, 16.f);
      const Gelu g = gelu_parts(a);
      return {fmaxf(x, 0.f) - ac * g.tail, fmaf(copysignf(ac, x), 0.39894228040143268f * g.density, x < 0.f ? g.tail : 1.f - g.tail)};
    }
    default: return {x, 1.f};
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
DEVINL uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }  // one instruction
DEVINL Words philox(const Stream& s, uint64_t group) {
  uint32_t c0 = static_cast<uint32_t>(group), c1 = static_cast<uint32_t>(group >> 32), c2 = s.c2, c3 = s.c3;
  uint32_t k0 = s.k0, k1 = s.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u;
    const uint64_t p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = xor3(static_cast<uint32_t>(p1 >> 32), c1, k0);
    c1 = static_cast<uint32_t>(p1);
    c2 = xor3(static_cast<uint32_t>(p0 >> 32), c3, k1);
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}
DEVINL bool kept(const TailArgs& a, const Stream& s, int64_t i) {
  return philox(s, static_cast<uint64_t>(i) >> 2).w[i & 3] > a.last_dropped;
}

// v[j] of element first + j: 0 where dropped, else v[j] * scale.  An aligned start (first & 3 == 0) takes V / 4 calls of the
// generator, any other one more, its words moved down by first & 3.
template <int V>
DEVINL void drop_pack(const TailArgs& a, const Stream& s, int64_t first, bool aligned, float (&v)[V]) {
  uint32_t w[V + 4];
  const uint64_t group = static_cast<uint64_t>(first) >> 2;
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    const Words t = philox(s, group + q);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[4 * q + j] = t.w[j];
  }
  if (!aligned) {
    const Words t = philox(s, group + V / 4);
#pragma unroll
    for (int j = 0; j < 3; ++j) w[V + j] = t.w[j];
    const bool two = first & 2, one = first & 1;
#pragma unroll
    for (int j = 0; j < V + 1; ++j) w[j] = two ? w[j + 2] : w[j];
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = one ? w[j + 1] : w[j];
  }
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = w[j] > a.last_dropped ? v[j] * a.scale : 0.f;
}

// ---------------------------------------------------------------------------------------------------
// without the norm: elementwise over the flat tensor, 16 bytes a thread
// ---------------------------------------------------------------------------------------------------
template <class T, bool BWD>
__global__ __launch_bounds__(kBlock) void elementwise_kernel(TailArgs a) {
  constexpr int V = kVec<T>;
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  const int64_t n = a.rows * a.width;
  const T* x = static_cast<const T*>(a.x);
  const T* g = static_cast<const T*>(a.g);
  T* y = static_cast<T*>(a.y);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kBlock * V;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x) * V; i < n; i += step) {
    const int count = n - i < V ? static_cast<int>(n - i) : V;
    float v[V], xv[V];
    if (BWD) load_pack(g + i, count, v);
    if (!BWD || a.act != AMBER_ACT_NONE) load_pack(x + i, count, xv);
    if (!BWD) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = act_of(xv[j], a.act);
    }
    if (a.drop) drop_pack(a, s, i, true, v);
    if (BWD && a.act != AMBER_ACT_NONE) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] *= act_grad(xv[j], a.act).d;
    }
    store_pack(y + i, count, v);
  }
}

// ---------------------------------------------------------------------------------------------------
// with the norm: a block per row
// ---------------------------------------------------------------------------------------------------
// sum / D with inv = 1 / D rounded: one correction, so that a row of equal values has exactly that value as its mean
DEVINL float mean_of(float sum, float width, float inv) {
  const float m = sum * inv;
  return fmaf(fmaf(-m, width, sum), inv, m);
}
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
    const float mean = mean_of(block_sum(sum, box), static_cast<float>(a.width), inv);
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
        y[c] = from_f<T>(rstd * (h - s0 - n * s1) * act_grad(xv, a.act).d);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------
// with the norm, rows in registers: a team of G lanes (W = 1: 64 / G teams a wave) or of W waves holds a row, K packs a lane
// ---------------------------------------------------------------------------------------------------
template <int CTRL>
DEVINL float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// sum over the G lanes of a team, the same bits in every lane
template <int G>
DEVINL float team_sum(float v) {
  if (G >= 2) v += dpp<0xB1>(v);   // lane ^ 1
  if (G >= 4) v += dpp<0x4E>(v);   // lane ^ 2
  if (G >= 8) v += dpp<0x141>(v);  // mirrored in 8: the other four
  if (G >= 16) v += dpp<0x140>(v); // mirrored in 16: the other eight
  if (G >= 32) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
  }
  if (G >= 64) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = __builtin_bit_cast(float, static_cast<unsigned>(r[0])) + __builtin_bit_cast(float, static_cast<unsigned>(r[1]));
  }
  return v;
}

// SMOOTH: activations beyond none / relu / leakyrelu
template <bool SMOOTH>
DEVINL float act_sel(float x, int act) {
  if (SMOOTH) return act_of(x, act);
  return act == AMBER_ACT_NONE || x > 0.f ? x : act == AMBER_ACT_RELU ? act_of(x, AMBER_ACT_RELU) : 0.01f * x;
}
template <bool SMOOTH>
DEVINL ActGrad act_grad_sel(float x, int act) {
  if (SMOOTH) return act_grad(x, act);
  const bool on = act == AMBER_ACT_NONE || x > 0.f;
  return {act_sel<false>(x, act), on ? 1.f : act == AMBER_ACT_RELU ? 0.f : 0.01f};
}

template <class T, int G, int W, int K, int R, bool SMOOTH>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void norm_rows_forward(TailArgs a) {
  constexpr int V = kVec<T>, LANES = G * W, THREADS = W == 1 ? 256 : 64 * W, TEAMS = THREADS / LANES;
  __shared__ float box[2][R][W];
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const int width = static_cast<int>(a.width);
  const float inv = 1.f / static_cast<float>(width);
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  const bool aligned = (width & 3) == 0;
  int count[K];
  float w[K][V], b[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * LANES + lane) * V;
    count[k] = min(V, max(0, width - c));
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[k][j] = j < count[k] ? load_weight<T>(a.weight, a.weight_dtype == AMBER_DTYPE_F32, c + j, 1.f) : 0.f;
      b[k][j] = j < count[k] ? load_weight<T>(a.bias, a.weight_dtype == AMBER_DTYPE_F32, c + j, 0.f) : 0.f;
    }
  }
  const int64_t stride = static_cast<int64_t>(gridDim.x) * TEAMS;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * TEAMS; base < a.rows; base += stride * R) {
    float v[R][K][V], sum[R], mean[R], rstd[R];
    int64_t row[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      row[r] = base + r * stride + team;
      const T* x = static_cast<const T*>(a.x) + row[r] * a.ldx;
#pragma unroll
      for (int k = 0; k < K; ++k) load_pack(x + (k * LANES + lane) * V, row[r] < a.rows ? count[k] : 0, v[r][k]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sum[r] = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[r][k][j] = act_sel<SMOOTH>(v[r][k][j], a.act);
          sum[r] += v[r][k][j];
        }
      sum[r] = team_sum<G>(sum[r]);
    }
    if (W > 1) {
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int r = 0; r < R; ++r) box[0][r][threadIdx.x >> 6] = sum[r];
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        sum[r] = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) sum[r] += box[0][r][i];
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = mean_of(sum[r], static_cast<float>(width), inv);
      sum[r] = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          v[r][k][j] = j < count[k] ? v[r][k][j] - mean[r] : 0.f;
          sum[r] += v[r][k][j] * v[r][k][j];
        }
      sum[r] = team_sum<G>(sum[r]);
    }
    if (W > 1) {
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int r = 0; r < R; ++r) box[1][r][threadIdx.x >> 6] = sum[r];
      __syncthreads();  // everyone has read box[0]: the next rows may write it
#pragma unroll
      for (int r = 0; r < R; ++r) {
        sum[r] = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) sum[r] += box[1][r][i];
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      rstd[r] = 1.f / sqrtf(sum[r] * inv + a.eps);
      if (row[r] >= a.rows) continue;
      T* y = static_cast<T*>(a.y) + row[r] * width;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * LANES + lane) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) v[r][k][j] = v[r][k][j] * rstd[r] * w[k][j] + b[k][j];
        if (a.drop) drop_pack(a, s, row[r] * width + c, aligned, v[r][k]);
        store_pack(y + c, count[k], v[r][k]);
      }
      if (a.stats && lane == 0) {
        a.stats[2 * row[r]] = mean[r];
        a.stats[2 * row[r] + 1] = rstd[r];
      }
    }
  }
}

template <class T, int G, int W, int K, int R, bool SMOOTH>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void norm_rows_backward(TailArgs a) {
  constexpr int V = kVec<T>, LANES = G * W, THREADS = W == 1 ? 256 : 64 * W, TEAMS = THREADS / LANES;
  __shared__ float box[2][R][2][W];
  __shared__ float columns[W == 1 ? 2 * LANES * K * V : 1];
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const int width = static_cast<int>(a.width);
  const float inv = 1.f / static_cast<float>(width);
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  const bool aligned = (width & 3) == 0;
  int count[K];
  float w[K][V], dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * LANES + lane) * V;
    count[k] = min(V, max(0, width - c));
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[k][j] = j < count[k] ? load_weight<T>(a.weight, a.weight_dtype == AMBER_DTYPE_F32, c + j, 1.f) : 0.f;
      dw[k][j] = db[k][j] = 0.f;
    }
  }
  const int64_t stride = static_cast<int64_t>(gridDim.x) * TEAMS;
  int turn = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * TEAMS; base < a.rows; base += stride * R, turn ^= 1) {
    float xv[R][K][V], gv[R][K][V], dact[R][K][SMOOTH ? V : 1], mean[R], rstd[R], s0[R], s1[R];
    int64_t row[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      row[r] = base + r * stride + team;
      const bool in = row[r] < a.rows;
      const T* x = static_cast<const T*>(a.x) + row[r] * a.ldx;
      const T* g = static_cast<const T*>(a.g) + row[r] * a.ldg;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * LANES + lane) * V;
        load_pack(x + c, in ? count[k] : 0, xv[r][k]);
        load_pack(g + c, in ? count[k] : 0, gv[r][k]);
      }
      mean[r] = in ? a.stats[2 * row[r]] : 0.f;
      rstd[r] = in ? a.stats[2 * row[r] + 1] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s0[r] = s1[r] = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (a.drop) drop_pack(a, s, row[r] * width + (k * LANES + lane) * V, aligned, gv[r][k]);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float n;
          if (SMOOTH) {  // the activation is worth keeping: xv becomes n
            const ActGrad t = act_grad(xv[r][k][j], a.act);
            n = (t.a - mean[r]) * rstd[r];
            xv[r][k][j] = n;
            dact[r][k][j] = t.d;
          } else {
            n = (act_sel<SMOOTH>(xv[r][k][j], a.act) - mean[r]) * rstd[r];
          }
          const float h = gv[r][k][j] * w[k][j];
          dw[k][j] += gv[r][k][j] * n;
          db[k][j] += gv[r][k][j];
          s0[r] += h;
          s1[r] += h * n;
        }
      }
      s0[r] = team_sum<G>(s0[r]);
      s1[r] = team_sum<G>(s1[r]);
    }
    if (W > 1) {
      // the two boxes take turns: a wave writes one again only behind the barrier that follows everyone's reads of it
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          box[turn][r][0][threadIdx.x >> 6] = s0[r];
          box[turn][r][1][threadIdx.x >> 6] = s1[r];
        }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        s0[r] = s1[r] = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          s0[r] += box[turn][r][0][i];
          s1[r] += box[turn][r][1][i];
        }
      }
    }
    if (a.y) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (row[r] >= a.rows) continue;
        T* y = static_cast<T*>(a.y) + row[r] * width;
        const float m0 = s0[r] * inv, m1 = s1[r] * inv;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float d[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const ActGrad t = act_grad_sel<false>(xv[r][k][j], a.act);
            const float n = SMOOTH ? xv[r][k][j] : (t.a - mean[r]) * rstd[r];
            d[j] = rstd[r] * (gv[r][k][j] * w[k][j] - m0 - n * m1) * (SMOOTH ? dact[r][k][j] : t.d);
          }
          store_pack(y + (k * LANES + lane) * V, count[k], d);
        }
      }
    }
  }
  if (!a.partial) return;
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * width;
  if (W > 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * LANES + lane) * V;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < count[k]) {
          out[c + j] = dw[k][j];
          out[width + c + j] = db[k][j];
        }
    }
    return;
  }
  // teams of a wave, then the waves one after the other through LDS: a fixed order
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int m = G; m < 64; m <<= 1) {
        dw[k][j] += __shfl_xor(dw[k][j], m, 64);
        db[k][j] += __shfl_xor(db[k][j], m, 64);
      }
  for (int wave = 0; wave < THREADS / 64; ++wave) {
    if (static_cast<int>(threadIdx.x >> 6) == wave && (threadIdx.x & 63) < G) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = (k * LANES + lane) * V + j;
          columns[c] = wave ? columns[c] + dw[k][j] : dw[k][j];
          columns[LANES * K * V + c] = wave ? columns[LANES * K * V + c] + db[k][j] : db[k][j];
        }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < width; c += THREADS) {
    out[c] = columns[c];
    out[width + c] = columns[LANES * K * V + c];
  }
}

inline unsigned blocks_for(int64_t work, int64_t limit) { return static_cast<unsigned>(work < 1 ? 1 : work < limit ? work : limit); }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a row is held: G lanes of a wave (W = 1) or W waves, K packs of V elements a lane.  The smallest team that holds the row with
// at most 16 elements a lane; wider rows than 16 waves hold are read from memory three times (G = 0).
struct Shape {
  int g, w, k;
};
inline Shape shape_for(int64_t width, int vec) {
  const int64_t packs = cdiv(width, vec);
  for (int g = 1; g <= 64; g *= 2)
    if (packs <= g) return {g, 1, 1};
  const int most = 16 / vec;
  for (int w = 1; w <= 16; w *= w == 1 ? 4 : 2)
    for (int k = 1; k <= most; ++k)
      if (packs <= 64 * w * k) return {64, w, k};
  return {0, 0, 0};
}
inline int vec_of(int dtype) { return dtype == AMBER_DTYPE_F32 ? 4 : 8; }
inline int64_t teams_in_block(const Shape& h) { return h.w > 1 ? 1 : 256 / h.g; }
inline int64_t forward_blocks(const TailArgs& a, const Shape& h) { return blocks_for(cdiv(a.rows, teams_in_block(h)), 2048 / (h.w > 1 ? h.w / 4 : 1)); }
inline int64_t backward_blocks(const TailArgs& a, const Shape& h) { return blocks_for(cdiv(a.rows, teams_in_block(h)), 1024 / (h.w > 1 ? h.w / 4 : 1)); }

template <class T, int G, int W, int K, bool SMOOTH>
void launch_rows(const TailArgs& a, const Shape& h, bool backward, hipStream_t s) {
  constexpr int RF = K == 1 ? 4 : K == 2 ? 2 : 1, RB = K == 1 ? 2 : 1;
  const dim3 block(W == 1 ? 256 : 64 * W);
  if (backward)
    hipLaunchKernelGGL((norm_rows_backward<T, G, W, K, W == 1 ? RB : 1, SMOOTH>), dim3(static_cast<unsigned>(backward_blocks(a, h))), block, 0, s, a);
  else
    hipLaunchKernelGGL((norm_rows_forward<T, G, W, K, W == 1 ? RF : 1, SMOOTH>), dim3(static_cast<unsigned>(forward_blocks(a, h))), block, 0, s, a);
}
template <class T, bool SMOOTH>
void launch_shape(const TailArgs& a, const Shape& h, bool backward, hipStream_t s) {
  constexpr int MOST = 16 / kVec<T>;
#define AMBER_ROWS(G, W, K) \
  if (h.g == G && h.w == W && h.k == K) return launch_rows<T, G, W, (K <= MOST ? K : 1), SMOOTH>(a, h, backward, s)
  AMBER_ROWS(1, 1, 1);
  AMBER_ROWS(2, 1, 1);
  AMBER_ROWS(4, 1, 1);
  AMBER_ROWS(8, 1, 1);
  AMBER_ROWS(16, 1, 1);
  AMBER_ROWS(32, 1, 1);
  AMBER_ROWS(64, 1, 1);
  AMBER_ROWS(64, 1, 2);
  AMBER_ROWS(64, 4, 1);
  AMBER_ROWS(64, 4, 2);
  AMBER_ROWS(64, 8, 1);
  AMBER_ROWS(64, 8, 2);
  AMBER_ROWS(64, 16, 1);
  AMBER_ROWS(64, 16, 2);
  if constexpr (MOST >= 4) {
    AMBER_ROWS(64, 1, 3);
    AMBER_ROWS(64, 1, 4);
    AMBER_ROWS(64, 4, 3);
    AMBER_ROWS(64, 4, 4);
    AMBER_ROWS(64, 8, 3);
    AMBER_ROWS(64, 8, 4);
    AMBER_ROWS(64, 16, 3);
    AMBER_ROWS(64, 16, 4);
  }
#undef AMBER_ROWS
}
template <class T>
bool launch_in_registers(const TailArgs& a, bool backward, hipStream_t s) {
  const Shape h = shape_for(a.width, kVec<T>);
  if (h.g == 0) return false;
  const bool smooth = a.act != AMBER_ACT_NONE && a.act != AMBER_ACT_RELU && a.act != AMBER_ACT_LEAKYRELU;
  if (smooth) launch_shape<T, true>(a, h, backward, s);
  else launch_shape<T, false>(a, h, backward, s);
  return true;
}

template <class T>
hipError_t tail_forward_t(const TailArgs& a, bool normalize, hipStream_t s) {
  if (!normalize)
    hipLaunchKernelGGL((elementwise_kernel<T, false>), dim3(blocks_for(cdiv(a.rows * a.width, kBlock * kVec<T>), kMaxBlocks)), dim3(kBlock), 0,
                       s, a);
  else if (!launch_in_registers<T>(a, false, s))
    hipLaunchKernelGGL((norm_forward_kernel<T>), dim3(blocks_for(a.rows, kMaxBlocks)), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}
// dx and, into a.partial, the blocks' sums for the weights' gradients
template <class T>
hipError_t tail_backward_t(const TailArgs& a, bool normalize, hipStream_t s) {
  if (!normalize)
    hipLaunchKernelGGL((elementwise_kernel<T, true>), dim3(blocks_for(cdiv(a.rows * a.width, kBlock * kVec<T>), kMaxBlocks)), dim3(kBlock), 0,
                       s, a);
  else if (!launch_in_registers<T>(a, true, s))
    hipLaunchKernelGGL((norm_backward_kernel<T>), dim3(static_cast<unsigned>(tail_partial_blocks(a))), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

}  // namespace
}  // namespace amber
