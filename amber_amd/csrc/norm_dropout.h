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

// Accesses past the caches (STREAM).  CACHE = 0: none.  1: the stores, where a call touches more than 1.5 times the 256 MB of the
// memory-side cache: what it writes would not stay there for who reads it next, and would drive out what it still has to read
// (32768 x 4096 bf16 dropout 102 -> 86 us).  2: the loads too, where the inputs alone do not fit (1.44 M x 128 fp32 LayerNorm
// forward 250 -> 243 us, backward 409 -> 372, 6.0 TB/s).  Smaller calls are slower for it (5003 x 4099 bf16 backward 38 -> 46 us).
template <bool STREAM, class T>
DEVINL Pack<T> load_raw(const T* p) {
  const LoosePack<T>* const q = reinterpret_cast<const LoosePack<T>*>(p);
  if constexpr (STREAM) return __builtin_nontemporal_load(q);
  else return *q;
}

// the first `count` of V elements (count >= V: all of them); the rest are 0
template <bool STREAM, class T, int V = kVec<T>>
DEVINL void load_pack(const T* p, int count, float (&v)[V]) {
  if (count >= V) {
    const Pack<T> q = load_raw<STREAM>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_f(q[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = j < count ? to_f(p[j]) : 0.f;
  }
}
template <bool STREAM, class T, int V = kVec<T>>
DEVINL void store_pack(T* p, int count, const float (&v)[V]) {
  if (count >= V) {
    Pack<T> q;
#pragma unroll
    for (int j = 0; j < V; ++j) q[j] = from_f<T>(v[j]);
    LoosePack<T>* const to = reinterpret_cast<LoosePack<T>*>(p);
    if constexpr (STREAM) __builtin_nontemporal_store(q, to);
    else *to = q;
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
// relu / leakyrelu / elu the derivative from the left), on the hardware's 2^x and reciprocal (1 unit in the last place, 2^-23):
//   exp(x) = 2^t (1 + d), t = x log2 e rounded, d = x - t ln 2 what the rounding left: relative error (4 + |x| / 20) 2^-24, so that
//         silu, mish, gelu and elu's derivative keep their relative accuracy where they fall like exp(-|x|) (without d 58 2^-24 at
//         -60).  In 16 bits (T) without it: 1.5 |x| 2^-24 more, far below the output's own 2^-12
//   tanh: x P(x^2) below 1/2 (relative error 1.3e-8), 1 - 2 / (1 + e^2|x|) above
//   expm1: x P(x) above -1/2 (1.4e-9), exp(x) - 1 below
//   mish: tanh(log(1 + w)) = n / (n + 2) with w = e^x, n = w (w + 2): no cancellation; beyond x = 20 it is 1 in fp32
//   gelu: Phi(-a) = e^(-a^2/2) t Q(t), t = 1 / (1 + 0.3 a), a = |x| (Q's fit: 5e-8 up to a = 9; all of it within 20 2^-24): the tail
//         itself is approximated, so x Phi(x) keeps its relative accuracy for negative x, and the derivative shares the exponential
// The polynomials are least-maximum fits of these functions.
// ---------------------------------------------------------------------------------------------------
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;
template <class T>
DEVINL float exp_of(float x) {
  const float t = x * kLog2e, e = __builtin_amdgcn_exp2f(t);
  if (sizeof(T) < 4) return e;
  // |d| < 2^-15 wherever e is neither 0 nor infinite; beyond that it may be anything (inf - inf) and is held there
  return e * (1.f + __builtin_amdgcn_fmed3f(fmaf(t, -kLn2, x), -0x1p-15f, 0x1p-15f));
}
DEVINL float rcp_of(float x) { return __builtin_amdgcn_rcpf(x); }
template <class T>
DEVINL float tanh_of(float x) {
  const float a = fabsf(x), z = x * x;
  float p = 0.01715129399739507f;
  p = fmaf(p, z, -0.05299422865708484f);
  p = fmaf(p, z, 0.13324906927244848f);
  p = fmaf(p, z, -0.3333307579068465f);
  p = fmaf(p, z, 0.99999998737373f);
  const float far = fmaf(-2.f, rcp_of(1.f + exp_of<T>(2.f * a)), 1.f);
  return a < 0.5f ? x * p : copysignf(far, x);
}
template <class T>
DEVINL float expm1_of(float x) {  // x <= 0
  float p = 0.0011216346774701612f;
  p = fmaf(p, x, 0.008187385691190183f);
  p = fmaf(p, x, 0.04162908900354672f);
  p = fmaf(p, x, 0.16666224080228778f);
  p = fmaf(p, x, 0.4999998074594835f);
  p = fmaf(p, x, 0.9999999986263833f);
  return x > -0.5f ? x * p : exp_of<T>(x) - 1.f;
}
struct Gelu {
  float tail, density;  // Phi(-|x|), e^(-x^2 / 2)
};
template <class T>
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
  if (sizeof(T) < 4) {
    const float e = __builtin_amdgcn_exp2f(a * a * (-0.5f * kLog2e));
    return {t * q * e, e};
  }
  const float c = fminf(a, 16.f), n = -0.5f * c, h = n * c, u = h * kLog2e;  // h = -c^2 / 2; beyond 16 e is 0 (and NaN comes from t)
  const float d = fmaf(u, -kLn2, h) + fmaf(n, c, -h), g = __builtin_amdgcn_exp2f(u), e = fmaf(g, d, g);
  return {t * q * e, e};
}
template <class T>
DEVINL float act_of(float x, int act) {
  switch (act) {
    case AMBER_ACT_RELU: return x < 0.f ? 0.f : x;  // NaN stays NaN
    case AMBER_ACT_LEAKYRELU: return x > 0.f ? x : 0.01f * x;
    case AMBER_ACT_TANH: return tanh_of<T>(x);
    case AMBER_ACT_ELU: return x > 0.f ? x : expm1_of<T>(x);
    case AMBER_ACT_SILU: return x * rcp_of(1.f + exp_of<T>(-x));
    case AMBER_ACT_MISH: {
      const float w = exp_of<T>(x > 20.f ? 20.f : x), n = w * (w + 2.f);
      return x * (n * rcp_of(n + 2.f));
    }
    case AMBER_ACT_GELU: {
      const float a = fabsf(x);
      return fmaf(-fminf(a, 16.f), gelu_parts<T>(a).tail, fmaxf(x, 0.f));
    }
    default: return x;
  }
}
struct ActGrad {
  float a, d;  // act(x), act'(x)
};
template <class T>
DEVINL ActGrad act_grad(float x, int act) {
  switch (act) {
    case AMBER_ACT_RELU: return {x < 0.f ? 0.f : x, x > 0.f ? 1.f : 0.f};
    case AMBER_ACT_LEAKYRELU: return x > 0.f ? ActGrad{x, 1.f} : ActGrad{0.01f * x, 0.01f};
    case AMBER_ACT_TANH: {
      const float t = tanh_of<T>(x);
      return {t, fmaf(-t, t, 1.f)};
    }
    case AMBER_ACT_ELU: return x > 0.f ? ActGrad{x, 1.f} : ActGrad{expm1_of<T>(x), exp_of<T>(x)};
    case AMBER_ACT_SILU: {
      const float s = rcp_of(1.f + exp_of<T>(-x));
      return {x * s, s * fmaf(x, 1.f - s, 1.f)};
    }
    case AMBER_ACT_MISH: {
      const float c = x > 20.f ? 20.f : x, w = exp_of<T>(c), n = w * (w + 2.f), r = rcp_of(n + 2.f), t = n * r;
      return {x * t, fmaf(c * r, 4.f * w * (w + 1.f) * r, t)};
    }
    case AMBER_ACT_GELU: {
      const float a = fabsf(x), ac = fminf(a, 16.f);
      const Gelu g = gelu_parts<T>(a);
      return {fmaf(-ac, g.tail, fmaxf(x, 0.f)), fmaf(copysignf(ac, x), 0.39894228040143268f * g.density, x < 0.f ? g.tail : 1.f - g.tail)};
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
// v[j] of element first + j: +0 where dropped, else kept(j).  A wave whose lanes all start at multiples of 4 takes V / 4 calls of the
// generator, any other one more, its words moved down by first & 3.
template <int V, class Kept>
DEVINL void select_pack(const TailArgs& a, const Stream& s, int64_t first, float (&v)[V], const Kept& kept) {
  uint32_t w[V + 4];
  const uint64_t group = static_cast<uint64_t>(first) >> 2;
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    const Words t = philox(s, group + q);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[4 * q + j] = t.w[j];
  }
  if (__any(static_cast<int>(first) & 3)) {
    uint32_t shift = static_cast<uint32_t>(first) & 3;
    asm volatile("" : "+v"(shift));  // keeps this a branch: computed for all and selected, the extra call would cost every row
    const Words t = philox(s, static_cast<uint64_t>(first - shift + V) >> 2);
#pragma unroll
    for (int j = 0; j < 3; ++j) w[V + j] = t.w[j];
    const bool two = shift & 2, one = shift & 1;
#pragma unroll
    for (int j = 0; j < V + 1; ++j) {
      const uint32_t here = w[j], there = w[j + 2];
      w[j] = two ? there : here;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t here = w[j], there = w[j + 1];
      w[j] = one ? there : here;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = w[j] > a.last_dropped ? kept(j) : 0.f;
}
template <int V>
DEVINL void drop_pack(const TailArgs& a, const Stream& s, int64_t first, float (&v)[V]) {
  select_pack(a, s, first, v, [&](int j) { return v[j] * a.scale; });
}

// v = act(v), d = act'(v) (if wanted) on N values: the choice is uniform and made outside the loops.  SMOOTH: the activations beyond
// none / relu / leakyrelu, in kernels of their own (they need more registers).
template <class T, int ACT, bool GRAD, int N>
DEVINL void act_loop(float (&v)[N], float (&d)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (GRAD) {
      const ActGrad t = act_grad<T>(v[j], ACT);
      v[j] = t.a;
      d[j] = t.d;
    } else {
      v[j] = act_of<T>(v[j], ACT);
    }
  }
}
template <class T, bool SMOOTH, bool GRAD, int N>
DEVINL void act_pack(int act, float (&v)[N], float (&d)[N]) {
  if (SMOOTH) {
    switch (act) {
      case AMBER_ACT_TANH: return act_loop<T, AMBER_ACT_TANH, GRAD>(v, d);
      case AMBER_ACT_ELU: return act_loop<T, AMBER_ACT_ELU, GRAD>(v, d);
      case AMBER_ACT_SILU: return act_loop<T, AMBER_ACT_SILU, GRAD>(v, d);
      case AMBER_ACT_MISH: return act_loop<T, AMBER_ACT_MISH, GRAD>(v, d);
      default: return act_loop<T, AMBER_ACT_GELU, GRAD>(v, d);
    }
  }
  switch (act) {
    case AMBER_ACT_RELU: return act_loop<T, AMBER_ACT_RELU, GRAD>(v, d);
    case AMBER_ACT_LEAKYRELU: return act_loop<T, AMBER_ACT_LEAKYRELU, GRAD>(v, d);
    default: return act_loop<T, AMBER_ACT_NONE, GRAD>(v, d);
  }
}

inline __host__ __device__ bool is_smooth(int act) { return act != AMBER_ACT_NONE && act != AMBER_ACT_RELU && act != AMBER_ACT_LEAKYRELU; }
template <class T, bool GRAD, int N>
DEVINL void act_any(int act, float (&v)[N], float (&d)[N]) {
  if (is_smooth(act)) act_pack<T, true, GRAD>(act, v, d);
  else act_pack<T, false, GRAD>(act, v, d);
}

// ---------------------------------------------------------------------------------------------------
// without the norm: elementwise over the flat tensor, 16 bytes a thread, the next 16 on their way while these are worked on
// (32768 x 4096 fp32 dropout 189 -> 177 us, 6.1 TB/s; 1.44 M x 128 fp32 with an activation 264 -> 245 forward, 446 -> 370 backward).
// Bound by the memory; relu and leaky relu cost nothing beside it, gelu in fp32 2 % (248 us forward), in 16 bits
// more (1000003 x 333 fp16 with dropout 4.0 TB/s).
// ---------------------------------------------------------------------------------------------------
template <class T, bool BWD, bool SMOOTH, int CACHE>
__global__ __launch_bounds__(kBlock) void elementwise_kernel(TailArgs a) {
  constexpr int V = kVec<T>;
  const int64_t n = a.rows * a.width, packs = n / V;
  const T* x = static_cast<const T*>(a.x);
  const T* g = static_cast<const T*>(a.g);
  T* y = static_cast<T*>(a.y);
  const bool needs_x = !BWD || a.act != AMBER_ACT_NONE;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kBlock;
  int64_t p = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
  Pack<T> xn, gn;
  if (p < packs) {
    if (needs_x) xn = load_raw<CACHE == 2>(x + p * V);
    if (BWD) gn = load_raw<CACHE == 2>(g + p * V);
  }
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  // v = what the dropout applies to, z = the pre-activation
  const auto work = [&](float (&v)[V], float (&z)[V], int64_t first) {
    if (!BWD) act_pack<T, SMOOTH, false>(a.act, v, v);
    if (BWD && a.act != AMBER_ACT_NONE) {
      float d[V];
      act_pack<T, SMOOTH, true>(a.act, z, d);
      if (a.drop) {  // selected last: the derivative may be negative (-0), NaN or infinite where the gradient is 0
        select_pack(a, s, first, v, [&](int j) { return v[j] * a.scale * d[j]; });
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= d[j];
      }
    } else if (a.drop) {
      drop_pack(a, s, first, v);
    }
  };
  for (; p < packs; p += step) {
    float v[V], z[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      v[j] = to_f(BWD ? gn[j] : xn[j]);
      if (BWD && needs_x) z[j] = to_f(xn[j]);
    }
    if (p + step < packs) {  // on their way while this pack is worked on
      if (needs_x) xn = load_raw<CACHE == 2>(x + (p + step) * V);
      if (BWD) gn = load_raw<CACHE == 2>(g + (p + step) * V);
    }
    work(v, z, p * V);
    store_pack<CACHE >= 1>(y + p * V, V, v);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0 && packs * V < n) {  // what is left of a pack
    const int count = static_cast<int>(n - packs * V);
    float v[V], z[V];
    load_pack<false>((BWD ? g : x) + packs * V, count, v);
    if (BWD && needs_x) load_pack<false>(x + packs * V, count, z);
    work(v, z, packs * V);
    store_pack<false>(y + packs * V, count, v);
  }
}

// ---------------------------------------------------------------------------------------------------
// with the norm
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
// Sums of N values over the waves of a block, in the waves' order (W = 1: nothing to do).  `box` is used again only behind another
// barrier: callers alternate two boxes.
template <int W, int N>
DEVINL void join_waves(float (&v)[N], float (&box)[W][N]) {
  if (W == 1) return;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) box[threadIdx.x >> 6][i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = box[0][i];
#pragma unroll
    for (int w = 1; w < W; ++w) v[i] += box[w][i];
  }
}
// 1 / sqrt(v): the hardware's estimate (1 unit in the last place) and one Newton step.  The estimate takes no subnormal numbers,
// the step no infinity: a variance below 2^-96 is scaled (only where eps leaves one: uniform), an overflown one gives 0.
DEVINL float rsqrt_normal(float v) {
  const float r = __builtin_amdgcn_rsqf(v);
  return v > 3.0e38f ? r : r * fmaf(-0.5f * v * r, r, 1.5f);
}
DEVINL float rsqrt_of(float v, float least) {
  if (least >= 0x1p-96f) return rsqrt_normal(v);
  return v < 0x1p-96f ? rsqrt_normal(v * 0x1p96f) * 0x1p48f : rsqrt_normal(v);
}
// sum / D with inv = 1 / D rounded: one correction, so that the quotient is good to half a step
DEVINL float mean_of(float sum, float width, float inv) {
  const float m = sum * inv;
  return fmaf(fmaf(-m, width, sum), inv, m);
}
// What the differences d = a - m from a first mean m add up to: m carries the rounding errors of its sum (some 2^-24 |m|, which next to
// a small deviation is much: rows of 1000.1 with eps = 1e-5 came out at 0.04 instead of 0 for 1021 features), and the mean of d takes
// them off again (1440000 x 128 fp32 forward 237 us either way, 243 -> 250 with dropout, which asks for its vector instructions; 5003 x
// 4099 bf16 19.7 -> 20.5).  The variance is that of a: mean(d^2) - mean(d)^2, where the second term is as small as m's error.
struct Spread {
  float shift, rstd;  // mean(d): n = (d - shift) rstd, the row's mean is m + shift
};
DEVINL Spread spread_of(float sum, float squares, float inv, float eps) {
  const float shift = sum * inv;
  const float left = squares - fminf(shift * sum, 3.0e38f);  // not a difference of two infinities
  return {shift, rsqrt_of(fmaf(fmaxf(left, 0.f), inv, eps), eps)};  // left = NaN: m is, and so is every n
}
// A sum of many terms one after the other, with the rounding errors of its additions beside it (Knuth's two-sum): good to some 2^-24 of
// the terms' magnitude however many there are.  For rows whose lanes add more than a handful of packs (20 x 999983 fp32 forward 708 us
// before, 693 with it and a pack's terms added pairwise).
struct LongSum {
  float s = 0.f, e = 0.f;
  DEVINL void add(float v) {
    const float t = s + v, z = t - s;
    e += (s - (t - z)) + (v - z);
    s = t;
  }
  DEVINL float value() const { return s - s == 0.f ? s + e : s; }  // infinite or NaN: e is NaN
};
template <int V>
DEVINL float pack_sum(const float (&v)[V]) {
  float s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = v[j];
#pragma unroll
  for (int n = V / 2; n >= 1; n /= 2)
#pragma unroll
    for (int j = 0; j < n; ++j) s[j] += s[j + n];
  return s[0];
}

// Rows that no team holds in registers (beyond 16384 features): a block of 16 waves reads a row three times forward and twice
// backward (a row is in its XCD's cache by then), and gathers the weights' gradients in its part of `partial`.
constexpr int kWide = 1024;
template <class T>
__global__ __launch_bounds__(kWide) void norm_forward_kernel(TailArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float box[kWide / 64][1], boxes[kWide / 64][2];
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  const int width = static_cast<int>(a.width), fp32 = a.weight_dtype == AMBER_DTYPE_F32;
  const float inv = 1.f / static_cast<float>(width);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    T* y = static_cast<T*>(a.y) + row * a.width;
    float sum[1], both[2], v[V];
    const auto load = [&](int c) {
      load_pack<false>(x + c, width - c, v);
      act_any<T, false>(a.act, v, v);  // 0 where the row has ended: act(0) = 0
    };
    LongSum first;
    for (int c = threadIdx.x * V; c < width; c += kWide * V) {
      load(c);
      first.add(pack_sum(v));
    }
    sum[0] = team_sum<64>(first.value());
    join_waves<kWide / 64, 1>(sum, box);
    const float mean = mean_of(sum[0], static_cast<float>(width), inv);
    LongSum rest, squares;
    for (int c = threadIdx.x * V; c < width; c += kWide * V) {
      load(c);
      float q[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[j] = c + j < width ? v[j] - mean : 0.f;
        q[j] = v[j] * v[j];
      }
      rest.add(pack_sum(v));
      squares.add(pack_sum(q));
    }
    both[0] = team_sum<64>(rest.value());
    both[1] = team_sum<64>(squares.value());
    join_waves<kWide / 64, 2>(both, boxes);
    const Spread sp = spread_of(both[0], both[1], inv, a.eps);
    for (int c = threadIdx.x * V; c < width; c += kWide * V) {
      load(c);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < width)
          v[j] = fmaf((v[j] - mean - sp.shift) * sp.rstd, load_weight<T>(a.weight, fp32, c + j, 1.f),
                      load_weight<T>(a.bias, fp32, c + j, 0.f));
      if (a.drop) drop_pack(a, s, row * a.width + c, v);
      store_pack<false>(y + c, width - c, v);
    }
    if (a.stats && threadIdx.x == 0) {
      a.stats[2 * row] = mean + sp.shift;
      a.stats[2 * row + 1] = sp.rstd;
    }
  }
}

template <class T>
__global__ __launch_bounds__(kWide) void norm_backward_kernel(TailArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float box[2][kWide / 64][2];
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  const int width = static_cast<int>(a.width), fp32 = a.weight_dtype == AMBER_DTYPE_F32;
  const float inv = 1.f / static_cast<float>(width);
  float* pw = a.partial ? a.partial + static_cast<int64_t>(blockIdx.x) * 2 * width : nullptr;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* g = static_cast<const T*>(a.g) + row * a.ldg;
    const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
    float sums[2], n[V], h[V], d[V];
    LongSum hs, hns;
    const auto load = [&](int c) {
      load_pack<false>(x + c, width - c, n);
      load_pack<false>(g + c, width - c, h);
      act_any<T, true>(a.act, n, d);
      if (a.drop) drop_pack(a, s, row * a.width + c, h);
#pragma unroll
      for (int j = 0; j < V; ++j) n[j] = (n[j] - mean) * rstd;
    };
    for (int c = threadIdx.x * V; c < width; c += kWide * V) {
      load(c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (c + j >= width) {
          h[j] = n[j] = 0.f;
          continue;
        }
        if (pw) {  // a thread's own columns: nobody else touches them
          float* const at = pw + c + j;
          const bool first = row == blockIdx.x;
          at[0] = first ? h[j] * n[j] : fmaf(h[j], n[j], at[0]);
          at[width] = first ? h[j] : at[width] + h[j];
        }
        h[j] *= load_weight<T>(a.weight, fp32, c + j, 1.f);
        n[j] *= h[j];
      }
      hs.add(pack_sum(h));
      hns.add(pack_sum(n));
    }
    sums[0] = team_sum<64>(hs.value());
    sums[1] = team_sum<64>(hns.value());
    join_waves<kWide / 64, 2>(sums, box[turn]);
    if (!a.y) continue;
    T* y = static_cast<T*>(a.y) + row * a.width;
    const float m0 = sums[0] * inv, m1 = sums[1] * inv;
    for (int c = threadIdx.x * V; c < width; c += kWide * V) {
      load(c);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < width)
          d[j] = rstd * fmaf(-n[j], m1, fmaf(h[j], load_weight<T>(a.weight, fp32, c + j, 1.f), -m0)) * d[j];
      store_pack<false>(y + c, width - c, d);
    }
  }
}

// ---------------------------------------------------------------------------------------------------
// with the norm, rows in registers: a team of G lanes (W = 1: 64 / G teams a wave) or of W waves holds a row, K packs a lane
// ---------------------------------------------------------------------------------------------------
// A lane's columns: pack k starts at (k LANES + lane) V, moved back to width - V where it would pass the row's end.  The lane then
// holds columns that its neighbours hold too: they take no part in sums (element j of the last pack counts iff j >= skip) and are
// stored twice with the same bits (the compiler may not fuse multiplications and additions by itself here: it could do so for one
// pack and not for another).  So every access is one full pack and no lane needs a path of its own.  NARROW (width < V, a
// lane per row): element by element.
template <class T, int LANES, int K, bool NARROW, int CACHE>
struct Columns {
  static constexpr int V = kVec<T>;
  using Raw = Pack<T>;
  int at[K], skip, width;
  DEVINL Columns(int lane, int width_) : width(width_) {
#pragma unroll
    for (int k = 0; k < K; ++k) at[k] = NARROW ? 0 : min((k * LANES + lane) * V, width - V);
    skip = NARROW ? 0 : ((K - 1) * LANES + lane) * V - at[K - 1];
  }
  DEVINL bool ragged() const { return NARROW || width != LANES * K * V; }  // uniform
  DEVINL bool counts(int k, int j) const { return NARROW ? j < width : k < K - 1 || j >= skip; }
  DEVINL bool stores(int k) const { return k < K - 1 || skip < V; }
  DEVINL void load(const T* row, Raw (&raw)[K]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (NARROW) {
#pragma unroll
        for (int j = 0; j < V; ++j) raw[k][j] = j < width ? row[j] : from_f<T>(0.f);
      } else {
        raw[k] = load_raw<CACHE == 2>(row + at[k]);
      }
    }
  }
  DEVINL void store(T* row, int k, const float (&v)[V]) const {
    if (!stores(k)) return;
    store_pack<CACHE >= 1>(row + at[k], NARROW ? width : V, v);
  }
  // weight or bias of pack k in fp32
  DEVINL void load_weight_pack(const void* w, bool fp32, float missing, int k, float (&v)[V]) const {
    if (!w || NARROW) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = NARROW && j >= width ? 0.f : load_weight<T>(w, fp32, at[k] + j, missing);
    } else if (fp32) {
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        const Pack<float> p = *reinterpret_cast<const LoosePack<float>*>(static_cast<const float*>(w) + at[k] + q);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[q + j] = p[j];
      }
    } else {
      const Raw p = *reinterpret_cast<const LoosePack<T>*>(static_cast<const T*>(w) + at[k]);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = to_f(p[j]);
    }
  }
  DEVINL void load_weights(const void* w, bool fp32, float missing, float (&v)[K][V]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) load_weight_pack(w, fp32, missing, k, v[k]);
  }
};

// One row per team and sweep; the next sweep's loads are issued before this one's arithmetic.  (Two rows a sweep, or four, were
// slower: 1.44 M x 128 fp32 forward 292 us instead of 250, cached.)
template <class T, int G, int W, int K, bool SMOOTH, int CACHE>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void norm_rows_forward(TailArgs a) {
  constexpr int V = kVec<T>, LANES = G * W, THREADS = W == 1 ? 256 : 64 * W, TEAMS = THREADS / LANES;
  __shared__ float box[W][1], boxes[W][2];
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const Columns<T, LANES, K, LANES == 1, CACHE> cols(lane, static_cast<int>(a.width));
  const bool ragged = cols.ragged(), last = W == 1 || __any(cols.stores(K - 1));  // a wave without columns in the last pack skips it
  const float width = static_cast<float>(cols.width), inv = 1.f / width;
  const T* x = static_cast<const T*>(a.x);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * TEAMS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * TEAMS + team;
  Pack<T> next[K];
  if (row < a.rows) cols.load(x + row * a.ldx, next);
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  float w[K][V], b[K][V];
  cols.load_weights(a.weight, a.weight_dtype == AMBER_DTYPE_F32, 1.f, w);
  cols.load_weights(a.bias, a.weight_dtype == AMBER_DTYPE_F32, 0.f, b);
  for (; row < a.rows; row += stride) {  // W > 1: uniform over the block, which meets at the barriers
    float v[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) v[k][j] = to_f(next[k][j]);
    if (row + stride < a.rows) cols.load(x + (row + stride) * a.ldx, next);
    float sum[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k == K - 1 && !last) break;
      act_pack<T, SMOOTH, false>(a.act, v[k], v[k]);
      if (k < K - 1 || !ragged) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[0] += v[k][j];
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[0] += cols.counts(k, j) ? v[k][j] : 0.f;
      }
    }
    sum[0] = team_sum<G>(sum[0]);
    join_waves<W, 1>(sum, box);
    const float mean = mean_of(sum[0], width, inv);
    float both[2] = {0.f, 0.f};  // of the differences, of their squares
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k == K - 1 && !last) break;
#pragma unroll
      for (int j = 0; j < V; ++j) v[k][j] -= mean;
      if (k < K - 1 || !ragged) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          both[0] += v[k][j];
          both[1] = fmaf(v[k][j], v[k][j], both[1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float c = cols.counts(k, j) ? v[k][j] : 0.f;
          both[0] += c;
          both[1] = fmaf(c, c, both[1]);
        }
      }
    }
    both[0] = team_sum<G>(both[0]);
    both[1] = team_sum<G>(both[1]);
    join_waves<W, 2>(both, boxes);
    const Spread sp = spread_of(both[0], both[1], inv, a.eps);
    const float back = -sp.shift * sp.rstd;
    T* y = static_cast<T*>(a.y) + row * cols.width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k == K - 1 && !last) break;
#pragma unroll
      for (int j = 0; j < V; ++j) v[k][j] = fmaf(fmaf(v[k][j], sp.rstd, back), w[k][j], b[k][j]);
      if (a.drop) drop_pack(a, s, row * cols.width + cols.at[k], v[k]);
      cols.store(y, k, v[k]);
    }
    if (a.stats && lane == 0) {
      a.stats[2 * row] = mean + sp.shift;
      a.stats[2 * row + 1] = sp.rstd;
    }
  }
}

// Needs x, the gradient and two statistics of a row; the gradients of weight and bias gather over a team's rows, in registers (W = 16,
// rows beyond 8192 features: 128 registers a lane are too few, so in LDS, where every thread adds to places of its own), and are
// joined over the block at its end.  Two rows on their way instead of one changed nothing (20000 x 8192 fp32 381 us, 385).
template <class T, int G, int W, int K, bool SMOOTH, int CACHE>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void norm_rows_backward(TailArgs a) {
  constexpr int V = kVec<T>, LANES = G * W, THREADS = W == 1 ? 256 : 64 * W, TEAMS = THREADS / LANES;
  constexpr bool IN_LDS = W == 16, AHEAD = !(IN_LDS && K * V == 16);
  __shared__ float box[2][W][2];
  // W = 1: [2][columns] for the join of the block's waves; IN_LDS: [2][K][V / 4][threads] packs of 4 sums
  __shared__ __attribute__((aligned(16))) float columns[W == 1 || IN_LDS ? 2 * LANES * K * V : 4];
  Pack<float>* const mine = reinterpret_cast<Pack<float>*>(columns) + threadIdx.x;
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  const Columns<T, LANES, K, LANES == 1, CACHE> cols(lane, static_cast<int>(a.width));
  const bool ragged = cols.ragged(), last = W == 1 || __any(cols.stores(K - 1)), fp32 = a.weight_dtype == AMBER_DTYPE_F32;
  const float inv = 1.f / static_cast<float>(cols.width);
  const T* x = static_cast<const T*>(a.x);
  const T* g = static_cast<const T*>(a.g);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * TEAMS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * TEAMS + team;
  Pack<T> xn[K], gn[K];
  float mean_next = 0.f, rstd_next = 0.f;
  const auto fetch = [&](int64_t r) {
    cols.load(x + r * a.ldx, xn);
    cols.load(g + r * a.ldg, gn);
    mean_next = a.stats[2 * r];
    rstd_next = a.stats[2 * r + 1];
  };
  if (AHEAD && row < a.rows) fetch(row);
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  float w[K][V], dw[IN_LDS ? 1 : K][V], db[IN_LDS ? 1 : K][V];
  cols.load_weights(a.weight, fp32, 1.f, w);
  if (IN_LDS) {
#pragma unroll
    for (int i = 0; i < 2 * K * V / 4; ++i) mine[i * THREADS] = Pack<float>{0.f, 0.f, 0.f, 0.f};
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) dw[IN_LDS ? 0 : k][j] = db[IN_LDS ? 0 : k][j] = 0.f;
  }
  for (int turn = 0; row < a.rows; row += stride, turn ^= 1) {
    if (!AHEAD) fetch(row);
    const float mean = mean_next, rstd = rstd_next;
    float n[K][V], h[K][V], dact[K][V], sums[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        n[k][j] = to_f(xn[k][j]);
        h[k][j] = to_f(gn[k][j]);
      }
    if (AHEAD && row + stride < a.rows) fetch(row + stride);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k == K - 1 && !last) break;
      if (a.drop) drop_pack(a, s, row * cols.width + cols.at[k], h[k]);
      act_pack<T, SMOOTH, true>(a.act, n[k], dact[k]);
#pragma unroll
      for (int j = 0; j < V; ++j) n[k][j] = (n[k][j] - mean) * rstd;
      if (IN_LDS) {
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
          Pack<float> tw = mine[(k * (V / 4) + q) * THREADS], tb = mine[((K + k) * (V / 4) + q) * THREADS];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            tw[j] = fmaf(h[k][4 * q + j], n[k][4 * q + j], tw[j]);
            tb[j] += h[k][4 * q + j];
          }
          mine[(k * (V / 4) + q) * THREADS] = tw;
          mine[((K + k) * (V / 4) + q) * THREADS] = tb;
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          dw[IN_LDS ? 0 : k][j] = fmaf(h[k][j], n[k][j], dw[IN_LDS ? 0 : k][j]);
          db[IN_LDS ? 0 : k][j] += h[k][j];
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) h[k][j] *= w[k][j];
      if (k < K - 1 || !ragged) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          sums[0] += h[k][j];
          sums[1] = fmaf(h[k][j], n[k][j], sums[1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float c = cols.counts(k, j) ? h[k][j] : 0.f;
          sums[0] += c;
          sums[1] = fmaf(c, n[k][j], sums[1]);
        }
      }
    }
    sums[0] = team_sum<G>(sums[0]);
    sums[1] = team_sum<G>(sums[1]);
    // the boxes take turns: a wave writes one again only behind the barrier that follows everyone's reads of it
    join_waves<W, 2>(sums, box[turn]);
    if (!a.y) continue;
    T* y = static_cast<T*>(a.y) + row * cols.width;
    const float m0 = sums[0] * inv, m1 = sums[1] * inv;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (k == K - 1 && !last) break;
      float d[V];
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = rstd * fmaf(-n[k][j], m1, h[k][j] - m0) * dact[k][j];
      cols.store(y, k, d);
    }
  }
  if (!a.grad_weight && !a.grad_bias) return;
  // the block's sums of column c: to its part of `partial`, or (the only block) where they belong
  float* const out = a.partial ? a.partial + static_cast<int64_t>(blockIdx.x) * 2 * cols.width : nullptr;
  const auto give = [&](int c, float sw, float sb) {
    if (out) {
      out[c] = sw;
      out[cols.width + c] = sb;
    } else {
      store_weight<T>(a.grad_weight, fp32, c, sw);
      store_weight<T>(a.grad_bias, fp32, c, sb);
    }
  };
  if constexpr (W > 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (cols.counts(k, j))
          give(cols.at[k] + j, IN_LDS ? mine[(k * (V / 4) + j / 4) * THREADS][j % 4] : dw[IN_LDS ? 0 : k][j],
               IN_LDS ? mine[((K + k) * (V / 4) + j / 4) * THREADS][j % 4] : db[IN_LDS ? 0 : k][j]);
    return;
  }
  // the teams of a wave, then the waves one after the other through LDS: a fixed order
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int m = LANES; m < 64; m <<= 1) {
        dw[k][j] += __shfl_xor(dw[k][j], m, 64);
        db[k][j] += __shfl_xor(db[k][j], m, 64);
      }
  for (int wave = 0; wave < THREADS / 64; ++wave) {
    if (static_cast<int>(threadIdx.x >> 6) == wave && (threadIdx.x & 63) < LANES) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (cols.counts(k, j)) {
            const int c = cols.at[k] + j;
            columns[c] = wave ? columns[c] + dw[k][j] : dw[k][j];
            columns[LANES * K * V + c] = wave ? columns[LANES * K * V + c] + db[k][j] : db[k][j];
          }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < cols.width; c += THREADS) give(c, columns[c], columns[LANES * K * V + c]);
}

inline unsigned blocks_for(int64_t work, int64_t limit) { return static_cast<unsigned>(work < 1 ? 1 : work < limit ? work : limit); }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a row is held: G lanes of a wave (W = 1) or W waves, K packs of V elements a lane, at most 16 elements.  The smallest team that
// holds the row; a row that 16 waves cannot hold (G = 0) is read from memory three times.  K - 1 packs a lane never hold the row.
struct Shape {
  int g, w, k;
};
inline int vec_of(int dtype) { return dtype == AMBER_DTYPE_F32 ? 4 : 8; }
inline Shape shape_for(int64_t width, int vec) {
  if (width < vec) return {1, 1, 1};
  const int64_t packs = cdiv(width, vec);
  for (int g = 2; g <= 64; g *= 2)
    if (packs <= g) return {g, 1, 1};
  const int most = 16 / vec;
  for (int w = 1; w <= 16; w *= w == 1 ? 4 : 2)
    for (int k = 1; k <= most; ++k)
      if (packs <= 64 * w * k) return {64, w, k};
  return {0, 0, 0};
}
inline int64_t teams_in_block(const Shape& h) { return h.w > 1 ? 1 : 256 / h.g; }
// Blocks of a launch: each takes rows in turn and has the next ones on their way, so their number sets the bytes in flight.  About
// 4 MB forward and 6 MB backward (x and the gradient) are best; more only spread the accesses over more pages: 1.44 M x 128 fp32
// forward 250 us with 1024 blocks, 311 with 512, 328 with 2048 (before its accesses went past the caches: 237 us now, 6.2 TB/s);
// 100000 x 1024 fp32 backward 219 with 256, 237 with 1024.
// The generator and the smooth activations ask for more waves than that: 100000 x 2048 bf16 forward with dropout 197 us with 1024
// blocks, 187 with 1280; 100000 x 1024 fp32 169 with 256, 143 with 768.  Measured from 32 to 16384 features, 1000 to 2 M rows, fp32
// and bf16, with and without dropout, in steps of 256 blocks: a CU more or less than the others counts (100000 x 1020 fp32 forward
// 136 us with 256 blocks, 175 with 257).  Backward teams of 8 and 16 waves fit once on a CU.
inline int64_t clamped(int64_t v, int64_t low, int64_t high) { return v < low ? low : v > high ? high : v; }
inline int64_t even(int64_t blocks) { return (blocks + 128) / 256 * 256; }  // a whole number of them on each of the 256 CUs
inline int64_t block_bytes(const TailArgs& a, const Shape& h) { return teams_in_block(h) * a.width * (16 / vec_of(a.dtype)); }
inline int64_t forward_blocks(const TailArgs& a, const Shape& h) {
  const bool half = a.dtype != AMBER_DTYPE_F32;
  const int64_t least = a.drop && half ? 1280 : a.drop || is_smooth(a.act) ? 768 : 256;
  return blocks_for(cdiv(a.rows, teams_in_block(h)), clamped(even((4 << 20) / block_bytes(a, h)), least, 2048));
}
inline int64_t backward_blocks(const TailArgs& a, const Shape& h) {
  const bool half = a.dtype != AMBER_DTYPE_F32;
  const int64_t least = a.drop && half && h.w < 8 ? 512 : 256;
  int64_t blocks = clamped(even((6 << 20) / (2 * block_bytes(a, h))), least, h.w < 8 ? 768 : 256);
  const int64_t sweeps = cdiv(a.rows, teams_in_block(h));
  // A block's partial sums cost 8 bytes a feature each way, and its join some microseconds: at least 3 sweeps a block, and where a block
  // takes one row at a time 12 rows of one pack a lane, 16 of more.  us with the rule, with that many rows, with that many:
  //   3:  6000 x 256 bf16 10.6, with 1 12.3, with 12 10.7; 2000 x 1021 bf16 13.1, 16.2, 13.2; 20736 x 64 fp32 10.2, 10.5, 11.1;
  //       30000 x 128 fp32 13.9, 14.1, 14.8
  //   12: 5003 x 1500 bf16 20.5, with 3 21.1, with 24 24.7; 3000 x 2000 18.5, 21.2, 18.2; 10000 x 1200 24.8, 24.8, 27.7
  //   16: 5003 x 4096 bf16 32.6, with 12 35.1, with 32 32.6; 8000 x 3000 36.3, 36.4, 42.5; 5003 x 2000 fp32 24.7, 25.6, 24.7
  blocks = clamped(even(sweeps / (h.w == 1 ? 3 : h.k == 1 ? 12 : 16)), 256, blocks);
  return sweeps <= 4 ? 1 : blocks_for(sweeps, blocks);  // a few rows: one block, no partial sums and no second launch
}

inline int cache_mode(const TailArgs& a, int inputs) {
  const int64_t bytes = a.rows * a.width * (16 / vec_of(a.dtype));
  return inputs * bytes > 300000000 ? 2 : (inputs + 1) * bytes > 384000000 ? 1 : 0;
}

template <class T, int G, int W, int K, bool SMOOTH, int CACHE>
void launch_rows(const TailArgs& a, const Shape& h, bool backward, hipStream_t s) {
  const dim3 block(W == 1 ? 256 : 64 * W);
  if (backward)
    hipLaunchKernelGGL((norm_rows_backward<T, G, W, K, SMOOTH, CACHE>), dim3(static_cast<unsigned>(backward_blocks(a, h))), block, 0, s, a);
  else
    hipLaunchKernelGGL((norm_rows_forward<T, G, W, K, SMOOTH, CACHE>), dim3(static_cast<unsigned>(forward_blocks(a, h))), block, 0, s, a);
}
template <class T, bool SMOOTH, int CACHE>
void launch_shape(const TailArgs& a, const Shape& h, bool backward, hipStream_t s) {
#define AMBER_ROWS(G, W, K) \
  if (h.g == G && h.w == W && h.k == K) return launch_rows<T, G, W, K, SMOOTH, CACHE>(a, h, backward, s)
  AMBER_ROWS(1, 1, 1);
  AMBER_ROWS(2, 1, 1);
  AMBER_ROWS(4, 1, 1);
  AMBER_ROWS(8, 1, 1);
  AMBER_ROWS(16, 1, 1);
  AMBER_ROWS(32, 1, 1);
  AMBER_ROWS(64, 1, 1);
  AMBER_ROWS(64, 1, 2);
  if constexpr (kVec<T> == 4) {  // 4 packs of 4 elements
    AMBER_ROWS(64, 1, 3);
    AMBER_ROWS(64, 1, 4);
    AMBER_ROWS(64, 4, 2);
    AMBER_ROWS(64, 4, 3);
    AMBER_ROWS(64, 4, 4);
    AMBER_ROWS(64, 8, 3);
    AMBER_ROWS(64, 8, 4);
    AMBER_ROWS(64, 16, 3);
    AMBER_ROWS(64, 16, 4);
  } else {  // 2 packs of 8
    AMBER_ROWS(64, 4, 1);
    AMBER_ROWS(64, 4, 2);
    AMBER_ROWS(64, 8, 2);
    AMBER_ROWS(64, 16, 2);
  }
#undef AMBER_ROWS
}
template <class T, bool BWD, bool SMOOTH>
void launch_elementwise(const TailArgs& a, hipStream_t s) {
  const int inputs = BWD && a.act != AMBER_ACT_NONE ? 2 : 1;
  // about as many bytes in flight for two inputs as for one: 1.44 M x 128 fp32 with leaky relu 245 us with 1024 blocks, 267 with 1536,
  // 274 with 2048; its backward 383, 434, 438, and 372 with 768.  Where a pack asks for more work, more waves: 32768 x 4096 bf16
  // dropout 91 us with 1024, 79 with 1280.  Small calls do not care (20736 x 512 fp32 13.8 us with 768 to 2048)
  const bool half = a.dtype != AMBER_DTYPE_F32;
  const int64_t most = half && (SMOOTH || (a.drop && inputs == 1)) ? 1280 : inputs == 2 ? 768 : 1024;
  const dim3 grid(blocks_for(cdiv(a.rows * a.width, kBlock * kVec<T>), most));
  switch (cache_mode(a, inputs)) {
    case 0: hipLaunchKernelGGL((elementwise_kernel<T, BWD, SMOOTH, 0>), grid, dim3(kBlock), 0, s, a); break;
    case 1: hipLaunchKernelGGL((elementwise_kernel<T, BWD, SMOOTH, 1>), grid, dim3(kBlock), 0, s, a); break;
    default: hipLaunchKernelGGL((elementwise_kernel<T, BWD, SMOOTH, 2>), grid, dim3(kBlock), 0, s, a);
  }
}
template <class T, bool SMOOTH>
bool launch_in_registers(const TailArgs& a, bool backward, hipStream_t s) {
  const Shape h = shape_for(a.width, kVec<T>);
  if (h.g == 0) return false;
  switch (cache_mode(a, backward ? 2 : 1)) {
    case 0: launch_shape<T, SMOOTH, 0>(a, h, backward, s); break;
    case 1: launch_shape<T, SMOOTH, 1>(a, h, backward, s); break;
    default: launch_shape<T, SMOOTH, 2>(a, h, backward, s);
  }
  return true;
}

template <class T>
hipError_t tail_forward_t(const TailArgs& a, bool normalize, hipStream_t s) {
  const bool smooth = is_smooth(a.act);
  if (!normalize)
    smooth ? launch_elementwise<T, false, true>(a, s) : launch_elementwise<T, false, false>(a, s);
  else if (!(smooth ? launch_in_registers<T, true>(a, false, s) : launch_in_registers<T, false>(a, false, s)))
    hipLaunchKernelGGL((norm_forward_kernel<T>), dim3(blocks_for(a.rows, 512)), dim3(kWide), 0, s, a);
  return hipGetLastError();
}
// dx and, into a.partial, the blocks' sums for the weights' gradients
template <class T>
hipError_t tail_backward_t(const TailArgs& a, bool normalize, hipStream_t s) {
  const bool smooth = is_smooth(a.act);
  if (!normalize)
    smooth ? launch_elementwise<T, true, true>(a, s) : launch_elementwise<T, true, false>(a, s);
  else if (!(smooth ? launch_in_registers<T, true>(a, true, s) : launch_in_registers<T, false>(a, true, s)))
    hipLaunchKernelGGL((norm_backward_kernel<T>), dim3(static_cast<unsigned>(tail_partial_blocks(a))), dim3(kWide), 0, s, a);
  return hipGetLastError();
}

}  // namespace
}  // namespace amber
