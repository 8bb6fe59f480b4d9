// What is common to all element types of the activation -> LayerNorm -> dropout operators (norm_dropout.h): the generator's state,
// its mask, the join of the weights' gradients, the choice of the type.
#include "norm_dropout.h"

namespace amber {
hipError_t tail_forward_f32(const TailArgs& a, bool normalize, hipStream_t s);
hipError_t tail_forward_bf16(const TailArgs& a, bool normalize, hipStream_t s);
hipError_t tail_forward_f16(const TailArgs& a, bool normalize, hipStream_t s);
hipError_t tail_backward_f32(const TailArgs& a, bool normalize, hipStream_t s);
hipError_t tail_backward_bf16(const TailArgs& a, bool normalize, hipStream_t s);
hipError_t tail_backward_f16(const TailArgs& a, bool normalize, hipStream_t s);

namespace {

__global__ void generator_take_kernel(int64_t* state, int64_t count, int64_t* taken) {
  taken[0] = state[0];
  taken[1] = static_cast<int64_t>(atomicAdd(reinterpret_cast<unsigned long long*>(state + 1), static_cast<unsigned long long>(count)));
}

__global__ __launch_bounds__(kBlock) void keep_mask_kernel(TailArgs a, uint8_t* out) {
  Stream s{};
  if (a.drop) s = stream_of(a.state, a.sequence);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kBlock * 4;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x) * 4; i < a.rows; i += step) {
    uint32_t bytes = 0x01010101u;
    if (a.drop) {
      const Words w = philox(s, static_cast<uint64_t>(i) >> 2);
      bytes = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) bytes |= w.w[j] > a.last_dropped ? 1u << (8 * j) : 0u;
    }
    if (i + 4 <= a.rows && (reinterpret_cast<uintptr_t>(out) & 3) == 0) {
      *reinterpret_cast<uint32_t*>(out + i) = bytes;
    } else {
      for (int j = 0; j < 4 && i + j < a.rows; ++j) out[i + j] = static_cast<uint8_t>(bytes >> (8 * j));
    }
  }
}

// gradients of weight and bias: the blocks' partial sums [blocks][2 width].  A block of 1024 threads takes C columns, Q = 1024 / C
// threads each: thread q adds blocks q, q + Q, ... in order, then a tree over q (always the same one).  Few columns are cut small, so
// that more than a handful of CUs works on them; many wide, for whole cache lines (16 for all: 768 x 128 4.1 us, now 3.5; 256 x 8198
// 6.6, now 4.7; 256 x 16384 8.0, now 5.0).  A launch of its own: a last block that joins would need a counter that someone clears.
template <int C>
__global__ __launch_bounds__(1024) void weight_gradient_kernel(TailArgs a, int64_t blocks) {
  constexpr int Q = 1024 / C, LANES = Q < 64 ? Q : 64, PER = Q / LANES;
  __shared__ float box[C][Q + 1];
  const int c = threadIdx.x % C, q = threadIdx.x / C;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * C, columns = 2 * a.width;
  float sum = 0.f;
  if (first + c < columns) {
    const float* p = a.partial + q * columns + first + c;
#pragma unroll 8
    for (int64_t b = q; b < blocks; b += Q, p += Q * columns) sum += *p;
  }
  box[c][q] = sum;
  __syncthreads();
  const int mine = threadIdx.x / LANES, lane = threadIdx.x % LANES;  // LANES lanes join a column
  if (mine >= C) return;
  sum = box[mine][lane];
#pragma unroll
  for (int i = 1; i < PER; ++i) sum += box[mine][lane + i * LANES];
  sum = team_sum<LANES>(sum);
  const int64_t out = first + mine;
  if (lane != 0 || out >= columns) return;
  void* to = out < a.width ? a.grad_weight : a.grad_bias;
  const int64_t i = out < a.width ? out : out - a.width;
  if (a.weight_dtype == AMBER_DTYPE_F32) store_weight<float>(to, 1, i, sum);
  else if (a.weight_dtype == AMBER_DTYPE_BF16) store_weight<bf16>(to, 0, i, sum);
  else store_weight<f16>(to, 0, i, sum);
}
template <int C>
void launch_weight_gradient(const TailArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((weight_gradient_kernel<C>), dim3(static_cast<unsigned>(cdiv(2 * a.width, C))), dim3(1024), 0, s, a,
                     a.rows > 0 ? tail_partial_blocks(a) : 0);
}

}  // namespace

int64_t tail_partial_blocks(const TailArgs& a) {
  const Shape h = shape_for(a.width, vec_of(a.dtype));
  return h.g ? backward_blocks(a, h) : blocks_for(a.rows, 256);
}
int64_t tail_partial_floats(const TailArgs& a) {
  if (a.rows == 0) return 0;
  const int64_t blocks = tail_partial_blocks(a);
  return blocks == 1 && shape_for(a.width, vec_of(a.dtype)).g ? 0 : 2 * a.width * blocks;
}

hipError_t launch_tail_forward(const TailArgs& a, bool normalize, hipStream_t s) {
  switch (a.dtype) {
    case AMBER_DTYPE_F32: return tail_forward_f32(a, normalize, s);
    case AMBER_DTYPE_BF16: return tail_forward_bf16(a, normalize, s);
    default: return tail_forward_f16(a, normalize, s);
  }
}
hipError_t launch_tail_backward(const TailArgs& a, bool normalize, hipStream_t s) {
  if (a.rows > 0) {
    hipError_t e;
    switch (a.dtype) {
      case AMBER_DTYPE_F32: e = tail_backward_f32(a, normalize, s); break;
      case AMBER_DTYPE_BF16: e = tail_backward_bf16(a, normalize, s); break;
      default: e = tail_backward_f16(a, normalize, s); break;
    }
    if (e != hipSuccess) return e;
  }
  if ((a.grad_weight || a.grad_bias) && (a.partial || a.rows == 0)) {  // no rows: zeros
    if (a.width <= 256) launch_weight_gradient<4>(a, s);
    else if (a.width <= 1024) launch_weight_gradient<16>(a, s);
    else launch_weight_gradient<64>(a, s);
  }
  return hipGetLastError();
}
hipError_t launch_keep_mask(const TailArgs& a, uint8_t* out, hipStream_t s) {
  hipLaunchKernelGGL(keep_mask_kernel, dim3(blocks_for(cdiv(a.rows, 4 * kBlock), kMaxBlocks)), dim3(kBlock), 0, s, a, out);
  return hipGetLastError();
}
hipError_t launch_generator_take(int64_t* state, int64_t count, int64_t* taken, hipStream_t s) {
  hipLaunchKernelGGL(generator_take_kernel, dim3(1), dim3(1), 0, s, state, count, taken);
  return hipGetLastError();
}

}  // namespace amber
