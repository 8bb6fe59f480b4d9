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

// gradients of weight and bias: the blocks' partial sums [blocks][2 width].  A block takes 16 columns, 64 threads each of them:
// thread q adds blocks q, q + 64, ... in order, then a tree over q.
__global__ __launch_bounds__(1024) void weight_gradient_kernel(TailArgs a, int64_t blocks) {
  __shared__ float box[16][65];
  const int c = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int64_t column = static_cast<int64_t>(blockIdx.x) * 16 + c, columns = 2 * a.width;
  float sum = 0.f;
  if (column < columns) {
#pragma unroll 8
    for (int64_t b = q; b < blocks; b += 64) sum += a.partial[b * columns + column];
  }
  box[c][q] = sum;
  __syncthreads();
  const int wave = threadIdx.x >> 6;
  sum = team_sum<64>(box[wave][threadIdx.x & 63]);
  const int64_t out = static_cast<int64_t>(blockIdx.x) * 16 + wave;
  if ((threadIdx.x & 63) != 0 || out >= columns) return;
  void* to = out < a.width ? a.grad_weight : a.grad_bias;
  const int64_t i = out < a.width ? out : out - a.width;
  if (a.weight_dtype == AMBER_DTYPE_F32) store_weight<float>(to, 1, i, sum);
  else if (a.weight_dtype == AMBER_DTYPE_BF16) store_weight<bf16>(to, 0, i, sum);
  else store_weight<f16>(to, 0, i, sum);
}

}  // namespace

int64_t tail_partial_blocks(const TailArgs& a) {
  const Shape h = shape_for(a.width, vec_of(a.dtype));
  return h.g ? backward_blocks(a, h) : blocks_for(a.rows, 256);
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
  if (a.grad_weight || a.grad_bias)  // no rows: zeros
    hipLaunchKernelGGL(weight_gradient_kernel, dim3(static_cast<unsigned>(cdiv(2 * a.width, 16))), dim3(1024), 0, s, a,
                       a.rows > 0 ? tail_partial_blocks(a) : 0);
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
