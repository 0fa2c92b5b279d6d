// The norms around a transformer block's output, fused with the block's gate, the residual add
// and, for the INT8 path, the per-token quantiser of the next product's activations (no
// counterpart in the reference, whose src/rms_norm_w_residual.cu:40-75 is one norm after one
// add):
//
//   u = x                    or  x * rsqrt(mean(x^2) + eps) * post_weight     the block's own norm
//   u = u * gate             (optional; one gate row per `rows_per_gate` tokens)
//   z = residual_scale * residual + u                                       the residual stream
//   y = z * rsqrt(mean(z^2) + eps) * weight                                 the next block's norm
//   out: y and z, or q = rint(y / scale), scale = max(amax|y|, 2^-100) / 127 and z.
//
// All of it in FP32.  z is rounded once, to the residual's type, on its way to memory; y is
// computed from the unrounded z, so that a 16-bit residual stream costs y nothing.
//
// Bound by HBM bandwidth: a row lives in registers between the reductions (row_ops.cuh), so
// every input byte is read once and every output byte written once.
#include <cstdint>
#include <cuda_runtime.h>

#include "host_common.h"
#include "ptx.cuh"
#include "row_ops.cuh"

namespace texo {
namespace bn {

struct Args {
  const void *x, *residual, *weight, *post_weight, *gate;
  void *y, *z;
  int8_t* q;
  float* scale;
  long long N;
  int C;
  long long rows_per_gate;
  int gate_per_channel;  // 0: one value per gate row
  float eps, residual_scale;
  int weights_f32;  // weight, post_weight and gate are FP32 (else they have x's type)
};

// Eight values of a weight-like row, in either of its two types.
template <bool VECTOR, typename X>
__device__ __forceinline__ void load_weights(const void* base, bool f32, size_t offset, int C, int thread,
                                             int threads, int i, float (&v)[8]) {
  if (f32)
    row::load_shared_group<VECTOR>(static_cast<const float*>(base) + offset, C, thread, threads, i, v);
  else
    row::load_shared_group<VECTOR>(static_cast<const X*>(base) + offset, C, thread, threads, i, v);
}

// The row in registers.  blockDim = (threads of a row, rows of the block).
template <typename X, typename R, bool QUANT, bool VECTOR, int UNITS>
__global__ void __launch_bounds__(UNITS == 4 ? 512 : 1024)
    row_kernel(const Args a) {
  __shared__ float sum_scratch[2][row::MAX_WARPS];
  __shared__ unsigned max_scratch[row::MAX_WARPS];
  const long long n = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (n >= a.N) return;  // only blocks of one-warp rows reach past N; they meet at no barrier
  const int t = threadIdx.x, threads = blockDim.x, warps = threads / 32, C = a.C;
  const size_t at = size_t(n) * C;
  const X* x = static_cast<const X*>(a.x) + at;
  const R* residual = static_cast<const R*>(a.residual) + at;

  row::Raw8<X> xr[UNITS];
  row::Raw8<R> rr[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) xr[i] = row::load_group<VECTOR>(x, C, t, threads, i);
#pragma unroll
  for (int i = 0; i < UNITS; ++i) rr[i] = row::load_group<VECTOR>(residual, C, t, threads, i);

  float v[UNITS][8];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = row::to_float(xr[i].v[j]);
  }
  if (a.post_weight) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[i][j] * v[i][j];
    }
    const float inv = rsqrtf(row::row_sum(sum, sum_scratch[0], warps) / float(C) + a.eps);
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      float w[8];
      load_weights<VECTOR, X>(a.post_weight, a.weights_f32, 0, C, t, threads, i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= inv * w[j];
    }
  }
  if (a.gate) {
    const size_t row = size_t(n / a.rows_per_gate);
    if (a.gate_per_channel) {
#pragma unroll
      for (int i = 0; i < UNITS; ++i) {
        float g[8];
        load_weights<VECTOR, X>(a.gate, a.weights_f32, row * C, C, t, threads, i, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= g[j];
      }
    } else {
      const float g = a.weights_f32 ? static_cast<const float*>(a.gate)[row]
                                    : row::to_float(static_cast<const X*>(a.gate)[row]);
#pragma unroll
      for (int i = 0; i < UNITS; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= g;
      }
    }
  }
  float sum = 0.f;
  R* z = static_cast<R*>(a.z) + at;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // values past the row's end are products with a zero: not for a gate that is infinite or NaN
      const bool in = row::position<VECTOR>(t, threads, i, j) < C;
      v[i][j] = in ? __fmaf_rn(a.residual_scale, row::to_float(rr[i].v[j]), v[i][j]) : 0.f;
      sum += v[i][j] * v[i][j];
    }
    row::store_group<VECTOR>(z, C, t, threads, i, v[i]);
  }
  const float inv = rsqrtf(row::row_sum(sum, sum_scratch[1], warps) / float(C) + a.eps);
  unsigned amax = 0;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    float w[8];
    load_weights<VECTOR, X>(a.weight, a.weights_f32, 0, C, t, threads, i, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i][j] *= inv * w[j];
      if (QUANT && row::position<VECTOR>(t, threads, i, j) < C) amax = max(amax, __float_as_uint(fabsf(v[i][j])));
    }
    if (!QUANT) row::store_group<VECTOR>(static_cast<X*>(a.y) + at, C, t, threads, i, v[i]);
  }
  if (QUANT) {
    const row::TokenScale s = row::token_scale(row::row_max(amax, max_scratch, warps));
    if (t == 0) a.scale[n] = s.scale;
#pragma unroll
    for (int i = 0; i < UNITS; ++i) row::store_quantised<VECTOR>(a.q + at, C, t, threads, i, v[i], s.inverse);
  }
}

// Rows that the registers do not hold: the values are computed again from x and residual in
// every pass (from L2 after the first).  z and y may lie over residual and x as in the kernel
// above: the last pass alone writes, each element after its own thread has read it.
constexpr int LONG_THREADS = 1024;
template <typename X, typename R, bool QUANT>
__global__ void __launch_bounds__(LONG_THREADS) long_row_kernel(const Args a) {
  __shared__ float sum_scratch[2][row::MAX_WARPS];
  __shared__ unsigned max_scratch[row::MAX_WARPS];
  constexpr int WARPS = LONG_THREADS / 32;
  const long long n = blockIdx.x;
  const int C = a.C;
  const size_t at = size_t(n) * C;
  const X* x = static_cast<const X*>(a.x) + at;
  const R* residual = static_cast<const R*>(a.residual) + at;
  auto weight = [&](const void* base, size_t i) {
    return a.weights_f32 ? static_cast<const float*>(base)[i] : row::to_float(static_cast<const X*>(base)[i]);
  };
  float post_inv = 1.f;
  if (a.post_weight) {
    float sum = 0.f;
    for (int c = threadIdx.x; c < C; c += LONG_THREADS) {
      const float v = row::to_float(x[c]);
      sum += v * v;
    }
    post_inv = rsqrtf(row::row_sum(sum, sum_scratch[0], WARPS) / float(C) + a.eps);
  }
  const size_t gate_row = a.gate ? size_t(n / a.rows_per_gate) : 0;
  auto z_at = [&](int c) {
    float v = row::to_float(x[c]);
    if (a.post_weight) v *= post_inv * weight(a.post_weight, c);
    if (a.gate) v *= weight(a.gate, a.gate_per_channel ? gate_row * C + c : gate_row);
    return __fmaf_rn(a.residual_scale, row::to_float(residual[c]), v);
  };
  float sum = 0.f;
  for (int c = threadIdx.x; c < C; c += LONG_THREADS) {
    const float v = z_at(c);
    sum += v * v;
  }
  const float inv = rsqrtf(row::row_sum(sum, sum_scratch[1], WARPS) / float(C) + a.eps);
  row::TokenScale s = {0.f, 0.f};
  if (QUANT) {
    unsigned amax = 0;
    for (int c = threadIdx.x; c < C; c += LONG_THREADS)
      amax = max(amax, __float_as_uint(fabsf(z_at(c) * (inv * weight(a.weight, c)))));
    s = row::token_scale(row::row_max(amax, max_scratch, WARPS));
    if (threadIdx.x == 0) a.scale[n] = s.scale;
  }
  for (int c = threadIdx.x; c < C; c += LONG_THREADS) {
    const float z = z_at(c);
    const float y = z * (inv * weight(a.weight, c));
    static_cast<R*>(a.z)[at + c] = row::from_float<R>(z);
    if (QUANT)
      a.q[at + c] = int8_t(__float2int_rn(__fmul_rn(y, s.inverse)));
    else
      static_cast<X*>(a.y)[at + c] = row::from_float<X>(y);
  }
}

template <typename X, typename R, bool QUANT>
static cudaError_t launch(const Args& a, cudaStream_t stream) {
  const row::RowPlan p = row::plan_row(a.N, a.C);
  auto aligned = [](const void* ptr, size_t n) { return (reinterpret_cast<uintptr_t>(ptr) & (n - 1)) == 0; };
  ++launch_counter();
  if (p.units == 0) {
    long_row_kernel<X, R, QUANT><<<unsigned(a.N), LONG_THREADS, 0, stream>>>(a);
    return cudaPeekAtLastError();
  }
  // rows of 16-bit values that are a multiple of eight long all start at 16-byte boundaries
  const bool vector = a.C % 8 == 0 && aligned(a.x, 16) && aligned(a.residual, 16) && aligned(a.weight, 16) &&
                      aligned(a.post_weight, 16) && (aligned(a.gate, 16) || !a.gate_per_channel) &&
                      aligned(a.z, 16) && (QUANT ? aligned(a.q, 8) : aligned(a.y, 16));
  const dim3 block(p.threads(), p.rows_per_block());
  const unsigned grid = unsigned((a.N + p.rows_per_block() - 1) / p.rows_per_block());
  if (vector) {
    if (p.units == 1) row_kernel<X, R, QUANT, true, 1><<<grid, block, 0, stream>>>(a);
    else if (p.units == 2) row_kernel<X, R, QUANT, true, 2><<<grid, block, 0, stream>>>(a);
    else row_kernel<X, R, QUANT, true, 4><<<grid, block, 0, stream>>>(a);
  } else {
    if (p.units == 1) row_kernel<X, R, QUANT, false, 1><<<grid, block, 0, stream>>>(a);
    else if (p.units == 2) row_kernel<X, R, QUANT, false, 2><<<grid, block, 0, stream>>>(a);
    else row_kernel<X, R, QUANT, false, 4><<<grid, block, 0, stream>>>(a);
  }
  return cudaPeekAtLastError();
}

template <bool QUANT>
static int solve(const Args& a, int x_type, int residual_type, cudaStream_t stream) {
  if (a.N <= 0 || a.N > 0x7fffffffLL || a.C <= 0 || !a.x || !a.residual || !a.weight || !a.z ||
      (QUANT ? !a.q || !a.scale : !a.y) || (a.gate && a.rows_per_gate <= 0) ||
      (residual_type != x_type && residual_type != row::TYPE_F32))
    return -1;
  cudaError_t err;
  if (x_type == row::TYPE_F16)
    err = residual_type == row::TYPE_F32 ? launch<__half, float, QUANT>(a, stream)
                                         : launch<__half, __half, QUANT>(a, stream);
  else if (x_type == row::TYPE_BF16)
    err = residual_type == row::TYPE_F32 ? launch<__nv_bfloat16, float, QUANT>(a, stream)
                                         : launch<__nv_bfloat16, __nv_bfloat16, QUANT>(a, stream);
  else if (x_type == row::TYPE_F32)
    err = launch<float, float, QUANT>(a, stream);
  else
    return -1;
  if (err != cudaSuccess) {
    cudaGetLastError();
    return -3;
  }
  return 0;
}

}  // namespace bn
}  // namespace texo

extern "C" int texo_block_norm_solve(const void* x, const void* residual, const void* weight,
                                     const void* post_weight, const void* gate, void* y, void* z, int N, int C,
                                     int gate_rows, int gate_per_channel, float eps, float residual_scale,
                                     int x_type, int residual_type, int weights_f32, void* stream) {
  if (gate && (gate_rows <= 0 || N % gate_rows != 0)) return -1;
  texo::bn::Args a = {x, residual, weight, post_weight, gate, y, z, nullptr, nullptr, N, C,
                      gate ? N / gate_rows : 1, gate_per_channel, eps, residual_scale, weights_f32};
  return texo::bn::solve<false>(a, x_type, residual_type, static_cast<cudaStream_t>(stream));
}

extern "C" int texo_block_norm_quant_solve(const void* x, const void* residual, const void* weight,
                                           const void* post_weight, const void* gate, int8_t* q, float* scale,
                                           void* z, int N, int C, int gate_rows, int gate_per_channel, float eps,
                                           float residual_scale, int x_type, int residual_type, int weights_f32,
                                           void* stream) {
  if (gate && (gate_rows <= 0 || N % gate_rows != 0)) return -1;
  texo::bn::Args a = {x, residual, weight, post_weight, gate, nullptr, z, q, scale, N, C,
                      gate ? N / gate_rows : 1, gate_per_channel, eps, residual_scale, weights_f32};
  return texo::bn::solve<true>(a, x_type, residual_type, static_cast<cudaStream_t>(stream));
}
