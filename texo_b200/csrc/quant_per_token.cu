// Per-token INT8 quantisers of activations, plain and behind the SwiGLU product (no counterpart
// in the reference, whose quantised operators take one scale per tensor; the SwiGLU formula is
// that of its src/swiglu.cu:15-18):
//
//   y = x                          quant_per_token
//   y = gate / (1 + exp(-gate)) * up   swiglu_quant_per_token, gate / up interleaved or as halves
//   scale = max(amax|y|, 2^-100) / 127,  q = rint(y / scale)
//
// One scale per row needs the row's maximum before its first output, so the row stays in
// registers between the two (row_ops.cuh): bound by HBM bandwidth, each byte crosses once.
#include <cstdint>
#include <cuda_runtime.h>

#include "host_common.h"
#include "ptx.cuh"
#include "row_ops.cuh"

namespace texo {
namespace qt {

enum Form { PLAIN = 0, SWIGLU_INTERLEAVED = 1, SWIGLU_HALVES = 2 };

struct Args {
  const void* x;
  int8_t* q;
  float* scale;
  long long N;
  int C;  // outputs per row
  long long stride;  // elements between rows of x
};

// gate and up are never multiplied first: their product can overflow where the result does not.
// __expf and __fdividef are within a few units in the last place; a denominator beyond 2^126
// (gate < -87) gives 0 where the value is below 2^-118.
__device__ __forceinline__ float swiglu(float gate, float up) {
  return __fdividef(gate, 1.f + __expf(-gate)) * up;
}

// Group i of the row, as y.
template <typename X, int FORM, bool VECTOR>
__device__ __forceinline__ void load_y(const X* x, int C, int t, int threads, int i, float (&y)[8]) {
  if (FORM == PLAIN) {
    const row::Raw8<X> r = row::load_group<VECTOR>(x, C, t, threads, i);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = row::to_float(r.v[j]);
  } else if (FORM == SWIGLU_HALVES) {
    const row::Raw8<X> g = row::load_group<VECTOR>(x, C, t, threads, i);
    const row::Raw8<X> u = row::load_group<VECTOR>(x + C, C, t, threads, i);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = swiglu(row::to_float(g.v[j]), row::to_float(u.v[j]));
  } else if (VECTOR) {
    const int c = row::position<true>(t, threads, i, 0);
    if (c < C) {
      const row::Raw8<X> lo = row::load8(x + 2 * c), hi = row::load8(x + 2 * c + 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = swiglu(row::to_float(lo.v[2 * j]), row::to_float(lo.v[2 * j + 1]));
        y[4 + j] = swiglu(row::to_float(hi.v[2 * j]), row::to_float(hi.v[2 * j + 1]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = row::position<false>(t, threads, i, j);
      y[j] = c < C ? swiglu(row::to_float(__ldcs(x + 2 * size_t(c))), row::to_float(__ldcs(x + 2 * size_t(c) + 1)))
                   : 0.f;
    }
  }
}

template <typename X, int FORM, bool VECTOR, int UNITS>
__global__ void __launch_bounds__(UNITS == 4 ? 512 : 1024) row_kernel(const Args a) {
  __shared__ unsigned scratch[row::MAX_WARPS];
  const long long n = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (n >= a.N) return;  // only blocks of one-warp rows reach past N; they meet at no barrier
  const int t = threadIdx.x, threads = blockDim.x;
  const X* x = static_cast<const X*>(a.x) + n * a.stride;
  float y[UNITS][8];
  unsigned amax = 0;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) load_y<X, FORM, VECTOR>(x, a.C, t, threads, i, y[i]);
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(fabsf(y[i][j])));
  }
  const row::TokenScale s = row::token_scale(row::row_max(amax, scratch, threads / 32));
  if (t == 0) a.scale[n] = s.scale;
  int8_t* q = a.q + size_t(n) * a.C;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) row::store_quantised<VECTOR>(q, a.C, t, threads, i, y[i], s.inverse);
}

// Rows that the registers do not hold: y is computed twice.
constexpr int LONG_THREADS = 1024;
template <typename X, int FORM>
__global__ void __launch_bounds__(LONG_THREADS) long_row_kernel(const Args a) {
  __shared__ unsigned scratch[row::MAX_WARPS];
  const long long n = blockIdx.x;
  const X* x = static_cast<const X*>(a.x) + n * a.stride;
  auto y_at = [&](int c) {
    if (FORM == PLAIN) return row::to_float(x[c]);
    const size_t g = FORM == SWIGLU_INTERLEAVED ? 2 * size_t(c) : c;
    const size_t u = FORM == SWIGLU_INTERLEAVED ? 2 * size_t(c) + 1 : size_t(a.C) + c;
    return swiglu(row::to_float(x[g]), row::to_float(x[u]));
  };
  unsigned amax = 0;
  for (int c = threadIdx.x; c < a.C; c += LONG_THREADS) amax = max(amax, __float_as_uint(fabsf(y_at(c))));
  const row::TokenScale s = row::token_scale(row::row_max(amax, scratch, LONG_THREADS / 32));
  if (threadIdx.x == 0) a.scale[n] = s.scale;
  int8_t* q = a.q + size_t(n) * a.C;
  for (int c = threadIdx.x; c < a.C; c += LONG_THREADS) q[c] = int8_t(__float2int_rn(__fmul_rn(y_at(c), s.inverse)));
}

template <typename X, int FORM>
static cudaError_t launch(const Args& a, cudaStream_t stream) {
  const row::RowPlan p = row::plan_row(a.N, a.C);
  ++launch_counter();
  if (p.units == 0) {
    long_row_kernel<X, FORM><<<unsigned(a.N), LONG_THREADS, 0, stream>>>(a);
    return cudaPeekAtLastError();
  }
  const bool vector = a.C % 8 == 0 && a.stride * sizeof(X) % 16 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 &&
                      (reinterpret_cast<uintptr_t>(a.q) & 7) == 0;
  const dim3 block(p.threads(), p.rows_per_block());
  const unsigned grid = unsigned((a.N + p.rows_per_block() - 1) / p.rows_per_block());
  if (vector) {
    if (p.units == 1) row_kernel<X, FORM, true, 1><<<grid, block, 0, stream>>>(a);
    else if (p.units == 2) row_kernel<X, FORM, true, 2><<<grid, block, 0, stream>>>(a);
    else row_kernel<X, FORM, true, 4><<<grid, block, 0, stream>>>(a);
  } else {
    if (p.units == 1) row_kernel<X, FORM, false, 1><<<grid, block, 0, stream>>>(a);
    else if (p.units == 2) row_kernel<X, FORM, false, 2><<<grid, block, 0, stream>>>(a);
    else row_kernel<X, FORM, false, 4><<<grid, block, 0, stream>>>(a);
  }
  return cudaPeekAtLastError();
}

template <int FORM>
static int solve(const Args& a, int x_type, cudaStream_t stream) {
  const long long width = FORM == PLAIN ? a.C : 2LL * a.C;
  if (a.N <= 0 || a.C <= 0 || a.stride < width || !a.x || !a.q || !a.scale) return -1;
  cudaError_t err;
  if (x_type == row::TYPE_F16) err = launch<__half, FORM>(a, stream);
  else if (x_type == row::TYPE_BF16) err = launch<__nv_bfloat16, FORM>(a, stream);
  else if (x_type == row::TYPE_F32) err = launch<float, FORM>(a, stream);
  else return -1;
  if (err != cudaSuccess) {
    cudaGetLastError();
    return -3;
  }
  return 0;
}

}  // namespace qt
}  // namespace texo

extern "C" int texo_quant_per_token_solve(const void* x, int8_t* q, float* scale, int N, int C, long long row_stride,
                                          int x_type, void* stream) {
  const texo::qt::Args a = {x, q, scale, N, C, row_stride};
  return texo::qt::solve<texo::qt::PLAIN>(a, x_type, static_cast<cudaStream_t>(stream));
}

extern "C" int texo_swiglu_quant_per_token_solve(const void* gate_up, int8_t* q, float* scale, int N, int F,
                                                 long long row_stride, int interleaved, int x_type, void* stream) {
  const texo::qt::Args a = {gate_up, q, scale, N, F, row_stride};
  return interleaved ? texo::qt::solve<texo::qt::SWIGLU_INTERLEAVED>(a, x_type, static_cast<cudaStream_t>(stream))
                     : texo::qt::solve<texo::qt::SWIGLU_HALVES>(a, x_type, static_cast<cudaStream_t>(stream));
}
