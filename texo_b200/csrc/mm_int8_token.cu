// INT8 product with one scale per token and one per output channel, floating output (no
// counterpart in the reference, whose INT8 operator is per-tensor: src/mm_int8.cu:530-535):
//
//   Y[m,n] = round(float(sum_k A[m,k] B[k,n]) * scale_A[m] * scale_B[n] (+ bias[n]))
//
// A [M,K], B [K,N] int8 row-major, Y [M,N] FP16, BF16 or FP32.  The integer dot is exact; it is
// rounded once to FP32, scaled by two FP32 multiplies (the second one fused with the bias add)
// and rounded once to Y's type.  Both operands are symmetric, so there is no zero-point
// identity and no sum over A or B beside the dot.
#include <algorithm>
#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "host_common.h"
#include "ptx.cuh"
#include "row_ops.cuh"

namespace texo {
namespace i8t {

struct Scales {
  const float* a;     // [M]
  const float* b;     // [N]
  const float* bias;  // [N] or null
};

// The one formula of every path below.
__device__ __forceinline__ float scaled(float dot, float sa, float sb, float bias) {
  return __fmaf_rn(__fmul_rn(dot, sa), sb, bias);
}

// -------------------------------------------------------------- generic path
// Any shape, any byte alignment, K = 0, and K >= 2^17, where an int32 can overflow: 64x64 SIMT
// tiles, dp4a on words packed in shared memory, int32 windows of 2^15 k flushed into int64.
constexpr int GT = 64, GK = 64, GKW = GK / 4, G_THREADS = 256;
constexpr int G_FLUSH_TILES = 512;

template <typename Y>
__global__ void __launch_bounds__(G_THREADS)
    generic_kernel(const int8_t* __restrict__ A, const int8_t* __restrict__ B, Y* __restrict__ out, int M, int N,
                   int K, Scales s) {
  __shared__ int As[GT][GKW + 1];  // four consecutive k of a row of A per word
  __shared__ int Bs[GT][GKW + 1];  // four consecutive k of a column of B per word
  const int t = threadIdx.x, ty = t / 16, tx = t % 16;
  const int row0 = blockIdx.y * GT, col0 = blockIdx.x * GT;
  int acc[4][4] = {};
  long long total[4][4] = {};
  const int tiles_k = (K + GK - 1) / GK;
  int since_flush = 0;
  for (int kt = 0; kt < tiles_k; ++kt) {
    const int k0 = kt * GK;
    {
      const int m = row0 + t / 4, kb = (t % 4) * 16;
      const int8_t* src = A + size_t(m) * K + k0 + kb;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        unsigned word = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned v = (m < M && k0 + kb + w * 4 + e < K) ? uint8_t(src[w * 4 + e]) : 0u;
          word |= v << (8 * e);
        }
        As[t / 4][kb / 4 + w] = int(word);
      }
    }
    {
      unsigned word[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = k0 + ty * 4 + e;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = col0 + tx * 4 + j;
          const unsigned v = (k < K && n < N) ? uint8_t(B[size_t(k) * N + n]) : 0u;
          word[j] |= v << (8 * e);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) Bs[tx * 4 + j][ty] = int(word[j]);
    }
    __syncthreads();
#pragma unroll
    for (int kw = 0; kw < GKW; ++kw) {
      int a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = As[ty * 4 + i][kw];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = Bs[tx * 4 + j][kw];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
      }
    }
    __syncthreads();
    if (++since_flush == G_FLUSH_TILES || kt + 1 == tiles_k) {
      since_flush = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          total[i][j] += acc[i][j];
          acc[i][j] = 0;
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = row0 + ty * 4 + i;
    if (m >= M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = col0 + tx * 4 + j;
      if (n >= N) continue;
      const float y = scaled(float(total[i][j]), s.a[m], s.b[n], s.bias ? s.bias[n] : 0.f);
      out[size_t(m) * N + n] = row::from_float<Y>(y);
    }
  }
}

// ------------------------------------------------------------------ dispatch
enum Path { PATH_AUTO = 0, PATH_GENERIC = 1 };
inline int& forced_path() {
  static int path = 0;
  return path;
}
inline int& last_path() {
  static int path = 0;
  return path;
}

template <typename Y>
static bool launch_generic(const int8_t* A, const int8_t* B, Y* out, int M, int N, int K, const Scales& s,
                           cudaStream_t stream) {
  // gridDim.y is limited to 65535 tiles per launch
  constexpr int ROWS = 65535 * GT;
  for (int m0 = 0; m0 < M; m0 += ROWS) {
    const int rows = std::min(M - m0, ROWS);
    const dim3 grid((N + GT - 1) / GT, (rows + GT - 1) / GT);
    const Scales part = {s.a + m0, s.b, s.bias};
    generic_kernel<Y><<<grid, G_THREADS, 0, stream>>>(A + size_t(m0) * K, B, out + size_t(m0) * N, rows, N, K, part);
    ++launch_counter();
    if (m0 > M - ROWS) break;  // m0 + ROWS would pass the int range
  }
  last_path() = PATH_GENERIC;
  return cudaPeekAtLastError() == cudaSuccess;
}

template <typename Y>
static int solve(const int8_t* A, const int8_t* B, Y* out, int M, int N, int K, const Scales& s,
                 cudaStream_t stream) {
  if (!launch_generic(A, B, out, M, N, K, s, stream)) {
    cudaGetLastError();
    return -3;
  }
  return 0;
}

}  // namespace i8t
}  // namespace texo

extern "C" int texo_mm_int8_solve_per_token(const int8_t* A, const int8_t* B, void* Y, int M, int N, int K,
                                            const float* scale_A, const float* scale_B, const float* bias,
                                            int out_type, void* stream) {
  using namespace texo;
  if (M <= 0 || N <= 0 || K < 0 || !Y || !scale_A || !scale_B || (K > 0 && (!A || !B))) return -1;
  const i8t::Scales s = {scale_A, scale_B, bias};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (out_type) {
    case row::TYPE_F16: return i8t::solve(A, B, static_cast<__half*>(Y), M, N, K, s, st);
    case row::TYPE_BF16: return i8t::solve(A, B, static_cast<__nv_bfloat16*>(Y), M, N, K, s, st);
    case row::TYPE_F32: return i8t::solve(A, B, static_cast<float*>(Y), M, N, K, s, st);
    default: return -1;
  }
}

extern "C" int texo_mm_int8_per_token_last_path(void) { return texo::i8t::last_path(); }
extern "C" void texo_mm_int8_per_token_force_path(int path) { texo::i8t::forced_path() = path; }
