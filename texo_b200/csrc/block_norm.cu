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
// Bound by HBM bandwidth: a row lives in registers between the reductions, so every input byte
// is read once and every output byte written once (row_ops.cuh).
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
  int N, C;
  int rows_per_gate;
  int gate_per_channel;  // 0: one value per gate row
  float eps, residual_scale;
  float inv_c;  // 1 / C
  int weights_f32;  // weight, post_weight and gate are FP32 (else they have x's type)
};

// Group i of a weight-like row, in either of its two types.
template <typename X, row::Layout L>
__device__ __forceinline__ void load_weights(const row::Spread<L>& s, const void* base, bool f32, size_t offset, int i,
                                             float (&v)[8]) {
  if (f32)
    s.template load<false>(static_cast<const float*>(base) + offset, i, v);
  else
    s.template load<false>(static_cast<const X*>(base) + offset, i, v);
}

template <int UNITS>
__device__ __forceinline__ float squares(const float (&v)[UNITS][8]) {
  float sum[8];
  row::mul8(sum, v[0], v[0]);
#pragma unroll
  for (int i = 1; i < UNITS; ++i) row::fma8(sum, v[i], v[i], sum);
  return ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
}

// x (group i) -> u: the block's own norm and the gate, whose row is `gate_row`.
template <typename X, row::Layout L>
__device__ __forceinline__ void to_u(const Args& a, size_t gate_row, const row::Spread<L>& s, int i, float post_inv,
                                     float (&v)[8]) {
  if (a.post_weight) {
    float w[8];
    load_weights<X>(s, a.post_weight, a.weights_f32, 0, i, w);
    row::mul8(w, w, post_inv);
    row::mul8(v, v, w);
  }
  if (a.gate) {
    if (a.gate_per_channel) {
      float g[8];
      load_weights<X>(s, a.gate, a.weights_f32, gate_row * a.C, i, g);
      row::mul8(v, v, g);
    } else {
      const float g = a.weights_f32 ? static_cast<const float*>(a.gate)[gate_row]
                                    : row::to_float(static_cast<const X*>(a.gate)[gate_row]);
      row::mul8(v, v, g);
    }
  }
}

// u and the residual (group i) -> z, in registers and to the row at `z`.  Values past the row's end become
// zero whatever they were.
template <typename R, row::Layout L>
__device__ __forceinline__ void to_z(const Args& a, R* z, const row::Spread<L>& s, int i, const float (&r)[8],
                                     float (&v)[8]) {
  row::fma8(v, r, a.residual_scale, v);
  s.mask(i, v);
  s.store(z, i, v);
}

// z -> the outputs, to the row at `y` or `q`.
template <typename X, bool QUANT, row::Layout L, int UNITS>
__device__ __forceinline__ void finish(const Args& a, int n, X* y, int8_t* q, const row::Spread<L>& s,
                                       float (&v)[UNITS][8], float* sum_scratch, unsigned* max_scratch) {
  const int warps = s.threads / 32;
  const float inv = rsqrtf(row::row_sum(squares(v), sum_scratch, s.t, warps) * a.inv_c + a.eps);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    float w[8];
    load_weights<X>(s, a.weight, a.weights_f32, 0, i, w);
    row::mul8(w, w, inv);
    row::mul8(v[i], v[i], w);
    if (QUANT) {
      s.mask(i, v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = row::max_abs(amax, v[i][j]);
    } else {
      s.store(y, i, v[i]);
    }
  }
  if (QUANT) {
    amax = row::row_max(amax, max_scratch, s.t, warps);
    const row::TokenScale scale = row::token_scale(amax);
    if (s.t == 0) a.scale[n] = scale.scale;
    row::shrink_huge(v, scale);
#pragma unroll
    for (int i = 0; i < UNITS; ++i) s.store_quantised(q, i, v[i], scale);
  }
}

struct Scratch {
  float post[row::MAX_WARPS], sum[row::MAX_WARPS];
  unsigned max[row::MAX_WARPS];
};

// A block (or a warp) per row.  blockDim = (threads of a row, rows of the block), LIMIT threads at most.
// Two blocks of 576 leave 56 registers instead of 64, hence three blocks of 384 on an SM instead of
// two (4096 x 6144 BF16, both norms, gate, quantised: 52.5 -> 42.4 us; 5999: 88.5 -> 73.2); where that
// spills (wider residual, y not quantised: 4096 x 8192 67.6 -> 70.4 us) it is not done.
constexpr int SHORT = 576;
template <typename X, typename R, bool QUANT, row::Layout L, int UNITS, int LIMIT>
__global__ void __launch_bounds__(LIMIT, LIMIT == SHORT ? 2 : 1) row_kernel(const Args a) {
  __shared__ Scratch scratch;
  grid_dependency_trigger();
  const long long row_number = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (row_number >= a.N) return;  // only blocks of one-warp rows reach past N; they meet at no barrier
  const int n = int(row_number);
  const row::Spread<L> s = {int(threadIdx.x), int(blockDim.x), a.C};
  const size_t gate_row = a.gate ? size_t(unsigned(n) / unsigned(a.rows_per_gate)) : 0;
  const size_t at = size_t(n) * a.C;
  R* z = static_cast<R*>(a.z) + at;
  X* y = static_cast<X*>(a.y) + at;
  int8_t* q = a.q + at;
  grid_dependency_wait();
  float v[UNITS][8], r[UNITS][8];
  if constexpr (L == row::ALIGNED) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) s.template load<true>(static_cast<const X*>(a.x) + at, i, v[i]);
#pragma unroll
    for (int i = 0; i < UNITS; ++i) s.template load<true>(static_cast<const R*>(a.residual) + at, i, r[i]);
  } else {
    // x's room takes y or q afterwards, the residual's z
    extern __shared__ __align__(16) uint8_t staging[];
    uint8_t* staged_r = staging + row::staged_bytes((long long)a.C * sizeof(X));
    auto fetch = [&](const void* base, int size, uint8_t* to) {
      const uintptr_t begin = reinterpret_cast<uintptr_t>(base), src = begin + at * size;
      row::fetch_row(smem_u32(to), src, a.C * size, begin, begin + size_t(a.N) * a.C * size, s.t, s.threads);
      return unsigned(src & 15);
    };
    const unsigned x_offset = fetch(a.x, sizeof(X), staging), r_offset = fetch(a.residual, sizeof(R), staged_r);
    row::fetched();
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      if (s.at(i, 0) < a.C) {
        row::read_staged<X>(smem_u32(staging), x_offset, s.at(i, 0), v[i]);
        row::read_staged<R>(smem_u32(staged_r), r_offset, s.at(i, 0), r[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = r[i][j] = 0.f;
      }
      s.mask(i, v[i]);  // (what lies past the row's end is arbitrary)
    }
    __syncthreads();
    z = reinterpret_cast<R*>(staged_r);
    y = reinterpret_cast<X*>(staging);
    q = reinterpret_cast<int8_t*>(staging);
  }
  float post_inv = 1.f;
  if (a.post_weight)
    post_inv = rsqrtf(row::row_sum(squares(v), scratch.post, s.t, s.threads / 32) * a.inv_c + a.eps);
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    to_u<X>(a, gate_row, s, i, post_inv, v[i]);
    to_z(a, z, s, i, r[i], v[i]);
  }
  finish<X, QUANT>(a, n, y, q, s, v, scratch.sum, scratch.max);
  if constexpr (L == row::STAGED) {
    __syncthreads();
    row::send_row(reinterpret_cast<uintptr_t>(static_cast<R*>(a.z) + at), smem_u32(z), a.C * int(sizeof(R)), s.t, s.threads);
    if (QUANT) row::send_row(reinterpret_cast<uintptr_t>(a.q + at), smem_u32(q), a.C, s.t, s.threads);
    else row::send_row(reinterpret_cast<uintptr_t>(static_cast<X*>(a.y) + at), smem_u32(y), a.C * int(sizeof(X)), s.t, s.threads);
  }
}

// Rows that the registers do not hold: the values are computed again from x and residual in
// every pass (from L2 after the first).  z and y may lie over residual and x as in the kernel
// above: the last pass alone writes, each element after its own thread has read it.
constexpr int LONG_THREADS = 1024;
template <typename X, typename R, bool QUANT>
__global__ void __launch_bounds__(LONG_THREADS) long_row_kernel(const Args a) {
  __shared__ Scratch scratch;
  grid_dependency_trigger();
  grid_dependency_wait();
  constexpr int WARPS = LONG_THREADS / 32;
  const int n = blockIdx.x;
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
    post_inv = rsqrtf(row::row_sum(sum, scratch.post, threadIdx.x, WARPS) / float(C) + a.eps);
  }
  const size_t gate_row = a.gate ? size_t(unsigned(n) / unsigned(a.rows_per_gate)) : 0;
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
  const float inv = rsqrtf(row::row_sum(sum, scratch.sum, threadIdx.x, WARPS) / float(C) + a.eps);
  row::TokenScale scale = {0.f, 0.f, 0.f};
  if (QUANT) {
    float amax = 0.f;
    for (int c = threadIdx.x; c < C; c += LONG_THREADS) amax = row::max_abs(amax, z_at(c) * (inv * weight(a.weight, c)));
    amax = row::row_max(amax, scratch.max, threadIdx.x, WARPS);
    scale = row::token_scale(amax);
    if (threadIdx.x == 0) a.scale[n] = scale.scale;
  }
  for (int c = threadIdx.x; c < C; c += LONG_THREADS) {
    const float z = z_at(c);
    const float y = z * (inv * weight(a.weight, c));
    static_cast<R*>(a.z)[at + c] = row::from_float<R>(z);
    if (QUANT)
      a.q[at + c] = row::quantise(y, scale);
    else
      static_cast<X*>(a.y)[at + c] = row::from_float<X>(y);
  }
}

template <typename X, typename R, bool QUANT>
static bool launch(const Args& a, cudaStream_t stream) {
  auto aligned = [](const void* ptr, size_t n) { return (reinterpret_cast<uintptr_t>(ptr) & (n - 1)) == 0; };
  // rows that are a multiple of eight values long all start at 16-byte boundaries
  const bool aligned_rows = a.C % 8 == 0 && aligned(a.x, 16) && aligned(a.residual, 16) && aligned(a.weight, 16) &&
                      aligned(a.post_weight, 16) && (aligned(a.gate, 16) || !a.gate_per_channel) &&
                      aligned(a.z, 16) && (QUANT ? aligned(a.q, 8) : aligned(a.y, 16));
  // Both norms, gate, quantised, BF16: 4096 x 8192 92 / 59 / 71 us for one / two / four groups per
  // thread, 128 x 8191 7.6 / 9.1 for one / two, 300 x 8191 20 / 16.
  row::RowPlan r = row::plan_row(a.C, 1, 1024, 1, aligned_rows);
  if (!row::at_once(r, a.N, 1024)) r = row::plan_row(a.C, 2, 1024, 1, aligned_rows);
  if (r.units == 0) return launch_on_stream(long_row_kernel<X, R, QUANT>, unsigned(a.N), LONG_THREADS, 0, 1, stream, a);
  const dim3 block(r.threads, r.rows_per_block);
  const unsigned grid = unsigned(((long long)a.N + r.rows_per_block - 1) / r.rows_per_block);
  constexpr bool HAS_SHORT = QUANT || sizeof(R) == sizeof(X);
  if (aligned_rows) {
    auto rows = [&](auto* kernel) { return launch_on_stream(kernel, grid, block, 0, 1, stream, a); };
    if (r.units == 1) return rows(row_kernel<X, R, QUANT, row::ALIGNED, 1, 1024>);
    if constexpr (HAS_SHORT)
      if (r.threads <= SHORT) return rows(row_kernel<X, R, QUANT, row::ALIGNED, 2, SHORT>);
    return rows(row_kernel<X, R, QUANT, row::ALIGNED, 2, 1024>);
  }
  const int room = row::staged_bytes((long long)a.C * sizeof(X)) + row::staged_bytes((long long)a.C * sizeof(R));
  auto rows = [&](auto* kernel) { return row::launch_staged(kernel, grid, block, room, stream, a); };
  if (r.units == 1) return rows(row_kernel<X, R, QUANT, row::STAGED, 1, 1024>);
  if constexpr (HAS_SHORT)
    if (r.threads <= SHORT) return rows(row_kernel<X, R, QUANT, row::STAGED, 2, SHORT>);
  return rows(row_kernel<X, R, QUANT, row::STAGED, 2, 1024>);
}

template <bool QUANT>
static int solve(const Args& a, int x_type, int residual_type, cudaStream_t stream) {
  if (a.N <= 0 || a.C <= 0 || !a.x || !a.residual || !a.weight || !a.z ||
      (QUANT ? !a.q || !a.scale : !a.y) || (a.gate && a.rows_per_gate <= 0) ||
      (residual_type != x_type && residual_type != row::TYPE_F32))
    return -1;
  if (a.C > row::MAX_C) return -2;
  if (x_type != row::TYPE_F16 && x_type != row::TYPE_BF16 && x_type != row::TYPE_F32) return -1;
  const bool f32 = residual_type == row::TYPE_F32;
  bool ok;
  if (x_type == row::TYPE_F16)
    ok = f32 ? launch<__half, float, QUANT>(a, stream) : launch<__half, __half, QUANT>(a, stream);
  else if (x_type == row::TYPE_BF16)
    ok = f32 ? launch<__nv_bfloat16, float, QUANT>(a, stream)
             : launch<__nv_bfloat16, __nv_bfloat16, QUANT>(a, stream);
  else
    ok = launch<float, float, QUANT>(a, stream);
  return ok ? 0 : -3;
}

}  // namespace bn
}  // namespace texo

extern "C" int texo_block_norm_solve(const void* x, const void* residual, const void* weight,
                                     const void* post_weight, const void* gate, void* y, void* z, int N, int C,
                                     int gate_rows, int gate_per_channel, float eps, float residual_scale,
                                     int x_type, int residual_type, int weights_f32, void* stream) {
  if (gate && (gate_rows <= 0 || N % gate_rows != 0)) return -1;
  texo::bn::Args a = {x, residual, weight, post_weight, gate, y, z, nullptr, nullptr, N, C,
                      gate ? N / gate_rows : 1, gate_per_channel, eps, residual_scale, 1.f / float(C), weights_f32};
  return texo::bn::solve<false>(a, x_type, residual_type, static_cast<cudaStream_t>(stream));
}

extern "C" int texo_block_norm_quant_solve(const void* x, const void* residual, const void* weight,
                                           const void* post_weight, const void* gate, int8_t* q, float* scale,
                                           void* z, int N, int C, int gate_rows, int gate_per_channel, float eps,
                                           float residual_scale, int x_type, int residual_type, int weights_f32,
                                           void* stream) {
  if (gate && (gate_rows <= 0 || N % gate_rows != 0)) return -1;
  texo::bn::Args a = {x, residual, weight, post_weight, gate, nullptr, z, q, scale, N, C,
                      gate ? N / gate_rows : 1, gate_per_channel, eps, residual_scale, 1.f / float(C), weights_f32};
  return texo::bn::solve<true>(a, x_type, residual_type, static_cast<cudaStream_t>(stream));
}
