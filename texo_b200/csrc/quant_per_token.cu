// Per-token INT8 quantisers of activations, plain and behind the SwiGLU product (no counterpart
// in the reference, whose quantised operators take one scale per tensor; the SwiGLU formula is
// that of its src/swiglu.cu:15-18):
//
//   y = x                          quant_per_token
//   y = gate / (1 + exp(-gate)) * up   swiglu_quant_per_token, gate / up interleaved or as halves
//   scale = max(amax|y|, 2^-100) / 127,  q = rint(y / scale)
//
// One scale per row needs the row's maximum before its first output, so the row stays in
// registers between the two: bound by HBM bandwidth, each byte crosses once (row_ops.cuh).
// Long rows are shared by a cluster of blocks that exchange their maxima.
#include <cmath>
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

// y = gate up / (1 + e^-gate), and e^-gate = 2^(-gate log2 e).  Errors in multiples of U = 2^-24,
// relative to the value: rounding log2 e and its product moves the exponent by 1.23 parts of itself, hence the
// power by 1.23 |gate|; PTX allows ex2.approx 4 (two ulps) and rcp.approx 2; the sum takes 1, the
// products 1 each, the first one none where the inputs have 16 bits.  Together 9 + 1.23 |gate|, far
// below the quantiser's half step: 20 of 117,440,512 outputs fall on the other side of a tie than with
// expf and an IEEE division, which take 181 us instead of 120 (4096 x 28672 BF16 pairs).
// Both instructions flush subnormals, which saves the scaling around them: a denominator beyond 2^126
// (gate < -87.3) would make y zero, where a large `up` may make it any value.  And gate * up can
// overflow where y does not.  Rows with either are done again (careful_row below).
constexpr float LOG2_E = 1.44269504f;
constexpr float LOWEST_GATE = -87.f;
__device__ __forceinline__ float swiglu(float gate, float up) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(gate, -LOG2_E)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(1.f, e)));
  return __fmul_rn(r, __fmul_rn(gate, up));
}
// The same of eight, in packed arithmetic (and the same bits), and the lowest gate.
__device__ __forceinline__ void swiglu8(const float (&gate)[8], const float (&up)[8], float (&y)[8], float& lowest) {
  float t[8], product[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) asm("min.f32 %0, %0, %1, %2;" : "+f"(lowest) : "f"(gate[j]), "f"(gate[j + 1]));
  row::mul8(t, gate, -LOG2_E);
#pragma unroll
  for (int j = 0; j < 8; ++j) asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t[j]));
  row::fma8(t, t, 1.f, 1.f);
#pragma unroll
  for (int j = 0; j < 8; ++j) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(t[j]));
  row::mul8(product, gate, up);
  row::mul8(y, t, product);
}
// The same, two values after two: the registers of gate and up are free sooner, which rows in halves,
// whose operands come from two places, are short of (4096 x 14336 FP16 60 -> 54.8 us; pairs of 28672
// BF16 take 125 us so instead of 120).
__device__ __forceinline__ void swiglu8_by_twos(const float (&gate)[8], const float (&up)[8], float (&y)[8], float& lowest) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    asm("min.f32 %0, %0, %1, %2;" : "+f"(lowest) : "f"(gate[j]), "f"(gate[j + 1]));
    const unsigned long long g = row::pair_of(gate[j], gate[j + 1]);
    const unsigned long long product = row::mul2(g, row::pair_of(up[j], up[j + 1]));
    float a, b;
    row::from_pair(row::mul2(g, row::pair_of(-LOG2_E, -LOG2_E)), a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    row::from_pair(row::fma2(row::pair_of(a, b), row::pair_of(1.f, 1.f), row::pair_of(1.f, 1.f)), a, b);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
    row::from_pair(row::mul2(row::pair_of(a, b), product), y[j], y[j + 1]);
  }
}
// For any finite gate and up, and the same bits where `swiglu` is good.  Below -87, 1 + e^-gate is e^-gate, and
// y = (gate h) (h up) with h = e^(gate / 2): no factor leaves the range unless y does (h is subnormal
// below -174, where |y| < 2^-115 whatever up is, a hundredth of the smallest scale).  Where the product
// overflows the quotient comes first.
__device__ __forceinline__ float careful_swiglu(float gate, float up) {
  if (gate < LOWEST_GATE) {
    const float h = expf(0.5f * gate);
    return (gate * h) * (h * up);
  }
  const float y = swiglu(gate, up);
  return fabsf(y) < INFINITY ? y : gate / (1.f + expf(-gate)) * up;
}

// Eight outputs from sixteen interleaved inputs.
__device__ __forceinline__ void swiglu_pairs(const float (&lo)[8], const float (&hi)[8], float (&y)[8], float& lowest) {
  const float gate[8] = {lo[0], lo[2], lo[4], lo[6], hi[0], hi[2], hi[4], hi[6]};
  const float up[8] = {lo[1], lo[3], lo[5], lo[7], hi[1], hi[3], hi[5], hi[7]};
  swiglu8(gate, up, y, lowest);
}

// Group i of an aligned row in global memory, as y; values past the end are zero.  `lowest` goes down to its
// lowest gate.
template <typename X, int FORM>
__device__ __forceinline__ void load_y(const X* x, const row::Spread<row::ALIGNED>& s, int i, float (&y)[8],
                                       float& lowest) {
  if (FORM == PLAIN) {
    s.template load<true>(x, i, y);
  } else if (FORM == SWIGLU_HALVES) {
    float g[8], u[8];
    s.template load<true>(x, i, g);
    s.template load<true>(x + s.C, i, u);
    swiglu8_by_twos(g, u, y, lowest);
  } else {
    // the sixteen inputs of eight outputs: two groups of a row of 2 C values
    const row::Spread<row::ALIGNED> wide = {0, 1, 2 * s.C};
    float lo[8], hi[8];
    const int c = s.at(i, 0);
    wide.template load<true>(x, c / 4, lo);
    wide.template load<true>(x, c / 4 + 1, hi);
    swiglu_pairs(lo, hi, y, lowest);
  }
}
// The same of a staged row: `first` holds x (or the gates, `second` the ups).  What lies past the row's end is
// arbitrary; in rows of SwiGLU operands, where it must not count as a gate, the thread that reads it makes
// it zero first (nobody else uses it).
template <typename X, int FORM>
__device__ __forceinline__ void read_y(uint32_t first, unsigned offset, uint32_t second, unsigned second_offset,
                                       const row::Spread<row::STAGED>& s, int i, float (&y)[8], float& lowest) {
  if (s.at(i, 0) >= s.C) {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = 0.f;
    return;
  }
  if (FORM == PLAIN) {
    row::read_staged<X>(first, offset, s.at(i, 0), y);
    s.mask(i, y);
    return;
  }
  if (s.at(i, 8) > s.C) {
    constexpr int WIDTH = FORM == SWIGLU_INTERLEAVED ? 2 : 1;
    row::clear_staged<X>(first, offset, WIDTH * s.C, WIDTH * s.at(i, 8));
    if (FORM == SWIGLU_HALVES) row::clear_staged<X>(second, second_offset, s.C, s.at(i, 8));
  }
  if (FORM == SWIGLU_INTERLEAVED) {
    float lo[8], hi[8];
    row::read_staged<X>(first, offset, 2 * s.at(i, 0), lo);
    row::read_staged<X>(first, offset, 2 * s.at(i, 0) + 8, hi);
    swiglu_pairs(lo, hi, y, lowest);
  } else {
    float g[8], u[8];
    row::read_staged<X>(first, offset, s.at(i, 0), g);
    row::read_staged<X>(second, second_offset, s.at(i, 0), u);
    swiglu8_by_twos(g, u, y, lowest);
  }
}

// Threads of a block at most.  Two blocks of 576 leave 56 registers instead of 64, hence three blocks of
// 352 instead of two: rows of 11008 30.6 -> 24.7 us, as halves 48.5 -> 41.9, staged pairs of 4000 x 11007
// 69.7 -> 58.2.  Interleaved pairs in aligned rows want the 64 (4096 x 28672: 120 us against 142).
constexpr int SHORT = 576;
__host__ __device__ constexpr int block_limit(int form, row::Layout layout, int units) {
  return layout == row::STAGED || units < 4 ? 1024 : form == SWIGLU_INTERLEAVED ? 512 : SHORT;
}

// A row whose y is computed twice, value by value, by `threads` threads in `blocks` blocks.
template <typename X, int FORM>
__device__ __forceinline__ void row_in_passes(const Args& a, long long n, int t, int threads, int blocks, unsigned* scratch,
                                              unsigned* maxima) {
  const X* x = static_cast<const X*>(a.x) + n * a.stride;
  auto y_at = [&](int c) {
    if (FORM == PLAIN) return row::to_float(x[c]);
    const size_t g = FORM == SWIGLU_INTERLEAVED ? 2 * size_t(c) : c;
    const size_t u = FORM == SWIGLU_INTERLEAVED ? 2 * size_t(c) + 1 : size_t(a.C) + c;
    return careful_swiglu(row::to_float(x[g]), row::to_float(x[u]));
  };
  float amax = 0.f;
  for (int c = t; c < a.C; c += threads) amax = row::max_abs(amax, y_at(c));
  amax = row::cluster_max(amax, scratch, threadIdx.x, blockDim.x / 32, maxima, blocks);
  const row::TokenScale scale = row::token_scale(amax);
  if (t == 0) a.scale[n] = scale.scale;
  int8_t* q = a.q + size_t(n) * a.C;
  for (int c = t; c < a.C; c += threads) q[c] = row::quantise(y_at(c), scale);
}
// Once more, for a row of SwiGLU products with a far gate, a huge value or one that is not finite.  The
// row's number comes from the special registers again, which keeps it and the row's addresses out of the registers
// until here (4096 x 28672 BF16 pairs 119.7 us, handed over 126.6).  Such a row costs five to seven others; in
// vectors it costs three, but then the others pay 14% (in line) or halves 10% (as a call).
template <typename X, int FORM>
__device__ __forceinline__ void careful_row(const Args& a, int blocks, unsigned* scratch, unsigned* maxima) {
  row::cluster_started(blocks);
  const long long n = (long long)cluster_id() * blockDim.y + threadIdx.y;
  row_in_passes<X, FORM>(a, n, int(cluster_ctarank() * blockDim.x + threadIdx.x), blocks * blockDim.x, blocks, scratch, maxima);
}

// A block, a warp or (blocks > 1) a cluster per row.  blockDim = (threads, rows of the block).
template <typename X, int FORM, row::Layout L, int UNITS, int LIMIT = block_limit(FORM, L, UNITS)>
__global__ void __launch_bounds__(LIMIT, LIMIT <= SHORT ? 2 : 1) row_kernel(const Args a, int blocks) {
  __shared__ unsigned scratch[2][row::MAX_WARPS], maxima[2][row::MAX_CLUSTER];
  grid_dependency_trigger();
  row::cluster_started(blocks);
  const int part = int(cluster_ctarank());  // of the row
  const long long n = (long long)cluster_id() * blockDim.y + threadIdx.y;
  if (n >= a.N) return;  // only blocks of one-warp rows reach past N; they meet at no barrier
  const int t = threadIdx.x, threads = blockDim.x;
  const row::Spread<L> s = {part * threads + t, blocks * threads, a.C};
  const X* x = static_cast<const X*>(a.x) + n * a.stride;
  int8_t* q = a.q + size_t(n) * a.C;
  grid_dependency_wait();
  float y[UNITS][8], lowest = 0.f;
  if constexpr (L == row::ALIGNED) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) load_y<X, FORM>(x, s, i, y[i], lowest);
  } else {  // a block per row; x's room takes q afterwards
    extern __shared__ __align__(16) uint8_t staging[];
    const uintptr_t begin = reinterpret_cast<uintptr_t>(a.x);
    const uintptr_t end = begin + size_t((a.N - 1) * a.stride + (long long)a.C * (FORM == PLAIN ? 1 : 2)) * sizeof(X);
    const int bytes = a.C * int(sizeof(X)) * (FORM == SWIGLU_INTERLEAVED ? 2 : 1);
    const uintptr_t first = reinterpret_cast<uintptr_t>(x), second = reinterpret_cast<uintptr_t>(x + a.C);
    const uint32_t to = smem_u32(staging), to_second = to + row::staged_bytes(bytes);
    row::fetch_row(to, first, bytes, begin, end, t, threads);
    if (FORM == SWIGLU_HALVES) row::fetch_row(to_second, second, bytes, begin, end, t, threads);
    row::fetched();
#pragma unroll
    for (int i = 0; i < UNITS; ++i)
      read_y<X, FORM>(to, unsigned(first & 15), to_second, unsigned(second & 15), s, i, y[i], lowest);
    __syncthreads();
    q = reinterpret_cast<int8_t*>(staging);
  }
  float amax = lowest < LOWEST_GATE ? INFINITY : 0.f;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = row::max_abs(amax, y[i][j]);
  }
  amax = row::cluster_max(amax, scratch[0], t, threads / 32, maxima[0], blocks);
  if (FORM != PLAIN && !(amax < row::HUGE_TOP)) {  // the same for all threads of the row
    careful_row<X, FORM>(a, blocks, scratch[1], maxima[1]);
    return;
  }
  const row::TokenScale scale = row::token_scale(amax);
  if (s.t == 0) a.scale[n] = scale.scale;
  if (FORM == PLAIN) row::shrink_huge(y, scale);
#pragma unroll
  for (int i = 0; i < UNITS; ++i) s.store_quantised(q, i, y[i], scale);
  if constexpr (L == row::STAGED) {
    __syncthreads();
    row::send_row(reinterpret_cast<uintptr_t>(a.q + size_t(n) * a.C), smem_u32(q), a.C, t, threads);
  }
}

// Rows that the registers do not hold.
constexpr int LONG_THREADS = 1024;
template <typename X, int FORM>
__global__ void __launch_bounds__(LONG_THREADS) long_row_kernel(const Args a) {
  __shared__ unsigned scratch[row::MAX_WARPS];
  grid_dependency_trigger();
  grid_dependency_wait();
  row_in_passes<X, FORM>(a, blockIdx.x, threadIdx.x, LONG_THREADS, 1, scratch, nullptr);
}

template <typename X, int FORM>
static bool launch(const Args& a, cudaStream_t stream) {
  const bool aligned_rows = a.C % 8 == 0 && a.stride * sizeof(X) % 16 == 0 &&
                            (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && (reinterpret_cast<uintptr_t>(a.q) & 7) == 0;
  auto launch_long = [&] { return launch_on_stream(long_row_kernel<X, FORM>, unsigned(a.N), LONG_THREADS, 0, 1, stream, a); };
  if (!aligned_rows) {
    const int bytes = a.C <= 32768 ? a.C * int(sizeof(X)) * (FORM == SWIGLU_INTERLEAVED ? 2 : 1) : 0;
    const int room = row::staged_bytes(bytes) * (FORM == SWIGLU_HALVES ? 2 : 1);
    // (4000 x 11007 BF16: 85 / 48 us for two / four groups per thread; pairs of 128 x 8191, 300 x 8191: 4.1,
    // 11 us for one, 7.2, 8 for four)
    row::RowPlan r = row::plan_row(a.C, 1, block_limit(FORM, row::STAGED, 1), 1, false);
    if (!row::at_once(r, a.N, 1536)) r = row::plan_row(a.C, 4, block_limit(FORM, row::STAGED, 4), 1, false);
    if (r.units == 0 || room > row::SMEM_LIMIT) return launch_long();
    auto rows = [&](auto* kernel) { return row::launch_staged(kernel, unsigned(a.N), dim3(r.threads), room, stream, a, 1); };
    if constexpr (FORM != PLAIN)
      if (r.units == 4 && r.threads <= SHORT) return rows(row_kernel<X, FORM, row::STAGED, 4, SHORT>);
    return r.units == 1 ? rows(row_kernel<X, FORM, row::STAGED, 1>) : rows(row_kernel<X, FORM, row::STAGED, 4>);
  }
  // 8192 x 8192 BF16: 60 / 41 / 35 us for one / two / four groups per thread; 4096 x 28672
  // interleaved pairs: 145 / 120 us for two / four; 450 x 4096, 300 x 14336: 4.2, 13.2 us for one,
  // 4.9, 6.6 for four.  (Clusters hold an SM's second block up.)
  row::RowPlan r = row::plan_row(a.C, 1, block_limit(FORM, row::ALIGNED, 1), row::MAX_CLUSTER, true);
  if (!row::at_once(r, a.N, r.cluster > 1 ? 1024 : 2048))
    r = row::plan_row(a.C, 4, block_limit(FORM, row::ALIGNED, 4), row::MAX_CLUSTER, true);
  if (r.units == 0 || a.N > 0x7fffffff / r.cluster) return launch_long();
  const dim3 block(r.threads, r.rows_per_block);
  const unsigned grid = unsigned((a.N + r.rows_per_block - 1) / r.rows_per_block) * r.cluster;
  auto rows = [&](auto* kernel) { return launch_on_stream(kernel, grid, block, 0, r.cluster, stream, a, r.cluster); };
  return r.units == 1 ? rows(row_kernel<X, FORM, row::ALIGNED, 1>) : rows(row_kernel<X, FORM, row::ALIGNED, 4>);
}

template <int FORM>
static int solve(const Args& a, int x_type, cudaStream_t stream) {
  const long long width = FORM == PLAIN ? a.C : 2LL * a.C;
  if (a.N <= 0 || a.C <= 0 || a.stride < width || !a.x || !a.q || !a.scale) return -1;
  if (width > row::MAX_C) return -2;
  if (x_type != row::TYPE_F16 && x_type != row::TYPE_BF16 && x_type != row::TYPE_F32) return -1;
  const bool ok = x_type == row::TYPE_F16    ? launch<__half, FORM>(a, stream)
                  : x_type == row::TYPE_BF16 ? launch<__nv_bfloat16, FORM>(a, stream)
                                             : launch<float, FORM>(a, stream);
  return ok ? 0 : -3;
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
