// Pieces shared by the row-wise producers of the INT8 path (block_norm.cu, quant_per_token.cu):
// element types, eight-element loads and stores, reductions over the threads of a row, and the
// per-token quantiser.
//
// A row of C values is held in registers by `threads` threads, UNITS groups of eight values
// each.  VECTOR: group u of the row is eight neighbouring values, moved in 16-byte pieces
// (every row starts at a 16-byte boundary).  Otherwise the eight values of a thread's group are
// `threads` apart, so that each load or store of a warp still covers neighbouring addresses.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "requant.cuh"

namespace texo {
namespace row {

// Element types of the C interface.
enum Type { TYPE_F16 = 0, TYPE_BF16 = 1, TYPE_F32 = 2 };
inline int type_size(int type) { return type == TYPE_F32 ? 4 : 2; }

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }

// Eight elements as they lie in memory.
template <typename T>
struct Raw8 {
  T v[8];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {  // 16-byte aligned
  Raw8<T> r;
  uint4* d = reinterpret_cast<uint4*>(&r);
#pragma unroll
  for (int i = 0; i < int(sizeof(Raw8<T>) / 16); ++i) d[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  return r;
}
template <typename T>
__device__ __forceinline__ Raw8<T> load8_cached(const T* p) {
  Raw8<T> r;
  uint4* d = reinterpret_cast<uint4*>(&r);
#pragma unroll
  for (int i = 0; i < int(sizeof(Raw8<T>) / 16); ++i) d[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  Raw8<T> r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r.v[j] = from_float<T>(v[j]);
  const uint4* s = reinterpret_cast<const uint4*>(&r);
#pragma unroll
  for (int i = 0; i < int(sizeof(Raw8<T>) / 16); ++i) __stcs(reinterpret_cast<uint4*>(p) + i, s[i]);
}

// Position in the row of value j of a thread's group i.
template <bool VECTOR>
__device__ __forceinline__ int position(int thread, int threads, int i, int j) {
  return VECTOR ? (thread + i * threads) * 8 + j : thread + (i * 8 + j) * threads;
}

// One group of a row of C values starting at `row`; values past the end read as zero.
template <bool VECTOR, typename T>
__device__ __forceinline__ Raw8<T> load_group(const T* row, int C, int thread, int threads, int i) {
  Raw8<T> r;
  if (VECTOR) {
    const int c = position<true>(thread, threads, i, 0);
    if (c < C) return load8(row + c);
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = from_float<T>(0.f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = position<false>(thread, threads, i, j);
      r.v[j] = c < C ? __ldcs(row + c) : from_float<T>(0.f);
    }
  }
  return r;
}
// The same for data that many rows share (weights, gates), as floats.
template <bool VECTOR, typename T>
__device__ __forceinline__ void load_shared_group(const T* row, int C, int thread, int threads, int i, float (&v)[8]) {
  if (VECTOR) {
    const int c = position<true>(thread, threads, i, 0);
    if (c < C) {
      const Raw8<T> r = load8_cached(row + c);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_float(r.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = position<false>(thread, threads, i, j);
      v[j] = c < C ? to_float(row[c]) : 0.f;
    }
  }
}
template <bool VECTOR, typename T>
__device__ __forceinline__ void store_group(T* row, int C, int thread, int threads, int i, const float (&v)[8]) {
  if (VECTOR) {
    const int c = position<true>(thread, threads, i, 0);
    if (c < C) store8(row + c, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = position<false>(thread, threads, i, j);
      if (c < C) __stcs(row + c, from_float<T>(v[j]));
    }
  }
}
// q: eight quantised values (VECTOR: q rows start at 8-byte boundaries).
template <bool VECTOR>
__device__ __forceinline__ void store_quantised(int8_t* row, int C, int thread, int threads, int i,
                                                const float (&v)[8], float inverse) {
  int r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = __float2int_rn(__fmul_rn(v[j], inverse));
  if (VECTOR) {
    const int c = position<true>(thread, threads, i, 0);
    if (c < C)
      __stcs(reinterpret_cast<uint2*>(row + c), make_uint2(i8::pack_sat_s8(r[0], r[1], r[2], r[3]),
                                                           i8::pack_sat_s8(r[4], r[5], r[6], r[7])));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = position<false>(thread, threads, i, j);
      if (c < C) row[c] = int8_t(r[j]);
    }
  }
}

// Reductions over the threads of one row: a warp (rows of a block share nothing), or all warps
// of the block.  `scratch` holds one word per warp and is not used again before the next
// barrier: consecutive reductions take different ones.  The order of the additions is fixed.
constexpr int MAX_WARPS = 32;
__device__ __forceinline__ float row_sum(float v, float* scratch, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (warps == 1) return v;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  float total = lane < warps ? scratch[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  return total;
}
// Largest bit pattern: for the bits of absolute values this is the largest value, infinity
// being above every finite value and NaN above infinity.
__device__ __forceinline__ unsigned row_max(unsigned v, unsigned* scratch, int warps) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (warps == 1) return v;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, lane < warps ? scratch[lane] : 0u);
}

// The per-token quantiser: scale = max(amax, 2^-100) / 127, q = rint(y * (127 / max(amax, 2^-100))).
// The floor keeps both quotients finite and non-zero for every row (a row of zeros gets q = 0).
// A row that holds a NaN or an infinity has no scale that stands for it: its scale is NaN and
// its q all zero, so that whatever the row is multiplied into shows it.
struct TokenScale {
  float scale, inverse;
};
__device__ __forceinline__ TokenScale token_scale(unsigned amax_bits) {
  TokenScale t;
  if (amax_bits >= 0x7f800000u) {
    t.scale = __int_as_float(0x7fffffff);
    t.inverse = 0.f;  // NaN * 0 and infinity * 0 convert to 0
  } else {
    const float top = fmaxf(__uint_as_float(amax_bits), 0x1p-100f);
    t.scale = __fdiv_rn(top, 127.f);
    t.inverse = __fdiv_rn(127.f, top);
  }
  return t;
}

// How a row is laid over threads: warps per row (1: four rows share a block of 128 threads) and
// groups of eight per thread.
struct RowPlan {
  int warps, units;  // units: 1, 2 or 4; 0: the row does not fit the registers
  int threads() const { return warps * 32; }
  int rows_per_block() const { return warps == 1 ? 4 : 1; }
};
constexpr int MAX_REGISTER_ROW = 16384;
inline RowPlan plan_row(long long N, int C) {
  RowPlan p = {1, 0};
  if (C > MAX_REGISTER_ROW) return p;
  const int groups = (C + 7) / 8;
  p.units = N < 512 ? 1 : groups <= 32 ? 1 : groups <= 64 ? 2 : 4;
  p.warps = (groups + 32 * p.units - 1) / (32 * p.units);
  if (p.warps > 32) {
    p.units = 2;
    p.warps = (groups + 63) / 64;
  }
  return p;
}

}  // namespace row
}  // namespace texo
