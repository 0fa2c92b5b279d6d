// Pieces shared by the row-wise producers of the INT8 path (block_norm.cu, quant_per_token.cu):
// element types, layouts of a row over threads, reductions over a row, the per-token quantiser.
//
// These kernels read each byte once and write each byte once, so HBM bounds them; what keeps a
// kernel from that bound is its instructions (a row of 16-bit values is ten to thirty per value, a staged
// one up to twice that) and above all its latencies: loads, one to three reductions and stores follow one
// another within a row (2.2 to 2.8 instructions per clock and SM of four, with a third to a half of the warps an
// SM holds).  The first is met by packed arithmetic, the second by many blocks: one row per block of up
// to 1024 threads, as few as the groups per thread allow, and as many blocks as an SM holds.  A persistent
// form (two to six blocks per SM, rows arriving through a ring of bulk copies one or more rows ahead)
// hid the loads but not the rest, and measured 89 us where this form takes 60 (4096 x 8192 BF16, both
// norms, gate, quantised).
#pragma once
#include <algorithm>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "host_common.h"
#include "ptx.cuh"
#include "requant.cuh"

namespace texo {
namespace row {

// Element types of the C interface.
enum Type { TYPE_F16 = 0, TYPE_BF16 = 1, TYPE_F32 = 2 };

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

// The two elements of a word.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return __half22float2(h);
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Eight elements as they lie in memory.
template <typename T>
struct Raw8 {
  T v[8];
};
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {  // 16-byte aligned
  Raw8<T> r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r.v[j] = from_float<T>(v[j]);
  const uint4* s = reinterpret_cast<const uint4*>(&r);
#pragma unroll
  for (int i = 0; i < int(sizeof(Raw8<T>) / 16); ++i) __stcs(reinterpret_cast<uint4*>(p) + i, s[i]);
}

// The per-token quantiser: scale = max(amax, 2^-100) / 127, q = rint(y / scale), both quotients
// rounded to FP32 first (y / scale from a value within 2^-46 of it, see below): values half way between two
// multiples of the scale are common where y has few bits, and a product with a rounded 127 / amax
// would take them off the tie.
// The floor keeps scale and reciprocal finite and non-zero for every row (a row of zeros gets
// q = 0).  A row that holds a NaN or an infinity has no scale that stands for it: its scale is
// NaN and its q all zero, so that whatever the row is multiplied into shows it.
constexpr float MIN_TOP = 0x1p-100f;
struct TokenScale {
  float scale;
  float hi, lo;  // 1 / scale in two terms; hi = 0: q is zero whatever y is
};
// Quotients by multiplication (Newton-Raphson on 1/b and on a/b with residuals that a fused
// multiply-add gives exactly; Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", 1990).  scale: q0 = a * RN(1/127) is within two ulps of a/127; q1 = q0 + (a - 127 q0) *
// RN(1/127) within one; the same step from there rounds correctly.  y / scale: one Newton step takes
// the approximate reciprocal r to hi = r + (1 - scale r) r, within half an ulp and a little; lo = (1 - scale hi)
// hi is the rest.  hi + lo is within 2^-47 of 1/scale, and y hi + RN(y lo) within 2^-46 of the quotient, so
// that it rounds like the quotient unless that lies so close to the middle between two FP32 values.  (The
// correction step once more instead of lo would round correctly and costs 3% of a plain quantiser's time.)
// From scale = 2^102 on lo would be subnormal and lose bits, so there hi, lo and y are those of a row
// 2^64 times smaller.  A few instructions that every thread can afford, where divisions take an eighth of
// a short row's time.
constexpr float HUGE_SCALE = 0x1p100f, HUGE_TOP = 0x1p106f /*below which no scale is huge*/, SHRINK = 0x1p-64f;
__device__ __forceinline__ TokenScale token_scale(float amax) {
  TokenScale s;
  if (__float_as_uint(amax) >= 0x7f800000u) {
    s.scale = __int_as_float(0x7fffffff);
    s.hi = s.lo = 0.f;
    return s;
  }
  const float top = fmaxf(amax, MIN_TOP);
  constexpr float BY_127 = 1.f / 127.f;
  float q = __fmul_rn(top, BY_127);
  q = __fmaf_rn(__fmaf_rn(-127.f, q, top), BY_127, q);
  s.scale = __fmaf_rn(__fmaf_rn(-127.f, q, top), BY_127, q);
  float r;
  const float divisor = s.scale >= HUGE_SCALE ? s.scale * SHRINK : s.scale;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(divisor));
  s.hi = __fmaf_rn(__fmaf_rn(-divisor, r, 1.f), r, r);
  s.lo = __fmul_rn(__fmaf_rn(-divisor, s.hi, 1.f), s.hi);
  return s;
}
// Adding this (1.5 * 2^23) to |t| < 2^22 rounds t to the nearest integer, whose low byte is then the
// sum's (a conversion instruction runs at an eighth of the rate).
constexpr float ROUND_TO_INTEGER = 12582912.f;
__device__ __forceinline__ int8_t quantise(float v, const TokenScale& s) {
  if (s.scale >= HUGE_SCALE) v *= SHRINK;
  const float quotient = __fmaf_rn(v, s.hi, __fmul_rn(v, s.lo));
  return s.hi == 0.f ? int8_t(0) : int8_t(uint8_t(__float_as_uint(__fadd_rn(quotient, ROUND_TO_INTEGER))));
}

// Packed FP32 arithmetic, two values an instruction (each rounded like the scalar one): these
// kernels are near the issue limit.
__device__ __forceinline__ unsigned long long pair_of(float a, float b) {
  unsigned long long p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void from_pair(unsigned long long p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// v = a * b + c, each of them eight values or one.
__device__ __forceinline__ float lane8(const float (&v)[8], int j) { return v[j]; }
__device__ __forceinline__ float lane8(float v, int) { return v; }
template <typename A, typename B, typename C>
__device__ __forceinline__ void fma8(float (&v)[8], const A& a, const B& b, const C& c) {
#pragma unroll
  for (int j = 0; j < 8; j += 2)
    from_pair(fma2(pair_of(lane8(a, j), lane8(a, j + 1)), pair_of(lane8(b, j), lane8(b, j + 1)),
                   pair_of(lane8(c, j), lane8(c, j + 1))),
              v[j], v[j + 1]);
}
// v = a * b.
template <typename A, typename B>
__device__ __forceinline__ void mul8(float (&v)[8], const A& a, const B& b) {
#pragma unroll
  for (int j = 0; j < 8; j += 2)
    from_pair(mul2(pair_of(lane8(a, j), lane8(a, j + 1)), pair_of(lane8(b, j), lane8(b, j + 1))), v[j], v[j + 1]);
}

// A thread's values as the scale's hi and lo expect them (a branch that no ordinary row takes).
template <int UNITS>
__device__ __forceinline__ void shrink_huge(float (&v)[UNITS][8], const TokenScale& s) {
  if (s.scale >= HUGE_SCALE) {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) mul8(v[i], v[i], float(SHRINK));
  }
}

// A row of C values over `threads` threads, this one being thread t: group i is the eight values
// from at(i, 0) on.
//   ALIGNED  rows start at 16-byte boundaries and are a multiple of eight long
//   STAGED   any rows: they pass through shared memory (see below)
enum Layout { ALIGNED, STAGED };
template <Layout L>
struct Spread {
  int t, threads, C;
  __device__ __forceinline__ int at(int i, int j) const { return (i * threads + t) * 8 + j; }

  // Makes the values past the row's end zero.
  __device__ __forceinline__ void mask(int i, float (&v)[8]) const {
    if (at(i, 8) <= C) return;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at(i, j) >= C) v[j] = 0.f;
  }

  // Group i of a row in global memory; values past the end read as zero.  ONCE: not worth caching.
  template <bool ONCE, typename T>
  __device__ __forceinline__ void load(const T* row, int i, float (&v)[8]) const {
    Raw8<T> r;
    if (L == ALIGNED || ((reinterpret_cast<uintptr_t>(row) & 15) == 0 && at(i, 8) <= C)) {
      uint4* d = reinterpret_cast<uint4*>(&r);
      const uint4* s = reinterpret_cast<const uint4*>(row + at(i, 0));
      const bool in = at(i, 0) < C;
#pragma unroll
      for (int k = 0; k < int(sizeof(Raw8<T>) / 16); ++k)
        d[k] = !in ? make_uint4(0, 0, 0, 0) : ONCE ? __ldcs(s + k) : __ldg(s + k);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) r.v[j] = at(i, j) < C ? row[at(i, j)] : from_float<T>(0.f);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_float(r.v[j]);
  }

  // ALIGNED: group i to the row in global memory.  STAGED: to a shared-memory copy of the row
  // (send_row takes it from there), where the last group may reach seven values past the end.
  template <typename T>
  __device__ __forceinline__ void store(T* row, int i, const float (&v)[8]) const {
    Raw8<T> r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = from_float<T>(v[j]);
    if (at(i, 0) >= C) return;
    const uint4* s = reinterpret_cast<const uint4*>(&r);
#pragma unroll
    for (int k = 0; k < int(sizeof(Raw8<T>) / 16); ++k) {
      if (L == ALIGNED) __stcs(reinterpret_cast<uint4*>(row + at(i, 0)) + k, s[k]);
      else reinterpret_cast<uint4*>(row + at(i, 0))[k] = s[k];
    }
  }

  // The same for v (after shrink_huge) quantised (ALIGNED: rows start at 8-byte boundaries).
  __device__ __forceinline__ void store_quantised(int8_t* row, int i, const float (&v)[8], const TokenScale& scale) const {
    uint32_t r[8] = {};
    if (scale.hi != 0.f) {
      float t[8];
      mul8(t, v, scale.lo);
      fma8(t, v, scale.hi, t);
      fma8(t, t, 1.f, float(ROUND_TO_INTEGER));
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = __float_as_uint(t[j]);
    }
    if (at(i, 0) >= C) return;
    const uint2 q = make_uint2(
        __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410),
        __byte_perm(__byte_perm(r[4], r[5], 0x0040), __byte_perm(r[6], r[7], 0x0040), 0x5410));
    if (L == ALIGNED) __stcs(reinterpret_cast<uint2*>(row + at(i, 0)), q);
    else *reinterpret_cast<uint2*>(row + at(i, 0)) = q;
  }
};

// ------------------------------------------------------------------ staged rows
// Rows that start anywhere: the bytes move in aligned 16-byte granules between global and shared
// memory, and are shifted by the row's offset (the same for the whole row) between shared memory
// and registers.  Loads and stores of single values took twice as long (quant_per_token on 4000 x
// 11007 BF16: 106 us against 49).

// A staged input's room: its granules and four more.  The last group's shift reads farthest past the row's
// end, of interleaved FP32 pairs (C = 8 k + 1: the group's second eight values start 24 bytes behind the
// row's end and come in three granules, 72 bytes in all; 44 in the 16-bit types).
__host__ __device__ constexpr int staged_bytes(long long bytes) { return int((bytes + 15) / 16 * 16 + 64); }

// Starts copying the granules that hold [src, src + bytes) to shared memory.  Bytes of granules that reach
// outside [begin, end) are loaded singly.
__device__ __forceinline__ void fetch_row(uint32_t dst, uintptr_t src, int bytes, uintptr_t begin, uintptr_t end, int t,
                                          int threads) {
  const uintptr_t first = src & ~uintptr_t(15);
  const int granules = int((src + bytes + 15 - first) / 16);
  auto copy = [&](int g, uintptr_t at) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + g * 16), "l"(at) : "memory");
  };
  if (first >= begin && first + size_t(granules) * 16 <= end) {
    uintptr_t at = first + size_t(t) * 16;
    for (int g = t; g < granules; g += threads, at += size_t(threads) * 16) copy(g, at);
    return;
  }
  for (int g = t; g < granules; g += threads) {
    const uintptr_t at = first + size_t(g) * 16;
    if (at >= begin && at + 16 <= end) {
      copy(g, at);
    } else {
      uint32_t w[4] = {};
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (at + e >= begin && at + e < end) w[e / 4] |= uint32_t(*reinterpret_cast<const uint8_t*>(at + e)) << (e % 4 * 8);
#pragma unroll
      for (int k = 0; k < 4; ++k) sts32(dst + g * 16 + k * 4, w[k]);
    }
  }
}
__device__ __forceinline__ void fetched() {
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
}

// Words from byte `offset` (0 to 15, the same for all threads) of the granules at `from` on.
template <int WORDS>
__device__ __forceinline__ void shifted_words(uint32_t from, unsigned offset, uint32_t (&out)[WORDS]) {
  uint32_t w[WORDS + 4];
#pragma unroll
  for (int k = 0; k < WORDS / 4 + 1; ++k) {
    const int4 x = lds128(from + k * 16);
    w[4 * k] = x.x, w[4 * k + 1] = x.y, w[4 * k + 2] = x.z, w[4 * k + 3] = x.w;
  }
#pragma unroll
  for (int k = 0; k < WORDS + 2; ++k) w[k] = offset & 8 ? w[k + 2] : w[k];
#pragma unroll
  for (int k = 0; k < WORDS + 1; ++k) w[k] = offset & 4 ? w[k + 1] : w[k];
#pragma unroll
  for (int k = 0; k < WORDS; ++k) out[k] = __funnelshift_r(w[k], w[k + 1], (offset & 3) * 8);
}
// Eight values of type T, `index` values into a fetched row.
template <typename T>
__device__ __forceinline__ void read_staged(uint32_t row, unsigned offset, int index, float (&v)[8]) {
  uint32_t w[2 * int(sizeof(T))];
  shifted_words(row + index * int(sizeof(T)), offset, w);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (sizeof(T) == 4) {
      v[2 * k] = __uint_as_float(w[2 * k]);
      v[2 * k + 1] = __uint_as_float(w[2 * k + 1]);
    } else {
      const float2 p = unpack2<T>(w[k]);
      v[2 * k] = p.x;
      v[2 * k + 1] = p.y;
    }
  }
}

// Makes the values from `begin` to `end` of a fetched row zero.
template <typename T>
__device__ __forceinline__ void clear_staged(uint32_t row, unsigned offset, int begin, int end) {
  for (int i = begin; i < end; ++i) {
    const uint32_t at = row + offset + i * int(sizeof(T));
    if (sizeof(T) == 4) sts32(at, 0u);
    else sts16(at, 0);
  }
}

// Writes `bytes` bytes at shared-memory address `from` (16-byte aligned) to dst, whatever its alignment: whole
// granules, and the bytes of the row's first and last one singly.
__device__ __forceinline__ void send_row(uintptr_t dst, uint32_t from, int bytes, int t, int threads) {
  const int head = min(bytes, int(-dst & 15));  // bytes before the first whole granule
  const int whole = (bytes - head) / 16;
  for (int g = t; g < whole; g += threads) {
    uint32_t w[4];
    shifted_words(from + g * 16, unsigned(head), w);
    __stcs(reinterpret_cast<uint4*>(dst + head + size_t(g) * 16), make_uint4(w[0], w[1], w[2], w[3]));
  }
  const int tail = bytes - head - whole * 16;
  if (t < head + tail) {  // at most 30
    const int b = t < head ? t : whole * 16 + t;
    *reinterpret_cast<uint8_t*>(dst + b) = uint8_t(lds32(from + b / 4 * 4) >> (b % 4 * 8));
  }
}

// Reductions over the threads of one row: a warp, or all warps of a block.  `scratch` holds one
// word per warp and serves one reduction.  The order of the additions is fixed.
constexpr int MAX_WARPS = 32;
__device__ __forceinline__ float row_sum(float v, float* scratch, int t, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (warps == 1) return v;
  const int lane = t % 32;
  if (lane == 0) scratch[t / 32] = v;
  __syncthreads();
  float total = lane < warps ? scratch[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  return total;
}
// The larger of two absolute values, NaN if either is.
__device__ __forceinline__ float max_abs(float a, float b) {
  asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %1;\n\tmax.NaN.f32 %0, %0, t;\n\t}" : "+f"(a) : "f"(b));
  return a;
}
// Largest of non-negative values, by their bits: infinity is above every finite value and NaN
// (as max_abs gives it) above infinity.
__device__ __forceinline__ float row_max(float v, unsigned* scratch, int t, int warps) {
  unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
  if (warps == 1) return __uint_as_float(bits);
  const int lane = t % 32;
  if (lane == 0) scratch[t / 32] = bits;
  __syncthreads();
  return __uint_as_float(__reduce_max_sync(0xffffffffu, lane < warps ? scratch[lane] : 0u));
}

// The same over a cluster of `blocks` blocks that share a row: each hands its maximum to all.  A
// block's shared memory is there for the others only once it has started, so every block calls
// cluster_started first and cluster_max waits for the others' calls.
constexpr int MAX_CLUSTER = 8;
__device__ __forceinline__ void cluster_started(int blocks) {
  if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ float cluster_max(float v, unsigned* scratch, int t, int warps, unsigned* maxima, int blocks) {
  v = row_max(v, scratch, t, warps);
  if (blocks == 1) return v;
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (t < blocks)
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to_cta(smem_u32(maxima + cluster_ctarank()), t)),
                 "r"(__float_as_uint(v))
                 : "memory");
  cluster_sync_all();  // (the last access to another block's shared memory lies before it)
  unsigned bits = 0;
  for (int b = 0; b < blocks; ++b) bits = max(bits, maxima[b]);
  return __uint_as_float(bits);
}

// ------------------------------------------------------------------- host side
constexpr int MAX_C = 0x7fffffff - 4096;  // positions a block's width past the end do not wrap
// How rows are laid over threads and blocks: `units` groups of eight per thread at most, blocks of
// at most `most_threads`, clusters of at most `most_blocks`.
struct RowPlan {
  int units = 0;    // groups of eight per thread; 0: the row does not fit the registers
  int threads = 0;  // of a block
  int rows_per_block = 1;
  int cluster = 1;  // blocks of a row
};
inline RowPlan plan_row(int C, int units, int most_threads, int most_blocks, bool aligned_rows) {
  RowPlan p;
  const int groups = (C + 7) / 8;
  auto threads = [&] { return (groups + 32 * units * p.cluster - 1) / (32 * units * p.cluster) * 32; };
  while (threads() > most_threads && p.cluster < most_blocks) p.cluster *= 2;
  if (threads() > most_threads) return p;
  p.units = units;
  p.threads = threads();
  p.rows_per_block = p.threads == 32 && p.cluster == 1 && aligned_rows ? 4 : 1;
  return p;
}
// Whether all rows are in work at once, on the 148 SMs of a whole B200 (on a part of one the rule
// sets in later, which costs time but no correctness) that hold `threads_per_sm` threads each.  Until
// then the shortest way through a row wins, one group of eight per thread; after that more groups
// per thread do, which spread a thread's fixed work over more values.
inline bool at_once(const RowPlan& p, long long N, int threads_per_sm) {
  return p.units > 0 && N * p.cluster <= 148LL * (threads_per_sm / p.threads);
}
constexpr int STATIC_ROOM = 2048;  // what the kernels' own few words take at most
constexpr int SMEM_LIMIT = 232448 - STATIC_ROOM;
// Launches a kernel on staged rows; the attribute is set before every launch that needs it, which
// costs less than keeping track of devices and kernels.
template <typename... Params, typename... Args>
static bool launch_staged(void (*kernel)(Params...), unsigned grid, dim3 block, int bytes, cudaStream_t stream,
                          Args... args) {
  if (bytes > 48 * 1024 - STATIC_ROOM &&  // both together may be 48 KiB without the attribute
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return launch_on_stream(kernel, grid, block, bytes, 1, stream, args...);
}

}  // namespace row
}  // namespace texo
