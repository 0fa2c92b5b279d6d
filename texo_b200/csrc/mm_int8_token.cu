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
#include <type_traits>
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

// ----------------------------------------------------------- streaming path
// Few rows (decode, small batches) or few tiles: the job is to stream B from HBM once with all
// SMs pulling.  Operand roles are swapped, as in skinny.cuh: two 128-column boxes of B side by
// side are the 128-row MMA operands (N-major in memory = M-major operand), up to 128 rows of A
// the narrow one, so an accumulator lane is an output column.
//
// A tile (256 columns x R rows) is worked on by a cluster of c CTAs, each on its own part of K.
// There is no workspace: every CTA pushes its int32 partials straight into the shared memory of
// the CTA that finishes the row (row r of a 32-row chunk belongs to CTA r % c), an mbarrier
// there counts the pushes, and the owner adds the c copies, scales and stores.  Integer sums, so
// the split changes no bit, and nothing is shared between calls: any streams, any graphs.
//
// Shared memory is nearly all ring: an SM has to keep about 100 KiB in flight to cover HBM
// latency at its share of the bandwidth.
//
// GATHER: rows of A or B that do not start at 16-byte boundaries cannot be moved by TMA.  Eight
// or sixteen warps then build the same swizzled tiles: aligned 4-byte words, coalesced over the
// lanes, shifted into place with their neighbour's word.
constexpr int S_BK = 128;                // k per ring stage = one 128-byte swizzle row
constexpr int S_BOX = 128 * 128;         // 128 k rows x 128 columns of B
constexpr int S_W_BYTES = 2 * S_BOX;     // the two boxes of a tile
constexpr int S_TILE_N = 256;
constexpr int S_MAX_STAGES = 6;
constexpr int S_EPI_WARPS = 8;
constexpr int S_GATHER_GROUPS = 2, S_GATHER_WARPS = 8;  // stages are dealt to the groups in turn
constexpr int S_THREADS = 64 + S_EPI_WARPS * 32;
constexpr int S_GATHER_THREADS = S_THREADS + S_GATHER_GROUPS * S_GATHER_WARPS * 32;
constexpr int S_MAX_CLUSTER = 8;

__host__ __device__ constexpr int s_chunk_rows(int R) { return R < 32 ? R : 32; }
// Rows of a chunk that one CTA of the cluster finishes.
__host__ __device__ constexpr int s_slots(int R, int c) { return (s_chunk_rows(R) + c - 1) / c; }
__host__ __device__ constexpr int s_stages(int R) { return R == 16 ? 6 : R == 32 ? 5 : 4; }
__host__ __device__ constexpr int s_stage_bytes(int R) { return S_W_BYTES + R * 128; }
__host__ __device__ constexpr int s_push_bytes(int R, int c) { return c * s_slots(R, c) * S_TILE_N * 4; }
__host__ __device__ constexpr int s_smem_bytes(int R, int c) {
  return s_stages(R) * s_stage_bytes(R) + s_push_bytes(R, c) + 1024 /*alignment*/ + 256 /*barriers*/;
}
static_assert(s_smem_bytes(128, 8) <= 232448 && s_smem_bytes(64, 7) <= 232448 && s_smem_bytes(32, 7) <= 232448 &&
                  s_smem_bytes(16, 7) <= 232448 && s_smem_bytes(16, 5) <= 232448,
              "streaming kernel: shared memory over the limit");

struct StreamBarriers {
  uint64_t full[S_MAX_STAGES];
  uint64_t empty[S_MAX_STAGES];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t pushed;  // all partials of a chunk have arrived in this CTA
  uint64_t taken;   // all CTAs have finished reading a chunk's partials
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(StreamBarriers) <= 256, "StreamBarriers outgrew its shared-memory reserve");

__device__ __forceinline__ void store_cluster_u32(uint32_t cluster_addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

// After a wait gave up: gives the loads in flight a tenth of a second to land before the CTA's
// shared memory goes back.  `issued` loads went round the ring of `stages` barriers.
__device__ __forceinline__ void drain_loads(uint64_t* full, int stages, int issued) {
  const long long start = clock64();
  for (int i = 0; i < stages && i < issued; ++i) {
    const uint32_t parity = uint32_t((issued - i - 1) / stages) & 1;
    while (!mbar_try_wait(&full[i], parity) && clock64() - start < WAIT_BUDGET_CLOCKS / 10) {}
  }
}

// The aligned word at p, of which bytes outside [begin, end) are not read and come back as 0.
__device__ __forceinline__ uint32_t load_word(const uint8_t* p, const uint8_t* begin, const uint8_t* end) {
  if (p >= begin && p + 4 <= end) return __ldg(reinterpret_cast<const unsigned int*>(p));
  uint32_t v = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (p + e >= begin && p + e < end) v |= uint32_t(p[e]) << (8 * e);
  return v;
}

struct StreamShape {
  int M, N, K;
  int R, cluster, m_tiles, tiles;
  int vector_out;  // rows of the output start at 16-byte boundaries
};

template <typename Y, bool GATHER>
__global__ void __launch_bounds__(GATHER ? S_GATHER_THREADS : S_THREADS, 1)
    stream_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a,
                  const int8_t* __restrict__ A, const int8_t* __restrict__ B, Y* __restrict__ out, Scales s,
                  StreamShape p, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  grid_dependency_trigger();
  const int R = p.R, c = p.cluster;
  const int stages = s_stages(R), stage_bytes = s_stage_bytes(R);
  uint32_t* push = reinterpret_cast<uint32_t*>(smem + stages * stage_bytes);
  StreamBarriers* bars = reinterpret_cast<StreamBarriers*>(smem + stages * stage_bytes + s_push_bytes(R, c));
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = int(cluster_ctarank());
  const int first_tile = blockIdx.x / c, tile_step = gridDim.x / c;
  const int num_kb = (p.K + S_BK - 1) / S_BK;
  const int kb0 = int((long long)num_kb * rank / c), kb1 = int((long long)num_kb * (rank + 1) / c);
  const uint32_t tmem_cols = R <= 32 ? (R == 16 ? 64u : 128u) : (R == 64 ? 256u : 512u);

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&bars->full[i], GATHER ? S_GATHER_WARPS : 1);
      mbar_init(&bars->empty[i], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], S_EPI_WARPS);
    }
    mbar_init(&bars->pushed, c * S_EPI_WARPS);
    mbar_init(&bars->taken, c * S_EPI_WARPS);
    bars->abort_flag = 0;
    fence_barrier_init();
    if (!GATHER) {
      // B may still be in the making by the grid ahead, so all that is safe before the wait
      // is a hint: the first boxes are pulled into L2, where every SM's writes meet.
      for (int i = 0; i < stages && kb0 + i < kb1 && first_tile < p.tiles; ++i) {
        const int n0 = first_tile / p.m_tiles * S_TILE_N;
        tma_prefetch_l2_2d(&map_b, n0, (kb0 + i) * S_BK);
        if (n0 + 128 < p.N) tma_prefetch_l2_2d(&map_b, n0 + 128, (kb0 + i) * S_BK);
      }
    }
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the other CTAs' barriers exist before anything signals them
  tc_fence_after_sync();
  const uint32_t tmem_base = bars->tmem_base;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (!GATHER && lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      grid_dependency_wait();  // the operands may have been written by the grid ahead
      for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
        const int n0 = tile / p.m_tiles * S_TILE_N, m0 = tile % p.m_tiles * R;
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(&bars->empty[stage], phase ^ 1, abort_flag, status, STATUS_TIMEOUT_EMPTY);
          if (!ok) break;
          uint8_t* sw = smem + stage * stage_bytes;
          mbar_arrive_expect_tx(&bars->full[stage], stage_bytes);
          tma_load_2d(sw, &map_b, &bars->full[stage], n0, kb * S_BK);
          tma_load_2d(sw + S_BOX, &map_b, &bars->full[stage], n0 + 128, kb * S_BK);
          tma_load_2d(sw + S_W_BYTES, &map_a, &bars->full[stage], kb * S_BK, m0);
          issued = issued < 1 << 30 ? issued + 1 : issued + 1 - 2 * stages;  // same stages and parities
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) drain_loads(bars->full, stages, issued);
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      const uint32_t idesc = umma_idesc(/*D=s32*/ 2, /*A=s8*/ 1, /*B=s8*/ 1, /*A M-major*/ 1, /*B K-major*/ 0, 128,
                                        uint32_t(R));
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      bool ok = true;
      for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
        ok = mbar_wait(&bars->acc_empty[buf], buf_phase ^ 1, abort_flag, status, STATUS_TIMEOUT_TMEM_EMPTY);
        tc_fence_after_sync();
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          ok = mbar_wait(&bars->full[stage], phase, abort_flag, status, STATUS_TIMEOUT_FULL);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t sw = smem_u32(smem + stage * stage_bytes);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t tmem_d = tmem_base + (buf * 2 + half) * R;
#pragma unroll
            for (int j = 0; j < S_BK / 32; ++j) {
              const uint64_t dw = smem_desc(sw + half * S_BOX + j * 32 * 128, 16, 1024, SMEM_SWIZZLE_128B);
              const uint64_t da = smem_desc(sw + S_W_BYTES + j * 32, 16, 1024, SMEM_SWIZZLE_128B);
              umma_i8(tmem_d, dw, da, idesc, (kb == kb0 && j == 0) ? 0u : 1u);
            }
          }
          umma_commit(&bars->empty[stage]);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (ok) umma_commit(&bars->acc_full[buf]);
        if (++buf == 2) {
          buf = 0;
          buf_phase ^= 1;
        }
      }
    }
  } else if (warp < 2 + S_EPI_WARPS) {
    // ---------------------------------------------------------------- epilogue
    const int ew = warp - 2, quarter = warp % 4, half = ew / 4;
    const int column = half * 128 + quarter * 32 + lane;
    const int chunk_rows = s_chunk_rows(R), slots = s_slots(R, c);
    const uint32_t push_addr = smem_u32(push);
    int buf = 0, chunk_no = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    grid_dependency_wait();  // before the scales are read and the output is written
    for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
      const int n0 = tile / p.m_tiles * S_TILE_N, m0 = tile % p.m_tiles * R;
      const int rows = min(R, p.M - m0);
      ok = mbar_wait(&bars->acc_full[buf], buf_phase, abort_flag, status, STATUS_TIMEOUT_TMEM_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after_sync();
      for (int r0 = 0; r0 < rows; r0 += chunk_rows, ++chunk_no) {
        const int here = min(chunk_rows, rows - r0);
        uint32_t v[32];
        const uint32_t at = tmem_base + (buf * 2 + half) * R + r0 + (uint32_t(quarter * 32) << 16);
        if (R == 16) {
          uint32_t v16[16];
          tmem_ld_32x16(at, v16);
          tmem_ld_wait();
#pragma unroll
          for (int r = 0; r < 16; ++r) v[r] = v16[r];
        } else {
          tmem_ld_32x32(at, v);
          tmem_ld_wait();
        }
        if (r0 + chunk_rows >= rows) {  // the accumulator is in registers: its buffer is free
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->acc_empty[buf]);
        }
        if (chunk_no > 0) {  // the last chunk's partials have been read everywhere
          ok = mbar_wait_cluster(&bars->taken, (chunk_no - 1) & 1, abort_flag, status, STATUS_TIMEOUT_FLAG);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        {
          int owner = 0, slot = 0;
#pragma unroll
          for (int r = 0; r < 32; ++r) {
            if (r < here) {
              store_cluster_u32(map_to_cta(push_addr, owner) + uint32_t(((rank * slots + slot) * S_TILE_N + column) * 4),
                                v[r]);
              if (++owner == c) {
                owner = 0;
                ++slot;
              }
            }
          }
        }
        __syncwarp();
        if (lane < c) mbar_arrive_cluster(map_to_cta(smem_u32(&bars->pushed), lane));
        ok = mbar_wait_cluster(&bars->pushed, chunk_no & 1, abort_flag, status, STATUS_TIMEOUT_FLAG);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        for (int slot = ew; slot * c + rank < here; slot += S_EPI_WARPS) {
          const int m = m0 + r0 + slot * c + rank;
          const uint32_t* first = push + slot * S_TILE_N;
          const float sa = __ldg(s.a + m);
          Y* row_out = out + size_t(m) * p.N + n0;
          if (p.vector_out && n0 + lane * 8 + 8 <= p.N) {
            int total[8] = {};
            for (int copy = 0; copy < c; ++copy) {
              const int4* w = reinterpret_cast<const int4*>(first + copy * slots * S_TILE_N + lane * 8);
              const int4 lo = w[0], hi = w[1];
              total[0] += lo.x, total[1] += lo.y, total[2] += lo.z, total[3] += lo.w;
              total[4] += hi.x, total[5] += hi.y, total[6] += hi.z, total[7] += hi.w;
            }
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int n = n0 + lane * 8 + e;
              y[e] = scaled(float(total[e]), sa, __ldg(s.b + n), s.bias ? __ldg(s.bias + n) : 0.f);
            }
            row::store8(row_out + lane * 8, y);
          } else if (!p.vector_out) {
#pragma unroll 1
            for (int j = 0; j < 8; ++j) {
              const int n = j * 32 + lane;
              if (n0 + n >= p.N) break;
              int total = 0;
              for (int copy = 0; copy < c; ++copy) total += int(first[copy * slots * S_TILE_N + n]);
              row_out[n] = row::from_float<Y>(
                  scaled(float(total), sa, __ldg(s.b + n0 + n), s.bias ? __ldg(s.bias + n0 + n) : 0.f));
            }
          }
        }
        __syncwarp();
        if (lane < c) mbar_arrive_cluster(map_to_cta(smem_u32(&bars->taken), lane));
      }
      if (++buf == 2) {
        buf = 0;
        buf_phase ^= 1;
      }
    }
  } else {
    // ------------------------------------------------------------------ gather
    const int group = (warp - 2 - S_EPI_WARPS) / S_GATHER_WARPS, gw = (warp - 2 - S_EPI_WARPS) % S_GATHER_WARPS;
    const uint8_t *a_begin = reinterpret_cast<const uint8_t*>(A), *a_end = a_begin + size_t(p.M) * p.K;
    const uint8_t *b_begin = reinterpret_cast<const uint8_t*>(B), *b_end = b_begin + size_t(p.K) * p.N;
    int stage = 0, turn = 0;
    uint32_t phase = 0;
    bool ok = true;
    grid_dependency_wait();
    for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
      const int n0 = tile / p.m_tiles * S_TILE_N, m0 = tile % p.m_tiles * R;
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        if (turn == group) {
          constexpr int ROWS = S_BK / S_GATHER_WARPS;
          // this lane's words of sixteen k rows: bytes 4 * lane .. of either box
          uint32_t w[ROWS][2], tail[ROWS];
#pragma unroll
          for (int i = 0; i < ROWS; ++i) {
            const int k = kb * S_BK + gw + i * S_GATHER_WARPS;
            w[i][0] = w[i][1] = tail[i] = 0;
            if (k < p.K) {
              const uint8_t* src = b_begin + size_t(k) * p.N + n0;
              const uint8_t* word = src - (reinterpret_cast<uintptr_t>(src) & 3);
              w[i][0] = load_word(word + lane * 4, b_begin, b_end);
              w[i][1] = load_word(word + 128 + lane * 4, b_begin, b_end);
              if (lane == 31) tail[i] = load_word(word + 256, b_begin, b_end);
            }
          }
          ok = mbar_wait(&bars->empty[stage], phase ^ 1, abort_flag, status, STATUS_TIMEOUT_EMPTY);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          uint8_t* sw = smem + stage * stage_bytes;
#pragma unroll
          for (int i = 0; i < ROWS; ++i) {
            const int kr = gw + i * S_GATHER_WARPS;
            const unsigned shift = unsigned((reinterpret_cast<uintptr_t>(b_begin) + size_t(kb * S_BK + kr) * p.N + n0) & 3) * 8;
            // the word after this lane's: its neighbour's, or the next box's first, or the tail
            const uint32_t next0 = __shfl_sync(0xffffffffu, lane == 0 ? w[i][1] : w[i][0], (lane + 1) & 31);
            const uint32_t next1 = __shfl_sync(0xffffffffu, w[i][1], (lane + 1) & 31);
            const uint32_t v0 = __funnelshift_r(w[i][0], next0, shift);
            const uint32_t v1 = __funnelshift_r(w[i][1], lane == 31 ? tail[i] : next1, shift);
            const int at = kr * 128 + (((lane / 4) ^ (kr & 7)) << 4) + (lane % 4) * 4;
            *reinterpret_cast<uint32_t*>(sw + at) = v0;
            *reinterpret_cast<uint32_t*>(sw + S_BOX + at) = v1;
          }
          // activations: k of the row past K must be zero (what it meets in B is arbitrary)
          for (int r = gw; r < R && m0 + r < p.M; r += S_GATHER_WARPS) {
            const uint8_t* src = a_begin + size_t(m0 + r) * p.K + size_t(kb) * S_BK;
            const unsigned mis = unsigned(reinterpret_cast<uintptr_t>(src) & 3);
            const uint8_t* word = src - mis;
            const uint32_t mine = load_word(word + lane * 4, a_begin, a_end);
            uint32_t next = __shfl_down_sync(0xffffffffu, mine, 1);
            if (lane == 31) next = load_word(word + 128, a_begin, a_end);
            uint32_t v = __funnelshift_r(mine, next, mis * 8);
            const int left = p.K - (kb * S_BK + lane * 4);
            if (left < 4) v = left <= 0 ? 0u : v & ((1u << (8 * left)) - 1);
            *reinterpret_cast<uint32_t*>(sw + S_W_BYTES + r * 128 + (((lane / 4) ^ (r & 7)) << 4) + (lane % 4) * 4) = v;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->full[stage]);
        }
        if (++turn == S_GATHER_GROUPS) turn = 0;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while another may still push into it or signal it
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, tmem_cols);
  }
}

// --------------------------------------------------------------- tensor path
// Many tiles: clusters of two CTAs (cta_group::2) on 256x256 tiles, persistent, as the INT8
// operator's pair kernel (mm_int8.cu) but with nothing to sum beside the product: A 128 rows
// and B 128 columns per CTA and k block of 128 in a six-stage ring, two accumulators per CTA, so
// that a tile's drain overlaps the next one's MMAs.  The drain scales 32 columns at a time, and
// every warp's 32 rows x 128 bytes leave through shared memory by TMA in whole lines.
constexpr int P_STAGES = 6, P_RING = 4;
constexpr int P_A_BYTES = 128 * 128, P_B_BYTES = 128 * 128, P_STAGE_BYTES = P_A_BYTES + P_B_BYTES;
constexpr int P_EPI_WARPS = 8;
constexpr int P_THREADS = 64 + P_EPI_WARPS * 32;
constexpr int P_OUT_BYTES = 32 * 128;  // a warp's staging tile
constexpr int P_SMEM_BYTES = P_STAGES * P_STAGE_BYTES + P_EPI_WARPS * P_OUT_BYTES + 1024 + 256;
static_assert(P_SMEM_BYTES <= 232448, "pair kernel: shared memory over the limit");

struct PairBarriers {
  uint64_t full[P_STAGES];  // even CTA: both CTAs' bytes
  uint64_t ring[P_RING];    // commits, one for every second k block
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(PairBarriers) <= 256, "PairBarriers outgrew its shared-memory reserve");

template <typename Y>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

struct PairShape {
  int M, N, K, tiles_m, tiles_n, raster_rows;
};

template <typename Y>
__global__ void __launch_bounds__(P_THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_y, Scales s, PairShape p, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  grid_dependency_trigger();
  uint8_t* staging = smem + P_STAGES * P_STAGE_BYTES;
  PairBarriers* bars = reinterpret_cast<PairBarriers*>(staging + P_EPI_WARPS * P_OUT_BYTES);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = int(cluster_ctarank());  // 0: the CTA that issues the MMAs
  const int first_tile = blockIdx.x / 2, tile_step = gridDim.x / 2;
  const int tiles = p.tiles_m * p.tiles_n;
  const int num_kb = (p.K + 127) / 128;

  if (threadIdx.x == 0) {
    for (int i = 0; i < P_STAGES; ++i) mbar_init(&bars->full[i], 1);
    for (int r = 0; r < P_RING; ++r) mbar_init(&bars->ring[r], 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], 2 * P_EPI_WARPS);
    }
    bars->abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
    tma_prefetch_desc(&map_y);
  }
  if (warp == 1) {
    tmem_alloc_pair(&bars->tmem_base, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the partner's barriers exist before anything signals them
  tc_fence_after_sync();
  const uint32_t tmem_base = bars->tmem_base;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0, g = 0, observed = -1;  // g: number of the next k block over all tiles
      bool ok = true;
      grid_dependency_wait();
      for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
        int tm, tn;
        i8::pair_tile_coords(tile, p.tiles_m, p.tiles_n, p.raster_rows, tm, tn);
        for (int kb = 0; kb < num_kb; ++kb, ++g) {
          if (g >= P_STAGES) {
            // commit e follows even block 2e and covers it and its predecessor
            const int e = (g - P_STAGES + 1) >> 1;
            if (e > observed) {
              ok = mbar_wait(&bars->ring[e & (P_RING - 1)], (e >> 2) & 1, abort_flag, status, STATUS_TIMEOUT_EMPTY);
              if (!ok) break;
              observed = e;
            }
          }
          uint8_t* sa = smem + stage * P_STAGE_BYTES;
          const uint32_t full = map_to_cta(smem_u32(&bars->full[stage]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&bars->full[stage], 2 * P_STAGE_BYTES);
          tma_load_2d_pair(sa, &map_a, full, kb * 128, tm * 256 + rank * 128);
          tma_load_2d_pair(sa + P_A_BYTES, &map_b, full, tn * 256 + rank * 128, kb * 128);
          if (++stage == P_STAGES) stage = 0;
        }
      }
      // (the odd CTA's loads are counted by the even one, which it meets before it leaves)
      if (!ok && rank == 0) drain_loads(bars->full, P_STAGES, g);
    }
  } else if (warp == 1) {
    // ----------------------------------------------- MMA issuer (even CTA only)
    if (rank == 0 && lane == 0) {
      constexpr uint32_t IDESC = umma_idesc(/*D=s32*/ 2, /*A=s8*/ 1, /*B=s8*/ 1, /*A K-major*/ 0, /*B N-major*/ 1,
                                            256, 256);
      int stage = 0, g = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
        ok = mbar_wait_cluster(&bars->acc_empty[acc], acc_phase ^ 1, abort_flag, status, STATUS_TIMEOUT_TMEM_EMPTY);
        tc_fence_after_sync();
        for (int kb = 0; kb < num_kb && ok; ++kb, ++g) {
          ok = mbar_wait(&bars->full[stage], phase, abort_flag, status, STATUS_TIMEOUT_FULL);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t sa = smem_u32(smem + stage * P_STAGE_BYTES), sb = sa + P_A_BYTES;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint64_t da = smem_desc(sa + j * 32, 16, 1024, SMEM_SWIZZLE_128B);
            const uint64_t db = smem_desc(sb + j * 32 * 128, 16, 1024, SMEM_SWIZZLE_128B);
            umma_i8_pair(tmem_base + acc * 256, da, db, IDESC, (kb | j) != 0);
          }
          if ((g & 1) == 0) umma_commit_pair(&bars->ring[(g >> 1) & (P_RING - 1)], 3);
          if (++stage == P_STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (ok) umma_commit_pair(&bars->acc_full[acc], 3);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    constexpr int COLS = 128 / int(sizeof(Y));  // columns of a staging tile
    const int ew = warp - 2, quarter = warp % 4, half = ew / 4;
    uint8_t* stage_out = staging + ew * P_OUT_BYTES;
    uint8_t* my_row = stage_out + lane * 128;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    grid_dependency_wait();
    for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
      int tm, tn;
      i8::pair_tile_coords(tile, p.tiles_m, p.tiles_n, p.raster_rows, tm, tn);
      const int m0 = tm * 256 + rank * 128 + quarter * 32;  // this warp's first row
      const int n0 = tn * 256 + half * 128;                 // and column
      const float sa = m0 + lane < p.M ? __ldg(s.a + m0 + lane) : 0.f;
      ok = mbar_wait(&bars->acc_full[acc], acc_phase, abort_flag, status, STATUS_TIMEOUT_TMEM_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after_sync();
#pragma unroll 1
      for (int col = 0; col < 128; col += COLS) {
        if (m0 >= p.M || n0 + col >= p.N) break;  // warp-uniform
        if (lane == 0) tma_store_wait_read<0>();  // the last store has read the staging tile
        __syncwarp();
#pragma unroll
        for (int sub = 0; sub < COLS; sub += 32) {
          uint32_t v[32];
          tmem_ld_32x32(tmem_base + acc * 256 + half * 128 + col + sub + (uint32_t(quarter * 32) << 16), v);
          tmem_ld_wait();
          const int n = n0 + col + sub;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            // N is a multiple of 16 here: four columns are inside or outside as a whole
            float4 sb = make_float4(0.f, 0.f, 0.f, 0.f), bias = sb;
            if (n + g * 4 < p.N) {
              sb = __ldg(reinterpret_cast<const float4*>(s.b + n + g * 4));
              if (s.bias) bias = __ldg(reinterpret_cast<const float4*>(s.bias + n + g * 4));
            }
            const float y0 = scaled(float(int(v[g * 4])), sa, sb.x, bias.x);
            const float y1 = scaled(float(int(v[g * 4 + 1])), sa, sb.y, bias.y);
            const float y2 = scaled(float(int(v[g * 4 + 2])), sa, sb.z, bias.z);
            const float y3 = scaled(float(int(v[g * 4 + 3])), sa, sb.w, bias.w);
            if constexpr (sizeof(Y) == 4) {
              *reinterpret_cast<float4*>(my_row + ((g ^ (lane & 7)) << 4)) = make_float4(y0, y1, y2, y3);
            } else {
              *reinterpret_cast<uint2*>(my_row + (((sub / 8 + g / 2) ^ (lane & 7)) << 4) + (g & 1) * 8) =
                  make_uint2(pack2<Y>(y0, y1), pack2<Y>(y2, y3));
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&map_y, stage_out, n0 + col, m0);  // rows and columns outside Y are dropped
          tma_store_commit();
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&bars->acc_empty[acc]), 0));
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
  }

  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves (or frees TMEM) while its partner may still signal it
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ------------------------------------------------------------------ dispatch
enum Path { PATH_AUTO = 0, PATH_GENERIC = 1, PATH_STREAM = 2, PATH_STREAM_GATHER = 3, PATH_PAIR = 4 };
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

// Launch in clusters of `cluster` CTAs; the grid may be scheduled while the one ahead drains.
template <typename... Params, typename... Args>
static bool launch_clusters(void (*kernel)(Params...), int grid, int threads, int smem_bytes, int cluster,
                            cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = cluster;
  attrs[0].val.clusterDim.y = 1;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = 2;
  ++launch_counter();
  if (cudaLaunchKernelEx(&cfg, kernel, Params(args)...) == cudaSuccess) return true;
  cudaGetLastError();
  return false;
}

// Clusters of `cluster` CTAs that the device holds at once.
template <typename Kernel>
static int max_clusters(Kernel kernel, int threads, int smem_bytes, int cluster) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster * 64);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem_bytes;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  return n;
}

constexpr int R_CHOICES[4] = {16, 32, 64, 128};
struct DeviceSetup {
  bool ready = false;
  int clusters[2][4][S_MAX_CLUSTER + 1] = {};  // [gather][R][c]
  int pairs = 0;
};
static DeviceSetup setups[MAX_DEVICES];
template <typename Y>
static void configure_kernels() {
  cudaFuncSetAttribute(stream_kernel<Y, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
  cudaFuncSetAttribute(stream_kernel<Y, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
  cudaFuncSetAttribute(pair_kernel<Y>, cudaFuncAttributeMaxDynamicSharedMemorySize, P_SMEM_BYTES);
}
static DeviceSetup& device_setup(DeviceCtx& ctx) {
  DeviceSetup& d = setups[ctx.device];
  if (!d.ready) {
    configure_kernels<__half>();
    configure_kernels<__nv_bfloat16>();
    configure_kernels<float>();
    for (int r = 0; r < 4; ++r) {
      for (int c = 1; c <= S_MAX_CLUSTER; ++c) {
        const int R = R_CHOICES[r], bytes = s_smem_bytes(R, c);
        if (bytes > 232448) continue;
        d.clusters[0][r][c] = max_clusters(stream_kernel<__half, false>, S_THREADS, bytes, c);
        d.clusters[1][r][c] = max_clusters(stream_kernel<__half, true>, S_GATHER_THREADS, bytes, c);
      }
    }
    d.pairs = max_clusters(pair_kernel<__half>, P_THREADS, P_SMEM_BYTES, 2);
    cudaGetLastError();
    d.ready = true;
  }
  return d;
}

struct StreamPlan {
  int R = 0, cluster = 0, clusters = 0, m_tiles = 0, tiles = 0;
  double us = 1e30;  // estimate
};
static StreamPlan plan_stream(const DeviceSetup& d, bool gather, int M, int N, int K) {
  StreamPlan best;
  const int r = M <= 16 ? 0 : M <= 32 ? 1 : M <= 64 ? 2 : 3;
  const int R = R_CHOICES[r];
  const long long m_tiles = (M + R - 1) / R, tiles = m_tiles * ((N + S_TILE_N - 1) / S_TILE_N);
  const int num_kb = (K + S_BK - 1) / S_BK;
  if (tiles > 0x3fffffff) return best;
  for (int c = 1; c <= S_MAX_CLUSTER && c <= num_kb; ++c) {
    const int held = d.clusters[gather][r][c];
    if (held <= 0) continue;
    const int clusters = int(std::min<long long>(tiles, held));
    const double rounds = double((tiles + clusters - 1) / clusters);
    const double kb = (num_kb + c - 1) / c;
    const double rate = std::min(58e3, 6.4e6 / (clusters * c));  // bytes per us and SM
    const double us = rounds * (kb * s_stage_bytes(R) / rate + 1.0 + 0.3 * (c > 1) + 0.01 * R) + 3;
    if (us < best.us) best = {R, c, clusters, int(m_tiles), int(tiles), us};
  }
  return best;
}

template <typename Y, bool GATHER>
static bool launch_stream(DeviceCtx& ctx, const StreamPlan& plan, const int8_t* A, const int8_t* B, Y* out, int M,
                          int N, int K, const Scales& s, cudaStream_t stream) {
  CUtensorMap map_b = {}, map_a = {};
  if (!GATHER && (!make_tensor_map_2d(&map_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, B, K, N, N, S_BK, 128,
                                      CU_TENSOR_MAP_SWIZZLE_128B) ||
                  !make_tensor_map_2d(&map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, A, M, K, K, plan.R, S_BK,
                                      CU_TENSOR_MAP_SWIZZLE_128B)))
    return false;
  const StreamShape p = {M, N, K, plan.R, plan.cluster, plan.m_tiles, plan.tiles,
                         N % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0};
  last_path() = GATHER ? PATH_STREAM_GATHER : PATH_STREAM;
  return launch_clusters(stream_kernel<Y, GATHER>, plan.clusters * plan.cluster,
                         GATHER ? S_GATHER_THREADS : S_THREADS, s_smem_bytes(plan.R, plan.cluster), plan.cluster,
                         stream, map_b, map_a, A, B, out, s, p, ctx.status);
}

template <typename Y>
static bool launch_pair(DeviceCtx& ctx, const DeviceSetup& d, const int8_t* A, const int8_t* B, Y* out, int M, int N,
                        int K, const Scales& s, cudaStream_t stream) {
  CUtensorMap map_a, map_b, map_y;
  constexpr CUtensorMapDataType TYPE = std::is_same<Y, float>::value    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : std::is_same<Y, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (!make_tensor_map_2d(&map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, A, M, K, K, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_2d(&map_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, B, K, N, N, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_2d(&map_y, TYPE, sizeof(Y), out, M, N, size_t(N) * sizeof(Y), 32, 128 / sizeof(Y),
                          CU_TENSOR_MAP_SWIZZLE_128B))
    return false;
  const PairShape p = {M, N, K, (M + 255) / 256, (N + 255) / 256, i8::raster_group_rows(K)};
  const int clusters = std::min(p.tiles_m * p.tiles_n, d.pairs);
  last_path() = PATH_PAIR;
  return launch_clusters(pair_kernel<Y>, 2 * clusters, P_THREADS, P_SMEM_BYTES, 2, stream, map_a, map_b, map_y, s, p,
                         ctx.status);
}

template <typename Y>
static int solve(const int8_t* A, const int8_t* B, Y* out, int M, int N, int K, const Scales& s,
                 cudaStream_t stream) {
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  int device;
  if ((!device_ctx_entry(device).ready || !setups[device].ready) && is_capturing(stream)) return -4;
  DeviceCtx& ctx = device_ctx();
  const DeviceSetup& d = device_setup(ctx);
  const int force = forced_path();
  if (ctx.cc_major >= 10 && K > 0 && K < (1 << 17) && force != PATH_GENERIC) {
    const bool tma = K % 16 == 0 && N % 16 == 0 && aligned(A) && aligned(B);
    const bool pair_ok = tma && d.pairs > 0 && aligned(out) && aligned(s.b) && aligned(s.bias) &&
                         (long long)((M + 255) / 256) * ((N + 255) / 256) <= 0x3fffffff;
    const StreamPlan plan = plan_stream(d, !tma || force == PATH_STREAM_GATHER, M, N, K);
    if (pair_ok && force != PATH_STREAM && force != PATH_STREAM_GATHER) {
      const double rounds = ((long long)((M + 255) / 256) * ((N + 255) / 256) + d.pairs - 1) / d.pairs;
      const double us = 6 + rounds * (0.3 * ((K + 127) / 128) + 1);
      if ((force == PATH_PAIR || us < plan.us) && launch_pair(ctx, d, A, B, out, M, N, K, s, stream)) return 0;
    }
    if (plan.cluster > 0) {
      const bool gather = !tma || force == PATH_STREAM_GATHER;
      if (gather ? launch_stream<Y, true>(ctx, plan, A, B, out, M, N, K, s, stream)
                 : launch_stream<Y, false>(ctx, plan, A, B, out, M, N, K, s, stream))
        return 0;
    }
  }
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
