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

// Sizes stay this far below 2^31, so that a tile's coordinates past the end do not wrap.
constexpr int MAX_SIZE = 0x7fffffff - 1024;
inline int ceil_div(int a, int b) { return int(((long long)a + b - 1) / b); }

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
// There is no workspace: once all of them are through, every CTA pushes its int32 partials
// straight into the shared memory (the ring, idle by then) of the CTA that finishes the rows, four
// rows at a time (a 16-byte store per lane; 4-byte ones took 5.8 of 47 us at 128 x 8192 x
// 28672), quad g going to CTA g % c; an mbarrier there counts the pushes, and the owner adds the c
// copies, scales and stores.  Integer sums, so the split changes no bit, and nothing is shared between
// calls: any streams, any graphs.  With c = 1 the lanes, each one output column, scale and store
// from registers while the ring fills for the next tile.
//
// Shared memory is nearly all ring: an SM has to keep about 100 KiB in flight to cover HBM
// latency at its share of the bandwidth.
//
// GATHER: rows of A or B that do not start at 16-byte boundaries cannot be moved by a tensor map.
// Four warps then copy the 16-byte granules that hold a tile's part of each row into a raw ring
// (cp.async; untiled bulk copies, one per row, measured 75 clocks each, six times what HBM
// allows), and eight shift them into the swizzled tiles that the MMAs read.
constexpr int S_BK = 128;                // k per ring stage = one 128-byte swizzle row
constexpr int S_BOX = 128 * 128;         // 128 k rows x 128 columns of B
constexpr int S_W_BYTES = 2 * S_BOX;     // the two boxes of a tile
constexpr int S_TILE_N = 256;
constexpr int S_MAX_STAGES = 6, S_MAX_RAW_STAGES = 4;
constexpr int S_EPI_WARPS = 8;
constexpr int S_GATHER_GROUPS = 2, S_GATHER_WARPS = 4;  // stages are dealt to the groups in turn
constexpr int S_COPY_WARPS = 4;                         // warp 0 and the last three
constexpr int S_THREADS = 64 + S_EPI_WARPS * 32;
constexpr int S_GATHER_THREADS = S_THREADS + (S_GATHER_GROUPS * S_GATHER_WARPS + S_COPY_WARPS - 1) * 32;
constexpr int S_MAX_CLUSTER = 8;

__host__ __device__ constexpr int s_stages(int R, bool gather) {
  return gather ? 2 : R <= 32 ? 6 : R == 64 ? 5 : 4;
}
__host__ __device__ constexpr int s_stage_bytes(int R) { return S_W_BYTES + R * 128; }
// Raw ring: the granules that hold 256 bytes of each k row of B, at any offset, and 128 of each
// row of A.
constexpr int S_RAW_B_ROW = 256 + 16, S_RAW_A_ROW = 128 + 16;
__host__ __device__ constexpr int s_raw_bytes(int R) { return S_BK * S_RAW_B_ROW + R * S_RAW_A_ROW; }
__host__ __device__ constexpr int s_raw_stages(int R) { return R == 16 ? 4 : R == 128 ? 2 : 3; }
__host__ __device__ constexpr int s_ring_bytes(int R, bool gather) {
  return s_stages(R, gather) * s_stage_bytes(R) + (gather ? s_raw_stages(R) * s_raw_bytes(R) : 0);
}
__host__ __device__ constexpr int s_smem_bytes(int R, bool gather) {
  return s_ring_bytes(R, gather) + 1024 /*alignment*/ + 256 /*barriers*/;
}
// Row quads of a tile that one CTA of the cluster finishes, and the room that their partials take.
__host__ __device__ constexpr int s_slots(int R, int c) { return (R / 4 + c - 1) / c; }
__host__ __device__ constexpr int s_push_bytes(int R, int c) { return c * s_slots(R, c) * S_TILE_N * 16; }
constexpr int SMEM_LIMIT = 232448, S_SMEM_LIMIT = SMEM_LIMIT - S_EPI_WARPS * 128 * 4 /*row scales*/;
__host__ __device__ constexpr bool s_fits(int R, bool gather) {
  return s_smem_bytes(R, gather) <= S_SMEM_LIMIT && s_push_bytes(R, 7) <= s_ring_bytes(R, gather) &&
         s_push_bytes(R, 6) <= s_ring_bytes(R, gather) && s_push_bytes(R, 5) <= s_ring_bytes(R, gather) &&
         s_push_bytes(R, 3) <= s_ring_bytes(R, gather) && s_push_bytes(R, 8) <= s_ring_bytes(R, gather);
}
static_assert(s_fits(16, false) && s_fits(32, false) && s_fits(64, false) && s_fits(128, false) && s_fits(16, true) &&
                  s_fits(32, true) && s_fits(64, true) && s_fits(128, true),
              "streaming kernel: shared memory over the limit");

struct StreamBarriers {
  uint64_t full[S_MAX_STAGES];
  uint64_t empty[S_MAX_STAGES];
  uint64_t raw_full[S_MAX_RAW_STAGES];   // GATHER: a k block's granules have landed
  uint64_t raw_empty[S_MAX_RAW_STAGES];  // and have been shifted into place
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t ring_idle;  // c > 1: every CTA of the cluster is through with its part of K
  uint64_t pushed;     // all partials of a tile have arrived in this CTA
  uint64_t taken;      // and have been read: the ring may fill again
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(StreamBarriers) <= 256, "StreamBarriers outgrew its shared-memory reserve");

__device__ __forceinline__ void store_cluster_quad(uint32_t cluster_addr, uint32_t a, uint32_t b, uint32_t c,
                                                   uint32_t d) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
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

// A whole warp's wait.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status,
                                          int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code));
}
__device__ __forceinline__ bool warp_wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                                  int* status, int code) {
  return __all_sync(0xffffffffu, mbar_wait_cluster(bar, parity, abort_flag, status, code));
}

// Whether the phase has completed, without waiting for it.
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Sixteen bytes global -> shared, asynchronously and past L1; both addresses aligned.
__device__ __forceinline__ void copy_granule(uint32_t dst, uintptr_t src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but this thread's N last groups of copies have landed.
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uintptr_t floor16(uintptr_t a) { return a & ~uintptr_t(15); }
__device__ __forceinline__ uintptr_t ceil16(uintptr_t a) { return (a + 15) & ~uintptr_t(15); }

// The gathering form's view of a row-major operand: where a block of it starts and how far its
// rows are apart.  Rows that are sixteen apart start at the same offset in their granule
// (sixteen pitches are a multiple of sixteen bytes), so a thread that keeps to one row of
// sixteen works with constant offsets.
struct Block {
  uintptr_t corner;  // first byte of the block
  int pitch, rows;
  uintptr_t begin, end;  // of the operand
  __device__ uintptr_t row(int r) const { return corner + size_t(r) * pitch; }
  // Whether `bytes` from the granule of each row's first byte on lie in the operand: for a block
  // whose every row has that, or row by row.
  __device__ bool inside(int bytes) const {
    return corner - 15 >= begin && row(rows - 1) + bytes <= end;
  }
  __device__ bool row_inside(int r, int bytes) const {
    return floor16(row(r)) >= begin && floor16(row(r)) + bytes <= end;
  }
};

// Copies GRANULES + 1 granules from each row's first byte on, to (GRANULES + 1) * 16 apart in
// shared memory.  Thread t of S_COPY_WARPS * 32: granule t % GRANULES of every (threads /
// GRANULES)th row, then the last granule of row t.  What reaches outside the operand is left out
// (edge_word reads that).
template <int GRANULES>
__device__ __forceinline__ void copy_rows(uint32_t smem_dst, const Block& b, int t) {
  constexpr int ROWS = S_COPY_WARPS * 32 / GRANULES, ROW_BYTES = (GRANULES + 1) * 16;
  static_assert(16 % ROWS == 0 && S_COPY_WARPS * 32 >= 128, "a thread keeps to a few rows of sixteen");
  const int g = t % GRANULES;
  const size_t step = 16 * size_t(b.pitch);
  const bool inside = b.inside(ROW_BYTES);
#pragma unroll
  for (int part = 0; part < 16 / ROWS; ++part) {
    const int r0 = t / GRANULES + part * ROWS;
    uint32_t dst = smem_dst + r0 * ROW_BYTES + g * 16;
    uintptr_t from = floor16(b.row(r0)) + g * 16;
    if (inside) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (r0 + i * 16 < b.rows) copy_granule(dst + i * 16 * ROW_BYTES, from);
        from += step;
      }
    } else {
      for (int r = r0; r < b.rows; r += 16, from += step, dst += 16 * ROW_BYTES)
        if (from >= b.begin && from + 16 <= b.end) copy_granule(dst, from);
    }
  }
  if (t < b.rows) {
    const uintptr_t last = floor16(b.row(t)) + GRANULES * 16;
    if (inside || (last >= b.begin && last + 16 <= b.end))
      copy_granule(smem_dst + t * ROW_BYTES + GRANULES * 16, last);
  }
}

// Word `w` from a row's first granule on, which is `granules` in shared memory and at address
// `from`; where its granule reaches outside the operand its bytes come from memory.
__device__ __noinline__ uint32_t edge_word(uint32_t granules, uintptr_t from, int w, uintptr_t begin,
                                           uintptr_t end) {
  const uintptr_t granule = from + w / 4 * 16, at = from + w * 4;
  if (granule >= begin && granule + 16 <= end) return lds32(granules + w * 4);
  uint32_t v = 0;
  for (int e = 0; e < 4; ++e)
    if (at + e >= begin && at + e < end) v |= uint32_t(*reinterpret_cast<const uint8_t*>(at + e)) << (8 * e);
  return v;
}

// Shifts WORDS * 4 bytes (WORDS: 32 or 64) of each row of a block from their granules into
// 128-byte rows with the swizzle of the MMA's operands, the second 32 words S_BOX further on.
// A warp's share: the rows whose number mod 16 is within [OWN gw, OWN gw + OWN); a lane moves one
// word (or two) of each: two conflict-free loads, a funnel shift, a conflict-free store; four
// rows' loads before the first store.  `mask` keeps a lane's bytes that the rows still have.
template <int WORDS>
__device__ __forceinline__ void shift_rows(uint32_t to, uint32_t granules, const Block& b, int gw, int lane,
                                           uint32_t mask) {
  constexpr int ROW_BYTES = WORDS * 4 + 16, BOXES = WORDS / 32, OWN = 16 / S_GATHER_WARPS;
  const int sixteens = (b.rows + 15) / 16;  // (the ring has room for whole sixteens)
#pragma unroll
  for (int j = 0; j < OWN; ++j) {
    const int r0 = gw * OWN + j;
    const unsigned offset = unsigned(b.row(r0)) & 15, bits = (offset & 3) * 8;
    const uint32_t from = granules + r0 * ROW_BYTES + (offset & 12) + lane * 4;
    const uint32_t dst = to + r0 * 128 + (((lane / 4) ^ (r0 & 7)) << 4) + lane % 4 * 4;
#pragma unroll
    for (int i0 = 0; i0 < 8; i0 += 4) {
      if (i0 >= sixteens) break;
      uint32_t v[4][BOXES];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int h = 0; h < BOXES; ++h) {
          const uint32_t w = from + (i0 + i) * 16 * ROW_BYTES + h * 128;
          v[i][h] = i0 + i < sixteens ? __funnelshift_r(lds32(w), lds32(w + 4), bits) & mask : 0u;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r0 + (i0 + i) * 16 < b.rows) {  // warp-uniform
#pragma unroll
          for (int h = 0; h < BOXES; ++h) sts32(dst + (i0 + i) * 16 * 128 + h * S_BOX, v[i][h]);
        }
      }
    }
  }
  if (!b.inside(ROW_BYTES)) {  // once more for the rows at the operand's first and last bytes
    for (int r = gw * OWN; r < b.rows; r += (r % OWN == OWN - 1 ? 17 - OWN : 1)) {
      if (b.row_inside(r, ROW_BYTES)) continue;
      const unsigned offset = unsigned(b.row(r)) & 15;
      const uint32_t from = granules + r * ROW_BYTES;
      const uintptr_t first = floor16(b.row(r));
      for (int h = 0; h < BOXES; ++h) {
        const int w = h * 32 + lane + offset / 4;
        sts32(to + h * S_BOX + r * 128 + (((lane / 4) ^ (r & 7)) << 4) + lane % 4 * 4,
              __funnelshift_r(edge_word(from, first, w, b.begin, b.end), edge_word(from, first, w + 1, b.begin, b.end),
                              (offset & 3) * 8) & mask);
      }
    }
  }
}

struct StreamShape {
  int M, N, K;
  int R, cluster, m_tiles, tiles;
};

template <typename Y, bool GATHER>
__global__ void __launch_bounds__(GATHER ? S_GATHER_THREADS : S_THREADS, 1)
    stream_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a,
                  const int8_t* __restrict__ A, const int8_t* __restrict__ B, Y* __restrict__ out, Scales s,
                  StreamShape p, int* status) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ float row_scales[S_EPI_WARPS][128];  // scale_A of the tile's rows, a copy for each warp
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  grid_dependency_trigger();
  const int R = p.R, c = p.cluster;
  const int stages = s_stages(R, GATHER), stage_bytes = s_stage_bytes(R);
  const uint32_t push = smem_u32(smem);  // c > 1: partials, over the idle ring
  uint8_t* raw = smem + stages * stage_bytes;
  const int raw_stages = s_raw_stages(R), raw_bytes = s_raw_bytes(R);
  StreamBarriers* bars = reinterpret_cast<StreamBarriers*>(smem + s_ring_bytes(R, GATHER));
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
    for (int i = 0; GATHER && i < raw_stages; ++i) {
      mbar_init(&bars->raw_full[i], S_COPY_WARPS);
      mbar_init(&bars->raw_empty[i], S_GATHER_WARPS);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], S_EPI_WARPS);
    }
    mbar_init(&bars->ring_idle, c);
    mbar_init(&bars->pushed, c * S_EPI_WARPS);
    mbar_init(&bars->taken, S_EPI_WARPS);
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

  constexpr int FIRST_COPY_WARP = 2 + S_EPI_WARPS + S_GATHER_GROUPS * S_GATHER_WARPS;
  if (GATHER && (warp == 0 || warp >= FIRST_COPY_WARP)) {
    // ---------------------------------------------------------------- granules
    const int t = warp == 0 ? lane : (warp - FIRST_COPY_WARP + 1) * 32 + lane;
    const uintptr_t a_begin = reinterpret_cast<uintptr_t>(A), a_end = a_begin + size_t(p.M) * p.K;
    const uintptr_t b_begin = reinterpret_cast<uintptr_t>(B), b_end = b_begin + size_t(p.K) * p.N;
    int stage = 0, pending = 0, done = 0;  // k blocks under way; stage of the oldest of them
    uint32_t phase = 0, taken_phase = 0;
    bool ok = true;
    auto landed = [&]() {  // this thread's copies have landed: the warp's oldest block is complete
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->raw_full[done]);
      if (++done == raw_stages) done = 0;
      --pending;
    };
    auto all_landed = [&]() {
      wait_copies<0>();
      while (pending > 0) landed();
    };
    grid_dependency_wait();
    for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
      const int n0 = tile / p.m_tiles * S_TILE_N, m0 = tile % p.m_tiles * R;
      const int rows = min(R, p.M - m0);
      if (c > 1 && tile != first_tile) {
        ok = warp_wait(&bars->taken, taken_phase, abort_flag, status, STATUS_TIMEOUT_FLAG);
        if (!ok) break;
        taken_phase ^= 1;
      }
      for (int kb = kb0; kb < kb1; ++kb) {
        // before the warp waits for room it hands over what it has
        int room = 1;
        if (lane == 0) room = mbar_test_wait(&bars->raw_empty[stage], phase ^ 1);
        if (!__shfl_sync(0xffffffffu, room, 0)) {
          all_landed();
          ok = warp_wait(&bars->raw_empty[stage], phase ^ 1, abort_flag, status, STATUS_TIMEOUT_EMPTY);
          if (!ok) break;
        }
        const uint32_t block = smem_u32(raw) + stage * raw_bytes;
        const int k0 = kb * S_BK;
        const Block block_b = {b_begin + size_t(k0) * p.N + n0, p.N, min(S_BK, p.K - k0), b_begin, b_end};
        const Block block_a = {a_begin + size_t(m0) * p.K + k0, p.K, rows, a_begin, a_end};
        copy_rows<16>(block, block_b, t);
        copy_rows<8>(block + S_BK * S_RAW_B_ROW, block_a, t);
        commit_copies();
        if (++pending == 3) {
          wait_copies<2>();
          landed();
        }
        if (++stage == raw_stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      all_landed();
    }
    wait_copies<0>();
  } else if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0, taken_phase = 0;
      bool ok = true;
      grid_dependency_wait();  // the operands may have been written by the grid ahead
      for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
        const int n0 = tile / p.m_tiles * S_TILE_N, m0 = tile % p.m_tiles * R;
        if (c > 1 && tile != first_tile) {
          ok = mbar_wait(&bars->taken, taken_phase, abort_flag, status, STATUS_TIMEOUT_FLAG);
          if (!ok) break;
          taken_phase ^= 1;
        }
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
    const int column = half * 128 + quarter * 32 + lane;  // of the tile
    // The finished values are dealt out by columns: warp ew has 32 of each row (c = 1: those that its
    // lanes read from tensor memory).
    const int own_column = c == 1 ? column : ew * 32 + lane;
    float* scales_a = row_scales[ew];
    int buf = 0;
    uint32_t buf_phase = 0, tile_phase = 0;
    bool ok = true;
    grid_dependency_wait();  // before the scales are read and the output is written
    for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
      const int n0 = tile / p.m_tiles * S_TILE_N, m0 = tile % p.m_tiles * R;
      const int rows = min(R, p.M - m0);
      // the scales travel while the accumulator fills
      const int n = n0 + own_column;
      const bool in = n < p.N;
      const float sb = in ? __ldg(s.b + n) : 0.f, bias = in && s.bias ? __ldg(s.bias + n) : 0.f;
      __syncwarp();
      for (int r = lane; r < rows; r += 32) scales_a[r] = __ldg(s.a + m0 + r);
      __syncwarp();
      Y* column_out = out + size_t(m0) * p.N + n;
      ok = warp_wait(&bars->acc_full[buf], buf_phase, abort_flag, status, STATUS_TIMEOUT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t acc = tmem_base + (buf * 2 + half) * R + (uint32_t(quarter * 32) << 16);
      if (c == 1) {
        for (int r0 = 0; r0 < rows; r0 += 16) {
          uint32_t v[16];
          tmem_ld_32x16(acc + r0, v);
          tmem_ld_wait();
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            if (in && r0 + r < rows)
              column_out[size_t(r0 + r) * p.N] = row::from_float<Y>(scaled(float(int(v[r])), scales_a[r0 + r], sb, bias));
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->acc_empty[buf]);
      } else {
        // all of this CTA's loads have landed and all its MMAs have read them
        if (ew == 0 && lane < c) mbar_arrive_cluster(map_to_cta(smem_u32(&bars->ring_idle), lane));
        ok = warp_wait_cluster(&bars->ring_idle, tile_phase, abort_flag, status, STATUS_TIMEOUT_FLAG);
        if (!ok) break;
        const int slots = s_slots(R, c);
        const uint32_t to = push + uint32_t((rank * slots * S_TILE_N + column) * 16);
        int owner = 0;
        uint32_t slot_bytes = 0;
        for (int r0 = 0; r0 < rows; r0 += 16) {
          uint32_t v[16];
          tmem_ld_32x16(acc + r0, v);
          tmem_ld_wait();
#pragma unroll
          for (int r = 0; r < 16; r += 4) {
            if (r0 + r < rows) {
              store_cluster_quad(map_to_cta(to + slot_bytes, owner), v[r], v[r + 1], v[r + 2], v[r + 3]);
              if (++owner == c) {
                owner = 0;
                slot_bytes += S_TILE_N * 16;
              }
            }
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->acc_empty[buf]);
        if (lane < c) mbar_arrive_cluster(map_to_cta(smem_u32(&bars->pushed), lane));
        ok = warp_wait_cluster(&bars->pushed, tile_phase, abort_flag, status, STATUS_TIMEOUT_FLAG);
        if (!ok) break;
        for (int slot = 0; (slot * c + rank) * 4 < rows; ++slot) {
          const int r0 = (slot * c + rank) * 4;
          int total[4] = {};
          for (int copy = 0; copy < c; ++copy) {
            const int4 x = lds128(push + uint32_t(((copy * slots + slot) * S_TILE_N + own_column) * 16));
            total[0] += x.x, total[1] += x.y, total[2] += x.z, total[3] += x.w;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (in && r0 + e < rows)
              column_out[size_t(r0 + e) * p.N] = row::from_float<Y>(scaled(float(total[e]), scales_a[r0 + e], sb, bias));
          }
        }
        fence_proxy_async_smem();  // these accesses come before the loads that fill the ring again
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->taken);
        tile_phase ^= 1;
      }
      if (++buf == 2) {
        buf = 0;
        buf_phase ^= 1;
      }
    }
  } else {
    // ----------------------------------------------------------------- shifting
    const int group = (warp - 2 - S_EPI_WARPS) / S_GATHER_WARPS, gw = (warp - 2 - S_EPI_WARPS) % S_GATHER_WARPS;
    const uintptr_t a_begin = reinterpret_cast<uintptr_t>(A), a_end = a_begin + size_t(p.M) * p.K;
    const uintptr_t b_begin = reinterpret_cast<uintptr_t>(B), b_end = b_begin + size_t(p.K) * p.N;
    int stage = 0, raw_stage = 0, turn = 0;
    uint32_t phase = 0, raw_phase = 0;
    bool ok = true;
    grid_dependency_wait();
    for (int tile = first_tile; tile < p.tiles && ok; tile += tile_step) {
      const int n0 = tile / p.m_tiles * S_TILE_N, m0 = tile % p.m_tiles * R;
      const int rows = min(R, p.M - m0);
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        if (turn == group) {
          ok = warp_wait(&bars->empty[stage], phase ^ 1, abort_flag, status, STATUS_TIMEOUT_EMPTY) &&
               warp_wait(&bars->raw_full[raw_stage], raw_phase, abort_flag, status, STATUS_TIMEOUT_FULL);
          if (!ok) break;
          const uint32_t sw = smem_u32(smem) + stage * stage_bytes;
          const uint32_t block = smem_u32(raw) + raw_stage * raw_bytes;
          const int k0 = kb * S_BK;
          // What a tile of B holds past K, or past the last column, meets a zero of A or goes to no
          // output; A's bytes past K have to be zero.
          const Block block_b = {b_begin + size_t(k0) * p.N + n0, p.N, min(S_BK, p.K - k0), b_begin, b_end};
          const Block block_a = {a_begin + size_t(m0) * p.K + k0, p.K, rows, a_begin, a_end};
          const int left = p.K - k0 - lane * 4;
          shift_rows<64>(sw, block, block_b, gw, lane, 0xffffffffu);
          shift_rows<32>(sw + S_W_BYTES, block + S_BK * S_RAW_B_ROW, block_a, gw, lane,
                         left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bars->full[stage]);
            mbar_arrive(&bars->raw_empty[raw_stage]);
          }
        }
        if (++turn == S_GATHER_GROUPS) turn = 0;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
        if (++raw_stage == raw_stages) {
          raw_stage = 0;
          raw_phase ^= 1;
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
static_assert(P_SMEM_BYTES <= SMEM_LIMIT, "pair kernel: shared memory over the limit");

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

// TMA_OUT: rows of Y start at 16-byte boundaries, and the scales' at theirs.  Otherwise a warp
// reads its staging tile back row by row and stores element by element.
template <typename Y, bool TMA_OUT>
__global__ void __launch_bounds__(P_THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_y, Y* __restrict__ out, Scales s, PairShape p, int* status) {
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
    if (TMA_OUT) tma_prefetch_desc(&map_y);
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
    const uint32_t my_row = smem_u32(stage_out) + lane * 128;
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
      ok = warp_wait(&bars->acc_full[acc], acc_phase, abort_flag, status, STATUS_TIMEOUT_TMEM_FULL);
      if (!ok) break;
      tc_fence_after_sync();
#pragma unroll 1
      for (int col = 0; col < 128; col += COLS) {
        if (m0 >= p.M || n0 + col >= p.N) break;  // warp-uniform
        if (TMA_OUT && lane == 0) tma_store_wait_read<0>();  // the last store has read the staging tile
        __syncwarp();
#pragma unroll
        for (int sub = 0; sub < COLS; sub += 32) {
          uint32_t v[32];
          tmem_ld_32x32(tmem_base + acc * 256 + half * 128 + col + sub + (uint32_t(quarter * 32) << 16), v);
          tmem_ld_wait();
          const int n = n0 + col + sub;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            float4 sb = make_float4(0.f, 0.f, 0.f, 0.f), bias = sb;
            if (TMA_OUT) {  // N is a multiple of 16: four columns are inside or outside as a whole
              if (n + g * 4 < p.N) {
                sb = __ldg(reinterpret_cast<const float4*>(s.b + n + g * 4));
                if (s.bias) bias = __ldg(reinterpret_cast<const float4*>(s.bias + n + g * 4));
              }
            } else {
              float* sb_of = &sb.x;
              float* bias_of = &bias.x;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int at = min(n + g * 4 + e, p.N - 1);
                sb_of[e] = __ldg(s.b + at);
                if (s.bias) bias_of[e] = __ldg(s.bias + at);
              }
            }
            const float y0 = scaled(float(int(v[g * 4])), sa, sb.x, bias.x);
            const float y1 = scaled(float(int(v[g * 4 + 1])), sa, sb.y, bias.y);
            const float y2 = scaled(float(int(v[g * 4 + 2])), sa, sb.z, bias.z);
            const float y3 = scaled(float(int(v[g * 4 + 3])), sa, sb.w, bias.w);
            if constexpr (sizeof(Y) == 4) {
              sts128(my_row + ((g ^ (lane & 7)) << 4), y0, y1, y2, y3);
            } else {
              sts64(my_row + (((sub / 8 + g / 2) ^ (lane & 7)) << 4) + (g & 1) * 8, pack2<Y>(y0, y1), pack2<Y>(y2, y3));
            }
          }
        }
        if (TMA_OUT) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_y, stage_out, n0 + col, m0);  // rows and columns outside Y are dropped
            tma_store_commit();
          }
        } else {
          __syncwarp();
          const int rows = min(32, p.M - m0);
          for (int r = 0; r < rows; ++r) {
#pragma unroll
            for (int sub = 0; sub < COLS; sub += 32) {
              const int n = n0 + col + sub + lane, byte = (sub + lane) * int(sizeof(Y));
              const uint32_t at = smem_u32(stage_out) + r * 128 + (((byte / 16) ^ (r & 7)) << 4) + byte % 16;
              if (n < p.N) {
                if constexpr (sizeof(Y) == 4)
                  out[size_t(m0 + r) * p.N + n] = __uint_as_float(lds32(at));
                else
                  reinterpret_cast<unsigned short*>(out)[size_t(m0 + r) * p.N + n] = lds16(at);
              }
            }
          }
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
    if (TMA_OUT && lane == 0) tma_store_wait_all<0>();
  }

  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves (or frees TMEM) while its partner may still signal it
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ------------------------------------------------------------------- padding
// Copies of A and B whose rows start at 16-byte boundaries, in the caller's workspace: what the
// gathering kernel does per tile, once per call.  Rows of `width` bytes become rows of `pitch`
// (the next multiple of 16) bytes; the bytes between are arbitrary (tensor maps end at `width`).
// A lane makes sixteen bytes from the two granules that hold them; a warp takes 2 KiB of a row,
// four pieces at once, and a block eight rows.
struct Pad {
  const uint8_t* from;
  uint8_t* to;
  int rows, width, pitch;
  int parts() const { return (pitch + 2047) / 2048; }
};
constexpr int PAD_ROWS = 8, PAD_THREADS = PAD_ROWS * 32;
// The granule at `at`, of which bytes outside [begin, end) are not read and come back as 0.
__device__ __forceinline__ uint4 load_granule(uintptr_t at, uintptr_t begin, uintptr_t end) {
  if (at >= begin && at + 16 <= end) return __ldg(reinterpret_cast<const uint4*>(at));
  uint32_t w[4] = {};
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (at + e >= begin && at + e < end) w[e / 4] |= uint32_t(*reinterpret_cast<const uint8_t*>(at + e)) << (e % 4 * 8);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// blockIdx = (part of the row, rows, operand).
__global__ void __launch_bounds__(PAD_THREADS) pad_kernel(const Pad a, const Pad b) {
  grid_dependency_trigger();
  const Pad& p = blockIdx.z == 0 ? a : b;
  const int c0 = int(blockIdx.x) * 2048 + int(threadIdx.x % 32) * 16;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(p.from), end = begin + size_t(p.rows) * p.width;
  grid_dependency_wait();
  if (int(blockIdx.x) * 2048 >= p.pitch) return;
  for (long long row = (long long)blockIdx.y * PAD_ROWS + threadIdx.x / 32; row < p.rows;
       row += (long long)gridDim.y * PAD_ROWS) {
    const uintptr_t src = begin + size_t(row) * p.width + c0;
    const unsigned offset = unsigned(src & 15);
    uint4 lo[4], hi[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (c0 + u * 512 < p.pitch) {
        lo[u] = load_granule(floor16(src) + u * 512, begin, end);
        hi[u] = load_granule(floor16(src) + u * 512 + 16, begin, end);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (c0 + u * 512 < p.pitch) {
        uint32_t w[8] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w, hi[u].x, hi[u].y, hi[u].z, hi[u].w};
#pragma unroll
        for (int j = 0; j < 6; ++j) w[j] = offset & 8 ? w[j + 2] : w[j];
#pragma unroll
        for (int j = 0; j < 5; ++j) w[j] = offset & 4 ? w[j + 1] : w[j];
        const unsigned bits = (offset & 3) * 8;
        *reinterpret_cast<uint4*>(p.to + size_t(row) * p.pitch + c0 + u * 512) =
            make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                       __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
      }
    }
  }
}

// ------------------------------------------------------------------ dispatch
enum Path { PATH_AUTO = 0, PATH_GENERIC = 1, PATH_STREAM = 2, PATH_STREAM_GATHER = 3, PATH_PAIR = 4 };
inline std::atomic<int>& forced_path() {
  static std::atomic<int> path{0};
  return path;
}
inline std::atomic<int>& last_path() {
  static std::atomic<int> path{0};
  return path;
}

template <typename Y>
static bool launch_generic(const int8_t* A, const int8_t* B, Y* out, int M, int N, int K, const Scales& s,
                           cudaStream_t stream) {
  // gridDim.y is limited to 65535 tiles per launch
  constexpr int ROWS = 65535 * GT;
  for (int m0 = 0; m0 < M; m0 += ROWS) {
    const int rows = std::min(M - m0, ROWS);
    const dim3 grid(ceil_div(N, GT), ceil_div(rows, GT));
    const Scales part = {s.a + m0, s.b, s.bias};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(G_THREADS);
    cfg.stream = stream;
    // (the launch's own return code: the last error may be one of the caller's)
    if (cudaLaunchKernelEx(&cfg, generic_kernel<Y>, A + size_t(m0) * K, B, out + size_t(m0) * N, rows, N, K, part) !=
        cudaSuccess) {
      cudaGetLastError();
      return false;
    }
    ++launch_counter();
    if (m0 > M - ROWS) break;  // m0 + ROWS would pass the int range
  }
  last_path() = PATH_GENERIC;
  return true;
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
  std::atomic<bool> ready{false};
  int clusters[2][4][S_MAX_CLUSTER + 1] = {};  // [gather][R][c]
  int pairs = 0;
};
static DeviceSetup setups[MAX_DEVICES];
template <typename Y>
static void configure_kernels() {
  auto allow = [](auto* kernel, int smem_bytes) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes) != cudaSuccess)
      cudaGetLastError();
  };
  allow(stream_kernel<Y, false>, S_SMEM_LIMIT);
  allow(stream_kernel<Y, true>, S_SMEM_LIMIT);
  allow(pair_kernel<Y, true>, P_SMEM_BYTES);
  allow(pair_kernel<Y, false>, P_SMEM_BYTES);
}
static DeviceSetup& device_setup(DeviceCtx& ctx) {
  DeviceSetup& d = setups[ctx.device];
  if (d.ready) return d;
  std::lock_guard<std::mutex> lock(setup_mutex());
  if (!d.ready) {
    configure_kernels<__half>();
    configure_kernels<__nv_bfloat16>();
    configure_kernels<float>();
    for (int r = 0; r < 4; ++r) {
      for (int c = 1; c <= S_MAX_CLUSTER; ++c) {
        const int R = R_CHOICES[r];
        d.clusters[0][r][c] = max_clusters(stream_kernel<__half, false>, S_THREADS, s_smem_bytes(R, false), c);
        d.clusters[1][r][c] = max_clusters(stream_kernel<__half, true>, S_GATHER_THREADS, s_smem_bytes(R, true), c);
      }
    }
    d.pairs = max_clusters(pair_kernel<__half, true>, P_THREADS, P_SMEM_BYTES, 2);
    d.ready = true;
  }
  return d;
}

// The choice between the paths, and of R and c, is by estimated time in microseconds.  The constants
// are fits to measurements on B200 (kernels back to back, operands from HBM):
//   stream, per k block of 128: 0.42 + 0.0009 R, or its 32 KiB of B at 7.1 TB/s over all CTAs
//   gather, per k block: 1.4 up to R = 32, then 1.7 (64) and 2.6 (128): shared-memory bandwidth;
//     1.5 more per call
//   either, per round of tiles: 0.3 (c = 1) or 2.5, per call: 2.2 or 2 + 0.15 c, and 0.035 R for
//     the drain
//   pair, per k block 0.33 (0.42 once all SMs run: power), per call 7, per round of tiles 1
//   padding: 1.5 and twice the operand's bytes at 6 TB/s
// E.g. 512 x 512 x 1024: streaming at R = 16, 32, 128 6.5, 7.3, 12 us, pairs 10.7; 256 x 4096 x
// 4096: 15.7 against 19.6; 1024 x 4096 x 4096: 25 against 19.9.  Over 136 aligned sizes the choice costs 1%
// more than the best one, 18% at worst (202 x 176 x 11408: 14.3 for 12.1).
struct StreamPlan {
  int R = 0, cluster = 0, clusters = 0, m_tiles = 0, tiles = 0;
  double us = 1e30;
};
static StreamPlan plan_stream(const DeviceSetup& d, bool gather, int M, int N, int K) {
  StreamPlan best;
  const int num_kb = (K + S_BK - 1) / S_BK;
  for (int r = 0; r < 4; ++r) {
    const int R = R_CHOICES[r];
    const long long m_tiles = ceil_div(M, R), tiles = m_tiles * ceil_div(N, S_TILE_N);
    if (tiles > 0x3fffffff) continue;
    for (int c = 1; c <= S_MAX_CLUSTER && c <= num_kb; ++c) {
      const int held = d.clusters[gather][r][c];
      if (held <= 0) continue;
      const int clusters = int(std::min<long long>(tiles, held));
      const double rounds = double((tiles + clusters - 1) / clusters);
      const double block = gather ? (R <= 32 ? 1.4 : R == 64 ? 1.7 : 2.6)
                                  : std::max(0.42 + 0.0009 * R, 32768.0 * clusters * c / double(m_tiles) / 7.1e6);
      const double us = rounds * ((num_kb + c - 1) / c * block + (c > 1 ? 2.5 : 0.3)) + (c > 1 ? 2 + 0.15 * c : 2.2) +
                        0.035 * R + (gather ? 1.5 : 0);
      if (us < best.us) best = {R, c, clusters, int(m_tiles), int(tiles), us};
    }
    if (M <= R) break;  // a larger R only pads
  }
  return best;
}

struct Route {
  int path = PATH_GENERIC;
  bool pad_a = false, pad_b = false;
  StreamPlan stream;
  double us = 1e30;
};
static int padded(int width) { return (width + 15) & ~15; }
static long long pad_bytes(int M, int N, int K, bool a, bool b) {
  return (a ? (long long)M * padded(K) : 0) + (b ? (long long)K * padded(N) : 0);
}
// a_ok / b_ok: TMA can move the operand as it lies.
static Route choose_route(const DeviceSetup& d, int M, int N, int K, bool a_ok, bool b_ok, long long workspace,
                          int force) {
  Route best;
  if (K <= 0 || K >= (1 << 17) || force == PATH_GENERIC) return best;
  const long long pad = pad_bytes(M, N, K, !a_ok, !b_ok);
  if (pad <= workspace && force != PATH_STREAM_GATHER) {
    const double pad_us = pad ? 1.5 + 2.0 * double(pad) / 6e6 : 0;
    if (force != PATH_PAIR) {
      const StreamPlan plan = plan_stream(d, false, M, N, K);
      if (plan.cluster > 0) best = {PATH_STREAM, !a_ok, !b_ok, plan, plan.us + pad_us};
    }
    const long long tiles = (long long)ceil_div(M, 256) * ceil_div(N, 256);
    if (d.pairs > 0 && tiles <= 0x3fffffff && force != PATH_STREAM) {
      const double rounds = double((tiles + d.pairs - 1) / d.pairs);
      const double us = 7 + rounds * ((K + 127) / 128 * (rounds > 2 ? 0.42 : 0.33) + 1) + pad_us;
      if (us < best.us) best = {PATH_PAIR, !a_ok, !b_ok, StreamPlan(), us};
    }
  }
  if (force == PATH_STREAM_GATHER || (force == PATH_AUTO && pad > 0) || best.us > 1e29) {
    const StreamPlan plan = plan_stream(d, true, M, N, K);
    if (plan.cluster > 0 && plan.us < best.us) best = {PATH_STREAM_GATHER, false, false, plan, plan.us};
  }
  return best;
}

// An operand as a kernel gets it: its rows and how far they are apart.
struct Operand {
  const int8_t* p;
  int pitch;
};

template <typename Y, bool GATHER>
static bool launch_stream(DeviceCtx& ctx, const StreamPlan& plan, const Operand& A, const Operand& B, Y* out, int M,
                          int N, int K, const Scales& s, cudaStream_t stream) {
  CUtensorMap map_b = {}, map_a = {};
  if (!GATHER && (!make_tensor_map_2d(&map_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, B.p, K, N, B.pitch, S_BK, 128,
                                      CU_TENSOR_MAP_SWIZZLE_128B) ||
                  !make_tensor_map_2d(&map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, A.p, M, K, A.pitch, plan.R, S_BK,
                                      CU_TENSOR_MAP_SWIZZLE_128B)))
    return false;
  const StreamShape p = {M, N, K, plan.R, plan.cluster, plan.m_tiles, plan.tiles};
  return launch_on_stream(stream_kernel<Y, GATHER>, plan.clusters * plan.cluster,
                         GATHER ? S_GATHER_THREADS : S_THREADS, s_smem_bytes(plan.R, GATHER), plan.cluster, stream,
                         map_b, map_a, A.p, B.p, out, s, p, ctx.status);
}

template <typename Y>
static bool launch_pair(DeviceCtx& ctx, const DeviceSetup& d, const Operand& A, const Operand& B, Y* out, int M,
                        int N, int K, const Scales& s, cudaStream_t stream) {
  CUtensorMap map_a, map_b, map_y = {};
  constexpr CUtensorMapDataType TYPE = std::is_same<Y, float>::value    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : std::is_same<Y, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool tma_out = N % 16 == 0 && aligned(out) && aligned(s.b) && aligned(s.bias);
  if (!make_tensor_map_2d(&map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, A.p, M, K, A.pitch, 128, 128,
                          CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_2d(&map_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, B.p, K, N, B.pitch, 128, 128,
                          CU_TENSOR_MAP_SWIZZLE_128B) ||
      (tma_out && !make_tensor_map_2d(&map_y, TYPE, sizeof(Y), out, M, N, size_t(N) * sizeof(Y), 32, 128 / sizeof(Y),
                                      CU_TENSOR_MAP_SWIZZLE_128B)))
    return false;
  const PairShape p = {M, N, K, ceil_div(M, 256), ceil_div(N, 256), i8::raster_group_rows(K)};
  const int clusters = std::min(p.tiles_m * p.tiles_n, d.pairs);
  return tma_out ? launch_on_stream(pair_kernel<Y, true>, 2 * clusters, P_THREADS, P_SMEM_BYTES, 2, stream, map_a,
                                   map_b, map_y, out, s, p, ctx.status)
                 : launch_on_stream(pair_kernel<Y, false>, 2 * clusters, P_THREADS, P_SMEM_BYTES, 2, stream, map_a,
                                   map_b, map_y, out, s, p, ctx.status);
}

// Makes the padded copies in the workspace and points the operands at them.
static bool launch_pad(const Route& route, Operand& A, Operand& B, int M, int N, int K,
                       void* workspace, cudaStream_t stream) {
  uint8_t* to = static_cast<uint8_t*>(workspace);
  Pad pads[2] = {};
  int n = 0;
  if (route.pad_a) {
    pads[n++] = {reinterpret_cast<const uint8_t*>(A.p), to, M, K, padded(K)};
    A = {reinterpret_cast<int8_t*>(to), padded(K)};
    to += size_t(M) * padded(K);
  }
  if (route.pad_b) {
    pads[n++] = {reinterpret_cast<const uint8_t*>(B.p), to, K, N, padded(N)};
    B = {reinterpret_cast<int8_t*>(to), padded(N)};
  }
  const int rows = std::max(pads[0].rows, pads[1].rows);
  const dim3 grid(std::max(pads[0].parts(), pads[1].parts()), std::min(ceil_div(rows, PAD_ROWS), 65535), n);
  return launch_on_stream(pad_kernel, grid, PAD_THREADS, 0, 1, stream, pads[0], pads[1]);
}

static bool tma_can_move(const int8_t* p, int width) {
  return width % 16 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

template <typename Y>
static int solve(const int8_t* A, const int8_t* B, Y* out, int M, int N, int K, const Scales& s, void* workspace,
                 long long workspace_bytes, cudaStream_t stream) {
  int device;
  if ((!device_ctx_entry(device).ready || !setups[device].ready) && is_capturing(stream)) return -4;
  DeviceCtx& ctx = device_ctx();
  const DeviceSetup& d = device_setup(ctx);
  if (ctx.cc_major >= 10) {
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) workspace_bytes = 0;
    const Route route = choose_route(d, M, N, K, tma_can_move(A, K), tma_can_move(B, N), workspace_bytes, forced_path());
    Operand a = {A, K}, b = {B, N};
    if (route.path != PATH_GENERIC &&
        (!(route.pad_a || route.pad_b) || launch_pad(route, a, b, M, N, K, workspace, stream)) &&
        (route.path == PATH_PAIR     ? launch_pair(ctx, d, a, b, out, M, N, K, s, stream)
         : route.path == PATH_STREAM ? launch_stream<Y, false>(ctx, route.stream, a, b, out, M, N, K, s, stream)
                                     : launch_stream<Y, true>(ctx, route.stream, a, b, out, M, N, K, s, stream))) {
      last_path() = route.path;
      return 0;
    }
  }
  return launch_generic(A, B, out, M, N, K, s, stream) ? 0 : -3;
}

}  // namespace i8t
}  // namespace texo

extern "C" long long texo_mm_int8_per_token_workspace(const int8_t* A, const int8_t* B, int M, int N, int K) {
  using namespace texo;
  const bool a_ok = i8t::tma_can_move(A, K), b_ok = i8t::tma_can_move(B, N);
  int device;
  if (M <= 0 || N <= 0 || K <= 0 || M > i8t::MAX_SIZE || N > i8t::MAX_SIZE || (a_ok && b_ok) || !device_ctx_entry(device).ready || !i8t::setups[device].ready)
    return 0;
  const i8t::Route route =
      i8t::choose_route(i8t::setups[device], M, N, K, a_ok, b_ok, 0x7fffffffffffffffLL, i8t::forced_path());
  return i8t::pad_bytes(M, N, K, route.pad_a, route.pad_b);
}

extern "C" int texo_mm_int8_solve_per_token(const int8_t* A, const int8_t* B, void* Y, int M, int N, int K,
                                            const float* scale_A, const float* scale_B, const float* bias,
                                            int out_type, void* workspace, long long workspace_bytes, void* stream) {
  using namespace texo;
  if (M <= 0 || N <= 0 || K < 0 || !Y || !scale_A || !scale_B || (K > 0 && (!A || !B))) return -1;
  if (M > i8t::MAX_SIZE || N > i8t::MAX_SIZE || K > i8t::MAX_SIZE) return -2;
  const i8t::Scales s = {scale_A, scale_B, bias};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (out_type) {
    case row::TYPE_F16:
      return i8t::solve(A, B, static_cast<__half*>(Y), M, N, K, s, workspace, workspace_bytes, st);
    case row::TYPE_BF16:
      return i8t::solve(A, B, static_cast<__nv_bfloat16*>(Y), M, N, K, s, workspace, workspace_bytes, st);
    case row::TYPE_F32:
      return i8t::solve(A, B, static_cast<float*>(Y), M, N, K, s, workspace, workspace_bytes, st);
    default: return -1;
  }
}

extern "C" int texo_mm_int8_per_token_last_path(void) { return texo::i8t::last_path(); }
extern "C" void texo_mm_int8_per_token_force_path(int path) { texo::i8t::forced_path() = path; }
