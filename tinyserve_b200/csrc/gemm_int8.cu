// out[m, n] = (sum over k of x[m, k] * w[n, k]) * x_scales[m] * w_scales[n], x and w 8-bit integers: tcgen05.mma kind::i8, the
// sums exact in 32-bit integers in tensor memory (127 * 127 * K < 2^31 up to K = 133,143). Any M and N; K a multiple of 16 (the
// pitch of a TMA copy; rows of codes are padded to it), the tail of a block of 128 k is filled with zeros by the copy.
//
// Three forms. Up to 16 rows: mma.sync on 8-bit integers whose operands come straight from memory. Few rows: 128 rows of w are the
// A operand of tcgen05.mma and XN rows of x the B operand, K cut into the slices of a cluster. Both are bound by the stream of the
// weights. Many rows: pairs of CTAs, 256 x 256 tiles; bound by the tensor cores.
#define TS_PDL_CLASS PDL_SKINNY
#include <cooperative_groups.h>

#include "cache_map.cuh"
#include "int8.cuh"
#include "launch_list.cuh"
#include "tcgen05.cuh"

namespace ts {
namespace cg = cooperative_groups;

constexpr int GI_MOST_K = 131072;
constexpr int GI_BK = 128;          // 128 codes = 128 bytes = one swizzle row
constexpr int GI_BN = 128;          // rows of w that an instruction takes
constexpr int GI_MAX_SLICES = 8;

// Instruction descriptor: D = 32-bit integers, A = B = signed 8-bit, both K-major.
template <int M, int N>
constexpr uint32_t GI_IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}

// ---------------------------------------------------------------- up to 16 rows
// 16 rows of w a tile, K cut over KW of a CTA's eight warps (so 8 / KW tiles a CTA); the codes go from memory straight into the operands of mma.sync on 8-bit
// integers (w the M of it, rows of x the N, eight of them or sixteen). Which codes stand at which k is free as long as both
// operands agree, so a lane takes 16 neighbouring codes of a row. Bound by the stream of the weights: all that a warp takes of
// them in a pass is in flight at once, the first of it asked for in front of the wait, and tiles are so small that every SM has
// about as much to fetch. One row, 24,576 x 4,096: 18.1 us (5.6 TB/s), 20.2 us through the ring of the form below.
constexpr int SK_THREADS = 256, SK_WARPS = 8, SK_CHUNKS = 8;      // chunks of 64 k that a warp has in flight

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT, int KW, typename T>
__global__ void __launch_bounds__(SK_THREADS, 2) gemm_int8_skinny_kernel(const int8_t* __restrict__ x, const float* __restrict__ x_scales,
                                                                        const int8_t* __restrict__ w, const float* __restrict__ w_scales,
                                                                        T* __restrict__ out, int M, int N, int K) {
  __shared__ int sums[SK_WARPS][16 * 8 * NT];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = (blockIdx.x * (SK_WARPS / KW) + warp / KW) * 16;
  // The warp's stretch of K, in chunks of 64: 16 codes a lane.
  const int chunks = (K + 63) / 64, part = warp % KW, c0 = (int)((long long)chunks * part / KW), c1 = (int)((long long)chunks * (part + 1) / KW);
  const int8_t* w0 = w + (size_t)min(n0 + g, N - 1) * K + 16 * t;          // (rows beyond the last are computed and not stored)
  const int8_t* w1 = w + (size_t)min(n0 + 8 + g, N - 1) * K + 16 * t;
  int acc[NT][4] = {};
  const int4 none = make_int4(0, 0, 0, 0);
  int4 a0[SK_CHUNKS], a1[SK_CHUNKS];
  auto load_w = [&](int c) {
#pragma unroll
    for (int i = 0; i < SK_CHUNKS; ++i) {
      a0[i] = a1[i] = none;
      const int k = (c + i) * 64;
      if (c + i < c1 && k + 16 * t < K) {
        a0[i] = __ldcs(reinterpret_cast<const int4*>(w0 + k));
        a1[i] = __ldcs(reinterpret_cast<const int4*>(w1 + k));
      }
    }
  };
  load_w(c0);
  pdl_wait();
  for (int c = c0; c < c1; c += SK_CHUNKS) {
    if (c > c0) load_w(c);
#pragma unroll
    for (int i = 0; i < SK_CHUNKS; ++i) {
      const int k = (c + i) * 64 + 16 * t;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        int4 b = none;
        if (n * 8 + g < M && c + i < c1 && k < K) b = __ldg(reinterpret_cast<const int4*>(x + (size_t)(n * 8 + g) * K + k));
        mma_s8(acc[n], a0[i].x, a1[i].x, a0[i].y, a1[i].y, b.x, b.y);
        mma_s8(acc[n], a0[i].z, a1[i].z, a0[i].w, a1[i].w, b.z, b.w);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    // [row of x][row of w]
    int* s = sums[warp] + (n * 8 + 2 * t) * 16 + g;
    s[0] = acc[n][0];
    s[16] = acc[n][1];
    s[8] = acc[n][2];
    s[24] = acc[n][3];
  }
  __syncthreads();
  constexpr int TILE = 16 * 8 * NT;
  for (int i = threadIdx.x; i < SK_WARPS / KW * TILE; i += SK_THREADS) {
    const int tile = i / TILE, m = (i % TILE) >> 4, n = (blockIdx.x * (SK_WARPS / KW) + tile) * 16 + (i & 15);
    if (m < M && n < N) {
      int sum = 0;
#pragma unroll
      for (int v = 0; v < KW; ++v) sum += sums[tile * KW + v][i % TILE];
      out[(size_t)m * N + n] = from_float<T>((float)sum * (x_scales[m] * w_scales[n]));
    }
  }
}

// ---------------------------------------------------------------- few rows
// 128 rows of w fill the M of the instruction whatever the rows of x; TMA keeps a ring of blocks of 128 k in flight, the first
// weights asked for in front of the wait, and the slices of K add up through distributed shared memory, in their order. A CTA
// takes all of x for its tile, so an SM fetches w and its tiles' share of x: tiles of up to 256 rows, of the height that gives all
// SMs as much, with two accumulators. What an instruction reads behind a tile's rows is never looked at.
// Bound by the stream of the weights where they are many (64 rows, 49,152 x 4,096: 36.5 us, 5.5 TB/s; 24,576 x 4,096: 21.4 us,
// 4.7 TB/s), by the trip through the ring and the cluster where they are few (37 rows, 6,144 x 4,096: 8.9 us for 3.9 us of memory).
constexpr int FR_MAX_STAGES = 8;
// Shared memory of a ring: so much that two CTAs fit an SM, this kernel's or one of the next product's (whose first weights then
// come while this one ends; 4,096 x 4,096, 17 rows, one after the other: 6.8 us, with a ring that fills the SM 8.0); of tiles above 128
// rows, one for each SM, what one CTA can have (24,576 x 4,096, 64 rows: 24.6 / 21.0).
constexpr uint32_t FR_RING = 114176, FR_RING_ALONE = 200 * 1024;
constexpr uint32_t FR_ACC_BYTES = GI_BN * GI_BK;      // what one instruction reads of w, however many rows a tile has
// A tile of `cols` rows of w: up to 128, or up to 256 with two accumulators (and then twice the threads).
struct FewRows {
  int stages;
  uint32_t stage, smem;
  FewRows(int xn, int accs, int cols, long long ctas) {
    stage = (uint32_t)(cols + xn) * GI_BK;
    // the last stage's instructions read on behind its rows; the sums take the place of the ring
    for (stages = FR_MAX_STAGES; stages > 2; --stages)
      if (room(accs) <= (accs == 2 && ctas <= 148 ? FR_RING_ALONE : FR_RING)) break;
    smem = max(room(accs), (uint32_t)(GI_BN * (accs == 1 ? xn : 64) * 4)) + 1024;
  }
  uint32_t room(int accs) const { return (stages - 1) * stage + max(stage, accs * FR_ACC_BYTES); }
  static uint32_t max(uint32_t a, uint32_t b) { return a > b ? a : b; }
};

// COLS: the tile's rows of w where they are known here, and with them the stages, or 0 (6,144 x 4,096, 37 rows: 8.9 us, not known 9.6).
template <int XN> constexpr int FR_STAGES = FR_RING / ((GI_BN + XN) * GI_BK);
template <int XN, int ACCS, int COLS, typename T>
__global__ void __launch_bounds__(128 * ACCS) gemm_int8_rows_kernel(const __grid_constant__ CUtensorMap map_x,
                                                                    const __grid_constant__ CUtensorMap map_w,
                                                                    const float* __restrict__ x_scales, const float* __restrict__ w_scales,
                                                                    T* __restrict__ out, int all_rows, int N, int K, int given_cols, int given_stages,
                                                                    int* __restrict__ error_flag) {
  constexpr int THREADS = 128 * ACCS;
  const int cols = COLS > 0 ? COLS : given_cols, stages = COLS > 0 ? FR_STAGES<XN> : given_stages;
  constexpr uint32_t IDESC = GI_IDESC<GI_BN, XN>, TMEM_COLS = ACCS * (XN < 32 ? 32 : XN);      // (32 are read at a time)
  // Beside a CTA of the product that allocates in front of its wait (TMEM_WAITING_SMEM, 32 columns each, two to an SM at most) a
  // CTA of this kernel finds its columns, now or when the other one of its kind, which waits for nobody, is done (two accumulators
  // are not taken with slices); it takes no TMEM_ALONE_SMEM.
  static_assert(TMEM_COLS <= 512 - 2 * 32 && TMEM_WAITING_SMEM * 3 > 228 * 1024, "room for the columns beside CTAs that wait");
  extern __shared__ unsigned char smem_raw[];
  unsigned char* ring = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full_bar[FR_MAX_STAGES];
  __shared__ __align__(8) uint64_t empty_bar[FR_MAX_STAGES];
  __shared__ __align__(8) uint64_t acc_full;
  __shared__ uint32_t tmem_base_slot;
  __shared__ int failed;

  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slices = gridDim.y, slice = blockIdx.y, n0 = blockIdx.x * cols;
  const int m0 = blockIdx.z * XN, M = min(XN, all_rows - m0);
  const uint32_t w_bytes = (uint32_t)cols * GI_BK, stage = w_bytes + XN * GI_BK;
  out += (size_t)m0 * N;
  x_scales += m0;
  const int all_kb = (K + GI_BK - 1) / GI_BK;
  const int kb0 = (int)((long long)all_kb * slice / slices), num_kb = (int)((long long)all_kb * (slice + 1) / slices) - kb0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    mbar_init(&acc_full, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  if (warp == 0) {
    // ---------------- TMA producer (one lane)
    if (lane == 0 && !wait_test_unarmed()) {
      auto load_w = [&](int i, int s) {
        mbar_expect_tx(&full_bar[s], stage);
        tma_load_2d(ring + (size_t)s * stage, &map_w, &full_bar[s], (kb0 + i) * GI_BK, n0);
      };
      const int early = num_kb < stages ? num_kb : stages;
      for (int i = 0; i < early; ++i) load_w(i, i);       // weights: nothing before this kernel writes them
      pdl_wait();
      int i = 0, s = 0;
      uint32_t parity = 1;
      for (; i < num_kb; ++i) {
        if (i >= early) {
          if (!mbar_wait(&empty_bar[s], parity)) { *(volatile int*)&failed = 1; break; }
          load_w(i, s);
        }
        tma_load_2d(ring + (size_t)s * stage + w_bytes, &map_x, &full_bar[s], (kb0 + i) * GI_BK, m0);
        if (++s == stages) { s = 0; parity ^= 1; }
      }
      // after a failure: copies in flight may still land in this CTA's shared memory
      if (*(volatile int*)&failed)
        for (int j = i > stages ? i - stages : 0; j < i; ++j) mbar_wait(&full_bar[j % stages], (j / stages) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer (one lane)
    pdl_wait();
    tmem_alloc(&tmem_base_slot, TMEM_COLS);
    tc_fence_before();
    __syncwarp();
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t*)&tmem_base_slot;
    if (lane == 0) {
      bool ok = true;
      int s = 0;
      uint32_t parity = 0;
      for (int i = 0; i < num_kb && ok; ++i) {
        ok = mbar_wait(&full_bar[s], parity);
        if (!ok) {
          *(volatile int*)&failed = 1;
          // the copies of this turn of the ring may still be on their way, and their thread gone: stay for them, once more with the limit
          for (int j = i; j < num_kb && j < i + stages; ++j) mbar_wait(&full_bar[j % stages], (j / stages) & 1);
          break;
        }
        tc_fence_after();
        const uint32_t a_addr = smem_u32(ring + (size_t)s * stage);
        const uint64_t bdesc = sw128_desc(a_addr + w_bytes);
#pragma unroll
        for (int a = 0; a < ACCS; ++a) {
          const uint64_t adesc = sw128_desc(a_addr + a * FR_ACC_BYTES);
#pragma unroll
          for (int k = 0; k < GI_BK / 32; ++k) umma_i8(tmem + a * XN, adesc + 2 * k, bdesc + 2 * k, IDESC, (i | k) != 0);
        }
        umma_commit(&empty_bar[s]);
        if (++s == stages) { s = 0; parity ^= 1; }
      }
      if (ok) umma_commit(&acc_full);
    }
    __syncwarp();
  }

  // ---------------- epilogue, all warps: thread = row of the tile = column of the output
  pdl_wait();
  if (!mbar_wait(&acc_full, 0)) {
    if (lane == 0) atomicExch(error_flag, WAIT_FAILED_GEMM_TCGEN05);
  }
  tc_fence_after();
  __syncthreads();         // the ring is free: all its copies have arrived and all MMAs have read them
  const uint32_t tmem = tmem_base_slot;
  const uint32_t lane_tmem = tmem + ((uint32_t)(warp % 4 * 32) << 16) + (uint32_t)(warp / 4 * XN);
  if constexpr (ACCS == 2) {
    // 32 rows of the result at a time, as they will lie in memory
    T* rows = reinterpret_cast<T*>(ring);
    constexpr int V = Vec<T>::N;
    const bool whole = N % V == 0;
    const int live = min(cols, N - n0);
    const float ws = (int)threadIdx.x < live ? w_scales[n0 + threadIdx.x] : 0.f;
#pragma unroll 1
    for (int c = 0; c * 32 < M; ++c) {
      uint32_t v[32];
      tmem_ld_32(lane_tmem + (uint32_t)(c * 32), v);
      const int count = min(M - c * 32, XN < 32 ? XN : 32);
#pragma unroll
      for (int m = 0; m < (XN < 32 ? XN : 32); ++m)
        if (m < count) rows[m * 256 + threadIdx.x] = from_float<T>((float)(int)v[m] * (x_scales[c * 32 + m] * ws));
      __syncthreads();
      T* o = out + (size_t)(c * 32) * N + n0;
      if (whole) {
        const int per_row = (live + V - 1) / V;
        for (int i = threadIdx.x; i < count * per_row; i += THREADS) {
          const int m = i / per_row, n = (i - m * per_row) * V;
          Vec<T> x;
          x.load(rows + m * 256 + n);
          x.store(o + (size_t)m * N + n);
        }
      } else {
        for (int m = 0; m < count; ++m)
          if ((int)threadIdx.x < live) o[(size_t)m * N + threadIdx.x] = rows[m * 256 + threadIdx.x];
      }
      __syncthreads();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
  } else {
    int* sums = reinterpret_cast<int*>(ring);        // [row of x][row of the tile]
#pragma unroll 1
    for (int c = 0; c < (XN + 31) / 32; ++c) {
      if (c * 32 >= M) break;
      uint32_t v[32];
      tmem_ld_32(lane_tmem + (uint32_t)(c * 32), v);
#pragma unroll
      for (int m = 0; m < (XN < 32 ? XN : 32); ++m)
        if (c * 32 + m < M) sums[(c * 32 + m) * GI_BN + threadIdx.x] = (int)v[m];
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
    cg::cluster_group cluster = cg::this_cluster();
    if (slices > 1) cluster.sync();
    const int* of_slice[GI_MAX_SLICES];
#pragma unroll
    for (int q = 0; q < GI_MAX_SLICES; ++q) of_slice[q] = slices > 1 && q < slices ? cluster.map_shared_rank(sums, q) : sums;
    // four neighbouring columns a thread: a trip to another CTA's shared memory costs the same for one word or for four
    const int quads = cols / 4;
    const bool whole = N % 4 == 0;
#pragma unroll 2
    for (int idx = slice * THREADS + threadIdx.x; idx < quads * M; idx += slices * THREADS) {
      const int m = idx / quads, row = (idx - m * quads) * 4, n = n0 + row;
      int4 v[GI_MAX_SLICES];
#pragma unroll
      for (int q = 0; q < GI_MAX_SLICES; ++q)
        if (q < slices) v[q] = *reinterpret_cast<const int4*>(of_slice[q] + m * GI_BN + row);
      if (n >= N) continue;
      int s[4] = {0, 0, 0, 0};
#pragma unroll
      for (int q = 0; q < GI_MAX_SLICES; ++q)
        if (q < slices) { s[0] += v[q].x; s[1] += v[q].y; s[2] += v[q].z; s[3] += v[q].w; }
      const float xs = x_scales[m];
      T* o = out + (size_t)m * N + n;
      if (whole) {
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = (float)s[e] * (xs * w_scales[n + e]);
        Quad<T>::store(o, f);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < N) o[e] = from_float<T>((float)s[e] * (xs * w_scales[n + e]));
      }
    }
    if (slices > 1) cluster.sync();      // nobody leaves while its sums are still read
  }
}

// ---------------------------------------------------------------- many rows
constexpr int MR_THREADS = 192, MR_STAGES = 5, MR_BM = 128, MR_BN = 256;      // TMA warp, MMA warp, four epilogue warps
constexpr uint32_t MR_A_BYTES = MR_BM * GI_BK, MR_STAGE = 2 * MR_A_BYTES;       // per CTA: 128 rows of x, half of 256 rows of w
constexpr uint32_t MR_PIECE = 32 * 128;                                         // 32 rows of 128 bytes of the result
constexpr size_t MR_SMEM = (size_t)MR_STAGES * MR_STAGE + 8 * MR_PIECE + 1024;
static_assert(MR_SMEM >= TMEM_ALONE_SMEM, "no CTA that waits with tensor memory of its own fits beside one");

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(map), "r"(smem_u32(src)), "r"(x), "r"(y) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// One warp's 32 rows of an accumulator, 256 columns, scaled and stored. A row of the accumulator is a lane's, so that a store
// straight from the registers touches 32 lines of memory with 16 bytes each: 128 bytes of each row go through shared memory
// instead (two pieces in turn, swizzled as the copy expects them, so that eight lanes cover all banks) and out by TMA, which
// also leaves out what lies beyond M and N. `turn` counts a warp's pieces over all its tiles: a tile at the right edge may have an
// odd number of them, and the next tile's first piece is then the other one, not the one that may still be on its way out.
// Rows off the 16-byte grid are stored from there by the warp, an element a lane and a row after the other.
template <typename T>
__device__ __forceinline__ void drain_int8_tile(uint32_t tmem_acc, int row0, int M, int N, int n0, T* __restrict__ out, bool by_copy,
                                                const CUtensorMap* map_out, unsigned char* pieces, uint32_t& turn,
                                                const float* __restrict__ x_scales, const float* tile_scales) {
  constexpr int COLS = 128 / sizeof(T);      // of a piece
  const int lane = threadIdx.x & 31, row = row0 + lane;
  const float xs = row < M ? x_scales[row] : 0.f;
#pragma unroll 1
  for (int c = 0; c < MR_BN / COLS; ++c) {
    const int n = n0 + c * COLS;
    if (n >= N) return;
    uint32_t r[COLS];
#pragma unroll
    for (int j = 0; j < COLS; j += 32) tmem_ld_32_nowait(tmem_acc + (uint32_t)(c * COLS + j), r + j);
    unsigned char* piece = pieces + (turn++ & 1u) * MR_PIECE;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");      // the piece before the last has been read
    __syncwarp();
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < COLS; j += Vec<T>::N) {
      float f[Vec<T>::N];
#pragma unroll
      for (int e = 0; e < Vec<T>::N; e += 4) {
        const float4 ws = *reinterpret_cast<const float4*>(tile_scales + c * COLS + j + e);
        f[e] = (float)(int)r[j + e] * (xs * ws.x);
        f[e + 1] = (float)(int)r[j + e + 1] * (xs * ws.y);
        f[e + 2] = (float)(int)r[j + e + 2] * (xs * ws.z);
        f[e + 3] = (float)(int)r[j + e + 3] * (xs * ws.w);
      }
      Vec<T> v;
      v.pack(f);
      v.store(reinterpret_cast<T*>(piece + lane * 128 + (((j / Vec<T>::N) ^ (lane & 7)) << 4)));
    }
    if (by_copy) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tma_store_2d(map_out, piece, n, row0);
    } else {
      __syncwarp();
      // (eight rows' words are read before the first is stored; words of two elements where every row begins with one)
      const int rows = min(32, M - row0);
      if (sizeof(T) == 2 && N % 2 == 0) {
#pragma unroll 8
        for (int r = 0; r < rows; ++r)
          if (n + 2 * lane < N)
            *reinterpret_cast<uint32_t*>(out + (size_t)(row0 + r) * N + n + 2 * lane) =
                *reinterpret_cast<const uint32_t*>(piece + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
      } else {
#pragma unroll 8
        for (int r = 0; r < rows; ++r)
#pragma unroll
          for (int j = lane; j < COLS; j += 32)
            if (n + j < N)
              out[(size_t)(row0 + r) * N + n + j] =
                  *reinterpret_cast<const T*>(piece + r * 128 + (((j / Vec<T>::N) ^ (r & 7)) << 4) + (j % Vec<T>::N) * sizeof(T));
      }
      __syncwarp();
    }
  }
}

// Pairs of CTAs (clusters of two, cta_group::2), as the bf16 product by pairs: each CTA loads its 128 rows of x and its half of
// the tile's 256 rows of w; one thread of the even CTA issues the MMAs for both and commits to both CTAs' barriers; both CTAs'
// copies report to the even CTA's "full" barrier; each CTA drains its own tensor memory, two accumulators in turn. Bound by the
// tensor cores, then by the power cap: 2,048 x 24,576 x 4,096 in 136 us for one call (3.0 POP/s; with stores straight from the
// registers 176), 157 us when calls follow one another for long.
template <typename T>
__global__ void __launch_bounds__(MR_THREADS) gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap map_x,
                                                                    const __grid_constant__ CUtensorMap map_w,
                                                                    const __grid_constant__ CUtensorMap map_out, bool by_copy,
                                                                    const float* __restrict__ x_scales, const float* __restrict__ w_scales,
                                                                    T* __restrict__ out, int M, int N, int K, int* __restrict__ error_flag) {
  constexpr int PAIR_BM = 2 * MR_BM, STAGES = MR_STAGES;
  constexpr uint32_t IDESC = GI_IDESC<PAIR_BM, MR_BN>, TMEM_COLS = 2 * MR_BN;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full_bar[STAGES];      // used in the even CTA: the bytes of both CTAs' copies
  __shared__ __align__(8) uint64_t empty_bar[STAGES];     // in each CTA: the MMAs have read this stage
  __shared__ __align__(8) uint64_t acc_full[2];           // in each CTA: the accumulator is complete
  __shared__ __align__(8) uint64_t acc_empty[2];          // used in the even CTA: 2 x 4 epilogue warps are done with it
  __shared__ __align__(8) uint64_t peer_ready;            // used in the even CTA: the odd one has its tensor memory
  __shared__ __align__(16) float tile_scales[2][MR_BN];   // of the tile's rows of w, for the accumulator of the same number
  __shared__ uint32_t tmem_base_slot;
  __shared__ int failed;

  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_cta_rank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int tiles_m = (M + PAIR_BM - 1) / PAIR_BM, tiles_n = (N + MR_BN - 1) / MR_BN;
  const int num_tiles = tiles_m * tiles_n;
  const int num_kb = (K + GI_BK - 1) / GI_BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 8); }
    mbar_init(&peer_ready, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  cluster_sync_all();      // both CTAs' barriers exist before either uses the other's
  uint32_t tmem_base = 0;
  const uint32_t full0 = smem_of_cta(&full_bar[0], 0), acc_empty0 = smem_of_cta(&acc_empty[0], 0);

  if (warp == 0) {
    // ---------------- TMA producer (one lane in each CTA)
    if (lane == 0 && !wait_test_unarmed()) {
      auto load_w = [&](int s, int kb, int n0) {
        tma_load_2d_pair(tiles + (size_t)s * MR_STAGE + MR_A_BYTES, &map_w, full0 + 8u * s, kb * GI_BK, n0 + (int)rank * (MR_BN / 2));
      };
      // the weights do not depend on the kernel before this one
      int early = 0;
      if (pair < num_tiles) {
        const int n0 = (pair / tiles_m) * MR_BN;
        early = num_kb < STAGES ? num_kb : STAGES;
        for (int kb = 0; kb < early; ++kb) {
          if (leader) mbar_expect_tx(&full_bar[kb], 2 * MR_STAGE);
          load_w(kb, kb, n0);
        }
      }
      pdl_wait();
      int it = 0;
      for (int tile = pair; tile < num_tiles && !failed; tile += num_pairs) {
        const int m0 = (tile % tiles_m) * PAIR_BM + (int)rank * MR_BM, n0 = (tile / tiles_m) * MR_BN;
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int s = it % STAGES;
          if (it >= early) {
            if (!mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1)) { failed = 1; break; }
            if (leader) mbar_expect_tx(&full_bar[s], 2 * MR_STAGE);
            load_w(s, kb, n0);
          }
          tma_load_2d_pair(tiles + (size_t)s * MR_STAGE, &map_x, full0 + 8u * s, kb * GI_BK, m0);
        }
      }
      // the even CTA's last commits also arrive at this CTA's barriers: stay until they have
      for (int j = it > STAGES ? it - STAGES : 0; j < it && !failed; ++j)
        if (!mbar_wait(&empty_bar[j % STAGES], (j / STAGES) & 1)) failed = 1;
      // after a failure: copies in flight may still land in either CTA's shared memory (the even one's barriers count both's)
      if (failed && leader)
        for (int j = it > STAGES ? it - STAGES : 0; j < it; ++j) mbar_wait(&full_bar[j % STAGES], (j / STAGES) & 1);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (one lane of the even CTA)
    pdl_wait();
    tmem_alloc_pair(&tmem_base_slot, TMEM_COLS);
    tmem_meet<1, MR_THREADS - 32>();
    tmem_base = tmem_base_slot;
    if (lane == 0 && !leader) mbar_arrive_cluster(smem_of_cta(&peer_ready, 0));
    if (lane == 0 && leader) {
      int it = 0, t = 0;
      if (!mbar_wait(&peer_ready, 0)) failed = 1;
      for (int tile = pair; tile < num_tiles && !failed; tile += num_pairs, ++t) {
        const int b = t & 1;
        if (!mbar_wait(&acc_empty[b], ((t >> 1) & 1) ^ 1)) { failed = 1; break; }
        tc_fence_after();
        const uint32_t tmem_d = tmem_base + (uint32_t)(b * MR_BN);
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&full_bar[s], (it / STAGES) & 1)) { failed = 1; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(tiles + (size_t)s * MR_STAGE);
          const uint64_t adesc = sw128_desc(a_addr), bdesc = sw128_desc(a_addr + MR_A_BYTES);
#pragma unroll
          for (int k = 0; k < GI_BK / 32; ++k) umma_i8_pair(tmem_d, adesc + 2 * k, bdesc + 2 * k, IDESC, (kb | k) != 0);
          umma_commit_pair(&empty_bar[s]);
        }
        umma_commit_pair(&acc_full[b]);
      }
    }
  } else {
    // ---------------- epilogue: warps 2..5 of each CTA drain their own CTA's tensor memory
    pdl_wait();
    tmem_meet<1, MR_THREADS - 32>();
    tmem_base = tmem_base_slot;
    const int quad = warp & 3;
    unsigned char* pieces = tiles + (size_t)STAGES * MR_STAGE + quad * (2 * MR_PIECE);
    int t = 0;
    uint32_t turn = 0;
    for (int tile = pair; tile < num_tiles; tile += num_pairs, ++t) {
      const int b = t & 1;
      const int m0 = (tile % tiles_m) * PAIR_BM + (int)rank * MR_BM, n0 = (tile / tiles_m) * MR_BN;
      // (a warp that is still at the tile before reads the other of the two)
      for (int i = (int)threadIdx.x - 64; i < MR_BN; i += 128) tile_scales[b][i] = n0 + i < N ? w_scales[n0 + i] : 0.f;
      asm volatile("bar.sync 2, 128;" ::: "memory");
      if (!mbar_wait(&acc_full[b], (t >> 1) & 1) || failed) {
        if (lane == 0) atomicExch(error_flag, WAIT_FAILED_GEMM_TCGEN05);
        break;
      }
      tc_fence_after();
      drain_int8_tile<T>(tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * MR_BN), m0 + quad * 32, M, N, n0, out, by_copy, &map_out,
                         pieces, turn, x_scales, tile_scales[b]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty0 + 8u * b);
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  // neither CTA may leave, or free its tensor memory, while the other can still reach it
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) tmem_dealloc_pair(tmem_base, TMEM_COLS);
}

// ---------------------------------------------------------------- host side
// rows x K codes row-major; boxes of box_rows x 128, 128-byte swizzle, zero fill outside.
static bool int8_map(CUtensorMap* map, const void* base, int rows, int K, int box_rows, CUtensorMapL2promotion promotion) {
  DtEncodeFn fn = dt_encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)K};
  cuuint32_t box[2] = {(cuuint32_t)GI_BK, (cuuint32_t)box_rows};
  cuuint32_t elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The result, rows x N of T: boxes of 32 rows x 128 bytes, 128-byte swizzle.
template <typename T>
static bool out_map(CUtensorMap* map, void* base, int rows, int N) {
  DtEncodeFn fn = dt_encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)N * sizeof(T)};
  cuuint32_t box[2] = {(cuuint32_t)(128 / sizeof(T)), 32u};
  cuuint32_t elem[2] = {1, 1};
  return fn(map, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, base, dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KW, typename T>
static int launch_skinny_of(const int8_t* x, const float* xs, const int8_t* w, const float* ws, void* out, int M, int N, int K, cudaStream_t stream) {
  const dim3 grid((N + 16 * (SK_WARPS / KW) - 1) / (16 * (SK_WARPS / KW)));
  return M <= 8 ? launch(gemm_int8_skinny_kernel<1, KW, T>, grid, SK_THREADS, 0, stream, x, xs, w, ws, (T*)out, M, N, K)
                : launch(gemm_int8_skinny_kernel<2, KW, T>, grid, SK_THREADS, 0, stream, x, xs, w, ws, (T*)out, M, N, K);
}
template <typename T>
static int launch_skinny(const int8_t* x, const float* xs, const int8_t* w, const float* ws, void* out, int M, int N, int K, int warps,
                         cudaStream_t stream) {
  switch (warps) {
    case 1: return launch_skinny_of<1, T>(x, xs, w, ws, out, M, N, K, stream);
    case 2: return launch_skinny_of<2, T>(x, xs, w, ws, out, M, N, K, stream);
    case 4: return launch_skinny_of<4, T>(x, xs, w, ws, out, M, N, K, stream);
    case 8: return launch_skinny_of<8, T>(x, xs, w, ws, out, M, N, K, stream);
  }
  return TS_ERR_BAD_ARGUMENT;
}

template <int XN, int ACCS, int COLS, typename T>
static int launch_few(const void* x, const float* xs, const void* w, const float* ws, void* out, int M, int N, int K, int slices, int cols,
                      int* error_flag, cudaStream_t stream) {
  CUtensorMap mx, mw;
  if (!int8_map(&mx, x, M, K, XN, CU_TENSOR_MAP_L2_PROMOTION_L2_128B) || !int8_map(&mw, w, N, K, cols, CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
    return TS_ERR_UNSUPPORTED;
  const dim3 grid((N + cols - 1) / cols, slices, (M + XN - 1) / XN);
  if (grid.z > 65535) return TS_ERR_UNSUPPORTED;
  const FewRows f(XN, ACCS, cols, (long long)grid.x * grid.y * grid.z);
  auto kern = gemm_int8_rows_kernel<XN, ACCS, COLS, T>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)f.smem);
  if (e != cudaSuccess) return (int)e;
  if (slices == 1) return launch(kern, grid, 128 * ACCS, f.smem, stream, mx, mw, xs, ws, (T*)out, M, N, K, cols, f.stages, error_flag);
  return launch_cluster(kern, grid, 128 * ACCS, f.smem, stream, dim3(1, slices), mx, mw, xs, ws, (T*)out, M, N, K, cols, f.stages, error_flag);
}

template <typename T>
static int launch_many(const void* x, const float* xs, const void* w, const float* ws, void* out, int M, int N, int K, int* error_flag,
                       cudaStream_t stream) {
  CUtensorMap mx, mw, mo;
  if (!int8_map(&mx, x, M, K, MR_BM, CU_TENSOR_MAP_L2_PROMOTION_L2_128B) ||
      !int8_map(&mw, w, N, K, MR_BN / 2, CU_TENSOR_MAP_L2_PROMOTION_L2_128B))
    return TS_ERR_UNSUPPORTED;
  const bool by_copy = (size_t)N * sizeof(T) % 16 == 0;
  mo = mx;      // (unused where the result's rows are off the 16-byte grid)
  if (by_copy && !out_map<T>(&mo, out, M, N)) return TS_ERR_UNSUPPORTED;
  auto kern = gemm_int8_pair_kernel<T>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MR_SMEM);
  if (e != cudaSuccess) return (int)e;
  const long long num_tiles = (long long)((N + MR_BN - 1) / MR_BN) * ((M + 2 * MR_BM - 1) / (2 * MR_BM));
  if (num_tiles > 0x3fffffff) return TS_ERR_UNSUPPORTED;
  const int pairs = num_tiles < 74 ? (int)num_tiles : 74;      // one persistent CTA per SM, two SMs a pair
  return launch_cluster(kern, dim3(2 * pairs), dim3(MR_THREADS), MR_SMEM, stream, dim3(2, 1, 1), mx, mw, mo, by_copy, xs, ws, (T*)out, M, N, K, error_flag);
}

}  // namespace ts

using namespace ts;

// tile_rows: 0: up to 16 rows, K cut over `slices` (1, 2, 4 or 8) warps; 16, 32, 64 or 128 rows of x a tile with `cols` rows of w (a
// multiple of 8 up to 128) and K in 1 to 8 slices of a cluster, or up to 256 and one slice; or 256: pairs of CTAs.
extern "C" int ts_gemm_int8(const void* x, const float* x_scales, const void* w, const float* w_scales, void* out, int M, int N, int K,
                            int tile_rows, int slices, int cols, int dtype, int* error_flag, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K % 16 != 0 || K > GI_MOST_K || error_flag == nullptr) return TS_ERR_UNSUPPORTED;
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)out) & 15) return TS_ERR_UNSUPPORTED;
  const bool b = dtype == TS_DTYPE_BF16;
  if (tile_rows == 0) {
    if (M > 16) return TS_ERR_BAD_ARGUMENT;
    return b ? launch_skinny<bf16>((const int8_t*)x, x_scales, (const int8_t*)w, w_scales, out, M, N, K, slices, stream)
             : launch_skinny<float>((const int8_t*)x, x_scales, (const int8_t*)w, w_scales, out, M, N, K, slices, stream);
  }
  if (tile_rows == 256)
    return b ? launch_many<bf16>(x, x_scales, w, w_scales, out, M, N, K, error_flag, stream)
             : launch_many<float>(x, x_scales, w, w_scales, out, M, N, K, error_flag, stream);
  if (slices < 1 || slices > GI_MAX_SLICES || slices > (K + GI_BK - 1) / GI_BK) return TS_ERR_BAD_ARGUMENT;
  if (cols < 8 || cols % 8 != 0 || cols > (slices == 1 ? 2 : 1) * GI_BN) return TS_ERR_BAD_ARGUMENT;
#define TS_FEW_OF(XN_, ACCS_, COLS_)                                                                                       \
  (b ? launch_few<XN_, ACCS_, COLS_, bf16>(x, x_scales, w, w_scales, out, M, N, K, slices, cols, error_flag, stream)       \
     : launch_few<XN_, ACCS_, COLS_, float>(x, x_scales, w, w_scales, out, M, N, K, slices, cols, error_flag, stream))
#define TS_FEW(XN_) return cols == GI_BN ? TS_FEW_OF(XN_, 1, GI_BN) : cols < GI_BN ? TS_FEW_OF(XN_, 1, 0) : TS_FEW_OF(XN_, 2, 0)
  switch (tile_rows) {
    case 16: TS_FEW(16);
    case 32: TS_FEW(32);
    case 64: TS_FEW(64);
    case 128: TS_FEW(128);
  }
#undef TS_FEW
#undef TS_FEW_OF
  return TS_ERR_BAD_ARGUMENT;
}
TS_LIST_ENTRY(ts_gemm_int8);
