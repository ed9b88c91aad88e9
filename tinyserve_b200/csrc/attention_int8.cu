// Causal attention over pages of 8-bit keys and values with a scale for every page and key/value head (cache_int8.cu):
//   s_j = scale * ks(page of j) * (q . ck_j) for the positions j that the query sees,  p = softmax(s),
//   out = sum over j of p_j * vs(page of j) * cv_j,
// the softmax by its running maximum and sum in 32 bits. A request without keys gets zeros.
//
// For few queries a request: single tokens, or as many that the cost is still the stream of the codes. A CTA takes a request, a
// key/value head and a tile of rows (the query heads of the group, for one query after the other); its warps take tiles of
// keys in turn, each with a running maximum and sum of its own. A request's keys are cut over the CTAs of a cluster, which add
// up through distributed shared memory: no scratch, no counter, the same order every time.
#define TS_PDL_CLASS PDL_ATTENTION
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "int8.cuh"
#include "launch_list.cuh"

namespace ts {
namespace cg = cooperative_groups;

constexpr float AI_LOG2E = 1.4426950408889634f;
constexpr int AI_MAX_SPLITS = 16;        // a cluster beyond eight CTAs has to be asked for, and is had on this GPU

struct Int8Attention {
  const int8_t *k, *v;
  const float *ks, *vs;
  const int* tables;
  const int *cu, *lens, *seqs;      // seqs null: all requests in their order
  int table_width, heads, kv_heads, dim, page_size, window;
  float scale;
};

// Where there are more CTAs than run at once, the long requests are begun first, so that no CTA that takes long comes last: block
// z takes the request with z longer ones, which every CTA finds by counting (1.5 us). 64 requests of 60 to 4,000 keys, 32 / 8
// heads of 128: 74.4 us in their own order, 54.3 so. (Spread over the CTAs in equal stretches of all requests' keys instead, the
// parts joined by a second kernel: 93 us; every piece of a stretch fills its ring anew.)
constexpr int AI_RANKED_MOST = 128;       // requests: one a thread
constexpr int AI_AT_ONCE = 296;           // CTAs: two on each of 148 SMs
__device__ __forceinline__ int request_of_block(const Int8Attention& a) {
  __shared__ int lens[AI_RANKED_MOST], found;
  const int requests = gridDim.z, i = threadIdx.x;
  if (requests > AI_RANKED_MOST || gridDim.x > 1 || gridDim.y * requests <= AI_AT_ONCE || a.window > 0) return blockIdx.z;
  const int mine = i < requests ? a.lens[a.seqs ? a.seqs[i] : i] : 0;
  if (i < requests) lens[i] = mine;
  __syncthreads();
  int longer = 0;
  for (int j = 0; j < requests; ++j) longer += lens[j] > mine || (lens[j] == mine && j < i);
  if (i < requests && longer == (int)blockIdx.z) found = i;
  __syncthreads();
  return found;
}

// What a row tile of a request looks at: its rows and the positions [from, to) that any of them sees.
struct RowTile {
  int seq, kv_head, row0, rows, first_token, first_place, from, to;
  __device__ __forceinline__ bool load(const Int8Attention& a, int per_tile, int request) {
    const int group = a.heads / a.kv_heads;
    seq = a.seqs ? a.seqs[request] : request;
    kv_head = blockIdx.y % a.kv_heads;
    row0 = (blockIdx.y / a.kv_heads) * per_tile;
    first_token = a.cu[seq];
    const int queries = a.cu[seq + 1] - first_token;
    rows = min(per_tile, queries * group - row0);
    if (rows <= 0) return false;
    first_place = a.lens[seq] - queries;
    to = first_place + (row0 + rows - 1) / group + 1;
    from = a.window > 0 ? max(0, first_place + row0 / group - a.window + 1) : 0;
    return true;
  }
  // the place of a row's query, and the row of q and out that it is
  __device__ __forceinline__ int place(const Int8Attention& a, int r) const { return first_place + (row0 + r) / (a.heads / a.kv_heads); }
  __device__ __forceinline__ size_t head_row(const Int8Attention& a, int r) const {
    const int group = a.heads / a.kv_heads, i = (row0 + r) / group;
    return (size_t)(first_token + i) * a.heads + kv_head * group + (row0 + r - i * group);
  }
};

// Joins the warps of a CTA and the CTAs of a cluster: m, l [warp][R], o [warp][R][dim] in shared memory hold each warp's running
// maximum (base 2), sum and weighted values, those of one warp `per_warp` behind those of the one before.
template <typename T, int R, int WARPS>
__device__ __forceinline__ void join_parts(const Int8Attention& a, const RowTile& tile, float* m, float* l, float* o, int per_warp,
                                           T* __restrict__ out) {
  __shared__ float top[R], sum[R];
  const int dim = a.dim, threads = WARPS * 32;
  __syncthreads();
  if (threadIdx.x < R) {
    float t = -INFINITY, s = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) t = fmaxf(t, m[w * R + threadIdx.x]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float mw = m[w * R + threadIdx.x], f = mw == -INFINITY ? 0.f : exp2f(mw - t);
      m[w * R + threadIdx.x] = f;
      s += f * l[w * R + threadIdx.x];
    }
    top[threadIdx.x] = t;
    sum[threadIdx.x] = s;
  }
  __syncthreads();
  const int splits = gridDim.x;
  const int count = tile.rows * dim;
  for (int i = threadIdx.x; i < count; i += threads) {
    const int r = i / dim;
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) x += m[w * R + r] * o[w * per_warp + i];
    if (splits == 1) out[tile.head_row(a, r) * dim + (i - r * dim)] = from_float<T>(sum[r] == 0.f ? 0.f : x / sum[r]);
    else o[i] = x;
  }
  if (splits == 1) return;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int rank = blockIdx.x;
  for (int i = rank * threads + threadIdx.x; i < count; i += splits * threads) {
    const int r = i / dim;
    float t = -INFINITY, s = 0.f, x = 0.f;
    float of[AI_MAX_SPLITS];
#pragma unroll
    for (int q = 0; q < AI_MAX_SPLITS; ++q) {
      of[q] = q < splits ? cluster.map_shared_rank(top, q)[r] : -INFINITY;
      t = fmaxf(t, of[q]);
    }
#pragma unroll
    for (int q = 0; q < AI_MAX_SPLITS; ++q)
      if (q < splits) {
        const float f = of[q] == -INFINITY ? 0.f : exp2f(of[q] - t);
        s += f * cluster.map_shared_rank(sum, q)[r];
        x += f * cluster.map_shared_rank(o, q)[i];
      }
    out[tile.head_row(a, r) * dim + (i - r * dim)] = from_float<T>(s == 0.f ? 0.f : x / s);
  }
  cluster.sync();      // nobody leaves while its parts are still read
}

// ---------------------------------------------------------------- CUDA cores: any type, head size and page size
// A lane takes a key for the scores (its row of codes against the queries in shared memory, so no sum crosses lanes) and
// stretches of the head for the values (a row of codes is read by the warp together, the weights come by shuffle).
// VEC: codes a load of a row can take (16, 4 or 1, by the head size).
template <typename T, int VEC, int R>
__global__ void __launch_bounds__(128) attention_int8_simt_kernel(const T* __restrict__ q, T* __restrict__ out, const Int8Attention a) {
  constexpr int WARPS = 4, VV = VEC == 1 ? 1 : 4, CHUNKS = 8 / VV;
  extern __shared__ float smem[];
  float* qs = smem;                                  // [R][dim], scaled
  float* m_at = qs + R * a.dim;
  float* l_at = m_at + WARPS * R;
  float* o_at = l_at + WARPS * R;                    // [WARPS][R][dim]
  pdl_trigger();
  pdl_wait();
  RowTile tile;
  if (!tile.load(a, R, request_of_block(a))) return;                      // (the whole cluster: it shares the row tile)
  const int dim = a.dim, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < R * dim; i += 128) {
    const int r = i / dim;
    qs[i] = r < tile.rows ? to_float(q[tile.head_row(a, r) * dim + (i - r * dim)]) * (a.scale * AI_LOG2E) : 0.f;
  }
  __syncthreads();
  float m[R], l[R], o[R][8];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[r][e] = 0.f;
  }
  const int* table = a.tables + (size_t)tile.seq * a.table_width;
  const int stride = gridDim.x * WARPS * 32;
  for (int j0 = tile.from + (blockIdx.x * WARPS + warp) * 32; j0 < tile.to; j0 += stride) {
    const int j = j0 + lane;
    const bool there = j < tile.to;
    float ks = 0.f, vs = 0.f;
    size_t at = 0;
    if (there) {
      const int page = table[j / a.page_size];
      const size_t group = (size_t)page * a.kv_heads + tile.kv_head;
      ks = a.ks[group];
      vs = a.vs[group];
      at = (group * a.page_size + j % a.page_size) * dim;
    }
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = 0.f;
    if (there) {
      const int8_t* row = a.k + at;
      for (int d = 0; d < dim; d += VEC) {
        alignas(16) int8_t c[VEC];
        if constexpr (VEC == 16) *reinterpret_cast<int4*>(c) = *reinterpret_cast<const int4*>(row + d);
        else if constexpr (VEC == 4) *reinterpret_cast<int*>(c) = *reinterpret_cast<const int*>(row + d);
        else c[0] = row[d];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float f = (float)c[e];
#pragma unroll
          for (int r = 0; r < R; ++r) s[r] += f * qs[r * dim + d + e];
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int place = tile.place(a, r);
      const bool seen = there && j <= place && (a.window <= 0 || j > place - a.window);
      s[r] = seen ? s[r] * ks : -INFINITY;
      const float top = fmaxf(m[r], warp_max(s[r]));
      // (a row whose keys so far are all hidden keeps its sums of zero)
      const float shrink = top == -INFINITY ? 1.f : exp2f(m[r] - top);
      s[r] = seen ? exp2f(s[r] - top) : 0.f;
      m[r] = top;
      l[r] = l[r] * shrink + s[r];
      s[r] = seen ? s[r] * vs : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[r][e] *= shrink;
    }
    const int keys = min(32, tile.to - j0);
#pragma unroll 4
    for (int i = 0; i < keys; ++i) {
      const size_t from = __shfl_sync(0xffffffffu, (unsigned long long)at, i);
      float p[R];
#pragma unroll
      for (int r = 0; r < R; ++r) p[r] = __shfl_sync(0xffffffffu, s[r], i);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int d = (lane + 32 * c) * VV;
        if (d < dim) {
          alignas(4) int8_t code[VV];
          if constexpr (VV == 4) *reinterpret_cast<int*>(code) = *reinterpret_cast<const int*>(a.v + from + d);
          else code[0] = a.v[from + d];
#pragma unroll
          for (int e = 0; e < VV; ++e) {
            const float f = (float)code[e];
#pragma unroll
            for (int r = 0; r < R; ++r) o[r][c * VV + e] += p[r] * f;
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] = warp_sum(l[r]);
    if (lane == 0) {
      m_at[warp * R + r] = m[r];
      l_at[warp * R + r] = l[r];
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int e = 0; e < VV; ++e) {
        const int d = (lane + 32 * c) * VV + e;
        if (d < dim) o_at[(warp * R + r) * dim + d] = o[r][c * VV + e];
      }
  }
  join_parts<T, R, WARPS>(a, tile, m_at, l_at, o_at, R * dim, out);
}

// ---------------------------------------------------------------- tensor cores: heads of 64, 96 or 128, pages of 8 n
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// With its sign bit flipped a code is itself plus 128, and behind 0x64 that is the fp16 number 1,152 + code. Four codes as two
// pairs of such numbers, in three instructions:
constexpr float AI_OFFSET = 1152.f;
__device__ __forceinline__ void codes_with_offset(uint32_t w, uint32_t& low, uint32_t& high) {
  w ^= 0x80808080u;
  low = __byte_perm(w, 0x64646464u, 0x4140);
  high = __byte_perm(w, 0x64646464u, 0x4342);
}
__device__ __forceinline__ uint32_t without_offset(uint32_t t) {
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(t) : "r"(0x64806480u));                                       // 1,152 in both halves
  return t;
}
// Two codes, in the low byte of each half, as two fp16, exactly.
__device__ __forceinline__ uint32_t codes_to_f16(uint32_t t) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(t), "r"(0x00ff00ffu), "r"(0x64806480u));      // (t & mask) ^ bits
  return without_offset(r);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// A run of codes of a lane, from a row in shared memory whose 16-byte pieces lie swapped about (`turn`).
template <int BYTES>
__device__ __forceinline__ void take_codes(uint32_t (&w)[BYTES / 4], const unsigned char* row, int from, int turn) {
  constexpr int UNIT = BYTES % 16 == 0 ? 16 : BYTES % 8 == 0 ? 8 : 4;
#pragma unroll
  for (int i = 0; i < BYTES / UNIT; ++i) {
    const int at = from + i * UNIT;
    const unsigned char* p = row + (((at >> 4) ^ turn) << 4) + (at & 15);
    if constexpr (UNIT == 16) {
      const uint4 x = *reinterpret_cast<const uint4*>(p);
      w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
    } else if constexpr (UNIT == 8) {
      const uint2 x = *reinterpret_cast<const uint2*>(p);
      w[2 * i] = x.x; w[2 * i + 1] = x.y;
    } else {
      w[i] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
}

// A warp's step is 32 keys, four runs of eight that each lie inside a page. Keys are the M of the first product (S^T = K Q^T) and
// the head's elements the M of the second (O^T = V^T P^T), query rows are the N of both, eight of them, or sixteen (NT = 2): no
// work is done for rows of a group that are not there beyond the next eight. Which element of the head stands at which k of the
// first product, and at which row of the second, is free as long as both operands agree: a lane takes runs of D/4 codes of a
// key and D/8 codes of a value, in words. The codes come by asynchronous copies into a ring of the warp's own, two steps
// ahead, so that what is in flight hangs neither on registers nor on how the compiler orders loads (loads into
// registers a step ahead: 3.1 us a step of 32 keys, uncontended); the 16-byte pieces of a row are swapped about by the row's
// number, so that reads of eight lanes cover all banks.
//
// Bound by the stream of the codes, as long as little is done to them: with both products in bf16 (four instructions a pair of
// codes) a step was bound by the integer pipe. So both are in fp16, which holds a code exactly for less. In the first
// product the codes keep their offset of 1,152, which comes off the sums again (1,152 times the sum of the query row): what that
// costs is some 2^-20 of sum |q| |1,152 + k|, far below what a score of a bf16 query is good for. A query row is brought to
// fp16 by a power of two, its largest element between 2^14 and 2^15: exactly, but for elements below 2^-31 of that. (As integers in
// two digits, mma.sync on 8-bit integers, without any conversion of keys: a third slower, that instruction is.) The weights of the
// second product, p_j vs(page), are made as 2^(s_j + log2 vs - m) with the running maximum m of those sums: at most 2^8 (a
// maximum is only raised when a weight passes it by more than that), times 2^6, so that only weights below 2^-20 of the
// largest lose bits and only those below 2^-31 count for nothing. The scale of a page's values counts as 2^-80 where it is
// smaller: an error below 2^-73. The accumulator of S^T becomes the second operand of O^T by 8 x 8 transposes.
//
// Queries of 32 bits: their elements as the sum of three fp16 numbers (exactly, but for what lies below 2^-39 of the row's
// largest), the codes without their offset, the weights as the sum of two (22 bits): three products for one and two for one, eight
// rows a CTA at most.
constexpr float AI_FLOOR = -3e38f;            // the running maximum of nothing: finite, so that hidden places need no care, and below all scores
constexpr float AI_LIFT = 6.f;
template <int D> constexpr int AI_PITCH = D <= 64 ? 64 : 128;                   // of a row in the ring
constexpr int AI_STAGES = 3, AI_TILES = 2, AI_KEYS = 16 * AI_TILES;
template <int D> constexpr int AI_STEP = 2 * AI_KEYS * AI_PITCH<D>;             // the keys of a step and their values
template <int D, int WARPS> constexpr size_t AI_SMEM = WARPS * (size_t)AI_STAGES * AI_STEP<D>;
template <typename T, int D, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 4 ? 2 : 1) attention_int8_mma_kernel(const T* __restrict__ q, T* __restrict__ out,
                                                                   const Int8Attention a) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int QP = EXACT ? 3 : 1, PP = EXACT ? 2 : 1;            // fp16 parts of a query's element and of a weight
  constexpr int R = 8 * NT, KS = D / 16, MT = D / 16, VW = D / 32, PITCH = AI_PITCH<D>, STAGES = AI_STAGES;
  constexpr int U = AI_TILES, KEYS = AI_KEYS, RUNS = 2 * U, SPAN = 32 / RUNS;
  static_assert(R * D * 4 <= STAGES * AI_STEP<D>, "a warp's results take the place of its ring");
  static_assert(STAGES - 1 <= SPAN / 2, "the scales looked up ahead are taken over before the next ones are");
  extern __shared__ __align__(128) unsigned char ring_smem[];
  __shared__ float m_at[WARPS * R], l_at[WARPS * R];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  RowTile tile;
  if (!tile.load(a, R, request_of_block(a))) return;                      // (the whole cluster: it shares the row tile)
  unsigned char* ring = ring_smem + (size_t)warp * (STAGES * AI_STEP<D>);
  const int* table = a.tables + (size_t)tile.seq * a.table_width;
  const int start = tile.from & ~7, steps = (tile.to - start + KEYS - 1) / KEYS, stride = gridDim.x * WARPS;
  const int first = blockIdx.x * WARPS + warp, mine = first < steps ? (steps - first + stride - 1) / stride : 0;

  // Lane i keeps where run i & 3 of step i / 4 of the next 8 lies, and its scales; the 8 after those are looked up while these
  // are worked on.
  const float scale = a.scale * AI_LOG2E;
  int row = 0, next_row = 0;
  float ks = 0.f, lv = 0.f, next_ks = 0.f, next_lv = 0.f;
  auto look_up = [&](int k, int& at) {               // the page, as the row of codes that the run starts with
    const int pos = start + (first + (k + lane / RUNS) * stride) * KEYS + (lane % RUNS) * 8;
    at = pos < tile.to ? (table[pos / a.page_size] * a.kv_heads + tile.kv_head) * a.page_size + pos % a.page_size : -1;
  };
  auto scales_of = [&](int& at, float& k_scale, float& v_log) {
    k_scale = v_log = 0.f;
    if (at >= 0) {
      // A page whose values are no numbers (v - v is none) makes a NaN of every row that sees it by its scores, which are masked
      // where a row does not: a weight of NaN would also reach the others. (Both scales are asked for at once.)
      const float k = a.ks[at / a.page_size] * scale, v = a.vs[at / a.page_size];
      k_scale = k + (v - v);
      v_log = log2f(fminf(fmaxf(v, 8.271806e-25f), 3e38f));
    } else {
      at = 0;                                        // nothing of it is seen; the cache's first rows are there to be read
    }
  };
  auto turn_of = [](int r) { return PITCH == 128 ? r & 7 : (r >> 1) & 3; };
  // The 16-byte pieces of a step that this lane copies lie at the same places of every band of BAND rows.
  constexpr int PIECES = D / 16, BAND = PIECES == 6 ? 16 : 8, PLACES = BAND * PIECES / 32;
  int run_of[PLACES], from_off[PLACES], to_off[PLACES];
#pragma unroll
  for (int p = 0; p < PLACES; ++p) {
    const int piece = lane + 32 * p, r = piece / PIECES, c = piece - r * PIECES;
    run_of[p] = r >> 3;
    from_off[p] = (r & 7) * D + c * 16;
    to_off[p] = r * PITCH + ((c ^ turn_of(r)) << 4);
  }
  auto fetch = [&](int k) {                          // step k into the ring, or nothing behind the last
    if (k < mine) {
      if (k % SPAN == 0 && k > 0) row = next_row;
      if (k % SPAN == 1) look_up(k + SPAN - 1, next_row);
      if (k % SPAN == SPAN / 2) scales_of(next_row, next_ks, next_lv);
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring + (k % STAGES) * AI_STEP<D>);
#pragma unroll
      for (int j = 0; j < KEYS / BAND; ++j) {
        int r = 0;
#pragma unroll
        for (int p = 0; p < PLACES; ++p) {
          // (rows of 96 codes: a place's row lies in the first or the second run of the band)
          if (p == 0 || BAND > 8) r = __shfl_sync(0xffffffffu, row, k % SPAN * RUNS + j * (BAND / 8) + (BAND > 8 ? run_of[p] : 0));
          const int8_t* from_k = a.k + (size_t)(uint32_t)r * D + from_off[p];
          const int8_t* from_v = a.v + (size_t)(uint32_t)r * D + from_off[p];
          const uint32_t at = to + j * (BAND * PITCH) + to_off[p];
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from_k) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + KEYS * PITCH), "l"(from_v) : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (mine > 0) {
    look_up(0, row);
    scales_of(row, ks, lv);
  }
  for (int k = 0; k < STAGES - 1; ++k) fetch(k);

  uint32_t qf[QP][NT][KS][2];                        // the lane's elements of row g
  float unit[NT][2], offset[NT][2];                  // of the rows 2 t and 2 t + 1: what 1 stands for, what the codes' offset adds
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = n * 8 + g;
    uint32_t most = 0;
    float x[EXACT ? KS : 1][4];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const T* p = q + (r < tile.rows ? tile.head_row(a, r) * D : 0) + (D / 4) * t + 4 * k;
      if constexpr (EXACT) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] = 0.f;
        if (r < tile.rows) Quad<T>::load(p, x[k]);
#pragma unroll
        for (int e = 0; e < 4; ++e) most = max(most, magnitude_bits(x[k][e]));
      } else {
        uint2 y = make_uint2(0u, 0u);
        if (r < tile.rows) y = *reinterpret_cast<const uint2*>(p);
        most = max(max(most, max((y.x << 16) & 0x7fffffffu, y.x & 0x7fff0000u)), max((y.y << 16) & 0x7fffffffu, y.y & 0x7fff0000u));
        qf[0][n][k][0] = y.x;
        qf[0][n][k][1] = y.y;
      }
    }
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int e = min(max((int)(most >> 23), 32), 254);                        // biased; a row below 2^-95 is as good as zeros
    const float inverse = __uint_as_float((uint32_t)(254 + 14 - e) << 23);
    const float one = most >= INT8_INF_BITS ? __uint_as_float(INT8_NAN_BITS) : __uint_as_float((uint32_t)(e - 14) << 23);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float lo, hi;
        if constexpr (EXACT) {
          lo = x[k][2 * i] * inverse;
          hi = x[k][2 * i + 1] * inverse;
        } else {
          lo = __uint_as_float(qf[0][n][k][i] << 16) * inverse;
          hi = __uint_as_float(qf[0][n][k][i] & 0xffff0000u) * inverse;
        }
#pragma unroll
        for (int p = 0; p < QP; ++p) {
          qf[p][n][k][i] = pack_f16(lo, hi);
          const __half2 held = *reinterpret_cast<const __half2*>(&qf[p][n][k][i]);
          if constexpr (EXACT) {
            lo -= __low2float(held);
            hi -= __high2float(held);
          } else {
            sum += __low2float(held) + __high2float(held);
          }
        }
      }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    sum *= AI_OFFSET;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      unit[n][i] = __shfl_sync(0xffffffffu, one, 8 * t + 4 * i);
      offset[n][i] = __shfl_sync(0xffffffffu, sum, 8 * t + 4 * i);
    }
  }
  float m[NT][2], l[NT][2], o[NT][MT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = AI_FLOOR;
    l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
  }
  // Positions below `inner_to` and from `inner_from` on are seen by every row of the tile.
  const int inner_to = tile.place(a, 0) + 1;
  const int inner_from = a.window > 0 ? tile.place(a, tile.rows - 1) - a.window + 1 : 0;

  for (int k = 0; k < mine; ++k) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();                                    // every lane's copies of this step are there, all have left the last one
    if (k % SPAN == 0 && k > 0) { ks = next_ks; lv = next_lv; }
    fetch(k + STAGES - 1);
    const unsigned char* keys = ring + (k % STAGES) * AI_STEP<D>;
    float raw[U][NT][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        raw[u][n][0] = raw[u][n][2] = -offset[n][0];
        raw[u][n][1] = raw[u][n][3] = -offset[n][1];
      }
      uint32_t kc[2][KS];
      take_codes<D / 4>(kc[0], keys + (16 * u + g) * PITCH, (D / 4) * t, turn_of(g));
      take_codes<D / 4>(kc[1], keys + (16 * u + 8 + g) * PITCH, (D / 4) * t, turn_of(8 + g));
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        uint32_t af[4];
        codes_with_offset(kc[0][i], af[0], af[2]);
        codes_with_offset(kc[1][i], af[1], af[3]);
        if constexpr (EXACT) {
#pragma unroll
          for (int e = 0; e < 4; ++e) af[e] = without_offset(af[e]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int p = QP - 1; p >= 0; --p) mma_f16(raw[u][n], af, qf[p][n][i]);
      }
    }
    float fks[RUNS], flv[RUNS];
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      fks[i] = __shfl_sync(0xffffffffu, ks, k % SPAN * RUNS + i);
      flv[i] = __shfl_sync(0xffffffffu, lv, k % SPAN * RUNS + i);
    }
    const int pos = start + (first + k * stride) * KEYS;
    const bool inner = pos >= inner_from && pos + KEYS <= inner_to;
    uint32_t pf[PP][U][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float s[U][4];
      float top[2] = {AI_FLOOR, AI_FLOOR};
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[u][e] = raw[u][n][e] * (fks[2 * u + e / 2] * unit[n][e & 1]);
          if (!inner) {
            const int at = pos + 16 * u + 8 * (e / 2) + g, place = tile.place(a, n * 8 + 2 * t + (e & 1));
            if (at > place || (a.window > 0 && at <= place - a.window)) s[u][e] = -INFINITY;
          }
          top[e & 1] = fmaxf(top[e & 1], s[u][e] + flv[2 * u + e / 2]);
        }
      if (__any_sync(0xffffffffu, top[0] > m[n][0] + 8.f || top[1] > m[n][1] + 8.f)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(top[e], m[n][e]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float shrink = exp2_approx(m[n][e] - x);
          m[n][e] = x;
          l[n][e] *= shrink;
#pragma unroll
          for (int i = 0; i < MT; ++i) { o[n][i][e] *= shrink; o[n][i][e + 2] *= shrink; }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[u][e] - m[n][e & 1];
          l[n][e & 1] += exp2_approx(x);
          w[e] = exp2_approx(x + (flv[2 * u + e / 2] + AI_LIFT));
        }
#pragma unroll
        for (int p = 0; p < PP; ++p)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t part = pack_f16(w[2 * i], w[2 * i + 1]);
            if constexpr (EXACT) {
              w[2 * i] -= __low2float(*reinterpret_cast<const __half2*>(&part));
              w[2 * i + 1] -= __high2float(*reinterpret_cast<const __half2*>(&part));
            }
            pf[p][u][n][i] = transpose_8x8(part);
          }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t vc[4][VW];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * u + 2 * t + (i & 1) + 8 * (i >> 1);
        take_codes<D / 8>(vc[i], keys + (KEYS + r) * PITCH, (D / 8) * g, turn_of(r));
      }
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // the elements 4 w + 2 h and the one after it of this lane's run
          const uint32_t even = h == 0 ? 0x0400 : 0x0602, odd = h == 0 ? 0x0501 : 0x0703;
          const uint32_t af[4] = {codes_to_f16(__byte_perm(vc[0][w], vc[1][w], even)), codes_to_f16(__byte_perm(vc[0][w], vc[1][w], odd)),
                                  codes_to_f16(__byte_perm(vc[2][w], vc[3][w], even)), codes_to_f16(__byte_perm(vc[2][w], vc[3][w], odd))};
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int p = PP - 1; p >= 0; --p) mma_f16(o[n][2 * w + h], af, pf[p][u][n]);
        }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();
  float* o_at = reinterpret_cast<float*>(ring);      // [R][D]
  const float drop = exp2f(-AI_LIFT);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[n][e];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const int r = n * 8 + 2 * t + e;
      if (g == 0) { m_at[warp * R + r] = m[n][e]; l_at[warp * R + r] = sum; }
#pragma unroll
      for (int i = 0; i < MT; ++i)
        *reinterpret_cast<float2*>(o_at + r * D + (D / 8) * g + 2 * i) = make_float2(o[n][i][e] * drop, o[n][i][e + 2] * drop);
    }
  join_parts<T, R, WARPS>(a, tile, m_at, l_at, reinterpret_cast<float*>(ring_smem), STAGES * AI_STEP<D> / 4, out);
}

template <typename K, typename T>
static int launch_split(K kern, dim3 grid, int threads, size_t smem, cudaStream_t stream, const void* q, void* out, const Int8Attention& a) {
  if (grid.x > 8) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return (int)e;
  }
  if (grid.x == 1) return launch(kern, grid, threads, smem, stream, (const T*)q, (T*)out, a);
  return launch_cluster(kern, grid, threads, smem, stream, dim3(grid.x), (const T*)q, (T*)out, a);
}

template <typename T, int VEC, int R>
static int launch_simt(dim3 grid, cudaStream_t stream, const void* q, void* out, const Int8Attention& a) {
  auto kern = attention_int8_simt_kernel<T, VEC, R>;
  const size_t smem = (size_t)(R * a.dim + 2 * 4 * R + 4 * R * a.dim) * sizeof(float);
  return launch_split<decltype(kern), T>(kern, grid, 128, smem, stream, q, out, a);
}
template <typename T>
static int launch_simt_of(int per_tile, dim3 grid, cudaStream_t stream, const void* q, void* out, const Int8Attention& a) {
  const int vec = a.dim % 16 == 0 ? 16 : a.dim % 4 == 0 ? 4 : 1;
#define TS_SIMT(R_)                                                                                                               \
  return vec == 16 ? launch_simt<T, 16, R_>(grid, stream, q, out, a) : vec == 4 ? launch_simt<T, 4, R_>(grid, stream, q, out, a)   \
                                                                                : launch_simt<T, 1, R_>(grid, stream, q, out, a)
  if (per_tile == 2) TS_SIMT(2);
  if (per_tile == 4) TS_SIMT(4);
  TS_SIMT(8);
#undef TS_SIMT
}
template <typename T, int D, int NT, int WARPS>
static int launch_mma(dim3 grid, cudaStream_t stream, const void* q, void* out, const Int8Attention& a) {
  auto kern = attention_int8_mma_kernel<T, D, NT, WARPS>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)AI_SMEM<D, WARPS>);
  if (e != cudaSuccess) return (int)e;
  return launch_split<decltype(kern), T>(kern, grid, WARPS * 32, AI_SMEM<D, WARPS>, stream, q, out, a);
}
template <int D>
static int launch_mma_of(bool bf, int per_tile, int warps, dim3 grid, cudaStream_t stream, const void* q, void* out, const Int8Attention& a) {
  if (!bf) return warps == 8 ? launch_mma<float, D, 1, 8>(grid, stream, q, out, a) : launch_mma<float, D, 1, 4>(grid, stream, q, out, a);
  if (warps == 8) return per_tile == 8 ? launch_mma<bf16, D, 1, 8>(grid, stream, q, out, a) : launch_mma<bf16, D, 2, 8>(grid, stream, q, out, a);
  return per_tile == 8 ? launch_mma<bf16, D, 1, 4>(grid, stream, q, out, a) : launch_mma<bf16, D, 2, 4>(grid, stream, q, out, a);
}

}  // namespace ts

using namespace ts;

// q and out [tokens, heads, dim] dt; seqs lists the requests that are worked on, max_query_len their most tokens; a request's keys
// are cut over `splits` (1 to 16) CTAs, of four warps or (on the tensor cores) eight.
extern "C" int ts_attention_int8(const void* q, void* out, const int8_t* k_cache, const int8_t* v_cache, const float* k_scales,
                                 const float* v_scales, const int* tables, int table_width, const int* cu_query_lens,
                                 const int* context_lens, const int* seqs, int num_seqs, int max_query_len, int heads, int kv_heads, int dim,
                                 int page_size, int num_pages, float scale, int window, int tile_rows, int splits, int warps,
                                 int dtype, cudaStream_t stream) {
  if (num_seqs <= 0 || max_query_len <= 0) return 0;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || page_size <= 0 || window < 0 || splits < 1 || splits > AI_MAX_SPLITS ||
      (warps != 4 && warps != 8))
    return TS_ERR_BAD_ARGUMENT;
  if (dim <= 0 || dim > 256 || num_seqs > 65535) return TS_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return TS_ERR_UNSUPPORTED;
  const Int8Attention a = {k_cache, v_cache, k_scales, v_scales, tables, cu_query_lens, context_lens, seqs, table_width, heads, kv_heads,
                           dim, page_size, window, scale};
  const int rows = heads / kv_heads * max_query_len;
  const bool bf = dtype == TS_DTYPE_BF16;
  // (rows of codes are counted in 32 bits there)
  const bool mma = (dim == 64 || dim == 96 || dim == 128) && page_size % 8 == 0 &&
                   (long long)num_pages * kv_heads * page_size < 0x7fffffffll;
  const int per_tile = mma ? (bf && tile_rows == 16 ? 16 : 8) : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
  const long long row_tiles = (rows + per_tile - 1) / per_tile;
  if (row_tiles * kv_heads > 65535) return TS_ERR_UNSUPPORTED;
  const dim3 grid(splits, (unsigned)(row_tiles * kv_heads), num_seqs);
  if (mma) {
    if (dim == 64) return launch_mma_of<64>(bf, per_tile, warps, grid, stream, q, out, a);
    if (dim == 96) return launch_mma_of<96>(bf, per_tile, warps, grid, stream, q, out, a);
    return launch_mma_of<128>(bf, per_tile, warps, grid, stream, q, out, a);
  }
  return bf ? launch_simt_of<bf16>(per_tile, grid, stream, q, out, a) : launch_simt_of<float>(per_tile, grid, stream, q, out, a);
}
TS_LIST_ENTRY(ts_attention_int8);

// How many clusters of `size` CTAs of eight warps the GPU runs at once: a cluster lies within one of its parts, whose sizes differ.
extern "C" int ts_attention_int8_clusters(int size) {
  auto kern = attention_int8_mma_kernel<bf16, 128, 1, 8>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)AI_SMEM<128, 8>);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  cudaLaunchAttribute shape[1];
  shape[0].id = cudaLaunchAttributeClusterDimension;
  shape[0].val.clusterDim = {(unsigned)size, 1, 1};
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(size);
  config.blockDim = dim3(256);
  config.dynamicSmemBytes = AI_SMEM<128, 8>;
  config.attrs = shape;
  config.numAttrs = 1;
  int clusters = 0;
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&clusters, kern, &config);
  return e == cudaSuccess ? clusters : -(int)e;
}
