// Keys and values of a paged cache as 8-bit integers, a scale for every page and key/value head (int8.cuh): the write of a
// step's new tokens, and pages read back as values for the attention of long portions. Codes [pages, kv_heads, page_size,
// head_dim], scales [pages, kv_heads].
//
// A page is filled over several steps. When a request's new tokens go on inside a page that holds earlier ones, the page's
// scale grows to what they need, s' = max(s, max|new| / 127), and where it grew the codes that are there are rounded once more,
// to rint(c s / s'): at most half a step of the new scale each time. A page that starts with a new token starts with that
// token's scale. Codes behind a request's last token are left as they are.
#define TS_PDL_CLASS PDL_SKINNY      // they stand between the products of that class
#include "int8.cuh"
#include "launch_list.cuh"

namespace ts {

// One CTA for each (page that gets tokens, key/value head, keys or values). A page belongs to one request of a step, so it is the only
// one that touches them, and there are no atomics and no order to depend on. (The exception is the page of the rows that fill up a
// recorded step: their CTAs write over one another there, and what they leave is read by those rows alone, whose results nobody
// reads. Each is a request of one token, so none reads a code or a scale that another writes.) A thread takes VEC neighbouring
// elements of a row at a time (the new rows are read twice, the second time from L1). Bound by latency: the lengths, the table, the
// rows and the old scale, then the codes; a token each for 64 requests with 8 heads of 128 takes 3.0 us, three portions of 683 tokens
// 7.4 us with their rows in L2 and 9.8 from memory (12.7 MB).
template <typename T, int VEC>
__global__ void __launch_bounds__(128) kv_write_int8_kernel(const T* __restrict__ k, const T* __restrict__ v, int8_t* __restrict__ k_cache,
                                                            int8_t* __restrict__ v_cache, float* __restrict__ k_scales,
                                                            float* __restrict__ v_scales, const int* __restrict__ tables, int table_width,
                                                            const int* __restrict__ cu_query_lens, const int* __restrict__ context_lens,
                                                            int kv_heads, int dim, int page_size, int num_pages) {
  __shared__ uint32_t most[4];
  pdl_trigger();
  pdl_wait();
  const int seq = blockIdx.z, head = blockIdx.y >> 1;
  const bool values = blockIdx.y & 1;
  const int first_row = cu_query_lens[seq], new_tokens = cu_query_lens[seq + 1] - first_row, end = context_lens[seq];
  const int first = end - new_tokens;                                  // position of the first new token
  if (new_tokens <= 0 || first < 0) return;
  const int block = first / page_size + blockIdx.x, begin = block * page_size;
  if (begin >= end || block >= table_width) return;
  const int page = tables[(size_t)seq * table_width + block];
  if ((unsigned)page >= (unsigned)num_pages) return;
  const int held = max(first - begin, 0), upto = min(end - begin, page_size);      // offsets [held, upto) are new
  const size_t group = (size_t)page * kv_heads + head;
  int8_t* codes = (values ? v_cache : k_cache) + group * page_size * dim;
  float* scale_at = (values ? v_scales : k_scales) + group;
  const T* rows = (values ? v : k) + ((size_t)(first_row + begin + held - first) * kv_heads + head) * dim;
  const size_t pitch = (size_t)kv_heads * dim;
  const int per_row = dim / VEC, count = (upto - held) * per_row;
  auto load = [&](int i, float* f) {
    const int r = i / per_row;
    const T* p = rows + r * pitch + (i - r * per_row) * VEC;
    if constexpr (VEC == 4) Quad<T>::load(p, f);
    else f[0] = to_float(p[0]);
  };
  const float before = held > 0 ? *scale_at : 0.f;
  uint32_t m = 0;
  for (int i = threadIdx.x; i < count; i += 128) {
    float f[VEC];
    load(i, f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) m = max(m, magnitude_bits(f[e]));
  }
  m = warp_max_bits(m);
  if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = m;
  __syncthreads();                                                     // also: every thread has read the old scale
  m = max(max(most[0], most[1]), max(most[2], most[3]));
  const float need = int8_scale(m);
  const bool lost = !(need < INFINITY) || !(before < INFINITY);        // an infinity or a NaN, now or earlier
  const float scale = lost ? __uint_as_float(INT8_NAN_BITS) : fmaxf(before, need);
  const float inverse = lost || scale == 0.f ? 0.f : 1.f / scale;
  // The quotient by the scale, rounded once: half of the largest of values with 8-bit mantissas is 63.5 steps, and products with the
  // rounded reciprocal alone fall to its other side more often. One correction by the remainder, which fma leaves whole (Markstein,
  // IBM J. Res. Dev. 34, 1990); portions of 3 x 683 tokens, the product alone / so / divided: 6.8 / 7.4 / 8.7 us. (A NaN becomes
  // the code 0.)
  auto code_of = [&](float v) {
    const float q = v * inverse;
    return (int8_t)__float2int_rn(fmaf(fmaf(-q, scale, v), inverse, q));
  };
  if (threadIdx.x == 0) *scale_at = scale;
  if (lost || scale > before) {
    for (int i = threadIdx.x * VEC; i < held * dim; i += 128 * VEC) {
      alignas(4) int8_t c[VEC];
      if constexpr (VEC == 4) *reinterpret_cast<int*>(c) = *reinterpret_cast<const int*>(codes + i);
      else c[0] = codes[i];
#pragma unroll
      for (int e = 0; e < VEC; ++e) c[e] = lost ? (int8_t)0 : code_of((float)c[e] * before);
      if constexpr (VEC == 4) *reinterpret_cast<int*>(codes + i) = *reinterpret_cast<const int*>(c);
      else codes[i] = c[0];
    }
  }
  for (int i = threadIdx.x; i < count; i += 128) {
    float f[VEC];
    load(i, f);
    alignas(4) int8_t c[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) c[e] = code_of(f[e]);
    if constexpr (VEC == 4) *reinterpret_cast<int*>(codes + held * dim + i * 4) = *reinterpret_cast<const int*>(c);
    else codes[held * dim + i] = c[0];
  }
}

// The pages that the prompt portions of a step look at, as values: request after request in k_out and v_out [out_pages, kv_heads,
// page_size, dim], with block tables [seqs, out_width] for them. A portion's attention is bound by arithmetic and looks at a page
// once for every tile of its queries, so the codes are turned into values once, in front of it. A CTA takes the keys or the
// values of a page. Of a page and head whose values are no numbers the keys become NaN and the values zeros: the queries that see
// it get NaN by their scores, and the others, whose scores there are masked, do not meet a NaN times their weight of 0.
// Two contexts of 2,500 to 4,100 keys, 8 heads of 128: 10.5 us for 46 MB, in front of 130 us of attention.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) kv_values_kernel(const int8_t* __restrict__ k_cache, const int8_t* __restrict__ v_cache,
                                                        const float* __restrict__ k_scales, const float* __restrict__ v_scales,
                                                        const int* __restrict__ tables, int table_width,
                                                        const int* __restrict__ cu_query_lens, const int* __restrict__ context_lens,
                                                        T* __restrict__ k_out, T* __restrict__ v_out, int* __restrict__ out_tables,
                                                        int out_width, int out_pages, int kv_heads, int dim, int page_size, int num_pages,
                                                        int window) {
  __shared__ int parts[8];
  pdl_trigger();
  pdl_wait();
  const int block = blockIdx.x, seq = blockIdx.z;
  // (asked for together: the page's entry is only used where the request has it)
  const int first = cu_query_lens[seq], last = cu_query_lens[seq + 1], len = context_lens[seq];
  const int page = block < table_width ? tables[(size_t)seq * table_width + block] : -1;
  const int queries = last - first;
  int* entry = out_tables + (size_t)seq * out_width + block;
  if (queries <= 1 || block * page_size >= len || block >= table_width) {
    if (threadIdx.x == 0 && blockIdx.y == 0) *entry = 0;
    return;
  }
  // The pages of the requests in front.
  int mine = 0;
  for (int i = threadIdx.x; i < seq; i += 256)
    if (cu_query_lens[i + 1] - cu_query_lens[i] > 1) mine += (context_lens[i] + page_size - 1) / page_size;
  mine = __reduce_add_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = mine;
  __syncthreads();
  int to = block;
#pragma unroll
  for (int w = 0; w < 8; ++w) to += parts[w];
  if (to >= out_pages) return;
  if (threadIdx.x == 0 && blockIdx.y == 0) *entry = to;
  if (window > 0 && (block + 1) * page_size <= len - queries - window + 1) return;       // no query sees it: it may be gone
  if ((unsigned)page >= (unsigned)num_pages) return;
  const int per_head = page_size * dim, count = per_head * kv_heads;
  const int8_t* codes = (blockIdx.y ? v_cache : k_cache) + (size_t)page * count;
  const float* of_keys = k_scales + (size_t)page * kv_heads;
  const float* of_values = v_scales + (size_t)page * kv_heads;
  T* out = (blockIdx.y ? v_out : k_out) + (size_t)to * count;
  auto scale_of = [&](int i) {
    const float ks = of_keys[i / per_head], vs = of_values[i / per_head];
    const bool lost = !(vs < INFINITY);
    return blockIdx.y ? (lost ? 0.f : vs) : (lost ? __uint_as_float(INT8_NAN_BITS) : ks);
  };
  if constexpr (VEC > 1) {
    // a thread's values are one store of 16 bytes, so that a warp's are one piece
    for (int i = threadIdx.x * VEC; i < count; i += 256 * VEC) {
      float f[VEC];
      if constexpr (VEC == 8) {
        const uint2 x = *reinterpret_cast<const uint2*>(codes + i);
        int8_floats(x.x, f);
        int8_floats(x.y, f + 4);
      } else {
        int8_floats(*reinterpret_cast<const uint32_t*>(codes + i), f);
      }
      const float s = scale_of(i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] *= s;
      Vec<T> v;
      v.pack(f);
      v.store(out + i);
    }
  } else {
    for (int i = threadIdx.x; i < count; i += 256) out[i] = from_float<T>((float)codes[i] * scale_of(i));
  }
}

template <typename T, int VEC, typename... Args>
static int launch_kv_values(dim3 grid, cudaStream_t stream, void* k_out, void* v_out, const int8_t* k, const int8_t* v, const float* ks,
                            const float* vs, const int* tables, int table_width, const int* cu, const int* lens, Args... args) {
  return launch(kv_values_kernel<T, VEC>, grid, 256, 0, stream, k, v, ks, vs, tables, table_width, cu, lens, (T*)k_out, (T*)v_out, args...);
}

}  // namespace ts

using namespace ts;

// k and v [tokens, kv_heads, dim] dt: the rows of the step's tokens, request after request.
extern "C" int ts_kv_write_int8(const void* k, const void* v, int8_t* k_cache, int8_t* v_cache, float* k_scales, float* v_scales,
                                const int* tables, int table_width, const int* cu_query_lens, const int* context_lens, int seqs,
                                int max_query_len, int kv_heads, int dim, int page_size, int num_pages, int dtype, cudaStream_t stream) {
  if (seqs <= 0 || max_query_len <= 0) return 0;
  if (kv_heads <= 0 || dim <= 0 || page_size <= 0 || num_pages <= 0 || table_width <= 0) return TS_ERR_BAD_ARGUMENT;
  if (2 * kv_heads > 65535 || seqs > 65535) return TS_ERR_UNSUPPORTED;
  const dim3 grid((max_query_len + page_size - 2) / page_size + 1, 2 * kv_heads, seqs);
  const bool vec = dim % 4 == 0 && (((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0;
#define TS_WRITE(T_, V_)                                                                                                             \
  launch(kv_write_int8_kernel<T_, V_>, grid, 128, 0, stream, (const T_*)k, (const T_*)v, k_cache, v_cache, k_scales, v_scales, tables, \
         table_width, cu_query_lens, context_lens, kv_heads, dim, page_size, num_pages)
  if (dtype == TS_DTYPE_BF16) return vec ? TS_WRITE(bf16, 4) : TS_WRITE(bf16, 1);
  return vec ? TS_WRITE(float, 4) : TS_WRITE(float, 1);
#undef TS_WRITE
}
TS_LIST_ENTRY(ts_kv_write_int8);

extern "C" int ts_kv_values_int8(const int8_t* k_cache, const int8_t* v_cache, const float* k_scales, const float* v_scales,
                                 const int* tables, int table_width, const int* cu_query_lens, const int* context_lens, void* k_out,
                                 void* v_out, int* out_tables, int out_width, int out_pages, int seqs, int kv_heads, int dim, int page_size,
                                 int num_pages, int window, int dtype, cudaStream_t stream) {
  if (seqs <= 0 || out_width <= 0) return 0;
  if (kv_heads <= 0 || dim <= 0 || page_size <= 0 || num_pages <= 0 || table_width <= 0 || out_pages <= 0) return TS_ERR_BAD_ARGUMENT;
  if (seqs > 65535 || (long long)kv_heads * page_size * dim > 0x7fffffffll) return TS_ERR_UNSUPPORTED;
  const dim3 grid(out_width, 2, seqs);
  const bool vec = page_size * dim % 16 == 0 && (((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0;
#define TS_VALUES(T_, V_)                                                                                                          \
  launch_kv_values<T_, V_>(grid, stream, k_out, v_out, k_cache, v_cache, k_scales, v_scales, tables, table_width, cu_query_lens,    \
                           context_lens, out_tables, out_width, out_pages, kv_heads, dim, page_size, num_pages, window)
  if (dtype == TS_DTYPE_BF16) return vec ? TS_VALUES(bf16, 8) : TS_VALUES(bf16, 1);
  return vec ? TS_VALUES(float, 4) : TS_VALUES(float, 1);
#undef TS_VALUES
}
TS_LIST_ENTRY(ts_kv_values_int8);
