// Rows as 8-bit integers with a scale each (int8.cuh): the residual sum with its RMSNorm, the gated activation of a
// feed-forward, or rows as they are; and codes read back as values. All arithmetic in 32 bits, rounded once, to the code.
#define TS_PDL_CLASS PDL_SKINNY      // they stand between the products of that class
#include "int8.cuh"
#include "launch_list.cuh"

namespace ts {

constexpr int ROW_NORM = 0, ROW_SILU = 1, ROW_GELU_TANH = 2, ROW_PLAIN = 3;

// Both activations are gate times a sigmoid: silu(z) = z / (1 + e^-z), and 0.5 z (1 + tanh u) = z / (1 + e^-2u). The exponential is
// good to |z| + 2 units; where |z| is large, either 1 + e^-z or the result hardly depends on it.
template <int MODE>
__device__ __forceinline__ float row_activation(float g, float u) {
  const float z = MODE == ROW_SILU ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
  return __fdividef(g, 1.f + __expf(-z)) * u;
}

// rint(v * inverse) as the low byte of a 32-bit value: behind 1.5 * 2^23 a unit is 1, and the sum is rounded to it.
__device__ __forceinline__ uint32_t code_byte(float v, float inverse) { return __float_as_uint(fmaf(v, inverse, 12582912.f)); }
__device__ __forceinline__ uint32_t four_codes(const float* v, float inverse) {
  const uint32_t lo = __byte_perm(code_byte(v[0], inverse), code_byte(v[1], inverse), 0x0040);
  const uint32_t hi = __byte_perm(code_byte(v[2], inverse), code_byte(v[3], inverse), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

// What a thread takes of a row at a time: N neighbouring values, 16 bytes of the widest input but for the 32-bit stream; one of a
// row off that grid.
template <typename T, int MODE> constexpr int ROW_VEC = MODE == ROW_NORM ? 4 : Vec<T>::N;
template <int N, int NV> constexpr int ROW_THREADS = N * NV > 16 ? 512 : 1024;      // so many at most
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* p, float* f) {
  if constexpr (N == 1) {
    f[0] = to_float(p[0]);
  } else if constexpr (N == 4) {
    Quad<T>::load(p, f);
  } else {
    Vec<T> v;
    v.load(p);
    v.unpack(f);
  }
}

// A CTA takes a row and keeps it in registers between its sums and its codes, a thread NV times N of its values; one
// barrier. Of a norm, y = x rstd w, the codes are those of x w, whose largest magnitude is found beside the sum of squares: rstd
// only enters the scale. Bound by memory where rows are many (the norm of 2,048 rows of 4,096 in bf16: 17.2 us, 5.4 TB/s of the
// 92 MB that it reads and writes), by latency where they are few (the weights are asked for in front of the wait). Rows off the
// grid of 4 or 8 values go value by value (1,763 rows of 3,653: 18.7 us; of 3,648: 9.5).
template <typename T, int MODE, int N, int NV>
__global__ void __launch_bounds__(ROW_THREADS<N, NV>) int8_rows_kernel(
    const T* __restrict__ in, float* __restrict__ resid, const T* __restrict__ delta, const T* __restrict__ weight,
    int8_t* __restrict__ out, float* __restrict__ scales, int width, int out_width, float eps) {
  __shared__ float parts[32];
  __shared__ uint32_t most[32];
  pdl_trigger();
  const size_t row = blockIdx.x;
  float v[NV][N];
  if constexpr (MODE == ROW_NORM) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (threadIdx.x + j * blockDim.x) * N;
#pragma unroll
      for (int e = 0; e < N; ++e) v[j][e] = 0.f;
      if (i < width) load_row<T, N>(weight + i, v[j]);
    }
  }
  pdl_wait();
  float ss = 0.f;
  uint32_t m = 0;
  if constexpr (MODE == ROW_NORM) {
    float* x = resid + row * width;
    const T* d = delta ? delta + row * width : nullptr;
    float a[NV][N], b[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (threadIdx.x + j * blockDim.x) * N;
#pragma unroll
      for (int e = 0; e < N; ++e) a[j][e] = b[j][e] = 0.f;
      if (i < width) {
        load_row<float, N>(x + i, a[j]);
        if (d) load_row<T, N>(d + i, b[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (threadIdx.x + j * blockDim.x) * N;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        a[j][e] += b[j][e];
        ss += a[j][e] * a[j][e];
        v[j][e] *= a[j][e];
        m = max(m, magnitude_bits(v[j][e]));
      }
      if (d && i < width) {
        if constexpr (N == 1) x[i] = a[j][0];
        else Quad<float>::store(x + i, a[j]);
      }
    }
  } else {
    const T* g = in + row * width * (MODE == ROW_PLAIN ? 1 : 2);
    float u[NV][N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (threadIdx.x + j * blockDim.x) * N;
#pragma unroll
      for (int e = 0; e < N; ++e) v[j][e] = u[j][e] = 0.f;
      if (i < width) {
        load_row<T, N>(g + i, v[j]);
        if constexpr (MODE != ROW_PLAIN) load_row<T, N>(g + width + i, u[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if constexpr (MODE != ROW_PLAIN) v[j][e] = row_activation<MODE>(v[j][e], u[j][e]);
        m = max(m, magnitude_bits(v[j][e]));
      }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  m = warp_max_bits(m);
  if constexpr (MODE == ROW_NORM) ss = warp_sum(ss);
  if (lane == 0) {
    most[warp] = m;
    parts[warp] = ss;
  }
  __syncthreads();
  m = warp_max_bits(lane < warps ? most[lane] : 0u);
  bool held = m < INT8_INF_BITS && m >= INT8_TINY_BITS;
  float scale = int8_scale(m);
  if constexpr (MODE == ROW_NORM) {
    ss = warp_sum(lane < warps ? parts[lane] : 0.f);
    const float rstd = 1.f / sqrtf(ss / (float)width + eps), most_y = rstd * __uint_as_float(m);
    // What is too small or no number is that of y. Where x w is too small for its reciprocal and y is not, x w is lifted first.
    held = m < INT8_INF_BITS && magnitude_bits(most_y) < INT8_INF_BITS && most_y >= __uint_as_float(INT8_TINY_BITS);
    scale = int8_scale(m >= INT8_INF_BITS ? m : magnitude_bits(most_y));
    if (held && m < INT8_TINY_BITS) {
      m = __float_as_uint(__uint_as_float(m) * 0x1p64f);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) v[j][e] *= 0x1p64f;
    }
  }
  const float inverse = int8_inverse(m);
  if (threadIdx.x == 0) scales[row] = scale;
  int8_t* o = out + row * out_width;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = (threadIdx.x + j * blockDim.x) * N;
    if (i < width) {
      if constexpr (N == 8) {
        *reinterpret_cast<uint2*>(o + i) = held ? make_uint2(four_codes(v[j], inverse), four_codes(v[j] + 4, inverse)) : make_uint2(0u, 0u);
      } else if constexpr (N == 4) {
        *reinterpret_cast<uint32_t*>(o + i) = held ? four_codes(v[j], inverse) : 0u;
      } else {
        o[i] = held ? (int8_t)code_byte(v[j][0], inverse) : (int8_t)0;
      }
    }
  }
  for (int i = width + threadIdx.x; i < out_width; i += blockDim.x) o[i] = 0;
}

// Many rows through an activation: the exponentials of a row take about as long as its bytes, so a CTA goes over rows and has the
// next one copied into shared memory meanwhile, by asynchronous copies of 16 bytes that the thread itself will read (no barrier
// between the copy and its use). 2,048 rows of 12,288, a CTA a row with its loads in front / so: 34 / 25 us
// (5.1 TB/s; half the SMs' issue slots are taken).
constexpr int STREAM_THREADS = 512;
template <typename T, int MODE, int NV>
__global__ void __launch_bounds__(STREAM_THREADS, 2) int8_rows_stream_kernel(const T* __restrict__ in, int8_t* __restrict__ out,
                                                                            float* __restrict__ scales, int rows, int width, int out_width) {
  constexpr int N = Vec<T>::N, PARTS = MODE == ROW_PLAIN ? 1 : 2;
  extern __shared__ __align__(16) unsigned char held_rows[];      // [2][PARTS][NV][threads] of 16 bytes
  __shared__ uint32_t most[2][STREAM_THREADS / 32];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto place = [&](int b, int part, int j) {
    return held_rows + ((((size_t)b * PARTS + part) * NV + j) * STREAM_THREADS + threadIdx.x) * 16;
  };
  auto fetch = [&](int row, int b) {
    if (row < rows) {
      const T* g = in + (size_t)row * width * PARTS;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = (threadIdx.x + j * STREAM_THREADS) * N;
        if (i < width) {
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                         ::"r"((uint32_t)__cvta_generic_to_shared(place(b, part, j))), "l"(g + part * width + i) : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(blockIdx.x, 0);
  int b = 0;
  for (int row = blockIdx.x; row < rows; row += gridDim.x, b ^= 1) {
    fetch(row + gridDim.x, b ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    float v[NV][N];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (threadIdx.x + j * STREAM_THREADS) * N;
#pragma unroll
      for (int e = 0; e < N; ++e) v[j][e] = 0.f;
      if (i < width) {
        Vec<T> x;
        x.load(reinterpret_cast<const T*>(place(b, 0, j)));
        x.unpack(v[j]);
        if constexpr (MODE != ROW_PLAIN) {
          float u[N];
          x.load(reinterpret_cast<const T*>(place(b, 1, j)));
          x.unpack(u);
#pragma unroll
          for (int e = 0; e < N; ++e) v[j][e] = row_activation<MODE>(v[j][e], u[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < N; ++e) m = max(m, magnitude_bits(v[j][e]));
    }
    m = warp_max_bits(m);
    if (lane == 0) most[b][warp] = m;
    __syncthreads();      // (the next row's go to the other half, the ones after that are behind the next barrier)
    m = warp_max_bits(lane < STREAM_THREADS / 32 ? most[b][lane] : 0u);
    const bool held = m < INT8_INF_BITS && m >= INT8_TINY_BITS;
    const float inverse = int8_inverse(m);
    if (threadIdx.x == 0) scales[row] = int8_scale(m);
    int8_t* o = out + (size_t)row * out_width;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = (threadIdx.x + j * STREAM_THREADS) * N;
      if (i < width) {
        if constexpr (N == 8) {
          *reinterpret_cast<uint2*>(o + i) = held ? make_uint2(four_codes(v[j], inverse), four_codes(v[j] + 4, inverse)) : make_uint2(0u, 0u);
        } else {
          *reinterpret_cast<uint32_t*>(o + i) = held ? four_codes(v[j], inverse) : 0u;
        }
      }
    }
    for (int i = width + threadIdx.x; i < out_width; i += STREAM_THREADS) o[i] = 0;
  }
}
template <typename T, int MODE, int NV>
static int launch_stream(const void* in, int8_t* out, float* scales, int rows, int width, int out_width, cudaStream_t stream) {
  auto kern = int8_rows_stream_kernel<T, MODE, NV>;
  constexpr size_t smem = 2 * (MODE == ROW_PLAIN ? 1 : 2) * NV * STREAM_THREADS * 16;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  const int per_sm = smem <= 48 * 1024 ? 3 : 2;
  return launch(kern, dim3(rows < 148 * per_sm ? rows : 148 * per_sm), STREAM_THREADS, smem, stream, (const T*)in, out, scales, rows, width, out_width);
}

// Rows of more than a CTA's registers hold: every pass reads its values again.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) int8_any_rows_kernel(const T* __restrict__ in, float* __restrict__ resid, const T* __restrict__ delta,
                                                            const T* __restrict__ weight, int8_t* __restrict__ out,
                                                            float* __restrict__ scales, int width, int out_width, float eps) {
  __shared__ float scratch[33];
  __shared__ uint32_t most[8];
  pdl_trigger();
  pdl_wait();
  const size_t row = blockIdx.x;
  const T* g = in ? in + row * width * (MODE == ROW_PLAIN ? 1 : 2) : nullptr;
  float* x = resid ? resid + row * width : nullptr;
  float rstd = 0.f;
  if constexpr (MODE == ROW_NORM) {
    float ss = 0.f;
    for (int i = threadIdx.x; i < width; i += blockDim.x) {
      float v = x[i];
      if (delta) x[i] = v += to_float(delta[row * width + i]);
      ss += v * v;
    }
    rstd = 1.f / sqrtf(block_sum(ss, scratch) / (float)width + eps);
  }
  auto value = [&](int i) {
    if constexpr (MODE == ROW_NORM) return x[i] * rstd * to_float(weight[i]);
    else if constexpr (MODE == ROW_PLAIN) return to_float(g[i]);
    else return row_activation<MODE>(to_float(g[i]), to_float(g[width + i]));
  };
  uint32_t m = 0;
  for (int i = threadIdx.x; i < width; i += blockDim.x) m = max(m, magnitude_bits(value(i)));
  m = warp_max_bits(m);
  if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = m;
  __syncthreads();
  m = warp_max_bits(most[threadIdx.x & 7]);
  if (threadIdx.x == 0) scales[row] = int8_scale(m);
  const float inverse = int8_inverse(m);
  for (int i = threadIdx.x; i < out_width; i += blockDim.x) out[row * out_width + i] = (int8_t)(i < width ? int8_code(value(i), inverse) : 0);
}

template <typename T, int MODE>
static int launch_rows(const void* in, float* resid, const void* delta, const void* weight, int8_t* out, float* scales, int rows, int width,
                       int out_width, float eps, cudaStream_t stream) {
  constexpr int N = ROW_VEC<T, MODE>;
  const bool aligned = (((uintptr_t)in | (uintptr_t)resid | (uintptr_t)delta | (uintptr_t)weight | (uintptr_t)out) & 15) == 0;
  const bool on_grid = aligned && width % N == 0 && out_width % N == 0, by_fours = N > 4 && !on_grid && aligned && width % 4 == 0 && out_width % 4 == 0;
  // Runs a thread: of few rows as few as a CTA's threads allow, of many rows as many as leave 256 threads to a row.
  const int runs = on_grid ? width / N : (width + 3) / 4, full = rows <= 148 ? 1024 : on_grid ? 256 : 512;
  const int nv = runs <= full ? 1 : runs <= 2 * full ? 2 : 4;
  const int threads = ((runs + nv - 1) / nv + 31) / 32 * 32;
  if constexpr (MODE != ROW_NORM) {
    if (on_grid && rows >= 4 * 148 && runs > 2 * 256 && runs <= 3 * STREAM_THREADS)
      return runs <= 2 * STREAM_THREADS ? launch_stream<T, MODE, 2>(in, out, scales, rows, width, out_width, stream)
                                        : launch_stream<T, MODE, 3>(in, out, scales, rows, width, out_width, stream);
  }
#define TS_ROWS(N_, NV_)                                                                                                          \
  if (threads <= ROW_THREADS<N_, NV_>)                                                                                            \
  return launch(int8_rows_kernel<T, MODE, N_, NV_>, dim3(rows), threads, 0, stream, (const T*)in, resid, (const T*)delta,          \
                (const T*)weight, out, scales, width, out_width, eps)
  if (on_grid) {
    if (nv == 1) TS_ROWS(N, 1);
    if (nv == 2) TS_ROWS(N, 2);
    if (nv == 4) TS_ROWS(N, 4);
  } else if (by_fours) {
    if constexpr (N > 4) {
      if (nv == 1) TS_ROWS(4, 1);
      if (nv == 2) TS_ROWS(4, 2);
      if (nv == 4) TS_ROWS(4, 4);
    }
  } else {
    if (nv == 1) TS_ROWS(1, 4);
    if (nv == 2) TS_ROWS(1, 8);
    if (nv == 4) TS_ROWS(1, 16);
  }
#undef TS_ROWS
  return launch(int8_any_rows_kernel<T, MODE>, dim3(rows), 256, 0, stream, (const T*)in, resid, (const T*)delta, (const T*)weight, out, scales,
                width, out_width, eps);
}

template <typename T>
static int rows_of(int mode, const void* in, int8_t* out, float* scales, int rows, int width, int out_width, cudaStream_t stream) {
  if (mode == ROW_SILU) return launch_rows<T, ROW_SILU>(in, nullptr, nullptr, nullptr, out, scales, rows, width, out_width, 0.f, stream);
  if (mode == ROW_GELU_TANH) return launch_rows<T, ROW_GELU_TANH>(in, nullptr, nullptr, nullptr, out, scales, rows, width, out_width, 0.f, stream);
  return launch_rows<T, ROW_PLAIN>(in, nullptr, nullptr, nullptr, out, scales, rows, width, out_width, 0.f, stream);
}

// out[i, h, c] = codes[rows ? rows[i] : i, h, c] * scales[.., h]: `heads` groups of in_width codes an item, of which the first
// out_width come out. An item outside the codes becomes NaN. A thread takes VEC neighbouring codes. Bound by memory: 2,048 rows of
// 4,096 to bf16 in 6.0 us (4.2 TB/s).
template <typename T, int VEC>
__global__ void __launch_bounds__(256) int8_values_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales,
                                                          const int* __restrict__ rows, T* __restrict__ out, int items, int heads,
                                                          int in_width, int out_width, long long total) {
  pdl_trigger();
  pdl_wait();
  const long long at = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * VEC;
  if (at >= total) return;
  long long to;          // the group of out that this is
  int c;
  if (total <= 0x7fffffffll) {
    to = (int)at / out_width;
    c = (int)at % out_width;
  } else {
    to = at / out_width;
    c = (int)(at - to * out_width);
  }
  const long long i = heads == 1 ? to : to / heads;
  const long long from = rows ? rows[i] : i;
  const bool there = from >= 0 && from < items;
  const size_t group = (size_t)(there ? from : 0) * heads + (to - i * heads);
  const float s = there ? scales[group] : __uint_as_float(INT8_NAN_BITS);
  const int8_t* p = codes + group * in_width + c;
  // (nothing is read for an item outside: there may be no codes at all)
  if constexpr (VEC == 1) {
    out[at] = from_float<T>((there ? (float)p[0] : 0.f) * s);
  } else {
    uint32_t w[VEC / 4] = {};
    if (there) {
      if constexpr (VEC == 16) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
      } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
      }
    }
    float f[VEC];
#pragma unroll
    for (int e = 0; e < VEC / 4; ++e) int8_floats(w[e], f + 4 * e);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] *= s;
    if constexpr (VEC == 16) {
#pragma unroll
      for (int e = 0; e < VEC; e += Vec<T>::N) {
        Vec<T> v;
        v.pack(f + e);
        v.store(out + at + e);
      }
    } else {
      Quad<T>::store(out + at, f);
    }
  }
}

// The same for groups off the grid of 4 codes, of a length that fills CTAs: one takes 1,024 of a group, a thread every 256th (1,763
// rows of 3,653 to bf16: 9.0 us; a division an element 30).
template <typename T>
__global__ void __launch_bounds__(256) int8_long_values_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales,
                                                               const int* __restrict__ rows, T* __restrict__ out, int items, int heads,
                                                               int in_width, int out_width, int per_group) {
  pdl_trigger();
  pdl_wait();
  const int to = blockIdx.x / per_group, c0 = (blockIdx.x - to * per_group) * 1024 + threadIdx.x, i = to / heads;
  const int from = rows ? rows[i] : i;
  const bool there = from >= 0 && from < items;
  const size_t group = (size_t)(there ? from : 0) * heads + (to - i * heads);
  const float s = there ? scales[group] : __uint_as_float(INT8_NAN_BITS);
  const int8_t* p = codes + group * in_width;
  T* o = out + (size_t)to * out_width;
  float f[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = there && c0 + 256 * e < out_width ? (float)p[c0 + 256 * e] : 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c0 + 256 * e < out_width) o[c0 + 256 * e] = from_float<T>(f[e] * s);
}

template <typename T>
static int launch_values(const int8_t* codes, const float* scales, const int* rows, void* out, int items, int count, int heads, int in_width,
                         int out_width, cudaStream_t stream) {
  const long long total = (long long)count * heads * out_width;
  const bool aligned = (((uintptr_t)codes | (uintptr_t)out) & 15) == 0;
  const int vec = aligned && out_width % 16 == 0 && in_width % 16 == 0 ? 16 : aligned && out_width % 4 == 0 && in_width % 4 == 0 ? 4 : 1;
  const int per_group = (out_width + 1023) / 1024;
  if (vec == 1 && out_width >= 256 && (long long)count * heads * per_group <= 0x7fffffffll)
    return launch(int8_long_values_kernel<T>, dim3((unsigned)(count * heads * per_group)), 256, 0, stream, codes, scales, rows, (T*)out, items,
                  heads, in_width, out_width, per_group);
  const long long blocks = (total / vec + 255) / 256;
  if (blocks > 0x7fffffffll) return TS_ERR_UNSUPPORTED;
#define TS_VALUES(V_)                                                                                                                  \
  launch(int8_values_kernel<T, V_>, dim3((unsigned)blocks), 256, 0, stream, codes, scales, rows, (T*)out, items, heads, in_width, out_width, \
         total)
  return vec == 16 ? TS_VALUES(16) : vec == 4 ? TS_VALUES(4) : TS_VALUES(1);
#undef TS_VALUES
}

}  // namespace ts

using namespace ts;

// resid [rows, width] float += delta (dt, may be null); y = resid / sqrt(mean(resid^2) + eps) * weight (dt) -> codes and scales.
// out is [rows, out_width] with out_width >= width; the columns from width on become 0.
extern "C" int ts_add_rms_norm_int8(float* resid, const void* delta, const void* weight, int8_t* out, float* scales, int rows, int width,
                                    int out_width, float eps, int dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (width <= 0 || out_width < width) return TS_ERR_BAD_ARGUMENT;
  if (dtype == TS_DTYPE_BF16)
    return launch_rows<bf16, ROW_NORM>(nullptr, resid, delta, weight, out, scales, rows, width, out_width, eps, stream);
  return launch_rows<float, ROW_NORM>(nullptr, resid, delta, weight, out, scales, rows, width, out_width, eps, stream);
}
TS_LIST_ENTRY(ts_add_rms_norm_int8);

// mode: 1 silu(gate) * up, 2 gelu_tanh(gate) * up (in is [rows, 2 width], gate first), 3 rows as they are (in is [rows, width]).
extern "C" int ts_act_mul_int8(const void* in, int8_t* out, float* scales, int rows, int width, int out_width, int mode, int dtype,
                               cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (width <= 0 || out_width < width || mode < ROW_SILU || mode > ROW_PLAIN) return TS_ERR_BAD_ARGUMENT;
  return dtype == TS_DTYPE_BF16 ? rows_of<bf16>(mode, in, out, scales, rows, width, out_width, stream)
                                : rows_of<float>(mode, in, out, scales, rows, width, out_width, stream);
}
TS_LIST_ENTRY(ts_act_mul_int8);

extern "C" int ts_int8_values(const int8_t* codes, const float* scales, const int* rows, void* out, int items, int count, int heads,
                              int in_width, int out_width, int dtype, cudaStream_t stream) {
  if (count <= 0) return 0;
  if (heads <= 0 || in_width <= 0 || out_width <= 0 || out_width > in_width) return TS_ERR_BAD_ARGUMENT;
  return dtype == TS_DTYPE_BF16 ? launch_values<bf16>(codes, scales, rows, out, items, count, heads, in_width, out_width, stream)
                                : launch_values<float>(codes, scales, rows, out, items, count, heads, in_width, out_width, stream);
}
TS_LIST_ENTRY(ts_int8_values);
