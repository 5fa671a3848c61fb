// Operators that stand around attention in a layer: the learned relative position bias by buckets, with the gradient of its
// table, and dropout of hidden states with the residual's addition.
//
// Relative bias.  bias[h, m, n] = table[bucket(n - m - offset), h] depends on the diagonal n - m only.  The forward is bound by its
// stores: a CTA works out the few hundred values its tile's diagonals have, and a thread then takes an N x N piece of the tile from
// 2N of them, held in registers and shifted by one element a row.  The backward is bound by reading the gradient once: a thread walks
// down the tile diagonal, so that the 2N - 1 diagonals of its N x N pieces stay the same and one register each sums them; a CTA sums
// those of its strip by buckets, and a second launch adds the CTAs' sums up in a fixed order (no atomics: the result does not
// depend on who comes first).
//
// Dropout.  Element i in logical (row-major) order takes word (0, 2, 1, 3)[i % 4] of Philox counter offset + i / 4, as the columns of a
// score row do (common.cuh): a mask follows from seed, offset and the logical index alone, not from strides, and is never stored; the
// backward draws it again.  Ten rounds of the generator serve four elements; beside them the kernel moves two to three elements' bytes each.
#include "launch.h"
#include "layer_ops.h"

namespace ab200 {
namespace {

constexpr int kThreads = 256;

template <typename T> struct alignas(16) Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  T e[N];
};

template <typename T>
__device__ __forceinline__ float table_entry(const RelativeBias& a, int bucket, int h) {
  return to_f32<T>(reinterpret_cast<const T*>(a.table)[(int64_t)bucket * a.table_stride[0] + (int64_t)h * a.table_stride[1]]);
}

// Bucket of distance d (key's position minus the query's).  `borders` in shared memory.
__device__ __forceinline__ int bucket_of(int64_t d, const int* borders, int per_direction, bool both) {
  const int64_t r = both ? (d < 0 ? -d : d) : (d < 0 ? -d : 0);
  int lo = 0, hi = per_direction - 1;      // the number of borders at or below r
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (borders[mid] <= r) lo = mid + 1;
    else hi = mid;
  }
  return lo + (both && d > 0 ? per_direction : 0);
}

// ---- relative bias, forward -----------------------------------------------------------------------------------
constexpr int kBiasRows = 64, kBiasCols = 512;

// Elements `first`..first + N - 1 of the 2N in w (first a constant).
template <typename T>
__device__ __forceinline__ uint4 window(const uint32_t (&w)[8], int first) {
  if constexpr (sizeof(T) == 4) return make_uint4(w[first], w[first + 1], w[first + 2], w[first + 3]);
  const int i = first >> 1;
  if ((first & 1) == 0) return make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  return make_uint4(__byte_perm(w[i], w[i + 1], 0x5432), __byte_perm(w[i + 1], w[i + 2], 0x5432), __byte_perm(w[i + 2], w[i + 3], 0x5432),
                    __byte_perm(w[i + 3], w[i + 4 < 8 ? i + 4 : 7], 0x5432));
}

// grid = (cdiv(sk, 512), cdiv(sq, 64), heads)
template <typename T, typename TT>
__global__ void __launch_bounds__(kThreads) relative_bias_kernel(const __grid_constant__ RelativeBias a) {
  wait_for_earlier_grids();
  constexpr int N = Vec<T>::N;
  __shared__ int borders[kMaxBorders];
  __shared__ __align__(16) T line[kBiasRows + kBiasCols];      // the value of diagonal n - m = n0 - m0 + i - kBiasRows
  const int tid = threadIdx.x, h = blockIdx.z;
  const int n0 = blockIdx.x * kBiasCols, m0 = blockIdx.y * kBiasRows;
  const int rows = min(kBiasRows, a.sq - m0), cols = min(kBiasCols, a.sk - n0);
  if (tid < a.per_direction - 1) borders[tid] = a.borders[tid];
  __syncthreads();
  for (int i = tid; i < kBiasRows + kBiasCols; i += kThreads) {
    const int64_t d = (int64_t)n0 - m0 + i - kBiasRows - a.offset;
    line[i] = from_f32<T>(table_entry<TT>(a, bucket_of(d, borders, a.per_direction, a.both != 0), h));
  }
  __syncthreads();
  T* out = reinterpret_cast<T*>(a.bias.ptr) + (int64_t)h * a.bias.s[1] + (int64_t)m0 * a.bias.s[2] + (int64_t)n0 * a.bias.s[3];
  if (!a.vec) {
    for (int r = 0; r < rows; ++r)
      for (int c = tid; c < cols; c += kThreads) out[(int64_t)r * a.bias.s[2] + (int64_t)c * a.bias.s[3]] = line[c - r + kBiasRows];
    return;
  }
  constexpr int kAcross = kBiasCols / N, kDown = kBiasRows / N;
#pragma unroll 1
  for (int i = tid; i < kAcross * kDown; i += kThreads) {
    const int r0 = i / kAcross * N, c0 = i % kAcross * N;
    if (r0 >= rows || c0 >= cols) continue;
    uint32_t w[8];
    *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(line + c0 - r0 + kBiasRows - N);
    *reinterpret_cast<uint4*>(w + 4) = *reinterpret_cast<const uint4*>(line + c0 - r0 + kBiasRows);
    T* dst = out + (int64_t)r0 * a.bias.s[2] + c0;
#pragma unroll
    for (int r = 0; r < N; ++r) {
      if (r0 + r >= rows) break;
      const uint4 v = window<T>(w, N - r);
      if (c0 + N <= cols) {
        *reinterpret_cast<uint4*>(dst + (int64_t)r * a.bias.s[2]) = v;
      } else {
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (c0 + k < cols) dst[(int64_t)r * a.bias.s[2] + k] = e[k];
      }
    }
  }
}

// ---- relative bias, gradient of the table -----------------------------------------------------------------------
// A strip: the diagonals n - m of 32 N columns' worth, seen from rows that are multiples of N.  Strip s of width W = 32 N starts at
// column W s - (rows rounded up to N) of row 0; its CTA's pieces touch the N - 1 diagonals before it as well.
template <typename T> struct Strip {
  static constexpr int N = Vec<T>::N, W = 32 * N, kWarps = kThreads / 32;
  static constexpr int kDiags = W + N - 1;      // diagonal i of a strip: n - m = first + i - (N - 1)
};
__host__ __device__ inline int64_t first_diagonal(int strip, int width, int rows) { return (int64_t)strip * width - (rows + 7) / 8 * 8; }

// grid = (strips * chunks, heads, batch_parts); partial[((h * batch_parts + part) * gridDim.x + x) * buckets + bucket]
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) relative_bias_sums_kernel(const __grid_constant__ RelativeBias a) {
  wait_for_earlier_grids();
  using S = Strip<T>;
  constexpr int N = S::N;
  __shared__ int borders[kMaxBorders];
  __shared__ float sums[S::kWarps][S::kDiags + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y, part = blockIdx.z;
  const int strip = blockIdx.x / a.chunks, chunk = blockIdx.x - strip * a.chunks;
  const int64_t first = first_diagonal(strip, S::W, a.sq);
  if (tid < a.per_direction - 1) borders[tid] = a.borders[tid];
  // rows some diagonal of the strip passes through; the chunk's share of them, in whole pieces
  const int64_t lo64 = -(first + S::W - 1), hi64 = (int64_t)a.sk - 1 - (first - (N - 1));
  const int row_lo = lo64 > 0 ? (int)(lo64 / N * N) : 0, row_hi = (int)min((int64_t)a.sq - 1, hi64);
  const int m_begin = row_lo + chunk * a.chunk_rows, m_end = (int)min((int64_t)row_hi + 1, (int64_t)m_begin + a.chunk_rows);
  const int b0 = (int)((int64_t)a.batch * part / a.batch_parts), b1 = (int)((int64_t)a.batch * (part + 1) / a.batch_parts);
  const T* g = reinterpret_cast<const T*>(a.bias.ptr) + (int64_t)h * a.bias.s[1];
  if constexpr (VEC) {
    float acc[2 * N - 1];      // acc[N - 1 + c - r]: column c, row r of a piece
#pragma unroll
    for (int i = 0; i < 2 * N - 1; ++i) acc[i] = 0.f;
    for (int b = b0; b < b1; ++b) {
      for (int m = m_begin + warp * N; m < m_end; m += S::kWarps * N) {
        const int64_t n = first + m + lane * N;
        if (n < 0 || n >= a.sk) continue;
        const T* src = g + (int64_t)b * a.bias.s[0] + (int64_t)m * a.bias.s[2] + n;
        Vec<T> v[N];
        if (n + N <= a.sk) {
#pragma unroll
          for (int r = 0; r < N; ++r) {
            if (m + r < m_end) *reinterpret_cast<uint4*>(&v[r]) = __ldcs(reinterpret_cast<const uint4*>(src + (int64_t)r * a.bias.s[2]));
            else *reinterpret_cast<uint4*>(&v[r]) = make_uint4(0u, 0u, 0u, 0u);
          }
        } else {
#pragma unroll
          for (int r = 0; r < N; ++r)
#pragma unroll
            for (int c = 0; c < N; ++c) v[r].e[c] = m + r < m_end && n + c < a.sk ? src[(int64_t)r * a.bias.s[2] + c] : from_f32<T>(0.f);
        }
#pragma unroll
        for (int r = 0; r < N; ++r)
#pragma unroll
          for (int c = 0; c < N; ++c) acc[N - 1 + c - r] += to_f32<T>(v[r].e[c]);
      }
    }
    // lane l's diagonals are strip entries N l .. N l + 2N - 2: neighbours overlap, so the even lanes write and the odd ones add
    float* mine = sums[warp];
    if ((lane & 1) == 0) {
#pragma unroll
      for (int i = 0; i < 2 * N - 1; ++i) mine[N * lane + i] = acc[i];
    }
    __syncwarp();
    if (lane & 1) {
      // (between two even lanes' entries lies one that neither wrote)
      mine[N * lane + N - 1] = acc[N - 1];
#pragma unroll
      for (int i = 0; i < 2 * N - 1; ++i)
        if (i != N - 1 && (lane < 31 || i < N - 1)) mine[N * lane + i] += acc[i];
      if (lane == 31) {
#pragma unroll
        for (int i = N; i < 2 * N - 1; ++i) mine[N * lane + i] = acc[i];
      }
    }
  } else {
    // a thread a diagonal (the strip's W, in passes of 256): rows whose starts are not 16-byte aligned
    float* flat = &sums[0][0];
    static_assert(S::W <= kThreads, "one pass");
    float acc = 0.f;
    const int64_t d = first + tid;
    if (tid < S::W) {
      const int lo = (int)max((int64_t)m_begin, -d), hi = (int)min((int64_t)m_end, (int64_t)a.sk - d);
      for (int b = b0; b < b1; ++b) {
        const T* src = g + (int64_t)b * a.bias.s[0] + (int64_t)lo * a.bias.s[2] + (lo + d) * a.bias.s[3];
        const int64_t step = a.bias.s[2] + a.bias.s[3];
        float part_sum[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) part_sum[i] = 0.f;
        int m = lo;
        for (; m + 8 <= hi; m += 8, src += 8 * step) {
#pragma unroll
          for (int i = 0; i < 8; ++i) part_sum[i] += to_f32<T>(__ldcs(src + i * step));
        }
        for (; m < hi; ++m, src += step) part_sum[0] += to_f32<T>(*src);
        acc += ((part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3])) + ((part_sum[4] + part_sum[5]) + (part_sum[6] + part_sum[7]));
      }
    }
    for (int i = tid; i < S::kDiags; i += kThreads) flat[i] = 0.f;
    __syncthreads();
    if (tid < S::W) flat[N - 1 + tid] = acc;
  }
  __syncthreads();
  if constexpr (VEC) {
    for (int i = tid; i < S::kDiags; i += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) s += sums[w][i];
      sums[0][i] = s;
    }
    __syncthreads();
  }
  // bucket by bucket: those between the strip's ends (buckets of a direction are intervals of distances)
  const int buckets = a.per_direction * (a.both ? 2 : 1);
  float* to = a.partial + (((int64_t)h * a.batch_parts + part) * gridDim.x + blockIdx.x) * buckets;
  const int64_t d0 = first - (N - 1) - a.offset;      // distance of entry 0
  for (int k = warp; k < buckets; k += S::kWarps) {
    const int j = k < a.per_direction ? k : k - a.per_direction;
    const int64_t r_lo = j > 0 ? borders[j - 1] : 0, r_hi = j + 1 < a.per_direction ? (int64_t)borders[j] - 1 : INT64_MAX / 2;
    // distances [x, y] of the bucket
    int64_t x, y;
    if (k >= a.per_direction) { x = max(r_lo, (int64_t)1); y = r_hi; }
    else { x = -r_hi; y = j == 0 && !a.both ? INT64_MAX / 2 : -r_lo; }
    const int i_lo = (int)max((int64_t)0, min(x - d0, (int64_t)S::kDiags)), i_hi = (int)min((int64_t)S::kDiags - 1, max(y - d0, (int64_t)-1));
    float s = 0.f;
    for (int i = i_lo + lane; i <= i_hi; i += 32) s += sums[0][i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) to[k] = s;
  }
}

// grid = (buckets, heads): the CTAs' sums, in their order
template <typename TT>
__global__ void __launch_bounds__(128) relative_bias_table_kernel(const __grid_constant__ RelativeBias a, int count) {
  wait_for_earlier_grids();
  __shared__ float sums[4];
  const int k = blockIdx.x, h = blockIdx.y, buckets = gridDim.x;
  const float* from = a.partial + (int64_t)h * count * buckets + k;
  float s = 0.f;
  for (int i = threadIdx.x; i < count; i += 128) s += from[(int64_t)i * buckets];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0)
    reinterpret_cast<TT*>(a.table)[(int64_t)k * a.table_stride[0] + (int64_t)h * a.table_stride[1]] =
        from_f32<TT>((sums[0] + sums[1]) + (sums[2] + sums[3]));
}

// ---- dropout ------------------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ T dropped(T x, bool keep, float scale, float residual) {
  // (selected, not multiplied by zero: what is dropped may be infinite, and so may be the scale)
  return from_f32<T>((keep ? to_f32<T>(x) * scale : 0.f) + residual);
}

// FLAT: everything is contiguous, one row.  Otherwise rows of cols elements, a multiple of N, with strides of their own.
template <typename T, bool FLAT, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const __grid_constant__ Dropout a, uint64_t vectors) {
  wait_for_earlier_grids();
  constexpr int N = Vec<T>::N, U = 16 / N;      // sixteen elements a thread: four counters in lockstep
  const uint64_t seed = a.seed + (a.seed_ptr ? *a.seed_ptr : 0ull), offset = a.offset + (a.offset_ptr ? *a.offset_ptr : 0ull);
  const bool keep_all = !a.on;
  const uint64_t v0 = (uint64_t)blockIdx.x * (kThreads * U) + threadIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* res = reinterpret_cast<const T*>(a.residual);
  T* out = reinterpret_cast<T*>(a.out);
  Vec<T> in[U], r[U];
  int64_t row[U], col[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t v = v0 + (uint64_t)u * kThreads;
    if (v >= vectors) continue;
    if constexpr (FLAT) { row[u] = 0; col[u] = (int64_t)v * N; }
    else {
      const uint64_t per = (uint64_t)a.cols / N;
      row[u] = vectors >> 32 ? (int64_t)(v / per) : (int64_t)((uint32_t)v / (uint32_t)per);
      col[u] = ((int64_t)v - row[u] * (int64_t)per) * N;
    }
    *reinterpret_cast<uint4*>(&in[u]) = __ldcs(reinterpret_cast<const uint4*>(x + row[u] * a.sx + col[u]));
    if constexpr (RESIDUAL) *reinterpret_cast<uint4*>(&r[u]) = __ldcs(reinterpret_cast<const uint4*>(res + row[u] * a.sr + col[u]));
  }
  uint32_t c[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint64_t counter = offset + (v0 + (uint64_t)(k / (N / 4)) * kThreads) * (N / 4) + (k % (N / 4));
    c[k][0] = (uint32_t)counter;
    c[k][1] = (uint32_t)(counter >> 32);
  }
  philox4x32_10_lockstep<4>(seed, c);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (v0 + (uint64_t)u * kThreads >= vectors) continue;
    Vec<T> w;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const uint32_t* words = c[u * (N / 4) + e / 4];
      const uint32_t word = (e & 3) == 0 ? words[0] : ((e & 3) == 1 ? words[2] : ((e & 3) == 2 ? words[1] : words[3]));
      w.e[e] = dropped<T>(in[u].e[e], keep_all || (int32_t)word > a.threshold, a.scale, RESIDUAL ? to_f32<T>(r[u].e[e]) : 0.f);
    }
    *reinterpret_cast<uint4*>(out + row[u] * a.so + col[u]) = *reinterpret_cast<const uint4*>(&w);
  }
}

// Any width, stride and alignment, from element `first` (a multiple of four) on: a warp takes 128 elements, one counter a lane, and
// hands the bits round so that its accesses are to consecutive elements.
template <typename T>
__global__ void __launch_bounds__(kThreads) dropout_elements_kernel(const __grid_constant__ Dropout a, uint64_t first) {
  wait_for_earlier_grids();
  const uint64_t seed = a.seed + (a.seed_ptr ? *a.seed_ptr : 0ull), offset = a.offset + (a.offset_ptr ? *a.offset_ptr : 0ull);
  const int lane = threadIdx.x & 31;
  const uint64_t n = (uint64_t)a.rows * (uint64_t)a.cols, base = first + ((uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * 128;
  if (base >= n) return;
  const Philox4 w = philox4x32_10(seed, offset + base / 4 + lane);
  const uint32_t mine = !a.on ? 15u
                              : ((int32_t)w.w[0] > a.threshold ? 1u : 0u) | ((int32_t)w.w[2] > a.threshold ? 2u : 0u) |
                                    ((int32_t)w.w[1] > a.threshold ? 4u : 0u) | ((int32_t)w.w[3] > a.threshold ? 8u : 0u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t keep = __shfl_sync(0xffffffffu, mine, 8 * j + (lane >> 2)) >> (lane & 3);
    const uint64_t i = base + 32 * j + lane;
    if (i >= n) continue;
    const int64_t row = n >> 32 ? (int64_t)(i / (uint64_t)a.cols) : (int64_t)((uint32_t)i / (uint32_t)a.cols), col = (int64_t)i - row * a.cols;
    const float r = a.residual ? to_f32<T>(reinterpret_cast<const T*>(a.residual)[row * a.sr + col]) : 0.f;
    reinterpret_cast<T*>(a.out)[row * a.so + col] = dropped<T>(reinterpret_cast<const T*>(a.x)[row * a.sx + col], keep & 1u, a.scale, r);
  }
}

// f.template operator()<T>() for the dtype's T
template <typename F>
cudaError_t with_type(int dtype, F f) {
  switch (dtype) {
    case 1: return f.template operator()<float>();
    case 2: return f.template operator()<__half>();
    case 3: return f.template operator()<__nv_bfloat16>();
  }
  return cudaErrorInvalidValue;
}

cudaError_t counted(cudaError_t e) {
  if (e == cudaSuccess) count_launch();
  return e;
}

}  // namespace

cudaError_t launch_relative_bias(int dtype, int table_dtype, const RelativeBias& a, cudaStream_t st) {
  if (a.sq <= 0 || a.sk <= 0 || a.heads <= 0) return cudaSuccess;
  const dim3 grid((a.sk + kBiasCols - 1) / kBiasCols, (a.sq + kBiasRows - 1) / kBiasRows, a.heads);
  return with_type(dtype, [&]<typename T>() {
    return with_type(table_dtype, [&]<typename TT>() { return counted(launch_kernel(relative_bias_kernel<T, TT>, grid, dim3(kThreads), 0, st, a)); });
  });
}

int64_t plan_relative_bias_backward(int dtype, RelativeBias& a, int sms) {
  if (a.sq <= 0 || a.sk <= 0 || a.heads <= 0 || a.batch <= 0) return 0;
  const int n = dtype == 1 ? 4 : 8, width = 32 * n;
  // strips cover the diagonals 1 - sq .. sk - 1
  const int64_t strips = ((int64_t)a.sk + (a.sq + 7) / 8 * 8 + width - 1) / width;
  const int most = a.sq < a.sk + width + 8 ? a.sq : a.sk + width + 8;      // rows of a strip
  a.chunk_rows = 512;
  a.strips = (int)strips;
  a.chunks = (most + n + a.chunk_rows - 1) / a.chunk_rows;
  a.batch_parts = a.batch;
  while (a.batch_parts > 1 && strips * a.chunks * a.heads * (int64_t)a.batch_parts > 16ll * sms) a.batch_parts = (a.batch_parts + 1) / 2;
  return strips * a.chunks * a.batch_parts * (int64_t)a.heads * a.per_direction * (a.both ? 2 : 1);
}

cudaError_t launch_relative_bias_backward(int dtype, int table_dtype, const RelativeBias& a, cudaStream_t st) {
  const int buckets = a.per_direction * (a.both ? 2 : 1);
  const bool empty = a.sq <= 0 || a.sk <= 0 || a.batch <= 0;
  if (!empty) {
    const dim3 grid(a.strips * a.chunks, a.heads, a.batch_parts);
    const cudaError_t e = with_type(dtype, [&]<typename T>() {
      return counted(launch_kernel(a.vec ? relative_bias_sums_kernel<T, true> : relative_bias_sums_kernel<T, false>, grid, dim3(kThreads), 0, st, a));
    });
    if (e != cudaSuccess) return e;
  }
  const int count = empty ? 0 : a.strips * a.chunks * a.batch_parts;
  return with_type(table_dtype, [&]<typename TT>() {
    return counted(launch_kernel(relative_bias_table_kernel<TT>, dim3(buckets, a.heads), dim3(128), 0, st, a, count));
  });
}

cudaError_t launch_dropout(int dtype, const Dropout& a, cudaStream_t st) {
  const int64_t total = a.rows * a.cols;
  if (total <= 0) return cudaSuccess;
  return with_type(dtype, [&]<typename T>() {
    constexpr int N = Vec<T>::N;
    auto aligned = [&](const void* p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % N == 0; };
    const bool one_row = a.rows == 1 || (a.sx == a.cols && a.so == a.cols && (a.residual == nullptr || a.sr == a.cols));
    const bool vec = one_row ? aligned(a.x, 0) && aligned(a.out, 0) && aligned(a.residual, 0)
                             : a.cols % N == 0 && aligned(a.x, a.sx) && aligned(a.out, a.so) && (a.residual == nullptr || aligned(a.residual, a.sr));
    uint64_t done = 0;
    if (vec && total >= N) {
      const uint64_t vectors = (uint64_t)(total / N), per = kThreads * (16 / N);
      const dim3 grid((unsigned)((vectors + per - 1) / per));
      auto kern = one_row ? (a.residual ? dropout_kernel<T, true, true> : dropout_kernel<T, true, false>)
                          : (a.residual ? dropout_kernel<T, false, true> : dropout_kernel<T, false, false>);
      const cudaError_t e = counted(launch_kernel(kern, grid, dim3(kThreads), 0, st, a, vectors));
      if (e != cudaSuccess) return e;
      done = vectors * N;
    }
    if ((int64_t)done == total) return cudaSuccess;
    const dim3 grid((unsigned)((total - done + 1023) / 1024));
    return counted(launch_kernel(dropout_elements_kernel<T>, grid, dim3(kThreads), 0, st, a, done));
  });
}

}  // namespace ab200
