// Operators that stand around attention in a layer: the learned relative position bias by buckets, with the gradient of its
// table, and dropout of hidden states with the residual's addition.
//
// Relative bias.  bias[h, m, n] = table[bucket(n - m - offset), h] depends on the diagonal n - m only.  The forward is bound by its
// stores: a CTA works out the few hundred values its tile's diagonals have, and a thread then takes an N x N piece of the tile from
// 2N of them, held in registers and shifted by one element a row.  16 heads x 2048 x 2048 bf16: 21.5 us, 6.2 TB/s.  The backward is bound by reading
// the gradient once: a warp walks down the diagonals in steps of eight rows, between which a 16-byte vector moves by whole vectors, so that each of its
// elements stays on its diagonal and one register a diagonal sums them; a CTA sums those of its band by buckets, and a second launch adds
// the CTAs' sums up in a fixed order (no atomics: the result does not depend on who comes first).  8 x 16 x 2048 x 2048 bf16, 1.07 GB: 185 to 188 us,
// 5.7 to 5.8 TB/s.  Short rows are far from that: of 16 x 12 x 391 x 391 fp16 (27 us, 2.2 TB/s) 55 % of what the bands cover lies inside the matrix, and
// nearly every step meets an edge.  (Pieces of 8 x 8 elements with 15 diagonals' registers took 217, and rows that start anywhere another kernel.)
//
// Dropout.  Element i in logical (row-major) order takes word (0, 2, 1, 3)[i % 4] of Philox counter offset + i / 4, as the columns of a
// score row do (common.cuh): a mask follows from seed, offset and the logical index alone, not from strides, and is never stored; the
// backward draws it again.  Ten rounds of the generator serve four elements, beside which two (with a residual three) elements' bytes each move: the
// wide multiplies, four of a round's eight issue slots' worth, and the exclusive ors bound the form without a residual in 16-bit types, memory the
// others.  64M elements of bf16: 55 to 58 us without a residual (4.6 to 4.9 TB/s), 65 with one (6.2 TB/s); fp32, 32M, 41 and 59 (6.6 and 6.8 TB/s).  (Round keys added up by each thread 68 and 74; CTAs that take several tiles in turn 57 to 63 and 64 to 75.)
#include <algorithm>
#include <type_traits>
#include "launch.h"
#include "layer_ops.h"
#include "sm100_ptx.cuh"

namespace ab200 {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kPhiloxA = 0xD2511F53u, kPhiloxB = 0xCD9E8D57u;

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
// A band: kBand diagonals, first .. first + kBand - 1, of one head, in STRIPS strips of 31 N side by side.  A CTA takes the rows that pass
// through it and have kResidues residues modulo 8 (kParts CTAs all of them), and of those chunk_rows' worth, counted through the batch (each of
// its elements has the band's rows, padded to whole steps).
template <typename T, int STRIPS> struct Band {
  static constexpr int N = Vec<T>::N, kStrips = STRIPS, kStrip = 31 * N, kBand = STRIPS * kStrip;
  static constexpr int kResidues = 8 / STRIPS, kParts = STRIPS, kStep = 64;      // rows of a step: eight of each residue
  int64_t first;
  int row_lo, rows;      // the rows some diagonal of the band passes through; `rows` in whole steps
  __host__ __device__ Band(int sq, int sk, int band) {
    first = (int64_t)band * kBand - (sq - 1);
    const int64_t lo = -(first + kBand - 1), hi = (int64_t)sk - 1 - first;
    row_lo = lo > 0 ? (int)lo : 0;
    const int row_hi = hi < sq - 1 ? (int)hi : sq - 1;
    rows = (row_hi - row_lo + kStep) / kStep * kStep;      // (at least one row: bands end with the last diagonal)
  }
  __host__ __device__ static int bands(int sq, int sk) { return (int)(((int64_t)sq + sk - 1 + kBand - 1) / kBand); }
};

// Two elements of a word as fp32.
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(__byte_perm(w, 0u, 0x1044)), __uint_as_float(w & 0xffff0000u));
}

// grid = (bands * chunks * kParts, heads); partial[(h * gridDim.x + x) * buckets + bucket], of chunks that have rows.
// UNIT: rows of unit stride.  A warp takes every eighth row, all of whose starts are as far from a 16-byte boundary, whatever the rows'
// stride: its lanes read aligned 16 bytes each, 32 of them from the one with the strip's first column on, and the diagonal of an element stays the
// same from row to row.  N registers sum them; nothing is shifted, and odd row lengths cost what even ones do.  (The last of the 32 only
// completes the first's: 31 N diagonals a strip.)  What is read beside the row lies in 16 bytes that hold some of it, and is not added.
template <typename T, int STRIPS, bool UNIT>
__global__ void __launch_bounds__(kThreads, 4) relative_bias_sums_kernel(const __grid_constant__ RelativeBias a) {
  wait_for_earlier_grids();
  using S = Band<T, STRIPS>;
  constexpr int N = S::N;
  __shared__ int borders[kMaxBorders];
  __shared__ float sums[S::kResidues][S::kBand];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y;
  const int part = blockIdx.x % S::kParts, item = blockIdx.x / S::kParts, band = item / a.chunks, chunk = item - band * a.chunks;
  const S st(a.sq, a.sk, band);
  const int64_t begin = (int64_t)chunk * a.chunk_rows, end = min(begin + a.chunk_rows, (int64_t)st.rows * a.batch);
  if (begin >= end) return;
  if (tid < a.per_direction - 1) borders[tid] = a.borders[tid];
  int b = (int)(begin / st.rows), row = (int)(begin - (int64_t)b * st.rows);      // the chunk's next step: rows row.. of the band's
  const T* g = reinterpret_cast<const T*>(a.bias.ptr) + (int64_t)h * a.bias.s[1];
  for (int i = tid; i < S::kResidues * S::kBand; i += kThreads) (&sums[0][0])[i] = 0.f;
  __syncthreads();
  if constexpr (UNIT) {
    const int strip = warp % STRIPS, residue = S::kResidues * part + warp / STRIPS;
    float* mine = sums[warp / STRIPS] + strip * S::kStrip;
    float2 acc[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) acc[i] = make_float2(0.f, 0.f);
    int shift = -1;      // of the rows summed so far: element e of lane l is the strip's diagonal N l + e - shift
    auto flush = [&] {
      if (shift < 0) return;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int i = N * lane + e - shift;
        if (i >= 0 && i < S::kStrip) mine[i] += (e & 1) ? acc[e / 2].y : acc[e / 2].x;
      }
    };
    const int64_t eight = 8 * (a.bias.s[2] + 1);
    for (int64_t at = begin; at < end; at += S::kStep) {
      const int m0 = st.row_lo + row + residue;
      const int n0 = (int)(st.first + m0) + strip * S::kStrip;                        // the strip's first column in row m0
      const T* p0 = g + (int64_t)b * a.bias.s[0] + (int64_t)m0 * a.bias.s[2];
      if ((row += S::kStep) == st.rows) { row = 0; ++b; }
      if (m0 >= a.sq || n0 - N >= a.sk || n0 + 56 + 32 * N <= 0) continue;      // (nothing of the row in the strip)
      const uintptr_t from = reinterpret_cast<uintptr_t>(p0 + n0);
      const int sh = (int)(from & 15) / (int)sizeof(T);
      if (sh != shift) {      // (another element of the batch, a whole one of which is not a multiple of 16 bytes)
        flush();
        __syncwarp();
#pragma unroll
        for (int i = 0; i < N / 2; ++i) acc[i] = make_float2(0.f, 0.f);
        shift = sh;
      }
      const int n = n0 - sh + N * lane;      // this lane's first column in row m0; one to the right in each further row
      const T* src = reinterpret_cast<const T*>(from & ~uintptr_t(15)) + N * lane;
      // adds a vector's elements; with `some`, those of them whose bits are set in `mask`
      auto add = [&](const uint4& v, auto some, uint32_t mask) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          float2 x;
          if constexpr (sizeof(T) == 2) x = unpack2<T>(w[i]);
          else x = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
          if constexpr (some.value) {
            if (!(mask & (1u << (2 * i)))) x.x = 0.f;
            if (!(mask & (2u << (2 * i)))) x.y = 0.f;
          }
          acc[i].x += x.x;
          acc[i].y += x.y;
        }
      };
      uint4 v[8];
      // (all of it inside: no element lies beside its row, no row behind the last)
      if (n0 - sh >= 0 && n0 - sh + 56 + 32 * N <= a.sk && m0 + 56 < a.sq) {
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = __ldg(reinterpret_cast<const uint4*>(src + r * eight));
#pragma unroll
        for (int r = 0; r < 8; ++r) add(v[r], std::false_type{}, 0u);
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const bool in = m0 + 8 * r < a.sq && n + 8 * r + N > 0 && n + 8 * r < a.sk;
          v[r] = in ? __ldg(reinterpret_cast<const uint4*>(src + r * eight)) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int before = -(n + 8 * r), behind = n + 8 * r + N - a.sk;      // elements of the vector on either side of the row, if above 0
          const uint32_t mask = (0xffu << min(max(before, 0), N)) & (0xffu >> (8 - N + min(max(behind, 0), N)));
          if (__any_sync(0xffffffffu, (before > 0 && before < N) || (behind > 0 && behind < N))) add(v[r], std::true_type{}, mask);
          else add(v[r], std::false_type{}, 0u);      // (whole vectors beside the row are zero)
        }
      }
    }
    flush();
    __syncthreads();
    for (int i = tid; i < S::kBand; i += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < S::kResidues; ++r) s += sums[r][i];
      sums[0][i] = s;
    }
  } else {
    // a thread a diagonal, in turns: elements that are not next to each other
    for (int64_t at = begin; at < end; at += S::kStep) {
      for (int i = tid; i < S::kBand; i += kThreads) {
        const int64_t d = st.first + i;
        float s = 0.f;
        const T* src = g + (int64_t)b * a.bias.s[0];
#pragma unroll 4
        for (int r = 0; r < 8 * S::kResidues; ++r) {
          const int m = st.row_lo + row + 8 * (r / S::kResidues) + S::kResidues * part + r % S::kResidues;
          const int64_t n = m + d;
          if (m < a.sq && n >= 0 && n < a.sk) s += to_f32<T>(src[(int64_t)m * a.bias.s[2] + n * a.bias.s[3]]);
        }
        sums[0][i] += s;
      }
      if ((row += S::kStep) == st.rows) { row = 0; ++b; }
    }
  }
  __syncthreads();
  // bucket by bucket (buckets of a direction are intervals of distances)
  const int buckets = a.per_direction * (a.both ? 2 : 1);
  float* to = a.partial + ((int64_t)h * gridDim.x + blockIdx.x) * buckets;
  const int64_t d0 = st.first - a.offset;      // distance of entry 0
  for (int k = warp; k < buckets; k += kThreads / 32) {
    const int j = k < a.per_direction ? k : k - a.per_direction;
    const int64_t r_lo = j > 0 ? borders[j - 1] : 0, r_hi = j + 1 < a.per_direction ? (int64_t)borders[j] - 1 : INT64_MAX / 2;
    // distances [x, y] of the bucket
    int64_t x, y;
    if (k >= a.per_direction) { x = max(r_lo, (int64_t)1); y = r_hi; }
    else { x = -r_hi; y = j == 0 && !a.both ? INT64_MAX / 2 : -r_lo; }
    const int i_lo = (int)max((int64_t)0, min(x - d0, (int64_t)S::kBand)), i_hi = (int)min((int64_t)S::kBand - 1, max(y - d0, (int64_t)-1));
    float s = 0.f;
    if (i_lo <= i_hi) {
      for (int i = i_lo + lane; i <= i_hi; i += 32) s += sums[0][i];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    if (lane == 0) to[k] = s;
  }
}

// grid = (buckets, heads): the CTAs' sums, in their order.  T: the gradient's type, which the bands' width goes by
template <typename T, int STRIPS, typename TT>
__global__ void __launch_bounds__(128) relative_bias_table_kernel(const __grid_constant__ RelativeBias a) {
  wait_for_earlier_grids();
  __shared__ float sums[4];
  const int k = blockIdx.x, h = blockIdx.y, buckets = gridDim.x, items = a.bands * a.chunks;
  const float* from = a.partial + (int64_t)h * items * Band<T, STRIPS>::kParts * buckets + k;
  float s = 0.f;
  for (int i = threadIdx.x; i < items; i += 128) {
    const int band = i / a.chunks;
    if ((int64_t)(i - band * a.chunks) * a.chunk_rows >= (int64_t)Band<T, STRIPS>(a.sq, a.sk, band).rows * a.batch) continue;
#pragma unroll
    for (int p = 0; p < Band<T, STRIPS>::kParts; ++p) s += from[((int64_t)i * Band<T, STRIPS>::kParts + p) * buckets];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0)
    reinterpret_cast<TT*>(a.table)[(int64_t)k * a.table_stride[0] + (int64_t)h * a.table_stride[1]] =
        from_f32<TT>((sums[0] + sums[1]) + (sums[2] + sums[3]));
}

// ---- dropout ------------------------------------------------------------------------------------------------------
// (selected, not multiplied by zero: what is dropped may be infinite, and so may be the scale)
template <typename T>
__device__ __forceinline__ float kept(T x, bool keep, float scale) { return keep ? to_f32<T>(x) * scale : 0.f; }

// Rounds FROM..9 of N counters of one seed side by side: c[n], four words in and out.  key(i): the i-th of the twenty round keys.
template <int FROM, int N, typename K>
__device__ __forceinline__ void philox_rounds(K key, uint32_t (&c)[N][4]) {
#pragma unroll
  for (int i = FROM; i < 10; ++i) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint64_t pa = (uint64_t)kPhiloxA * c[n][0], pb = (uint64_t)kPhiloxB * c[n][2];
      const uint32_t n0 = (uint32_t)(pb >> 32) ^ c[n][1] ^ key(2 * i), n2 = (uint32_t)(pa >> 32) ^ c[n][3] ^ key(2 * i + 1);
      c[n][1] = (uint32_t)pb; c[n][3] = (uint32_t)pa; c[n][0] = n0; c[n][2] = n2;
    }
  }
}
__host__ __device__ constexpr uint32_t round_key(uint64_t seed, int i) {
  return (i & 1) ? (uint32_t)(seed >> 32) + 0xBB67AE85u * (uint32_t)(i >> 1) : (uint32_t)seed + 0x9E3779B9u * (uint32_t)(i >> 1);
}
// The words of counters c[n][0..1], whatever they are.
template <int N>
__device__ __forceinline__ void philox_words(uint64_t seed, uint32_t (&c)[N][4]) {
#pragma unroll
  for (int n = 0; n < N; ++n) c[n][2] = c[n][3] = 0u;
  philox_rounds<0, N>([&](int i) { return round_key(seed, i); }, c);
}
// The same for a call that passes its seed by value and all of whose counters have one high word: the keys come from the call's parameters, where
// the exclusive ors read them for nothing, and of the first two rounds what the high word alone decides is in them already
// (dropout_keys).  c[n][0]: the counter's low word in.
template <int N>
__device__ __forceinline__ void philox_words_by_value(const uint32_t (&keys)[20], uint32_t (&c)[N][4]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const uint64_t pa = (uint64_t)kPhiloxA * c[n][0], pb = (uint64_t)kPhiloxB * ((uint32_t)(pa >> 32) ^ keys[1]);
    c[n][0] = (uint32_t)(pb >> 32) ^ keys[2];
    c[n][1] = (uint32_t)pb;
    c[n][2] = (uint32_t)pa ^ keys[3];
    c[n][3] = 0u;      // (in keys[5])
  }
  philox_rounds<2, N>([&](int i) { return keys[i]; }, c);
}
// Round 1 leaves c0 = high ^ keys[0], the same for all counters; its product in round 2 goes into keys[3] and keys[5].
void dropout_keys(uint64_t seed, uint32_t high, uint32_t (&keys)[20]) {
  for (int i = 0; i < 20; ++i) keys[i] = round_key(seed, i);
  const uint64_t product = (uint64_t)kPhiloxA * (high ^ keys[0]);
  keys[3] ^= (uint32_t)(product >> 32);
  keys[5] ^= (uint32_t)product;
}

// FLAT: everything is contiguous, one row.  Otherwise rows of cols elements, a multiple of N, with strides of their own.  BY_VALUE: seed and
// offset are the call's alone, and the counters' high word is one.
template <typename T, bool FLAT, bool RESIDUAL, bool BY_VALUE>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const __grid_constant__ Dropout a, uint64_t vectors) {
  wait_for_earlier_grids();
  constexpr int N = Vec<T>::N, U = 16 / N;      // sixteen elements a thread: four counters side by side
  uint64_t seed = a.seed, offset = a.offset;
  if constexpr (!BY_VALUE) {
    if (a.seed_ptr) seed += *a.seed_ptr;
    if (a.offset_ptr) offset += *a.offset_ptr;
  }
  const bool keep_all = !a.on;
  const uint64_t v0 = (uint64_t)blockIdx.x * (kThreads * U) + threadIdx.x;
  auto body = [&](auto whole) {      // (no bounds but in the last CTA)
    uint4 in[U], r[U], *to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t v = v0 + (uint64_t)u * kThreads;
      if (!whole.value && v >= vectors) continue;
      const uint4 *from = reinterpret_cast<const uint4*>(a.x), *add = reinterpret_cast<const uint4*>(a.residual);
      to[u] = reinterpret_cast<uint4*>(a.out);
      if constexpr (FLAT) {
        from += v0 + u * kThreads;
        add += v0 + u * kThreads;
        to[u] += v0 + u * kThreads;
      } else {
        const uint64_t per = (uint64_t)a.cols / N;
        const int64_t row = vectors >> 32 ? (int64_t)(v / per) : (int64_t)((uint32_t)v / (uint32_t)per), col = (int64_t)v - row * (int64_t)per;
        from += row * (a.sx / N) + col;
        add += row * (a.sr / N) + col;
        to[u] += row * (a.so / N) + col;
      }
      in[u] = __ldcs(from);
      if constexpr (RESIDUAL) r[u] = __ldcs(add);
    }
    uint32_t c[4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t counter = offset + v0 * (N / 4) + (k / (N / 4)) * kThreads * (N / 4) + (k % (N / 4));
      c[k][0] = (uint32_t)counter;
      c[k][1] = (uint32_t)(counter >> 32);
    }
    if constexpr (BY_VALUE) philox_words_by_value<4>(a.keys, c);
    else philox_words<4>(seed, c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!whole.value && v0 + (uint64_t)u * kThreads >= vectors) continue;
      const uint32_t x[4] = {in[u].x, in[u].y, in[u].z, in[u].w}, res[4] = {r[u].x, r[u].y, r[u].z, r[u].w};
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        constexpr int kPer = N / 4;      // elements of a word: one or two
        auto keep = [&](int e) {
          const uint32_t* words = c[u * (N / 4) + e / 4];
          return keep_all || (int32_t)((e & 3) == 0 ? words[0] : ((e & 3) == 1 ? words[2] : ((e & 3) == 2 ? words[1] : words[3]))) > a.threshold;
        };
        if constexpr (kPer == 1) {
          float y = keep(i) ? __uint_as_float(x[i]) * a.scale : 0.f;
          if constexpr (RESIDUAL) y += __uint_as_float(res[i]);
          w[i] = __float_as_uint(y);
        } else {
          float2 y = unpack2<T>(x[i]);
          y.x = keep(2 * i) ? y.x * a.scale : 0.f;
          y.y = keep(2 * i + 1) ? y.y * a.scale : 0.f;
          if constexpr (RESIDUAL) y = ptx::add2(y, unpack2<T>(res[i]));
          w[i] = pack2<T>(y.x, y.y);
        }
      }
      *to[u] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  };
  if ((uint64_t)(blockIdx.x + 1ull) * (kThreads * U) <= vectors) body(std::true_type{});
  else body(std::false_type{});
}

// Any width, stride and alignment, from element `first` (a multiple of four) on: a warp takes 256 elements, two counters a lane, and
// hands the bits round so that its accesses are to consecutive elements.  WIDE: rows of 256 elements or more, so that a warp's lie in one row or
// two.
constexpr int kElementsWarp = 256, kElementsCta = kElementsWarp * (kThreads / 32);
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) dropout_elements_kernel(const __grid_constant__ Dropout a, uint64_t first) {
  wait_for_earlier_grids();
  const uint64_t seed = a.seed + (a.seed_ptr ? *a.seed_ptr : 0ull), offset = a.offset + (a.offset_ptr ? *a.offset_ptr : 0ull);
  const int lane = threadIdx.x & 31;
  const uint64_t n = (uint64_t)a.rows * (uint64_t)a.cols, base = first + (uint64_t)blockIdx.x * kElementsCta + (threadIdx.x >> 5) * kElementsWarp;
  if (base >= n) return;
  constexpr int kPer = kElementsWarp / 32;
  const int left = (int)min(n - base, (uint64_t)kElementsWarp) - lane;      // element 32 j + lane is one where 32 j < left
  // this lane's first element, and where its elements lie in a tensor with a stride of s between rows
  uint64_t row = n >> 32 ? base / (uint64_t)a.cols : (uint64_t)((uint32_t)base / (uint32_t)a.cols);
  const int64_t col = (int64_t)(base - row * (uint64_t)a.cols) + lane;
  const int in_row = (int)min(a.cols - col, (int64_t)1 << 20);      // element j is in the next row where 32 j >= in_row (WIDE)
  auto at = [&](int64_t s, int j) -> int64_t {
    if constexpr (WIDE) return (int64_t)row * s + col + 32 * j + (32 * j >= in_row ? s - a.cols : 0);
    const int64_t c = col + 32 * j, down = c / a.cols;
    return ((int64_t)row + down) * s + c - down * a.cols;
  };
  const T *x = reinterpret_cast<const T*>(a.x), *res = reinterpret_cast<const T*>(a.residual);
  T *out = reinterpret_cast<T*>(a.out), in[kPer], r[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (32 * j < left) {
      in[j] = x[at(a.sx, j)];
      if (res) r[j] = res[at(a.sr, j)];
    }
  }
  uint32_t c[2][4], mine[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint64_t counter = offset + base / 4 + 32 * k + lane;
    c[k][0] = (uint32_t)counter;
    c[k][1] = (uint32_t)(counter >> 32);
  }
  philox_words<2>(seed, c);
#pragma unroll
  for (int k = 0; k < 2; ++k)
    mine[k] = !a.on ? 15u
                    : ((int32_t)c[k][0] > a.threshold ? 1u : 0u) | ((int32_t)c[k][2] > a.threshold ? 2u : 0u) |
                          ((int32_t)c[k][1] > a.threshold ? 4u : 0u) | ((int32_t)c[k][3] > a.threshold ? 8u : 0u);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const uint32_t keep = __shfl_sync(0xffffffffu, mine[j / 4], 8 * (j & 3) + (lane >> 2)) >> (lane & 3);
    if (32 * j >= left) continue;
    float y = kept<T>(in[j], keep & 1u, a.scale);
    if (res) y += to_f32<T>(r[j]);
    out[at(a.so, j)] = from_f32<T>(y);
  }
}

// f.template operator()<T>() for the dtype's T (the entry points let no other through)
template <typename F>
auto with_type(int dtype, F f) {
  return dtype == 1 ? f.template operator()<float>() : (dtype == 2 ? f.template operator()<__half>() : f.template operator()<__nv_bfloat16>());
}
template <typename F>
auto with_band(int dtype, const RelativeBias& a, F f) {
  return with_type(dtype, [&]<typename T>() { return a.strips == 4 ? f.template operator()<T, 4>() : f.template operator()<T, 1>(); });
}
// Four strips side by side, 2 KB of a row at once, where rows are long: memory gives 512 bytes here and there at 4.3 TB/s, 2 KB at 5.9.  In shorter
// rows most of such a band lies beside them.  Measured, us, whole backward with nothing in L2, four strips / one: bf16, 8 x 16 heads x 513 44.0 / 37.9,
// x 1000 75.8 / 67.6, 4 x 16 x 1536 80.9 / 77.8, x 2048 112.6 / 113.7, 8 x 16 x 2047 207.9 / 212.1; fp32, 8 x 16 x 768 72.8 / 72.7, x 1024 108.5 / 110.7,
// x 2048 356 / 382.
inline bool wide_bands(int dtype, const RelativeBias& a) { return (int64_t)std::min(a.sq, a.sk) * (dtype == 1 ? 4 : 2) >= 3584; }

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
  a.bands = a.chunks = a.chunk_rows = 0;
  if (a.sq <= 0 || a.sk <= 0 || a.heads <= 0 || a.batch <= 0) return 0;
  a.strips = wide_bands(dtype, a) ? 4 : 1;
  return with_band(dtype, a, [&]<typename T, int STRIPS>() {
    // Rows a CTA, whole steps: one round of the four CTAs an SM holds where the whole is small, three for long rows, whose bands are uneven.
    // (Device us with 4 / 6 / 8 / 12 / 16 CTAs an SM: 16 x 12 x 391 bf16 27.4 / 28.0 / 29.9 / 31.7 / 31.7, 8 x 16 x 768 33.6 / 37.7 / 35.4 / 38.4 /
    // 41.3, 4 x 16 x 2048 109.2 / 102.8 / 97.3 / 94.4 / 96.3.)  64 bands tell how many rows there are (neighbours differ little).
    using B = Band<T, STRIPS>;
    constexpr int step = B::kStep;
    const int bands = B::bands(a.sq, a.sk), probe = std::min(bands, 64);
    int64_t all = 0;
    for (int i = 0; i < probe; ++i) all += B(a.sq, a.sk, (int)((int64_t)bands * i / probe)).rows;
    const int64_t total = all * bands / probe * a.batch * a.heads * B::kParts, target = total / ((STRIPS == 4 ? 12ll : 4ll) * sms);
    const int64_t rows = std::min<int64_t>(std::max<int64_t>((target + step - 1) / step * step, step), 1 << 30);
    const int64_t most = (std::min<int64_t>(a.sq, (int64_t)a.sk + B::kBand - 1) + step - 1) / step * step;      // rows of a band
    a.bands = bands;
    a.chunk_rows = (int)rows;
    a.chunks = (int)((most * a.batch + rows - 1) / rows);
    return (int64_t)bands * a.chunks * B::kParts * a.heads * a.per_direction * (a.both ? 2 : 1);
  });
}

cudaError_t launch_relative_bias_backward(int dtype, int table_dtype, const RelativeBias& a, cudaStream_t st) {
  const int buckets = a.per_direction * (a.both ? 2 : 1);
  return with_band(dtype, a, [&]<typename T, int STRIPS>() {
    if (a.bands > 0) {
      const cudaError_t e = counted(launch_kernel(a.unit ? relative_bias_sums_kernel<T, STRIPS, true> : relative_bias_sums_kernel<T, STRIPS, false>,
                                                  dim3(a.bands * a.chunks * Band<T, STRIPS>::kParts, a.heads), dim3(kThreads), 0, st, a));
      if (e != cudaSuccess) return e;
    }
    return with_type(table_dtype, [&]<typename TT>() {
      return counted(launch_kernel(relative_bias_table_kernel<T, STRIPS, TT>, dim3(buckets, a.heads), dim3(128), 0, st, a));
    });
  });
}

cudaError_t launch_dropout(int dtype, const Dropout& given, cudaStream_t st) {
  Dropout a = given;
  const int64_t total = a.rows * a.cols;
  if (total <= 0) return cudaSuccess;
  const bool by_value = a.seed_ptr == nullptr && a.offset_ptr == nullptr && (a.offset >> 32) == ((a.offset + (uint64_t)(total - 1) / 4) >> 32);
  dropout_keys(a.seed, (uint32_t)(a.offset >> 32), a.keys);
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
      using Kernel = void (*)(Dropout, uint64_t);
      static constexpr Kernel kernels[2][2][2] = {      // [one row][residual][by value]
          {{dropout_kernel<T, false, false, false>, dropout_kernel<T, false, false, true>}, {dropout_kernel<T, false, true, false>, dropout_kernel<T, false, true, true>}},
          {{dropout_kernel<T, true, false, false>, dropout_kernel<T, true, false, true>}, {dropout_kernel<T, true, true, false>, dropout_kernel<T, true, true, true>}}};
      const Kernel kern = kernels[one_row][a.residual != nullptr][by_value];
      const cudaError_t e = counted(launch_kernel(kern, grid, dim3(kThreads), 0, st, a, vectors));
      if (e != cudaSuccess) return e;
      done = vectors * N;
    }
    if ((int64_t)done == total) return cudaSuccess;
    const dim3 grid((unsigned)((total - done + kElementsCta - 1) / kElementsCta));
    return counted(launch_kernel(a.cols >= kElementsWarp ? dropout_elements_kernel<T, true> : dropout_elements_kernel<T, false>, grid, dim3(kThreads), 0, st, a, done));
  });
}

}  // namespace ab200
