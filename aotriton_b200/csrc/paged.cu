// Operators over a cache in pages: block tables and slot maps, the writing of new tokens, attention for any type and size, the sum of a split
// sequence's pieces; and keys whose last columns all heads share.
#include <algorithm>
#include "launch.h"
#include "paged.h"
#include "paged_split.cuh"

namespace ab200 {
namespace {

// ---- block tables and slot maps --------------------------------------------------------------------------------
// Sequence z holds n tokens and takes m more; token i of them stands at position n + i, in page (n + i) / page of its row.  Pages that it has not
// got yet are the next of the free list, in order of sequence and position, so that a token finds its page from two running sums over the sequences
// ahead of it: tokens, which say whose it is, and pages taken.  Every CTA adds those up for itself, as far as its own tokens; nothing waits
// for anything, and one launch does.
constexpr int kTableThreads = 256, kTableTokens = 2048;

// RUN: tokens next to each other that a thread takes: 4 where sequences take many, most often of one sequence and one page; 1 where most take one (48 of
// one token 2.8 us, with 4 4.9; 590000 tokens of 300 sequences 7.0, with 1 9.6).
template <int RUN>
__global__ void __launch_bounds__(kTableThreads) block_tables_kernel(const __grid_constant__ BlockTables a) {
  wait_for_earlier_grids();
  __shared__ int64_t warp_tokens[kTableThreads / 32], warp_pages[kTableThreads / 32];
  __shared__ int64_t fresh[kTableThreads];
  __shared__ int start[kTableThreads], held[kTableThreads], pages_of[kTableThreads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t t0 = (int64_t)blockIdx.x * kTableTokens, t1 = min(t0 + kTableTokens, a.total);
  const bool sums = blockIdx.x == 0;
  int64_t tokens = 0, pages = a.taken != nullptr ? max(a.taken[0], 0) : 0;      // of the sequences so far
  for (int z0 = 0; z0 < a.batch && (sums || tokens < t1); z0 += kTableThreads) {
    const int z = z0 + tid;
    int n = 0, m = 0, have = 0, need = 0;
    // (of so many tokens; two numbers of 31 bits and a page's worth are within 32)
    auto pages_for = [&](unsigned count) { return (int)min(count / (unsigned)a.page + (count % (unsigned)a.page != 0u), (unsigned)a.width); };
    if (z < a.batch) {
      n = max(a.lengths[z], 0);
      m = max(a.new_tokens[z], 0);
      have = pages_for((unsigned)n);
      need = pages_for((unsigned)n + (unsigned)m) - have;
    }
    int64_t up_t = m, up_p = need;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, up_t, d), y = __shfl_up_sync(0xffffffffu, up_p, d);
      if (lane >= d) { up_t += x; up_p += y; }
    }
    __syncthreads();      // (the last chunk's tokens have been found)
    if (lane == 31) { warp_tokens[warp] = up_t; warp_pages[warp] = up_p; }
    __syncthreads();
    int64_t all_t = 0, all_p = 0;
    for (int w = 0; w < kTableThreads / 32; ++w) {
      if (w < warp) { up_t += warp_tokens[w]; up_p += warp_pages[w]; }
      all_t += warp_tokens[w];
      all_p += warp_pages[w];
    }
    start[tid] = (int)min(tokens + up_t - m, (int64_t)0x7fffffff);      // (of tokens below 2^31 alone)
    fresh[tid] = pages + up_p - need - have;
    held[tid] = n;
    pages_of[tid] = have;
    int got = m;      // its tokens with room among the slots: it holds those, and their pages are taken
    if (sums && tokens + all_t > a.total) {
      got = (int)min((int64_t)m, max(a.total - (tokens + up_t - m), (int64_t)0));
      int64_t fewer = (int64_t)pages_for((unsigned)n + (unsigned)got) - have - need;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) fewer += __shfl_xor_sync(0xffffffffu, fewer, d);
      __syncthreads();      // (the warps' pages have been added up)
      if (lane == 0) warp_pages[warp] = fewer;
      __syncthreads();
      for (int w = 0; w < kTableThreads / 32; ++w) all_p += warp_pages[w];
    }
    if (sums && z < a.batch) {
      if (z == 0) a.cu_seqlens[0] = 0;
      a.cu_seqlens[z + 1] = (int)min(tokens + up_t, (int64_t)0x7fffffff);
      a.new_lengths[z] = (int)min((int64_t)n + got, (int64_t)0x7fffffff);
    }
    __syncthreads();
    const int64_t from = max(tokens, t0), end = min(tokens + all_t, t1);
    for (int t = from < end ? (int)from + tid * RUN : 0x7fffffff; t < (int)end; t += kTableThreads * RUN) {
      int lo = -1, id = -1;
      unsigned page = 0u, in = 0u;
      bool looked = false;
#pragma unroll
      for (int k = 0; k < RUN; ++k) {
        const int tk = t + k;
        if (tk >= (int)end) break;
        if (lo < 0 || (lo + 1 < kTableThreads && start[lo + 1] <= tk)) {
          lo = 0;      // the last sequence that starts at or ahead of the token: it has tokens, those behind it start later
          for (int hi = kTableThreads - 1; lo < hi;) {
            const int mid = (lo + hi + 1) >> 1;
            if (start[mid] <= tk) lo = mid;
            else hi = mid - 1;
          }
          const unsigned p = (unsigned)held[lo] + (unsigned)(tk - start[lo]);
          page = p / (unsigned)a.page;
          in = p - page * (unsigned)a.page;
          looked = false;
        } else if (++in == (unsigned)a.page) {
          in = 0u;
          ++page;
          looked = false;
        }
        if (!looked) {
          looked = true;
          id = -1;
          if (page < (unsigned)a.width) {
            int32_t* entry = a.table + (int64_t)(z0 + lo) * a.table_stride + page;
            if ((int)page < pages_of[lo]) {
              id = *entry;
            } else {
              const int64_t i = fresh[lo] + page;
              id = i < a.num_free ? a.free_pages[i] : -1;
              if (in == 0u) *entry = id;      // (a page's first token enters it)
            }
          }
        }
        a.slots[tk] = id < 0 ? -1 : (int64_t)id * a.page + in;
      }
    }
    tokens += all_t;
    pages += all_p;
  }
  for (int64_t t = max(tokens, t0) + tid; t < t1; t += kTableThreads) a.slots[t] = -1;
  if (sums && tid == 0) {
    if (a.batch == 0) a.cu_seqlens[0] = 0;
    a.taken_out[0] = (int)min(pages, (int64_t)0x7fffffff);
  }
}

// ---- new tokens into their slots --------------------------------------------------------------------------------
// Rows are moved as they are: bound by their bytes, read once and written once.  A CTA takes a few tokens' rows, each thread kWriteBatch vectors whose
// loads are on the way together.
constexpr int kWriteThreads = 256, kWriteBatch = 4;

// I: what counts the vectors; 32 bits where they do (20000 latent rows of 576 11.9 us in 64 bits).
template <typename V, typename I>
__global__ void __launch_bounds__(kWriteThreads) paged_write_kernel(const __grid_constant__ PagedWrite a, int elt, I vectors) {
  wait_for_earlier_grids();
  const int per = (int)sizeof(V) / elt;      // elements of a vector
  const int vk = a.dk / per, vv = a.dv / per, of_k = a.heads * vk, of_token = of_k + a.heads * vv;
  const I first = (I)blockIdx.x * (kWriteBatch * kWriteThreads) + threadIdx.x;
  V value[kWriteBatch];
  V* to[kWriteBatch];
#pragma unroll
  for (int b = 0; b < kWriteBatch; ++b) {
    const I i = first + b * kWriteThreads;
    to[b] = nullptr;
    if (i >= vectors) continue;
    const int64_t t = i / (I)of_token;
    int e = (int)(i - (I)t * (I)of_token);
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.slots_total) continue;
    const I page = (I)slot / (I)a.page;      // (slots of a cache that 32 bits do not count: 64)
    const int in = (int)((I)slot - page * (I)a.page);
    const bool is_k = e < of_k;
    if (!is_k) e -= of_k;
    const int wide = is_k ? vk : vv, h = (int)((unsigned)e / (unsigned)wide), c = e - h * wide;
    const int64_t from = t * (is_k ? a.sk[0] : a.sv[0]) + h * (is_k ? a.sk[1] : a.sv[1]) + (int64_t)c * per;
    const int64_t dst = (int64_t)page * (is_k ? a.ck[0] : a.cv[0]) + in * (is_k ? a.ck[1] : a.cv[1]) + h * (is_k ? a.ck[2] : a.cv[2]) + (int64_t)c * per;
    value[b] = *reinterpret_cast<const V*>(reinterpret_cast<const char*>(is_k ? a.k : a.v) + from * elt);
    to[b] = reinterpret_cast<V*>(reinterpret_cast<char*>(is_k ? a.k_cache : a.v_cache) + dst * elt);
  }
#pragma unroll
  for (int b = 0; b < kWriteBatch; ++b)
    if (to[b] != nullptr) *to[b] = value[b];
}

// ---- attention, any type and size up to 1024 ----------------------------------------------------------------------
// For what has no tensor-core kernel: fp32, odd head dims and pages.  Bound by instructions (a fused multiply-add a score and column on the ordinary pipe, and its
// operands from shared memory).  16 sequences of 40 to 2000 fp32 keys, 32:8 heads of 128, 72 us (floor 21).
// Tiles of 32 keys: eight lanes form a key's scores with the unit's rows, a warp a row takes their softmax on, and a thread a column adds up
// the values; with fewer columns than threads, groups of threads share the keys.
constexpr int kGenThreads = 256, kGenRows = 8, kGenKeys = 32;

template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* src, float (&x)[N]) {
  if constexpr (N == 1) {
    x[0] = to_f32<T>(*src);
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(src);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32<T>(e[i]);
  }
}

// Blocks an SM, for which a call is cut.  Values of one column a thread: three, 80 registers (the case above with 112 and two blocks 111 us; 16-bit rows read 16 bytes at a
// time then keep 56 to 76 bytes in memory, and are faster all the same: 32 sequences of 100 to 4000 bf16 keys, 16:4 heads of 256, 291 us, with two blocks
// and nothing there 368).  More columns: two, 102 to 123 registers (cut for three, which do not fit, a wave and a half: heads of 512 1434 us for 1091, 8 sequences
// of 500 to 4000 fp32 latent rows x 16 heads 125 for 99).
__host__ __device__ constexpr int gen_blocks(int columns) { return columns == 1 ? 3 : 2; }

// J: columns of a thread.  N: elements of K that a lane reads at a time.
template <typename T, int N, int J>
__global__ void __launch_bounds__(kGenThreads, gen_blocks(J)) paged_general_kernel(const __grid_constant__ PagedAttn p) {
  wait_for_earlier_grids();
  extern __shared__ __align__(16) float q_s[];      // [kGenRows][dqk]
  __shared__ float scores[2][kGenRows][kGenKeys], alphas[2][kGenRows], m_s[kGenRows], l_s[kGenRows];      // (of a tile and the next one)
  __shared__ float meet[J == 1 ? kGenThreads * kGenRows : 1];
  // where a key and its value start in the caches (-1: nobody sees it), worked out once (with a division in every thread for every key the
  // sequences above took 166 us and not 112); a tile's, the last one's, which some may still read, and the next one's
  __shared__ int64_t places_k[3][kGenKeys], places_v[3][kGenKeys];
  __shared__ int scratch[kGenThreads / 32 + 2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Line line = find_in_line<kGenThreads>(p, -1, blockIdx.x / p.lanes, scratch);
  if (line.z >= p.batch) return;
  int width = 32;      // threads that share the columns
  while (width < p.dvo && width < kGenThreads) width <<= 1;
  const int groups = kGenThreads / width, group = tid / width, col = tid - group * width;
  Piece c(p, line);
  while (c.next(p)) {
    const Walk& w = c.w;
    const int z = c.z, hk = c.hk, first = c.first, last = c.last;
    const bool whole = c.whole();
    const Rows rows(p, w, c.chunk);
    if (first == 0 && c.chunk == 0) zero_rows_behind<T, kGenThreads>(p, w, z, hk, tid);
    if (rows.n == 0) continue;
    __syncthreads();
    for (int i = tid; i < rows.n * p.dqk; i += kGenThreads) {
      const int r = i / p.dqk, d = i - r * p.dqk;
      q_s[i] = to_f32<T>(reinterpret_cast<const T*>(p.q.ptr)[(int64_t)z * p.q.s[0] + (int64_t)rows.head(p, hk, r) * p.q.s[1] + (int64_t)rows.query(r) * p.q.s[2] + d]);
    }
    if (tid < kGenRows) { m_s[tid] = -INFINITY; l_s[tid] = 0.f; }
    float acc[kGenRows][J];
#pragma unroll
    for (int r = 0; r < kGenRows; ++r)
#pragma unroll
      for (int j = 0; j < J; ++j) acc[r][j] = 0.f;
    auto place_of = [&](int n, int64_t& at_k, int64_t& at_v) {
      at_k = at_v = -1;
      if (!w.seen(p, n)) return;
      const int page = (int)((unsigned)n / (unsigned)p.page), in = n - page * p.page, id = p.table[(int64_t)z * p.table_stride + page];
      if (id < 0 || id >= p.num_pages) return;
      at_k = id * p.k.s[0] + in * p.k.s[1] + hk * p.k.s[2];
      at_v = id * p.v.s[0] + in * p.v.s[1] + hk * p.v.s[2];
    };
    if (tid < kGenKeys) place_of(w.tile(first) * kGenKeys + tid, places_k[first % 3][tid], places_v[first % 3][tid]);
    __syncthreads();
    for (int i = first; i < last; ++i) {
      const int n0 = w.tile(i) * kGenKeys;
      const int64_t *at_k = places_k[i % 3], *at_v = places_v[i % 3];
      float(*s)[kGenKeys] = scores[i & 1];
      float* alpha = alphas[i & 1];
      int64_t next_k = -1, next_v = -1;      // (looked up while the keys are on their way)
      if (tid < kGenKeys && i + 1 < last) place_of(w.tile(i + 1) * kGenKeys + tid, next_k, next_v);
      {
        const int key = tid >> 3, l8 = tid & 7;
        const int64_t place = at_k[key];
        float dot[kGenRows];
#pragma unroll
        for (int r = 0; r < kGenRows; ++r) dot[r] = 0.f;
        if (place >= 0) {
          const T* kr = reinterpret_cast<const T*>(p.k.ptr) + place;
          constexpr int kAhead = 4;      // vectors of a lane on the way at a time
          for (int d0 = l8 * N; d0 < p.dqk; d0 += 8 * N * kAhead) {
            float x[kAhead][N];
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
              if (d0 + 8 * N * a < p.dqk) load_vec<T, N>(kr + d0 + 8 * N * a, x[a]);
              else
#pragma unroll
                for (int e = 0; e < N; ++e) x[a][e] = 0.f;
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
              const int d = d0 + 8 * N * a;
              if (d >= p.dqk) break;
#pragma unroll
              for (int r = 0; r < kGenRows; ++r) {
                if (r >= rows.n) break;
                const float* q = q_s + r * p.dqk + d;
                if constexpr (N % 4 == 0) {
#pragma unroll
                  for (int e = 0; e < N; e += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(q + e);
                    dot[r] = fmaf(y.x, x[a][e], dot[r]);
                    dot[r] = fmaf(y.y, x[a][e + 1], dot[r]);
                    dot[r] = fmaf(y.z, x[a][e + 2], dot[r]);
                    dot[r] = fmaf(y.w, x[a][e + 3], dot[r]);
                  }
                } else {
#pragma unroll
                  for (int e = 0; e < N; ++e) dot[r] = fmaf(q[e], x[a][e], dot[r]);
                }
              }
            }
          }
        }
#pragma unroll
        for (int r = 0; r < kGenRows; ++r) {
          if (r >= rows.n) break;
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) dot[r] += __shfl_xor_sync(0xffffffffu, dot[r], o);
          if (l8 == 0) s[r][key] = dot[r];
        }
      }
      if (tid < kGenKeys) { places_k[(i + 1) % 3][tid] = next_k; places_v[(i + 1) % 3][tid] = next_v; }
      __syncthreads();
      for (int r = warp; r < rows.n; r += kGenThreads / 32) {
        const int n = n0 + lane;
        const int64_t pos = (int64_t)w.len - w.queries + rows.query(r);
        const bool ok = at_k[lane] >= 0 && n <= pos && (n > pos - p.window || n < p.sinks);
        const float x = ok ? s[r][lane] * p.qk_scale : -INFINITY;
        float mx = x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float was = m_s[r], now = fmaxf(was, mx), ref = now == -INFINITY ? 0.f : now;
        const float e = exp2f(x - ref);
        float sum = e;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        s[r][lane] = e;
        __syncwarp();
        if (lane == 0) {
          alpha[r] = exp2f(was - ref);
          m_s[r] = now;
          l_s[r] = l_s[r] * alpha[r] + sum;
        }
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kGenRows; ++r)
        if (r < rows.n)
#pragma unroll
          for (int j = 0; j < J; ++j) acc[r][j] *= alpha[r];
      constexpr int kKeysAhead = J > 1 ? 4 : 8;      // values of a thread on the way at a time
      for (int k0 = group; k0 < kGenKeys; k0 += groups * kKeysAhead) {
        float x[kKeysAhead][J];
#pragma unroll
        for (int u = 0; u < kKeysAhead; ++u) {
          const int key = k0 + u * groups;
          const int64_t place = key < kGenKeys ? at_v[key] : -1;
          const T* vr = reinterpret_cast<const T*>(p.v.ptr) + place;
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const int d = col + j * kGenThreads;
            x[u][j] = place >= 0 && d < p.dvo ? to_f32<T>(vr[d]) : 0.f;
          }
        }
#pragma unroll
        for (int u = 0; u < kKeysAhead; ++u) {
          const int key = k0 + u * groups;
          if (key >= kGenKeys) break;
#pragma unroll
          for (int r = 0; r < kGenRows; ++r) {
            if (r >= rows.n) break;
            const float e = s[r][key];
#pragma unroll
            for (int j = 0; j < J; ++j) acc[r][j] = fmaf(e, x[u][j], acc[r][j]);
          }
        }
      }
    }
    __syncthreads();
    if constexpr (J == 1) {      // the groups' sums, in their order
      if (groups > 1) {
#pragma unroll
        for (int r = 0; r < kGenRows; ++r) meet[r * kGenThreads + tid] = acc[r][0];
        __syncthreads();
        if (group == 0)
#pragma unroll
          for (int r = 0; r < kGenRows; ++r)
            for (int g = 1; g < groups; ++g) acc[r][0] += meet[r * kGenThreads + g * width + col];
        __syncthreads();
      }
    }
    float* part = partial_of(p, c);
#pragma unroll
    for (int r = 0; r < kGenRows; ++r) {
      if (r >= rows.n) continue;
      const float l = l_s[r], inv = l > 0.f ? 1.f / l : 0.f;
      const int h = rows.head(p, hk, r), m = rows.query(r);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int d = col + j * kGenThreads;
        if (group != 0 || d >= p.dvo) continue;
        if (whole) out_row<T>(p, z, h, m)[d] = from_f32<T>(acc[r][j] * inv);
        else part[r * p.dvo + d] = acc[r][j];
      }
      if (tid == 0) {
        if (whole) put_lse(p, z, h, m, m_s[r], l);
        else { part[p.rows * p.dvo + r] = m_s[r]; part[p.rows * p.dvo + p.rows + r] = l; }
      }
    }
  }
}

// ---- the pieces of split units ----------------------------------------------------------------------------------------
// A warp takes 32 K vectors of a row; it weighs the pieces' rows by their maxima and adds them up in the order of the keys, several of them on the way at a
// time: what bounds it is how many loads stand one behind another.  V: float4, or float where the columns are not a multiple of 4.  K: 1 while there are
// too few rows to fill the GPU, 4 beyond (one sequence of 32768 keys, 128 heads of 512, 51 us with 4, 40 with 1; 128 short ones 70 and 78).
// grid = (batch * hk * chunks, some): a unit's blocks take its rows' pieces, `widths` a row, in turn.
constexpr int kJoinThreads = 128, kJoinWarps = kJoinThreads / 32, kJoinBlocks = 4736;      // (32 for each SM)

__device__ __forceinline__ void add_weighed(float& a, float w, const float& x) { a = fmaf(w, x, a); }
__device__ __forceinline__ void add_weighed(float4& a, float w, const float4& x) {
  a.x = fmaf(w, x.x, a.x); a.y = fmaf(w, x.y, a.y); a.z = fmaf(w, x.z, a.z); a.w = fmaf(w, x.w, a.w);
}

template <typename T, typename V, int K>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedAttn p, int widths) {
  constexpr int N = sizeof(V) / 4, kAhead = K > 1 ? 4 : 8;
  __shared__ int scratch[kJoinThreads / 32 + 2];
  const int tid = threadIdx.x, lane = tid & 31, units = p.hk * p.chunks;
  // (the lengths are older than the attention's launch, which has waited for what was ahead of it: the places are worked out while that still runs)
  const int z = (int)(blockIdx.x / (unsigned)units), u = (int)(blockIdx.x - (unsigned)z * units);
  const Line line = find_in_line<kJoinThreads>(p, z, 0, scratch);
  const Walk w(p, z);
  const int hk = u / p.chunks, chunk = u - hk * p.chunks, along = hk * (p.chunks / p.lanes) + chunk / p.lanes;
  const Rows rows(p, w, chunk);
  int c0, c1;
  pieces_of_unit(p, line, w, along, c0, c1);
  wait_for_earlier_grids();
  if (c0 == c1) return;      // (the unit was finished where it was formed)
  const unsigned int failed = p.status != nullptr ? *reinterpret_cast<volatile unsigned int*>(p.status) : 0u;
  const int64_t step = 2 * (int64_t)p.lanes * partial_floats(p);
  // (of the first piece the second place, of the others the first)
  const float* head = partial_of(p, 2 * ((int64_t)c0 * p.lanes + chunk % p.lanes) + 1);
  auto piece = [&](int i) { return i == 0 ? head : head + i * step - partial_floats(p); };
  const int n = c1 - c0 + 1;
  for (int job = blockIdx.y * kJoinWarps + tid / 32; job < rows.n * widths; job += gridDim.y * kJoinWarps) {
    const int r = (int)((unsigned)job / (unsigned)widths), d = ((job - r * widths) * 32 * K + lane) * N;
    const int64_t at_m = (int64_t)p.rows * p.dvo + r, at_l = at_m + p.rows, at_o = (int64_t)r * p.dvo;
    // the row's maximum, and of up to 32 pieces what each lane's weighs
    float m0 = -INFINITY, l0 = 0.f;
    if (lane < n) { m0 = piece(lane)[at_m]; l0 = piece(lane)[at_l]; }
    float mx = m0;
    for (int i = lane + 32; i < n; i += 32) mx = fmaxf(mx, piece(i)[at_m]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float ref = mx == -INFINITY ? 0.f : mx;
    V acc[K];
#pragma unroll
    for (int k = 0; k < K; ++k) acc[k] = V{};
    float l = 0.f;
    for (int from = 0; from < n; from += 32) {
      if (from > 0) {
        m0 = -INFINITY;
        l0 = 0.f;
        if (from + lane < n) { m0 = piece(from + lane)[at_m]; l0 = piece(from + lane)[at_l]; }
      }
      const float weight = exp2f(m0 - ref);
      l = fmaf(weight, l0, l);
      const int here = min(32, n - from);
      for (int i = 0; i < here; i += kAhead) {
        V x[kAhead][K];      // (all of them asked for ahead of the first use: behind the last piece and the last column, the last again)
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const float* row = piece(from + min(i + a, here - 1)) + at_o;
#pragma unroll
          for (int k = 0; k < K; ++k) x[a][k] = *reinterpret_cast<const V*>(row + min(d + 32 * N * k, p.dvo - N));
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const float f = __shfl_sync(0xffffffffu, weight, (i + a) & 31);
          if (i + a < here)
#pragma unroll
            for (int k = 0; k < K; ++k) add_weighed(acc[k], f, x[a][k]);
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (failed != 0u) return;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int h = rows.head(p, hk, r), m = rows.query(r);
    T* out = out_row<T>(p, z, h, m);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float* e = reinterpret_cast<const float*>(&acc[k]);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (d + 32 * N * k < p.dvo) out[d + 32 * N * k + j] = from_f32<T>(e[j] * inv);
    }
    if (d == 0) put_lse(p, z, h, m, mx, l);
  }
}

// ---- keys that share columns --------------------------------------------------------------------------------------
// out[b, h, s] = (k[b, h, s], shared[b, 0, s]): rows moved as they are, bound by their bytes.  V: the vector that all rows allow.  A block takes the
// vectors of a token's heads, each thread four at a time whose loads are on the way together; the shared ones are read again for each head, out of L1.
// grid = (batch * tokens, some)
constexpr int kColumnThreads = 128, kColumnBatch = 4;

template <typename V>
__global__ void __launch_bounds__(kColumnThreads) join_columns_kernel(const __grid_constant__ SharedColumns a, int elt) {
  wait_for_earlier_grids();
  const int per = (int)sizeof(V) / elt, vn = (int)a.k.n[3] / per, wide = vn + (int)a.shared.n[3] / per, items = (int)a.out.n[1] * wide;
  const int b = (int)(blockIdx.x / (unsigned)a.out.n[2]), s = (int)(blockIdx.x - (unsigned)b * (unsigned)a.out.n[2]);
  const char* k = reinterpret_cast<const char*>(a.k.ptr) + (b * a.k.s[0] + s * a.k.s[2]) * elt;
  const char* shared = reinterpret_cast<const char*>(a.shared.ptr) + (b * a.shared.s[0] + s * a.shared.s[2]) * elt;
  char* out = reinterpret_cast<char*>(a.out.ptr) + (b * a.out.s[0] + s * a.out.s[2]) * elt;
  for (int i0 = blockIdx.y * kColumnThreads * kColumnBatch + threadIdx.x; i0 < items; i0 += gridDim.y * kColumnThreads * kColumnBatch) {
    V x[kColumnBatch];
    V* to[kColumnBatch];
#pragma unroll
    for (int j = 0; j < kColumnBatch; ++j) {
      const int i = i0 + j * kColumnThreads, h = (int)((unsigned)i / (unsigned)wide), c = i - h * wide;
      to[j] = nullptr;
      if (i >= items) continue;
      x[j] = *reinterpret_cast<const V*>(c < vn ? k + h * a.k.s[1] * elt + (int64_t)c * sizeof(V) : shared + (int64_t)(c - vn) * sizeof(V));
      to[j] = reinterpret_cast<V*>(out + h * a.out.s[1] * elt + (int64_t)c * sizeof(V));
    }
#pragma unroll
    for (int j = 0; j < kColumnBatch; ++j)
      if (to[j] != nullptr) *to[j] = x[j];
  }
}

// Whether token `s` of batch element `b` is a key of a sequence.  dK's kernels write those alone, so that nothing is summed for the others.
__device__ __forceinline__ bool of_a_sequence(const KeyTokens& t, int64_t b, int64_t s) {
  if (t.varlen_mode == 0) return b < t.batch && s < t.max_sk;
  if (t.varlen_mode == 2) return b < t.batch && s < min(t.cu_k[b + 1] - t.cu_k[b], t.max_sk);
  const int32_t* starts = t.ss_k != nullptr ? t.ss_k : t.cu_k;
  int lo = 0;      // the last sequence that starts at or ahead of the token: of those that start together all but the last are empty
  for (int hi = t.batch - 1; lo < hi;) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= s) lo = mid;
    else hi = mid - 1;
  }
  return b == 0 && t.batch > 0 && s >= starts[lo] && s - starts[lo] < min(t.cu_k[lo + 1] - t.cu_k[lo], t.max_sk);
}

// shared[b, 0, s, c] = sum over the heads of out[b, h, s, dn + c], in their order, in 32 bits, rounded once.
template <typename T>
__global__ void __launch_bounds__(256) sum_columns_kernel(const __grid_constant__ SharedColumns a) {
  wait_for_earlier_grids();
  const int dr = (int)a.shared.n[3];
  const int64_t dn = a.out.n[3] - dr, total = a.shared.n[0] * a.shared.n[2] * dr;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / dr, b = row / a.shared.n[2], s = row - b * a.shared.n[2];
    const int c = (int)(i - row * dr);
    const T* src = reinterpret_cast<const T*>(a.out.ptr) + b * a.out.s[0] + s * a.out.s[2] + dn + c;
    float sum = 0.f;
    const int heads = of_a_sequence(a.tokens, b, s) ? (int)a.out.n[1] : 0;
#pragma unroll 8
    for (int h = 0; h < heads; ++h) sum += to_f32<T>(src[(int64_t)h * a.out.s[1]]);
    reinterpret_cast<T*>(a.shared.ptr)[b * a.shared.s[0] + s * a.shared.s[2] + c] = from_f32<T>(sum);
  }
}

// ... from columns in 32 bits, heads * rows * dr of them a batch element, dr a multiple of 4.  Many heads' loads on the way at a time: one by one and four bytes
// each, 32 heads x 4096 x 64 took 23 us.
template <typename T>
__global__ void __launch_bounds__(128) sum_tail_kernel(const __grid_constant__ SharedColumns a, const float* __restrict__ tail, int heads) {
  wait_for_earlier_grids();
  const View4& shared = a.shared;
  const int dr = (int)shared.n[3];
  const int64_t a_head = shared.n[2] * dr / 4, total = shared.n[0] * a_head;
  for (int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 128) {
    const int64_t b = i / a_head, at = i - b * a_head, s = at * 4 / dr;
    const float4* src = reinterpret_cast<const float4*>(tail) + b * heads * a_head + at;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const int terms = of_a_sequence(a.tokens, b, s) ? heads : 0;
#pragma unroll 16
    for (int h = 0; h < terms; ++h) {
      const float4 x = __ldcs(src + h * a_head);
      sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
    }
    T* dst = reinterpret_cast<T*>(shared.ptr) + b * shared.s[0] + s * shared.s[2] + (at * 4 - s * dr);
    dst[0] = from_f32<T>(sum.x); dst[1] = from_f32<T>(sum.y); dst[2] = from_f32<T>(sum.z); dst[3] = from_f32<T>(sum.w);
  }
}

unsigned grid_for(int64_t items, int64_t per) { return (unsigned)std::min<int64_t>((items + per - 1) / per, 0x7fffffff); }

template <typename... K, typename... A>
cudaError_t launch_counted(void (*kernel)(K...), dim3 grid, int threads, size_t smem, cudaStream_t st, A&&... args) {
  const cudaError_t e = launch_kernel(kernel, grid, dim3(threads), smem, st, std::forward<A>(args)...);
  if (e == cudaSuccess) count_launch();
  return e;
}

bool vec_rows(const View4& v, int elements) {
  if (reinterpret_cast<uintptr_t>(v.ptr) % 16 != 0 || v.n[3] % elements != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (v.n[i] > 1 && v.s[i] % elements != 0) return false;
  return true;
}

template <typename T, int N, int J>
cudaError_t launch_general_NJ(const PagedAttn& p, cudaStream_t st) {
  return launch_counted(paged_general_kernel<T, N, J>, dim3(p.ctas), kGenThreads, (size_t)kGenRows * p.dqk * sizeof(float), st, p);
}
template <typename T>
cudaError_t launch_general_T(const PagedAttn& p, cudaStream_t st) {
  constexpr int N = 16 / (int)sizeof(T);
  const bool vec = vec_rows(p.k, N);
  if (p.dvo <= kGenThreads) return vec ? launch_general_NJ<T, N, 1>(p, st) : launch_general_NJ<T, 1, 1>(p, st);
  return vec ? launch_general_NJ<T, N, 4>(p, st) : launch_general_NJ<T, 1, 4>(p, st);
}
template <typename T, typename V, int K>
cudaError_t launch_join_K(const PagedAttn& p, cudaStream_t st) {
  const int per = 32 * K * (int)(sizeof(V) / 4), widths = (p.dvo + per - 1) / per;
  const int64_t units = (int64_t)p.batch * p.hk * p.chunks, jobs = std::min<int64_t>(p.rows, (int64_t)p.group * p.sq) * widths;
  const int64_t blocks = std::max<int64_t>(1, std::min((jobs + kJoinWarps - 1) / kJoinWarps, kJoinBlocks / units));
  return launch_counted(paged_join_kernel<T, V, K>, dim3((unsigned)units, (unsigned)blocks), kJoinThreads, 0, st, p, widths);
}
template <typename T>
cudaError_t launch_join_T(const PagedAttn& p, cudaStream_t st) {
  if (p.dvo % 4 != 0) return launch_join_K<T, float, 1>(p, st);
  const int64_t warps = (int64_t)p.batch * p.hk * p.group * p.sq * ((p.dvo + 127) / 128);
  return warps > kJoinBlocks && p.dvo > 128 ? launch_join_K<T, float4, 4>(p, st) : launch_join_K<T, float4, 1>(p, st);
}

template <typename F>
auto with_type(int dtype, F f) {
  switch (dtype) {
    case 1: return f.template operator()<float>();
    case 2: return f.template operator()<__half>();
    default: return f.template operator()<__nv_bfloat16>();
  }
}

}  // namespace

cudaError_t launch_block_tables(const BlockTables& a, cudaStream_t st) {
  return launch_counted(a.total > (int64_t)8 * a.batch ? block_tables_kernel<4> : block_tables_kernel<1>, dim3(std::max(1u, grid_for(a.total, kTableTokens))),
                        kTableThreads, 0, st, a);
}

cudaError_t launch_paged_write(int dtype, const PagedWrite& a, cudaStream_t st) {
  const int elt = dtype == 1 ? 4 : 2, per = a.vec / elt;
  const int64_t vectors = a.tokens * a.heads * ((a.dk + a.dv) / per);
  if (vectors == 0) return cudaSuccess;
  const dim3 grid(grid_for(vectors, (int64_t)kWriteThreads * kWriteBatch));
  auto launch = [&]<typename I>() {
    switch (a.vec) {
      case 16: return launch_counted(paged_write_kernel<uint4, I>, grid, kWriteThreads, 0, st, a, elt, (I)vectors);
      case 4: return launch_counted(paged_write_kernel<uint32_t, I>, grid, kWriteThreads, 0, st, a, elt, (I)vectors);
      default: return launch_counted(paged_write_kernel<uint16_t, I>, grid, kWriteThreads, 0, st, a, elt, (I)vectors);
    }
  };
  // (room for the last block's indices)
  return vectors < 0x7fff0000 && a.slots_total < 0x7fff0000 ? launch.template operator()<uint32_t>() : launch.template operator()<int64_t>();
}

int64_t plan_paged(int dtype, PagedAttn& p, int sms) {
  if (!plan_paged_latent(dtype, p, sms) && !plan_paged_split(dtype, p, sms)) {
    p.kind = kPagedGeneral;
    p.rows = kGenRows;
    p.tile_log = 5;
    p.min_tiles = 2;
    p.extra = 1;
    p.ctas = sms * gen_blocks(p.dvo <= kGenThreads ? 1 : 4);
  }
  const int64_t chunks = ((int64_t)p.group * p.sq + p.rows - 1) / p.rows;
  p.chunks = (int)chunks;
  // (a last tile's keys are counted in 32 bits)
  p.max_len = (int32_t)std::min<int64_t>((int64_t)p.width * p.page, 0x7fffff00);
  const int64_t most = (p.max_len >> p.tile_log) + 2 + p.extra;      // tiles of a unit: a window may cross a border
  // What the tables have room for is all that is known here of the lengths: where that is more than 31 bits count, a few launches take some sequences each.
  const int64_t fit = 0x3fffffff / ((int64_t)p.hk * chunks * most);
  if (fit == 0) return -kPagedTooLarge;
  const int64_t launches = (p.batch + fit - 1) / fit;
  p.slice = (int32_t)((p.batch + launches - 1) / launches);
  const int64_t units = (int64_t)p.slice * p.hk * chunks;
  // A kv head's chunks side by side, so that its keys come from memory once, unless that left too few CTAs to share a line out evenly.
  p.lanes = chunks <= 8 ? (int)chunks : 1;
  p.ctas = (int)std::max<int64_t>(1, std::min<int64_t>(p.ctas / p.lanes, units / p.lanes * most / p.min_tiles + 1)) * p.lanes;
  return 2 * (int64_t)p.ctas * partial_floats(p);
}

static cudaError_t launch_paged_slice(int dtype, PagedAttn& p, cudaStream_t st) {
  cudaError_t e = p.kind == kPagedSplit    ? launch_paged_split(dtype, p, st)
                  : p.kind == kPagedLatent ? launch_paged_latent(dtype, p, st)
                                           : with_type(dtype, [&]<typename T>() { return launch_general_T<T>(p, st); });
  if (e == cudaSuccess) e = with_type(dtype, [&]<typename T>() { return launch_join_T<T>(p, st); });
  return e;
}
cudaError_t launch_paged(int dtype, PagedAttn& p, cudaStream_t st) {
  if (p.slice >= p.batch) return launch_paged_slice(dtype, p, st);
  const int64_t elt = dtype == 1 ? 4 : 2;
  for (int z = 0; z < p.batch; z += p.slice) {      // (one behind the other: they share the workspace)
    PagedAttn s = p;
    s.batch = std::min(p.slice, p.batch - z);
    for (View4* v : {&s.q, &s.out}) {
      v->ptr = static_cast<char*>(v->ptr) + z * v->s[0] * elt;
      v->n[0] = s.batch;
    }
    s.table += z * p.table_stride;
    s.lengths += z;
    if (s.query_lengths != nullptr) s.query_lengths += z;
    if (s.lse != nullptr) s.lse += (int64_t)z * p.hq * p.sq;
    if (const cudaError_t e = launch_paged_slice(dtype, s, st)) return e;
  }
  return cudaSuccess;
}

cudaError_t launch_join_columns(int dtype, const SharedColumns& a, cudaStream_t st) {
  const int elt = dtype == 1 ? 4 : 2;
  const bool vec = vec_rows(a.k, 16 / elt) && vec_rows(a.shared, 16 / elt) && vec_rows(a.out, 16 / elt);
  const int64_t items = a.out.n[1] * (a.out.n[3] / (vec ? 16 / elt : 1));
  const dim3 grid((unsigned)(a.out.n[0] * a.out.n[2]), (unsigned)std::min<int64_t>(65535, (items + kColumnThreads * kColumnBatch - 1) / (kColumnThreads * kColumnBatch)));
  if (vec) return launch_counted(join_columns_kernel<uint4>, grid, kColumnThreads, 0, st, a, elt);
  if (elt == 4) return launch_counted(join_columns_kernel<uint32_t>, grid, kColumnThreads, 0, st, a, elt);
  return launch_counted(join_columns_kernel<uint16_t>, grid, kColumnThreads, 0, st, a, elt);
}

cudaError_t launch_sum_tail(int dtype, const SharedColumns& a, const float* tail, int heads, cudaStream_t st) {
  const dim3 grid(grid_for(a.shared.n[0] * a.shared.n[2] * a.shared.n[3], 512));
  return with_type(dtype, [&]<typename T>() { return launch_counted(sum_tail_kernel<T>, grid, 128, 0, st, a, tail, heads); });
}

cudaError_t launch_sum_columns(int dtype, const SharedColumns& a, cudaStream_t st) {
  const dim3 grid(grid_for(a.shared.n[0] * a.shared.n[2] * a.shared.n[3], 256));
  return with_type(dtype, [&]<typename T>() { return launch_counted(sum_columns_kernel<T>, grid, 256, 0, st, a); });
}

}  // namespace ab200
