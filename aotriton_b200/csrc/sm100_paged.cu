// Attention of a few queries over a paged cache, fp16 and bf16, head dims up to 128.
//
// What bounds it: reading each key and value that is seen once, at the memory's rate.  So
//   * the query heads of a kv head, times the queries, are the rows of one tile (row r = head r / queries of the group, query r % queries), 16 or 32 of
//     them, and the products run as warp-level MMAs: a 128-row tensor-memory tile would be padding;
//   * the cache is streamed in tiles of 64 keys through a ring of TMA copies.  A tile is put together of boxes of as many slots as pages and tiles
//     have in common (64 slots of a page of 64, four boxes of 16 of pages of 16), each at its page's place: eight lanes of the producing
//     warp look up a page each, one tile ahead, and each issues its own copies.  Boxes that nobody sees -- behind the sequence, out of the window, of a page outside
//     the cache -- are copies of a page that does not exist: zeros, without a read;
//   * the ring knows no sequences: the producer runs ahead into the next unit while the consumers finish one, and paged_split.cuh gives every CTA the
//     same number of tiles whatever the lengths;
//   * four warps take 16 keys of a tile each with a softmax of their own, and meet at the end of a unit, 32 columns of the output at a time, so that
//     the ring keeps its room.
// Arithmetic: scores times sm_scale * log2(e) in fp32, hidden ones -inf, weights rounded to the value type before P V (half a step off each; the sum
// keeps 32 bits), fp32 sums.
// Measured, us of device a call with the join: 64 sequences of 100 to 8192 keys, 32:8 heads of 128, 167 (6.2 TB/s, 95 % of a copy's rate); 4 of about 110000 keys 286 (6.5);
// one of 1500 10.5, of which the places 1.1, queries and first tile 1.6, two tiles 1.3, the results 1.4 and the join 3; 24 of 40 to 6007 keys, four queries of 16:8
// heads of 64, window 2048, 26; with 32 rows a tile and heads of 128 (one CTA an SM, 255 registers) 32 of 100 to 8192, three queries of 64:8 heads, 209 (floor 83).
#include <atomic>
#include "launch.h"
#include "paged.h"
#include "paged_split.cuh"
#include "sm100_ptx.cuh"
#include "warp_mma.cuh"

namespace ab200 {

__device__ unsigned int g_sm100_paged_status = 0;

namespace {
using namespace ptx;

constexpr int kTileKeys = 64, kTileLog = 6, kConsumers = 4, kSplitThreads = (kConsumers + 1) * 32;
constexpr int kMergeCols = 32;

template <int HD, int MT>
struct SplitSmem {
  static constexpr int kRows = 16 * MT, kCtasPerSm = HD > 64 && MT > 1 ? 1 : 2;
  static constexpr int kTile = (HD / 64) * kTileKeys * 128;      // 64-column boxes, 128-byte rows
  static constexpr int kStages = HD > 64 ? (MT > 1 ? 6 : 3) : (MT > 1 ? 5 : 6);
  static constexpr int bFull = 0, bEmpty = kStages, bCount = 2 * kStages;
  static constexpr int kAbort = bCount * 8;
  static constexpr int kValid = kAbort + 8;                       // per stage: which eights of its keys are in the cache
  static constexpr int kScratch = (kValid + kStages * 4 + 15) & ~15;
  static constexpr int kMl = kScratch + (kSplitThreads / 32 + 3) * 4;
  static constexpr int kLdO = kMergeCols + 4;
  static constexpr int kMerge = (kMl + kConsumers * 2 * kRows * 4 + 15) & ~15;
  static constexpr int kRing = (kMerge + kConsumers * kRows * kLdO * 4 + 1023) & ~1023;
  static constexpr int kBytes = kRing + kStages * 2 * kTile + 1024;
  static_assert(kBytes <= (kCtasPerSm == 2 ? 115712 : 232448), "fits");
};

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); }
// ... and whether any of them says so
__device__ __forceinline__ bool consumers_any(bool x) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.b32 a, %1, 0;\n\tbarrier.cta.red.or.pred b, 1, %2, a;\n\tselp.b32 %0, 1, 0, b;\n\t}"
               : "=r"(r) : "r"((uint32_t)x), "n"(kConsumers * 32) : "memory");
  return r != 0;
}

template <typename T, int HD, int MT>
__global__ void __launch_bounds__(kSplitThreads, SplitSmem<HD, MT>::kCtasPerSm)
paged_split_kernel(const __grid_constant__ PagedAttn p, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  using L = SplitSmem<HD, MT>;
  constexpr int kBoxes = HD / 64, kKsteps = HD / 16, kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kAbort);
  volatile uint32_t* valid = reinterpret_cast<volatile uint32_t*>(smem + L::kValid);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) { prefetch_tmap(&tm_k); prefetch_tmap(&tm_v); }
  wait_for_earlier_grids();
  const unsigned int failed = tid == 0 ? *reinterpret_cast<volatile unsigned int*>(p.status) : 0u;
  if (tid == 0) {
    init_abort_and_limit(abort_flag, p.wait_limit_kcycles);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars[L::bFull + s], 1);
      mbar_init(&bars[L::bEmpty + s], kConsumers);
    }
    fence_barrier_init();
  }
  const Line line = find_in_line<kSplitThreads>(p, -1, blockIdx.x / p.lanes, reinterpret_cast<int*>(smem + L::kScratch));
  if (__syncthreads_or(failed != 0u)) return;
  if (line.z >= p.batch) return;
  Piece run(p, line);
  const Walk& w = run.w;

  if (warp == kConsumers) {
    // ================================ TMA producer ===================================
    const int octets = p.box / 8, group = lane / octets;      // a box's eights of keys
    const uint32_t mine = lane < 8 ? ((octets == 8 ? 0xffu : (1u << octets) - 1u) << (group * octets)) & 0xffu : 0u;
    int s = 0, ph = 1, issued = 0;
    bool stop = false, dropped = false;
    while (!stop && run.next(p)) {
      if (Rows(p, w, run.chunk).n == 0) continue;
      const int first = run.first, last = run.last, hk = run.hk;
      const int32_t* row = p.table + (int64_t)run.z * p.table_stride;
      // the page of this lane's eight keys in tile i, -1 where there is none; `seen`: whether any of them is seen
      auto look = [&](int i, bool& seen) {
        const int n = w.tile(i) * kTileKeys + lane * 8;
        seen = false;
        if (lane >= 8 || n >= w.len) return -1;
        seen = n < p.sinks || n + 7 >= w.lo;
        return row[n / p.page];
      };
      bool seen;
      int id = look(first, seen);
      for (int i = first; i < last; ++i) {
        const bool ok = seen && id >= 0 && id < p.num_pages;
        const uint32_t bits = __ballot_sync(0xffffffffu, ok);
        const int page = (bits & mine) != 0u ? id : p.num_pages;      // (a page that does not exist: zeros)
        const int slot = (w.tile(i) * kTileKeys + lane * 8) % p.page;
        if (i + 1 < last) id = look(i + 1, seen);
        if (!__all_sync(0xffffffffu, mbar_wait(&bars[L::bEmpty + s], (uint32_t)ph, abort_flag, p.status, 0x6000))) { stop = true; break; }
        const bool drop = p.drop_copy == 1 && run.z == 0 && run.hk == 0 && run.chunk == 0 && i == 0;      // (test hook: the first tile never arrives)
        dropped |= drop;
        if (!drop) {
          uint8_t* kt = smem + L::kRing + s * (2 * L::kTile);
          if (lane == 0) {
            valid[s] = bits;
            mbar_expect_tx(&bars[L::bFull + s], 2 * L::kTile);
          }
          __syncwarp();
          if (lane < 8 && lane % octets == 0) {
#pragma unroll
            for (int b = 0; b < kBoxes; ++b) tma_load_4d(kt + b * (kTileKeys * 128) + lane * 1024, &tm_k, &bars[L::bFull + s], b * 64, slot, hk, page);
#pragma unroll
            for (int b = 0; b < kBoxes; ++b)
              tma_load_4d(kt + L::kTile + b * (kTileKeys * 128) + lane * 1024, &tm_v, &bars[L::bFull + s], b * 64, slot, hk, page);
          }
        }
        ++issued;
        if (++s == kStages) { s = 0; ph ^= 1; }
      }
    }
    __syncwarp();
    if (*abort_flag && lane == 0) {      // copies that are still in flight land before the memory is used again
      for (int i = max(dropped ? 1 : 0, issued - kStages); i < issued; ++i)
        mbar_wait_quiet(&bars[L::bFull + i % kStages], (uint32_t)(i / kStages) & 1u, abort_flag);
    }
    return;
  }

  // ================================== consumers =====================================
  const int qr = lane >> 2, qc = (lane & 3) * 2;      // this lane's row (and row + 8) and column pair in a fragment
  const uint32_t smem_s = smem_u32(smem);
  // ldmatrix addresses inside a tile: 128-byte rows, 16-byte chunks XOR-swizzled with the row (the TMA layout).
  const int krow = warp * 16 + (lane & 7) + ((lane >> 4) << 3), kchunk = (lane >> 3) & 1;
  const int vrow = warp * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), vchunk = lane >> 4;
  float* ml = reinterpret_cast<float*>(smem + L::kMl);
  float* merge = reinterpret_cast<float*>(smem + L::kMerge);
  int s = 0, ph = 0;
  bool broken = false;
  while (!broken && run.next(p)) {
    const int z = run.z, hk = run.hk, first = run.first, last = run.last;
    const Rows rows(p, w, run.chunk);
    if (first == 0 && run.chunk == 0) zero_rows_behind<T, kConsumers * 32>(p, w, z, hk, tid);
    if (rows.n == 0) continue;
    // Q as A fragments, straight from global memory (rows and columns beyond the ends are zero)
    uint32_t q[MT][kKsteps][4];
    int row_lo[2 * MT], row_hi[2 * MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = t * 16 + half * 8 + qr;
        const bool in = r < rows.n;
        const int h = rows.head(p, hk, in ? r : 0), m = rows.query(in ? r : 0);
        const T* qp = reinterpret_cast<const T*>(p.q.ptr) + (int64_t)z * p.q.s[0] + (int64_t)h * p.q.s[1] + (int64_t)m * p.q.s[2];
#pragma unroll
        for (int kk = 0; kk < kKsteps; ++kk)
#pragma unroll
          for (int c8 = 0; c8 < 2; ++c8) {
            const int d = kk * 16 + c8 * 8 + qc;
            q[t][kk][c8 * 2 + half] = (in && d < p.dqk) ? __ldg(reinterpret_cast<const uint32_t*>(qp + d)) : 0u;
          }
        const int pos = in ? w.len - rows.queries + m : -1;
        const int64_t lo = (int64_t)pos - p.window + 1;
        row_hi[2 * t + half] = pos;
        row_lo[2 * t + half] = lo > 0 ? (int)lo : 0;
      }
    float m_run[2 * MT], l_run[2 * MT], o[MT][2 * kKsteps][4];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      m_run[2 * t] = m_run[2 * t + 1] = -INFINITY;
      l_run[2 * t] = l_run[2 * t + 1] = 0.f;
#pragma unroll
      for (int c = 0; c < 2 * kKsteps; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][c][e] = 0.f;
    }
    for (int i = first; i < last; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait(&bars[L::bFull + s], (uint32_t)ph, abort_flag, p.status, 0x6100))) { broken = true; break; }
      const uint32_t here = valid[s] >> (warp * 2);
      const int key0 = w.tile(i) * kTileKeys + warp * 16;      // first key of this warp's 16
      const uint32_t kt = smem_s + L::kRing + s * (2 * L::kTile) + krow * 128;
      const uint32_t vt = smem_s + L::kRing + s * (2 * L::kTile) + L::kTile + vrow * 128;
      if (key0 + 16 > w.len || (key0 < w.lo && key0 + 16 > p.sinks)) {
        // V rows that nobody sees hold whatever the cache has there: a zero weight times a non-finite value would poison the sum
        uint8_t* vtile = smem + L::kRing + s * (2 * L::kTile) + L::kTile + warp * 16 * 128;
#pragma unroll
        for (int r0 = 0; r0 < 16; r0 += 4) {      // (a lane 16 bytes of a row, a warp four rows)
          const int rr = r0 + (lane >> 3);
          if (!w.seen(p, key0 + rr))
#pragma unroll
            for (int b = 0; b < kBoxes; ++b) *reinterpret_cast<uint4*>(vtile + b * (kTileKeys * 128) + rr * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();      // (ahead of the copy that overwrites the stage)
        __syncwarp();
      }
      constexpr int kChains = MT == 1 ? 2 : 1;      // (two accumulators with one tile of rows: half the chain of dependent MMAs)
      float sc[MT][2][4], sc2[2][4];
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[t][0][e] = sc[t][1][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) sc2[0][e] = sc2[1][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < kKsteps; ++kk) {
        uint32_t kb[4];
        const int c = (kk & 3) * 2 + kchunk;
        ldsm4(kb, kt + (kk >> 2) * (kTileKeys * 128) + ((c ^ (krow & 7)) << 4));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const bool second = kChains == 2 && (kk & 1);
          mma_16816<T>(second ? sc2[0] : sc[t][0], q[t][kk], kb[0], kb[1]);
          mma_16816<T>(second ? sc2[1] : sc[t][1], q[t][kk], kb[2], kb[3]);
        }
      }
      if constexpr (kChains == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) { sc[0][0][e] += sc2[0][e]; sc[0][1][e] += sc2[1][e]; }
      }
      uint32_t pa[MT][4];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = key0 + j * 8 + qc + (e & 1), half = e >> 1;
            const bool ok = ((here >> j) & 1u) && n <= row_hi[2 * t + half] && (n >= row_lo[2 * t + half] || n < p.sinks);
            sc[t][j][e] = ok ? sc[t][j][e] * p.qk_scale : -INFINITY;
            mx[half] = fmaxf(mx[half], sc[t][j][e]);
          }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
          mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
        }
        const bool grow = mx[0] > m_run[2 * t] || mx[1] > m_run[2 * t + 1];
        if (__any_sync(0xffffffffu, grow)) {
          float al[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float mn = fmaxf(m_run[2 * t + half], mx[half]);
            al[half] = mn == -INFINITY ? 1.f : ex2(m_run[2 * t + half] - mn);
            m_run[2 * t + half] = mn;
            l_run[2 * t + half] *= al[half];
          }
#pragma unroll
          for (int c = 0; c < 2 * kKsteps; ++c) {
            o[t][c][0] *= al[0]; o[t][c][1] *= al[0];
            o[t][c][2] *= al[1]; o[t][c][3] *= al[1];
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float ms = m_run[2 * t + half] == -INFINITY ? 0.f : m_run[2 * t + half];
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float e0 = ex2(sc[t][j][2 * half] - ms), e1 = ex2(sc[t][j][2 * half + 1] - ms);
            sum += e0 + e1;
            pa[t][2 * j + half] = pack2<T>(e0, e1);
          }
          l_run[2 * t + half] += sum;      // this lane's columns; the quad's sums meet at the end of the unit
        }
      }
#pragma unroll
      for (int c = 0; c < kKsteps; ++c) {      // 16 columns of the head dim per step
        uint32_t vb[4];
        const int ch = (c & 3) * 2 + vchunk;
        ldsm4t(vb, vt + (c >> 2) * (kTileKeys * 128) + ((ch ^ (vrow & 7)) << 4));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          mma_16816<T>(o[t][2 * c], pa[t], vb[0], vb[1]);
          mma_16816<T>(o[t][2 * c + 1], pa[t], vb[2], vb[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[L::bEmpty + s]);
      if (++s == kStages) { s = 0; ph ^= 1; }
    }
    // ---- the four warps' results with a common row maximum ----
    // (a warp whose wait ran out takes the barriers too; they leave together)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float l = l_run[2 * t + half];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if ((lane & 3) == 0) {
          ml[warp * 2 * L::kRows + t * 16 + half * 8 + qr] = m_run[2 * t + half];
          ml[warp * 2 * L::kRows + L::kRows + t * 16 + half * 8 + qr] = l;
        }
      }
    const bool whole = run.whole();
    float* part = partial_of(p, run);
#pragma unroll
    for (int c0 = 0; c0 < HD; c0 += kMergeCols) {
      if (c0 >= p.dvo) break;
      if (c0 > 0) consumers_sync();
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int c = 0; c < kMergeCols / 8; ++c)
            *reinterpret_cast<float2*>(merge + (warp * L::kRows + t * 16 + half * 8 + qr) * L::kLdO + c * 8 + qc) =
                make_float2(o[t][c0 / 8 + c][2 * half], o[t][c0 / 8 + c][2 * half + 1]);
      consumers_sync();
      for (int i = tid; i < rows.n * (kMergeCols / 4); i += kConsumers * 32) {
        const int r = i / (kMergeCols / 4), c = (i % (kMergeCols / 4)) * 4, d = c0 + c;
        float mx = -INFINITY, l = 0.f;
#pragma unroll
        for (int k = 0; k < kConsumers; ++k) mx = fmaxf(mx, ml[k * 2 * L::kRows + r]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kConsumers; ++k) {
          const float a = mx == -INFINITY ? 0.f : ex2(ml[k * 2 * L::kRows + r] - mx);
          const float4 x = *reinterpret_cast<const float4*>(merge + (k * L::kRows + r) * L::kLdO + c);
          acc.x = fmaf(a, x.x, acc.x); acc.y = fmaf(a, x.y, acc.y);
          acc.z = fmaf(a, x.z, acc.z); acc.w = fmaf(a, x.w, acc.w);
          l = fmaf(a, ml[k * 2 * L::kRows + L::kRows + r], l);
        }
        if (d < p.dvo && !*abort_flag) {
          if (whole) {
            const float inv = l > 0.f ? 1.f / l : 0.f;
            const int h = rows.head(p, hk, r), m = rows.query(r);
            *reinterpret_cast<uint2*>(out_row<T>(p, z, h, m) + d) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
            if (d == 0) put_lse(p, z, h, m, mx, l);
          } else {
            *reinterpret_cast<float4*>(part + r * p.dvo + d) = acc;
            if (d == 0) { part[p.rows * p.dvo + r] = mx; part[p.rows * p.dvo + p.rows + r] = l; }
          }
        }
      }
    }
    broken = consumers_any(broken);      // (ml and the merge area are free for the next unit)
  }
}

// A cache as a (pages, heads, slots, columns) view, as the tile maps take it.
View4 as_tiles(const View4& c, int columns) {
  return View4{c.ptr, {c.n[0], c.n[2], c.n[1], columns}, {c.s[0], c.s[2], c.s[1], c.s[3]}};
}

template <typename T, int HD, int MT>
cudaError_t launch_split_T(PagedAttn& p, cudaStream_t st) {
  using L = SplitSmem<HD, MT>;
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  bool remember = false;
  cudaError_t e = paged_status_word(&p.status, &dev, &remember);
  if (e != cudaSuccess) return e;
  auto* kernel = paged_split_kernel<T, HD, MT>;
  if (!remember || !attr_set[dev].load(std::memory_order_acquire)) {
    if ((e = host().func_set_smem(reinterpret_cast<const void*>(kernel), L::kBytes)) != cudaSuccess) return e;
    if (remember) attr_set[dev].store(true, std::memory_order_release);
  }
  CUtensorMap tk, tv;
  const View4 k = as_tiles(p.k, p.dqk), v = as_tiles(p.v, p.dvo);
  if (!make_tile_map_16bit(&tk, k, p.dqk, p.page, p.box) || !make_tile_map_16bit(&tv, v, p.dvo, p.page, p.box)) return cudaErrorInvalidValue;
  e = launch_kernel(kernel, dim3(p.ctas), dim3(kSplitThreads), L::kBytes, st, p, tk, tv);
  if (e == cudaSuccess) count_launch();
  return e;
}

// f<HD, MT>() of the instantiation that takes the call
template <typename F>
auto with_split_tile(const PagedAttn& p, F f) {
  const bool small = p.dqk <= 64 && p.dvo <= 64, one = p.group * p.sq <= 16;
  if (small) return one ? f.template operator()<64, 1>() : f.template operator()<64, 2>();
  return one ? f.template operator()<128, 1>() : f.template operator()<128, 2>();
}

}  // namespace

cudaError_t paged_status_word(unsigned int** word, int* dev, bool* remember) {
  static std::atomic<unsigned int*> word_of[64];
  cudaError_t e = host().get_device(dev);
  if (e != cudaSuccess) return e;
  *remember = *dev >= 0 && *dev < 64 && !host_pretends();
  *word = *remember ? word_of[*dev].load(std::memory_order_acquire) : nullptr;
  if (*word == nullptr) {
    if ((e = host().symbol_address(reinterpret_cast<void**>(word), reinterpret_cast<const void*>(&g_sm100_paged_status))) != cudaSuccess) return e;
    if (*remember) word_of[*dev].store(*word, std::memory_order_release);
  }
  return cudaSuccess;
}

unsigned int sm100_paged_status(bool reset) {
  unsigned int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_sm100_paged_status, sizeof(v)) != cudaSuccess) { (void)cudaGetLastError(); return 0xffffffffu; }
  if (reset && v != 0) {
    unsigned int zero = 0;
    if (cudaMemcpyToSymbol(g_sm100_paged_status, &zero, sizeof(zero)) != cudaSuccess) (void)cudaGetLastError();
  }
  return v;
}

bool plan_paged_split(int dtype, PagedAttn& p, int sms) {
  if (dtype == 1 || p.dqk > 128 || p.dvo > 128 || p.dqk % 8 != 0 || p.dvo % 8 != 0 || p.page % 8 != 0 || !host().have_encoder()) return false;
  if (!tma_friendly(as_tiles(p.k, p.dqk)) || !tma_friendly(as_tiles(p.v, p.dvo))) return false;
  // Q is read and the output written 4 and 8 bytes at a time
  auto rows = [](const View4& t, int per) {
    if (reinterpret_cast<uintptr_t>(t.ptr) % (2 * per) != 0) return false;
    for (int i = 0; i < 3; ++i)
      if (t.n[i] > 1 && t.s[i] % per != 0) return false;
    return true;
  };
  if (!rows(p.q, 2) || !rows(p.out, 4)) return false;
  p.kind = kPagedSplit;
  p.box = 64;
  while (p.page % p.box != 0) p.box /= 2;
  p.tile_log = kTileLog;
  p.min_tiles = 2;
  p.extra = 3;
  with_split_tile(p, [&]<int HD, int MT>() {
    p.rows = SplitSmem<HD, MT>::kRows;
    p.ctas = sms * SplitSmem<HD, MT>::kCtasPerSm;
  });
  return true;
}

cudaError_t launch_paged_split(int dtype, PagedAttn& p, cudaStream_t st) {
  return with_split_tile(p, [&]<int HD, int MT>() {
    return dtype == 2 ? launch_split_T<__half, HD, MT>(p, st) : launch_split_T<__nv_bfloat16, HD, MT>(p, st);
  });
}

}  // namespace ab200
