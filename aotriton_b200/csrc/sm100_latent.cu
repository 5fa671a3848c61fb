// Latent attention over a paged cache in its absorbed form, fp16 and bf16: every head reads the same row of a key, whose first columns are the value.
//
// With 16 heads it is bound by reading the cache, with 128 the tensor cores have as much to do (2 x 128 x 1088 flop for a row of 1152 bytes).  Either way the
// accumulator is the difficulty: 512 columns of fp32 for each of 128 rows would take all of tensor memory.  So the products are turned round:
//   S^T = K Q^T   128 keys x N rows      A: a tile of 128 keys as it lies in shared memory, B: the queries
//   O^T += V^T P  128 columns x N rows   A: the same tile, 128 of its columns at a time, transposed by the descriptor, B: the weights
// with N = 16, 32 or 64 rows (heads times queries) in 5 N columns of tensor memory.  A key's scores are then a thread's: hiding a key costs nothing, and no
// lane idles with few heads.  What gets awkward is the maximum of a row, which runs across the lanes of four warps.  It is not taken: weights are formed
// against a row's reference, the maximum of the tiles up to the last one that raised it, and only if a score passes it by more than 8 (in base 2), which one vote a tile finds
// out, the four warps take the true maximum, and rescale.  Sums stay with the threads, per key's lane, until the end of a unit.
//
// A tile comes in blocks of 128 columns (32 KB, pairs of 64-column boxes) and the last columns, which are no values, by themselves; slots go back one by one as
// the second product has read them, so the next tile arrives under it.  (64 rows leave room for no more than one tile; the weights then take the last columns' slot,
// which are done with once the scores are formed.)
//
// Measured, us of device a call with the join, bf16, 576 and 512 columns: 64 sequences of 8000 keys x 16 heads 119 (4.9 TB/s; a tile takes what its bytes do, the rest is the
// start, when every SM asks for its first tile at once, and the end); 32 of 500 to 8192 x 128 heads 75, 64 heads 57, 32 heads 52; 8 of 500 to 6007 x 16 heads 21. With 64 rows a
// tile takes 6500 clocks, the tensor pipe 4250 of them (an MMA of 64 rows about 54); 128 heads read each row from memory once and from L2 twice.
//
// Roles: warps 0-3 (64 rows: 0-7) softmax and write-out (thread = key, then = value column), then one that copies, one that issues the products.
#include <atomic>
#include "launch.h"
#include "paged.h"
#include "paged_split.cuh"
#include "sm100_ptx.cuh"

namespace ab200 {
namespace {
using namespace ptx;

constexpr int kKeys = 128;
constexpr int kBox = kKeys * 128, kBlock = 2 * kBox;      // bytes: 64 columns of a tile, 128 columns
constexpr float kNoReference = -3.0e38f;                  // of a row that has seen nothing
constexpr float kSlack = 8.f;

template <int NR>
struct LatentSmem {
  static constexpr bool kAlias = NR > 16;                 // the weights lie in the last columns' slot
  static constexpr int kGroups = NR > 32 ? 2 : 1;         // warpgroups that share the rows' softmax and write-out
  static constexpr int kSoftmax = 128 * kGroups, kThreads = kSoftmax + 64, kOwn = NR / kGroups;
  static constexpr int kSlots = NR > 32 ? 4 : 5;
  static constexpr int bFull = 0, bEmpty = kSlots, bTailFull = 2 * kSlots, bTailEmpty = bTailFull + 1, bQ = bTailEmpty + 1, bS = bQ + 1, bP = bS + 1,
                       bO = bP + 1, bDrain = bO + 1, bQEmpty = bDrain + 1, bCount = bQEmpty + 1;
  static constexpr int kAbort = bCount * 8, kTmem = kAbort + 8;
  static constexpr int kScratch = (kTmem + 8 + 15) & ~15;
  static constexpr int kRef = (kScratch + (kThreads / 32 + 2) * 4 + 15) & ~15;      // [NR] references, rescales, inverse sums; [4][NR] of the warps
  static constexpr int kAlpha = kRef + NR * 4, kInv = kAlpha + NR * 4, kWarps = kInv + NR * 4;
  static constexpr int kPos = kWarps + 4 * NR * 4, kOut = kPos + NR * 4;                  // [NR] positions; offsets of the output's rows
  static constexpr int kQ = (kOut + NR * 8 + 1023) & ~1023;
  static constexpr int kQBox = NR * 128;
  static constexpr int kP = kQ + 9 * kQBox;
  static constexpr int kTail = kP + (kAlias ? 0 : kBox);
  static constexpr int kRing = kTail + kBox;
  static constexpr int kBytes = kRing + kSlots * kBlock + 1024;
  static constexpr uint32_t kOCol = 64, kTmemCols = NR > 32 ? 512 : (NR > 16 ? 256 : 128);
  static_assert(kBytes <= 232448 && kQBox % 1024 == 0 && kOCol + 4 * NR <= kTmemCols, "fits");
};

template <int N>
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory"); }
// ... and whether any thread says so
template <int N>
__device__ __forceinline__ bool softmax_any(bool x) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.b32 a, %1, 0;\n\tbarrier.cta.red.or.pred b, 1, %2, a;\n\tselp.b32 %0, 1, 0, b;\n\t}"
               : "=r"(r) : "r"((uint32_t)x), "n"(N) : "memory");
  return r != 0;
}

template <int NR>
__device__ __forceinline__ void tmem_row(uint32_t taddr, float (&x)[NR]) {
  if constexpr (NR == 16) tmem_ld16f(taddr, x);
  else tmem_ld32f(taddr, x);
  tmem_wait_ld();
}

// Combines x[c] over the lanes of a warp, halving the columns that a lane holds from step to step; that of lane_column(lane) is then in x[0].
template <int NR, typename Op>
__device__ __forceinline__ void across_lanes(float (&x)[NR], int lane, Op op) {
  int n = NR;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (n > 1) {
      n /= 2;
#pragma unroll
      for (int j = 0; j < NR / 2; ++j) {
        if (j >= n) break;
        const bool up = lane & o;
        const float keep = up ? x[j + n] : x[j], send = up ? x[j] : x[j + n];
        x[j] = op(keep, __shfl_xor_sync(0xffffffffu, send, o));
      }
    } else {
      x[0] = op(x[0], __shfl_xor_sync(0xffffffffu, x[0], o));
    }
  }
}
template <int NR>
__device__ __forceinline__ int lane_column(int lane) { return NR == 32 ? lane : lane >> 1; }

// p.rows = NR; p.dvo a multiple of 128 up to 512, the last 1 to 64 of p.dqk columns behind it
template <typename T, int NR>
__global__ void __launch_bounds__(LatentSmem<NR>::kThreads, 1) paged_latent_kernel(const __grid_constant__ PagedAttn p, const __grid_constant__ CUtensorMap tm, const __grid_constant__ CUtensorMap tm_q) {
  using L = LatentSmem<NR>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kAbort);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kTmem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    prefetch_tmap(&tm);
    if (p.q_tiles) prefetch_tmap(&tm_q);
  }
  wait_for_earlier_grids();
  const unsigned int failed = tid == 0 ? *reinterpret_cast<volatile unsigned int*>(p.status) : 0u;
  if (tid == 0) {
    init_abort_and_limit(abort_flag, p.wait_limit_kcycles);
    for (int b = 0; b < L::bCount; ++b) mbar_init(&bars[b], b == L::bP || (b == L::bQ && !p.q_tiles) ? 4 * L::kGroups : 1);
    fence_barrier_init();
  }
  const Line line = find_in_line<L::kThreads>(p, -1, blockIdx.x / p.lanes, reinterpret_cast<int*>(smem + L::kScratch));
  if (__syncthreads_or(failed != 0u)) return;
  if (line.z >= p.batch) return;
  if (warp == 4 * L::kGroups + 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Piece run(p, line);
  const Walk& w = run.w;
  const int blocks = p.dvo / 128, qboxes = (p.dqk + 63) / 64;

  if (warp == 4 * L::kGroups) {
    // ================================ TMA producer ===================================
    const int octets = p.box / 8;
    const bool leads = lane < 16 && lane % octets == 0;
    int vi = 0, ti = 0, units = 0;      // blocks, tails and units requested
    bool stop = false, dropped = false;
    while (!stop && run.next(p)) {
      if (Rows(p, w, run.chunk).n == 0) continue;
      const int first = run.first, last = run.last;
      if (p.q_tiles) {
        if (!__all_sync(0xffffffffu, mbar_wait(&bars[L::bQEmpty], ((uint32_t)units & 1u) ^ 1u, abort_flag, p.status, 0x7020))) { stop = true; break; }
        if (lane == 0) {
          mbar_expect_tx(&bars[L::bQ], qboxes * L::kQBox);
          for (int b = 0; b < qboxes; ++b) tma_load_4d(smem + L::kQ + b * L::kQBox, &tm_q, &bars[L::bQ], b * 64, run.chunk * NR, 0, run.z);
        }
        __syncwarp();
        ++units;
      }
      const int32_t* row = p.table + (int64_t)run.z * p.table_stride;
      auto look = [&](int i) {      // the page of this lane's eight keys in tile i
        const int n = i * kKeys + lane * 8;
        if (lane >= 16 || n >= w.len) return -1;
        const int id = row[n / p.page];
        return id;
      };
      int id = look(first);
      for (int i = first; i < last && !stop; ++i) {
        const int page = id >= 0 && id < p.num_pages ? id : p.num_pages;      // (a page that does not exist: zeros, without a read)
        const int slot = (i * kKeys + lane * 8) % p.page;
        if (i + 1 < last) {
          id = look(i + 1);
          // the next tile towards L2: there is no room for it yet, and memory would rest until there is
          const int next = id >= 0 && id < p.num_pages ? id : p.num_pages, at = ((i + 1) * kKeys + lane * 8) % p.page;
          if (leads && next < p.num_pages) {
            for (int b = run.lane; b < blocks; b += p.lanes) {
              tma_prefetch_4d(&tm, b * 128, at, 0, next);
              tma_prefetch_4d(&tm, b * 128 + 64, at, 0, next);
            }
            if (run.lane == 0) tma_prefetch_4d(&tm, p.dvo, at, 0, next);
          }
          __syncwarp();
        }
        auto tail = [&] {
          if (!__all_sync(0xffffffffu, mbar_wait(&bars[L::bTailEmpty], ((uint32_t)ti & 1u) ^ 1u, abort_flag, p.status, 0x7000))) { stop = true; return; }
          if (lane == 0) mbar_expect_tx(&bars[L::bTailFull], kBox);
          __syncwarp();
          if (leads) tma_load_4d(smem + L::kTail + lane * 1024, &tm, &bars[L::bTailFull], p.dvo, slot, 0, page);
          ++ti;
        };
        for (int b = 0; b < blocks && !stop; ++b) {
          if (!L::kAlias && b == 1) tail();
          if (stop) break;
          const int s = vi % L::kSlots;
          if (!__all_sync(0xffffffffu, mbar_wait(&bars[L::bEmpty + s], ((uint32_t)(vi / L::kSlots) & 1u) ^ 1u, abort_flag, p.status, 0x7010))) { stop = true; break; }
          const bool drop = p.drop_copy == 1 && run.z == 0 && run.chunk == 0 && i == 0 && b == 0;      // (test hook: the first block never arrives)
          dropped |= drop;
          if (!drop) {
            uint8_t* dst = smem + L::kRing + s * kBlock;
            if (lane == 0) mbar_expect_tx(&bars[L::bFull + s], kBlock);
            __syncwarp();
            if (leads) {
              tma_load_4d(dst + lane * 1024, &tm, &bars[L::bFull + s], b * 128, slot, 0, page);
              tma_load_4d(dst + kBox + lane * 1024, &tm, &bars[L::bFull + s], b * 128 + 64, slot, 0, page);
            }
          }
          ++vi;
        }
        if (!stop && (L::kAlias || blocks == 1)) tail();
      }
    }
    __syncwarp();
    if (*abort_flag && lane == 0) {      // copies that are still in flight land before the memory is used again
      for (int i = max(dropped ? 1 : 0, vi - L::kSlots); i < vi; ++i)
        mbar_wait_quiet(&bars[L::bFull + i % L::kSlots], (uint32_t)(i / L::kSlots) & 1u, abort_flag);
      if (units > 0) mbar_wait_quiet(&bars[L::bQ], (uint32_t)(units - 1) & 1u, abort_flag);
      if (ti > 0) mbar_wait_quiet(&bars[L::bTailFull], (uint32_t)(ti - 1) & 1u, abort_flag);
    }
    __syncwarp();
  } else if (warp == 4 * L::kGroups + 1) {
    // ================================ the products ===================================
    constexpr uint32_t kIdescS = instr_desc_f16(Fmt<T>::code, 128, NR, 0, 0), kIdescO = instr_desc_f16(Fmt<T>::code, 128, NR, 1, 1);
    const uint64_t ring_k = smem_desc_sw128(smem_u32(smem + L::kRing), 16, 1024), ring_mn = smem_desc_sw128(smem_u32(smem + L::kRing), kBox, 1024);
    const uint64_t tail_k = smem_desc_sw128(smem_u32(smem + L::kTail), 16, 1024), q_k = smem_desc_sw128(smem_u32(smem + L::kQ), 16, 1024);
    const uint64_t p_mn = smem_desc_sw128(smem_u32(smem + (L::kAlias ? L::kTail : L::kP)), kBox, 1024);
    const int tail_steps = (p.dqk - p.dvo + 15) / 16;
    int vi = 0, tiles = 0, units = 0;
    bool ok = true;
    auto wait = [&](int bar, uint32_t parity, uint32_t where) {
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&bars[bar], parity, abort_flag, p.status, where)) != 0;
      return ok;
    };
    while (ok && run.next(p)) {
      if (Rows(p, w, run.chunk).n == 0) continue;
      const int first = run.first, last = run.last;
      if (!wait(L::bQ, (uint32_t)units & 1u, 0x7100)) break;
      ++units;
      for (int i = first; i < last; ++i) {
        uint32_t acc = 0u;
        auto scores_tail = [&] {
          if (!wait(L::bTailFull, (uint32_t)tiles & 1u, 0x7110)) return;
          tc_fence_after();
          if (elect_one())
            for (int k = 0; k < tail_steps; ++k)
              mma_ss(tmem, tail_k + (uint64_t)(k * 2), q_k + (uint64_t)((2 * blocks * L::kQBox) >> 4) + (uint64_t)(k * 2), kIdescS, k > 0 ? 1u : acc);
          __syncwarp();
          acc = 1u;
        };
        for (int b = 0; b < blocks; ++b) {
          if (!L::kAlias && b == 1) scores_tail();
          const int s = (vi + b) % L::kSlots;
          if (!wait(L::bFull + s, (uint32_t)((vi + b) / L::kSlots) & 1u, 0x7120)) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              mma_ss(tmem, ring_k + (uint64_t)((s * kBlock + (k >> 2) * kBox) >> 4) + (uint64_t)((k & 3) * 2),
                     q_k + (uint64_t)(((2 * b + (k >> 2)) * L::kQBox) >> 4) + (uint64_t)((k & 3) * 2), kIdescS, k > 0 ? 1u : acc);
          }
          __syncwarp();
          acc = 1u;
        }
        if (ok && (L::kAlias || blocks == 1)) scores_tail();
        if (!ok) break;
        if (elect_one()) {
          if (!L::kAlias) mma_commit(&bars[L::bTailEmpty]);
          if (i + 1 == last) mma_commit(&bars[L::bQEmpty]);
          mma_commit(&bars[L::bS]);
        }
        __syncwarp();
        if (!wait(L::bP, (uint32_t)tiles & 1u, 0x7130)) break;
        tc_fence_after();
        if (elect_one()) {
          for (int b = 0; b < blocks; ++b) {
            const int s = (vi + b) % L::kSlots;
#pragma unroll
            for (int k = 0; k < 8; ++k)
              mma_ss(tmem + L::kOCol + b * NR, ring_mn + (uint64_t)((s * kBlock + k * 2048) >> 4), p_mn + (uint64_t)((k * 2048) >> 4), kIdescO,
                     k > 0 || i > first ? 1u : 0u);
            mma_commit(&bars[L::bEmpty + s]);
          }
          if (L::kAlias) mma_commit(&bars[L::bTailEmpty]);
          if (i + 1 == last) mma_commit(&bars[L::bO]);
        }
        __syncwarp();
        vi += blocks;
        ++tiles;
      }
    }
    if (!ok) {      // products in flight end before tensor memory is given back
      if (elect_one()) mma_commit(&bars[L::bDrain]);
      __syncwarp();
      mbar_wait_quiet(&bars[L::bDrain], 0u, abort_flag);
    }
    __syncwarp();
  } else {
    // ================================ softmax, write-out ===============================
    float* ref = reinterpret_cast<float*>(smem + L::kRef);
    float* alpha = reinterpret_cast<float*>(smem + L::kAlpha);
    float* inv = reinterpret_cast<float*>(smem + L::kInv);
    float* warps = reinterpret_cast<float*>(smem + L::kWarps);
    int* pos = reinterpret_cast<int*>(smem + L::kPos);
    int64_t* out_at = reinterpret_cast<int64_t*>(smem + L::kOut);
    uint8_t* ps = smem + (L::kAlias ? L::kTail : L::kP);
    // a warpgroup has kOwn of the rows, from `col` on; a thread of it a key, then a column of the values
    constexpr int kSoftmax = L::kSoftmax, kOwn = L::kOwn;
    const int col = warp / 4 * kOwn, key = tid & 127;
    const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16) + col;      // this warp's lanes
    int vi = 0, tiles = 0, units = 0;
    bool broken = false;
    while (!broken && run.next(p)) {
      const int z = run.z, first = run.first, last = run.last;
      const Rows rows(p, w, run.chunk);
      if (first == 0 && run.chunk == 0) zero_rows_behind<T, kSoftmax>(p, w, z, 0, tid);
      if (rows.n == 0) continue;
      // ---- the unit's queries, as the products read them, where they are not rows of a tile copy ----
      if (!p.q_tiles)
      for (int r = warp; r < NR; r += 4 * L::kGroups) {      // (a warp a row, a lane 16 bytes; those that there are none of are zero)
        const bool in = r < rows.n;
        const T* src = reinterpret_cast<const T*>(p.q.ptr);
        if (in) src += (int64_t)z * p.q.s[0] + (int64_t)rows.head(p, 0, r) * p.q.s[1] + (int64_t)rows.query(r) * p.q.s[2];
        for (int c = lane; c < qboxes * 8; c += 32)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem + L::kQ + (c >> 3) * L::kQBox + r * 128 + (((c ^ r) & 7) << 4))),
                       "l"(in && c * 8 < p.dqk ? src + c * 8 : reinterpret_cast<const T*>(p.q.ptr)), "r"(in && c * 8 < p.dqk ? 16 : 0) : "memory");
      }
      if (tid < NR) {
        ref[tid] = kNoReference;
        pos[tid] = tid < rows.n ? w.len - rows.queries + rows.query(tid) : 0x7fffffff;
        out_at[tid] = tid < rows.n ? (int64_t)z * p.out.s[0] + (int64_t)rows.head(p, 0, tid) * p.out.s[1] + (int64_t)rows.query(tid) * p.out.s[2] : 0;
      }
      if (!p.q_tiles) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[L::bQ]);
      }
      softmax_sync<kSoftmax>();
      float l[kOwn];
#pragma unroll
      for (int j = 0; j < kOwn; ++j) l[j] = 0.f;
      const int32_t* row = p.table + (int64_t)z * p.table_stride;
      for (int i = first; i < last; ++i) {
        const int n = i * kKeys + key;
        bool there = n < w.len;
        if (there) {
          const int id = row[n / p.page];
          there = id >= 0 && id < p.num_pages;
        }
        const bool some_hidden = (i + 1) * kKeys > w.len - rows.queries + 1;      // (warp-uniform: of the later queries' keys)
        const bool ok = mbar_wait(&bars[L::bS], (uint32_t)tiles & 1u, abort_flag, p.status, 0x7200);
        const bool came = __all_sync(0xffffffffu, ok) != 0;
        tc_fence_after();
        // this key's score with each row, in base 2
        auto scores = [&](float (&x)[kOwn]) {
          tmem_row<kOwn>(mine, x);
#pragma unroll
          for (int j = 0; j < kOwn; ++j) x[j] = there ? x[j] * p.qk_scale : -INFINITY;
          if (some_hidden)
#pragma unroll
            for (int j = 0; j < kOwn; ++j)
              if (n > pos[col + j]) x[j] = -INFINITY;
        };
        float x[kOwn], top = i > first ? -INFINITY : INFINITY;      // (a first tile has no reference)
        if (i > first) {
        scores(x);
#pragma unroll
        for (int j = 0; j < kOwn; j += 4) {
          const float4 m = *reinterpret_cast<const float4*>(ref + col + j);
          x[j] -= m.x; x[j + 1] -= m.y; x[j + 2] -= m.z; x[j + 3] -= m.w;
          top = fmaxf(top, fmaxf(fmaxf(x[j], x[j + 1]), fmaxf(x[j + 2], x[j + 3])));
        }
        }
        if (softmax_any<kSoftmax>(top > kSlack || !came)) {
          // ---- a score far above its row's reference (or the first of its row): the true maxima, and everything against them ----
          if (softmax_any<kSoftmax>(!came)) { broken = true; break; }
          scores(x);
          across_lanes<kOwn>(x, lane, [](float a, float b) { return fmaxf(a, b); });
          warps[(warp & 3) * NR + col + lane_column<kOwn>(lane)] = x[0];
          softmax_sync<kSoftmax>();
          if (tid < NR) {
            const float was = ref[tid];
            float now = fmaxf(fmaxf(warps[tid], warps[NR + tid]), fmaxf(warps[2 * NR + tid], warps[3 * NR + tid]));
            now = fmaxf(now, was);
            alpha[tid] = ex2(was - now);
            ref[tid] = now;
          }
          softmax_sync<kSoftmax>();
#pragma unroll
          for (int j = 0; j < kOwn; ++j) l[j] *= alpha[col + j];
          if (i > first) {      // (the last tile's product has ended: this one's scores were formed behind it)
            for (int b = 0; b < blocks; ++b) {
#pragma unroll
              for (int h = 0; h < kOwn; h += 16) {
                float o[16];
                uint32_t u[16];
                tmem_ld16f(mine + L::kOCol + b * NR + h, o);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) u[j] = __float_as_uint(o[j] * alpha[col + h + j]);
                tmem_st16(mine + L::kOCol + b * NR + h, u);
              }
            }
            tmem_wait_st();
          }
          scores(x);
#pragma unroll
          for (int j = 0; j < kOwn; ++j) x[j] -= ref[col + j];
        }
        // ---- weights, rounded to the value type (half a step off; the sums keep 32 bits) ----
#pragma unroll
        for (int j = 0; j < kOwn; j += 8) {
          float e[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            e[k] = ex2(x[j + k]);
            l[j + k] += e[k];
          }
          *reinterpret_cast<uint4*>(ps + key * 128 + (((((col + j) >> 3) ^ key) & 7) << 4)) =
              make_uint4(pack2<T>(e[0], e[1]), pack2<T>(e[2], e[3]), pack2<T>(e[4], e[5]), pack2<T>(e[6], e[7]));
        }
        if (n >= w.len)      // slots behind the sequence hold whatever the cache has there: a zero weight times a non-finite value would poison the sum
          for (int b = warp / 4; b < 2 * blocks; b += L::kGroups) {
            uint8_t* r = smem + L::kRing + (vi + b / 2) % L::kSlots * kBlock + (b & 1) * kBox + key * 128;
#pragma unroll
            for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(r + c * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[L::bP]);
        vi += blocks;
        ++tiles;
      }
      // ---- the unit's result ----
      bool done = !broken;
      if (done) done = __all_sync(0xffffffffu, mbar_wait(&bars[L::bO], (uint32_t)units & 1u, abort_flag, p.status, 0x7210)) != 0;
      ++units;
      if (broken || softmax_any<kSoftmax>(!done)) { broken = true; break; }
      tc_fence_after();
      across_lanes<kOwn>(l, lane, [](float a, float b) { return a + b; });
      if (kOwn != 16 || (lane & 1) == 0) warps[(warp & 3) * NR + col + lane_column<kOwn>(lane)] = l[0];
      softmax_sync<kSoftmax>();
      const bool whole = run.whole();
      float* part = partial_of(p, run);
      if (tid < rows.n) {
        const float sum = (warps[tid] + warps[NR + tid]) + (warps[2 * NR + tid] + warps[3 * NR + tid]);
        inv[tid] = whole ? (sum > 0.f ? 1.f / sum : 0.f) : 1.f;
        if (whole) {
          put_lse(p, z, rows.head(p, 0, tid), rows.query(tid), ref[tid], sum);
        } else {
          part[NR * p.dvo + tid] = ref[tid] == kNoReference ? -INFINITY : ref[tid];
          part[NR * p.dvo + NR + tid] = sum;
        }
      }
      softmax_sync<kSoftmax>();
      for (int b = 0; b < blocks; ++b) {
        float o[kOwn];
        tmem_row<kOwn>(mine + L::kOCol + b * NR, o);
        const int d = b * 128 + key;
        if (whole) {
          T* out = reinterpret_cast<T*>(p.out.ptr) + d;
#pragma unroll
          for (int j = 0; j < kOwn; ++j)
            if (col + j < rows.n) out[out_at[col + j]] = from_f32<T>(o[j] * inv[col + j]);
        } else {
#pragma unroll
          for (int j = 0; j < kOwn; ++j)
            if (col + j < rows.n) part[(col + j) * p.dvo + d] = o[j];
        }
      }
      tc_fence_before();
      softmax_sync<kSoftmax>();      // (the next unit's rows and queries take the place of these)
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4 * L::kGroups + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

// A call of one query each: the heads as the rows of a (batch, 1, heads, columns) view.
View4 query_rows(const PagedAttn& p) { return View4{p.q.ptr, {p.q.n[0], 1, p.q.n[1], p.dqk}, {p.q.s[0], p.q.s[1], p.q.s[1], p.q.s[3]}}; }

template <typename T, int NR>
cudaError_t launch_latent_T(PagedAttn& p, cudaStream_t st) {
  using L = LatentSmem<NR>;
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  bool remember = false;
  cudaError_t e = paged_status_word(&p.status, &dev, &remember);
  if (e != cudaSuccess) return e;
  auto* kernel = paged_latent_kernel<T, NR>;
  if (!remember || !attr_set[dev].load(std::memory_order_acquire)) {
    if ((e = host().func_set_smem(reinterpret_cast<const void*>(kernel), L::kBytes)) != cudaSuccess) return e;
    if (remember) attr_set[dev].store(true, std::memory_order_release);
  }
  CUtensorMap tm;
  const View4 k{p.k.ptr, {p.k.n[0], 1, p.k.n[1], p.dqk}, {p.k.s[0], p.k.s[2], p.k.s[1], p.k.s[3]}};
  if (!make_tile_map_16bit(&tm, k, p.dqk, p.page, p.box)) return cudaErrorInvalidValue;
  CUtensorMap tq = tm;
  if (p.q_tiles && !make_tile_map_16bit(&tq, query_rows(p), p.dqk, p.hq, NR)) return cudaErrorInvalidValue;
  e = launch_kernel(kernel, dim3(p.ctas), dim3(L::kThreads), L::kBytes, st, p, tm, tq);
  if (e == cudaSuccess) count_launch();
  return e;
}

}  // namespace

bool plan_paged_latent(int dtype, PagedAttn& p, int sms) {
  if (dtype == 1 || p.hk != 1 || p.v.ptr != p.k.ptr || p.dvo % 128 != 0 || p.dvo > 512 || p.dqk % 8 != 0 || p.dqk <= p.dvo || p.dqk > p.dvo + 64 ||
      p.page % 8 != 0 || p.window != INT32_MAX || !host().have_encoder())
    return false;
  for (int i = 0; i < 2; ++i)
    if (p.k.n[i] > 1 && p.k.s[i] != p.v.s[i]) return false;
  const View4 k{p.k.ptr, {p.k.n[0], 1, p.k.n[1], p.dqk}, {p.k.s[0], p.k.s[2], p.k.s[1], p.k.s[3]}};
  if (!tma_friendly(k) || !aligned16(p.q.ptr)) return false;
  for (int i = 0; i < 3; ++i)
    if (p.q.n[i] > 1 && p.q.s[i] % 8 != 0) return false;
  const int64_t rows = (int64_t)p.group * p.sq;
  p.kind = kPagedLatent;
  p.rows = rows <= 16 ? 16 : (rows <= 32 ? 32 : 64);
  p.box = 128;
  while (p.page % p.box != 0) p.box /= 2;
  p.tile_log = 7;
  p.q_tiles = p.sq == 1 && tma_friendly(query_rows(p));
  p.min_tiles = 1;
  p.extra = 2;
  p.ctas = sms;
  return true;
}

cudaError_t launch_paged_latent(int dtype, PagedAttn& p, cudaStream_t st) {
  auto with = [&]<typename T>() {
    return p.rows == 16 ? launch_latent_T<T, 16>(p, st) : (p.rows == 32 ? launch_latent_T<T, 32>(p, st) : launch_latent_T<T, 64>(p, st));
  };
  return dtype == 2 ? with.template operator()<__half>() : with.template operator()<__nv_bfloat16>();
}

}  // namespace ab200
