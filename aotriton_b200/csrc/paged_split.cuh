// How the attention kernels over a paged cache share a call out, and how pieces of a sequence meet.
//
// Sequences of one batch have lengths between one token and a hundred thousand, which only the device knows.  So nothing is cut by a
// bound on the lengths: the key tiles of all units -- (sequence, kv head, chunk of query rows) -- are put in one line, and each CTA takes an equal
// piece of it, whatever sequences that crosses.  A unit that lies within a piece is finished there; the pieces of others leave row maximum,
// row sum and unnormalised output in a workspace (at most two a CTA: of the unit it begins with and of the one it ends with, so that its size does not
// depend on the lengths), which a second launch adds up in the order of the keys.  Every CTA works out its place from the lengths alone.
//
// A unit costs a CTA more than its tiles: queries to fetch, a result to put together.  So its place in the line is p.extra tiles longer than it is (the first ones
// of it, which nobody works on), and a CTA gets many short sequences or few long ones for the same time.
#pragma once

#include "paged.h"

namespace ab200 {
namespace {

// What a sequence's queries see of its keys: the first `sinks` and those from `lo` on, in tiles of 2^p.tile_log keys.  At least one tile, so
// that every unit has an owner.
struct Walk {
  int len, queries, lo, first, n_sink, tiles;
  __device__ __forceinline__ Walk(const PagedAttn& p, int z) : Walk(p, p.lengths[z], p.query_lengths != nullptr ? p.query_lengths[z] : p.sq) {}
  __device__ __forceinline__ Walk(const PagedAttn& p, int length, int query_length) {
    len = min(max(length, 0), p.max_len);
    queries = min(max(query_length, 0), p.sq);
    if (len == 0 || queries == 0) { lo = first = n_sink = 0; tiles = 1; return; }
    const int64_t from = (int64_t)len - queries - p.window + 1;      // the first query's window
    lo = from > 0 ? (int)from : 0;
    first = lo >> p.tile_log;
    n_sink = min((min(p.sinks, lo) + (1 << p.tile_log) - 1) >> p.tile_log, first);
    tiles = n_sink + ((len - 1) >> p.tile_log) - first + 1;
  }
  __device__ __forceinline__ int tile(int i) const { return i < n_sink ? i : first + i - n_sink; }
  // Whether some query of the sequence sees key n, its page apart.
  __device__ __forceinline__ bool seen(const PagedAttn& p, int n) const { return n < len && (n >= lo || n < p.sinks); }
};

// Places in the line of a unit.
__device__ __forceinline__ int places(const PagedAttn& p, const Walk& w) { return w.tiles + p.extra; }

// The line of tiles as one thread block sees it; the host has seen to it that 31 bits hold it.  `lanes` CTAs next to each other take the same piece of
// a line without the chunks, a chunk each: they read the same keys at the same time.
struct Line {
  int total, share;      // tiles in all, and of a CTA
  int base;              // first tile of sequence z
  int z;
};

// A block of NT threads (a multiple of 32) finds sequence `z`, or the one that the first place of piece `piece` belongs to (z < 0).  `scratch`: NT / 32 + 2
// words.  Behind the last place, z is the batch's size.
template <int NT>
__device__ __forceinline__ Line find_in_line(const PagedAttn& p, int z, int piece, int* scratch) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int units = (int)((unsigned)(p.hk * p.chunks) / (unsigned)p.lanes), pieces = (int)((unsigned)p.ctas / (unsigned)p.lanes);
  Line r;
  if (p.batch <= 64) {      // each warp for itself: lane i has the sequences 2i and 2i + 1
    const int z0 = 2 * lane, a = z0 < p.batch ? places(p, Walk(p, z0)) : 0, b = z0 + 1 < p.batch ? places(p, Walk(p, z0 + 1)) : 0;
    int up = a + b;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, up, d);
      if (lane >= d) up += o;
    }
    r.total = __shfl_sync(0xffffffffu, up, 31) * units;
    r.share = max((int)((unsigned)(r.total + pieces - 1) / (unsigned)pieces), p.min_tiles);
    const int before = (up - a - b) * units, middle = before + a * units;
    const int64_t at = (int64_t)piece * r.share;
    const bool first = z >= 0 ? z == z0 : (a > 0 && at >= before && at < middle), second = z >= 0 ? z == z0 + 1 : (b > 0 && at >= middle && at < middle + b * units);
    const uint32_t owner = __ballot_sync(0xffffffffu, first || second);
    const int from = owner != 0u ? __ffs(owner) - 1 : 0;
    r.z = __shfl_sync(0xffffffffu, second ? z0 + 1 : z0, from);
    r.base = __shfl_sync(0xffffffffu, second ? middle : before, from);
    if (owner == 0u) r.z = p.batch;
    return r;
  }
  const int each = (p.batch + NT - 1) / NT, z0 = min(tid * each, p.batch), z1 = min(z0 + each, p.batch);
  int mine = 0;
  for (int i = z0; i < z1; ++i) mine += places(p, Walk(p, i));
  int up = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, up, d);
    if (lane >= d) up += o;
  }
  if (lane == 31) scratch[warp] = up;
  if (tid == 0) scratch[NT / 32] = p.batch;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    const int s = scratch[w];
    if (w < warp) before += s;
    total += s;
  }
  before += up - mine;
  r.total = total * units;
  r.share = max((int)((unsigned)(r.total + pieces - 1) / (unsigned)pieces), p.min_tiles);
  const int64_t at = (int64_t)piece * r.share;
  if (z >= 0 ? (z >= z0 && z < z1) : (mine > 0 && at >= before * units && at < (before + mine) * units)) {
    int b = before, i = z0;
    for (; i + 1 < z1; ++i) {
      if (i == z) break;
      const int t = places(p, Walk(p, i));
      if (z < 0 && at < (b + t) * units) break;
      b += t;
    }
    scratch[NT / 32] = i;
    scratch[NT / 32 + 1] = b * units;
  }
  __syncthreads();
  r.z = scratch[NT / 32];
  r.base = scratch[NT / 32 + 1];
  return r;
}

// A CTA's way along its piece of the line.
struct Piece {
  int at, end, z, base, lane;
  Walk w;
  int hk, chunk, first, last;      // the current unit, and its tiles in this piece
  __device__ __forceinline__ Piece(const PagedAttn& p, const Line& line)
      : at((int)(blockIdx.x / p.lanes) * line.share), end(min(at + line.share, line.total)), z(line.z), base(line.base),
        lane((int)(blockIdx.x % p.lanes)), w(p, line.z), hk(0), chunk(0), first(0), last(0) {}
  // The next unit with tiles in this piece, if there is one; `at` is moved behind it.
  __device__ __forceinline__ bool next(const PagedAttn& p) {
    const int chunks = (int)((unsigned)p.chunks / (unsigned)p.lanes), units = p.hk * chunks;
    while (at < end) {
      int n = places(p, w);
      while (at >= base + n * units) {
        base += n * units;
        w = Walk(p, ++z);
        n = places(p, w);
      }
      const int u = (int)((unsigned)(at - base) / (unsigned)n);
      hk = (int)((unsigned)u / (unsigned)chunks);
      chunk = (u - hk * chunks) * p.lanes + lane;
      const int unit = base + u * n + p.extra;      // its first tile's place
      first = max(at - unit, 0);
      last = min(end, unit + w.tiles) - unit;
      at = unit + last;
      if (last > 0) return true;
      at = end;      // (the piece ends ahead of the unit's first tile)
    }
    return false;
  }
  __device__ __forceinline__ bool whole() const { return first == 0 && last == w.tiles; }
};
// The pieces that have tiles of unit `along` (of its lane) of the sequence that `line` has found.
__device__ __forceinline__ void pieces_of_unit(const PagedAttn& p, const Line& line, const Walk& w, int along, int& first, int& last) {
  const int unit = line.base + along * places(p, w) + p.extra;
  first = (int)((unsigned)unit / (unsigned)line.share);
  last = (int)((unsigned)(unit + w.tiles - 1) / (unsigned)line.share);
}

// Rows of a unit's chunk: row r of it is query m of head h.
struct Rows {
  int row0, n, queries;
  __device__ __forceinline__ Rows(const PagedAttn& p, const Walk& w, int chunk) {
    queries = w.queries;
    row0 = chunk * p.rows;
    n = min(p.rows, p.group * w.queries - row0);
    if (n < 0) n = 0;
  }
  __device__ __forceinline__ int head(const PagedAttn& p, int hk, int r) const { return hk * p.group + (row0 + r) / queries; }
  __device__ __forceinline__ int query(int r) const { return (row0 + r) % queries; }
};

// Partial result `slot` (twice the CTA, one more for the unit that starts in it): rows x dvo outputs, then maxima, then sums.
__host__ __device__ __forceinline__ int64_t partial_floats(const PagedAttn& p) { return ((int64_t)p.rows * (p.dvo + 2) + 3) / 4 * 4; }
__device__ __forceinline__ float* partial_of(const PagedAttn& p, int64_t slot) { return p.partial + slot * partial_floats(p); }

// ... of the unit that a CTA is at
__device__ __forceinline__ float* partial_of(const PagedAttn& p, const Piece& c) { return partial_of(p, 2 * (int64_t)blockIdx.x + (c.first == 0 ? 1 : 0)); }

template <typename T>
__device__ __forceinline__ T* out_row(const PagedAttn& p, int z, int h, int m) {
  return reinterpret_cast<T*>(p.out.ptr) + (int64_t)z * p.out.s[0] + (int64_t)h * p.out.s[1] + (int64_t)m * p.out.s[2];
}
__device__ __forceinline__ void put_lse(const PagedAttn& p, int z, int h, int m, float mx, float l) {
  if (p.lse != nullptr) p.lse[((int64_t)z * p.hq + h) * p.sq + m] = l > 0.f ? (mx + log2f(l)) * kLn2 : INFINITY;
}

// Rows of a kv head's queries behind the sequence's last, by the block that starts the head's first chunk: zeros.
template <typename T, int NT>
__device__ __forceinline__ void zero_rows_behind(const PagedAttn& p, const Walk& w, int z, int hk, int tid) {
  const int behind = p.sq - w.queries;
  for (int r = tid / 32; r < p.group * behind; r += NT / 32) {
    const int h = hk * p.group + r / behind, m = w.queries + r % behind;
    for (int d = tid & 31; d < p.dvo; d += 32) out_row<T>(p, z, h, m)[d] = from_f32<T>(0.f);
    if ((tid & 31) == 0) put_lse(p, z, h, m, 0.f, 0.f);
  }
}

}  // namespace
}  // namespace ab200
