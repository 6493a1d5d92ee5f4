// How the attention kernels of a paged cache deal out their work (PagedAttn: kernels.h).
//
// A sequence's query rows (its tokens times the heads of a group) are cut into row tiles, its keys behind the shared pages into key tiles.  An entry
// is a (sequence, row tile), a pair an (entry, key/value head); a pair's key tiles are those that its newest token sees.  All key tiles of a
// launch, pair after pair, are dealt out evenly: block c takes `per` of them from c * per on, wherever that lies, so that long and short
// sequences in one batch fill the GPU alike.  Each block finds its place from the positions alone: nothing about lengths has to be known on the
// host.  On the tensor memory a pair of few tiles is not cut: it belongs to the block in whose share it begins.  A pair that lies within one block is
// finished there; of one that is cut every block leaves its part in a workspace (slot 2 c + 1 if the pair begins in block c, 2 c if it began before),
// and a second launch joins them.  Where there are shared pages, their rows are those of the whole
// batch, cut and dealt out in the same way by a launch of their own; then all results of either are parts (slot: the pair's number, or the
// number of pairs + c), and the last launch joins both kinds.  The launch over the shared pages goes first.  Its blocks let the next launch start
// when they have waited for everything before them, and that one, which reads nothing that they write, waits for them at its end alone: the two
// share the GPU.
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace nxd {
namespace paged {

NXD_DEVICE int new_tokens(const PagedAttn& p, int b) {
  const long n = p.lens ? p.lens[b] : p.W;
  return p.positions[b] < 0 ? 0 : (int)(n < 0 ? 0 : n > p.W ? p.W : n);
}
// Keys that token w of sequence b sees; what lies behind the page table's end nobody sees
NXD_DEVICE int visible_keys(const PagedAttn& p, int b, int w) {
  const long cap = (long)p.cols * p.ps, first = p.positions[b];
  return (int)(first < cap && first + w + 1 < cap ? first + w + 1 : cap);
}
// One past the last key of the sequence: none of its tokens sees more
NXD_DEVICE int all_keys(const PagedAttn& p, int b) {
  const int m = new_tokens(p, b);
  return m ? visible_keys(p, b, m - 1) : 0;
}
// Shared keys that some row of the batch sees (a whole warp asks): what lies behind them need not be finite
NXD_DEVICE int seen_of_shared(const PagedAttn& p, int lane) {
  int n = 0;
  for (int b = lane; b < p.B; b += 32) n = max(n, all_keys(p, b));
  return min(p.shared, __reduce_max_sync(0xffffffffu, n));
}
// Key tiles that rows [row0, row1) of a sequence see behind the shared pages
NXD_DEVICE int row_key_tiles(const PagedAttn& p, int b, int row0, int row1) {
  const int m = new_tokens(p, b);
  if (row0 / p.G >= m) return 0;
  const int n = visible_keys(p, b, min(m, (row1 + p.G - 1) / p.G) - 1) - p.shared;
  return n > 0 ? (n + p.tile_keys - 1) / p.tile_keys : 0;
}
NXD_DEVICE int entry_tiles(const PagedAttn& p, int e) {
  const int row0 = e % p.row_tiles * p.tile_rows;
  return row_key_tiles(p, e / p.row_tiles, row0, row0 + p.tile_rows);
}

// SHARED, here and below: the rows of the whole batch as one sequence's, over the shared pages; the cuts are the host's
template <bool SHARED> NXD_DEVICE int walk_tiles(const PagedAttn& p, int e) { return SHARED ? p.pre_tiles : entry_tiles(p, e); }

struct Place { int e; long tile; long per, total; };

// Where tile block * per lies: entry (all of them behind the last tile) and tile within the entry's pairs.  THREADS threads from FIRST on call it.
template <int THREADS, bool SHARED, int FIRST = 0>
NXD_DEVICE Place find_place(const PagedAttn& p, int grid, int block) {
  auto sync = [] {
    if constexpr (FIRST == 0) __syncthreads();
    else asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
  };
  if constexpr (SHARED) {
    const long t = (long)p.Hkv * p.pre_tiles, first = (long)block * p.pre_per;
    return Place{(int)(first / t), first % t, p.pre_per, t * p.pre_row_tiles};
  } else {
    __shared__ long sums[THREADS / 32];
    __shared__ long found[2];
    const int lane = threadIdx.x & 31, thread = threadIdx.x - FIRST, warp = thread >> 5, entries = p.B * p.row_tiles;
    const int each = (entries + THREADS - 1) / THREADS, e0 = min(entries, thread * each), e1 = min(entries, e0 + each);
    long mine = 0;
    for (int e = e0; e < e1; ++e) mine += entry_tiles(p, e);
    long scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long x = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += x;
    }
    if (lane == 31) sums[warp] = scan;
    if (thread == 0) { found[0] = entries; found[1] = 0; }
    sync();
    Place at;
    long before = scan - mine;
    at.total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += sums[w];
      at.total += sums[w];
    }
    at.total *= p.Hkv;
    at.per = max((long)p.min_tiles, (at.total + grid - 1) / grid);
    long left = block * at.per - before * p.Hkv;
    if (left >= 0 && left < mine * p.Hkv) {
      for (int e = e0; e < e1; ++e) {
        const long t = (long)entry_tiles(p, e) * p.Hkv;
        if (left < t) { found[0] = e; found[1] = left; break; }
        left -= t;
      }
    }
    sync();
    at.e = (int)found[0];
    at.tile = found[1];
    return at;
  }
}

// A block's walk over its share: the pair and the tile in it
struct Walk { int e, head, tile, tiles; };

template <bool SHARED>
NXD_DEVICE void next_pair(const PagedAttn& p, Walk& w) {
  w.tile = 0;
  if (++w.head < p.Hkv) return;
  w.head = 0;
  ++w.e;
  if constexpr (!SHARED)
    while ((w.tiles = w.e < p.B * p.row_tiles ? entry_tiles(p, w.e) : 1) == 0) ++w.e;
}

// Whether a pair is not cut, so that it belongs to the block in whose share it begins, however far it reaches into the next one's
template <bool SHARED> NXD_DEVICE bool whole(const PagedAttn& p, int tiles) { return !SHARED && tiles <= p.whole_tiles; }

// Slot of the part that block `block` leaves of pair `pair`
template <bool SHARED>
NXD_DEVICE long part_slot(const PagedAttn& p, long pair, int block, bool begins) {
  if (!SHARED && p.shared == 0) return 2l * block + begins;
  return begins ? pair : (long)p.Hkv * (SHARED ? p.pre_row_tiles : p.B * p.row_tiles) + block;
}

// Joins n parts of each of ROWS rows, D / 32 columns a lane; slot(x, r) is the row of part x of row r among all parts' rows, row(r) where it goes, null:
// nowhere.  A row that is not live is zeros.  The first eight (parts times rows) are asked for before their weights are known.
template <typename T, int D, int ROWS, typename F, typename G>
NXD_DEVICE void join_parts(const PagedAttn& p, int n, const bool (&live)[ROWS], F slot, G row) {
  constexpr int C = D / 32, AHEAD = 8 / ROWS;
  const int lane = threadIdx.x & 31;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  float m[ROWS], l[ROWS], acc[ROWS][C] = {};
#pragma unroll
  for (int r = 0; r < ROWS; ++r) { m[r] = -INFINITY; l[r] = 0.f; }
  for (int x0 = 0; x0 < n; x0 += 32) {
    const int here = min(32, n - x0);
    float v[AHEAD][ROWS][C], f[ROWS];
    auto ask = [&](int x1) {
#pragma unroll
      for (int x = 0; x < AHEAD; ++x)
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          if (x1 + x < here && live[r]) {
            const float* src = p.part_o + slot(x0 + x1 + x, r) * D + lane * C;
            if constexpr (C == 4) *reinterpret_cast<float4*>(v[x][r]) = *reinterpret_cast<const float4*>(src);
            else *reinterpret_cast<float2*>(v[x][r]) = *reinterpret_cast<const float2*>(src);
          }
    };
    ask(0);
    float2 a[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) a[r] = lane < here && live[r] ? ml[slot(x0 + lane, r)] : make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float mn = fmaxf(m[r], warp_max(a[r].x)), old = m[r] == -INFINITY ? 0.f : exp2f(m[r] - mn);
      f[r] = a[r].x == -INFINITY ? 0.f : exp2f(a[r].x - mn);
      l[r] = l[r] * old + warp_sum(a[r].y * f[r]);
      m[r] = mn;
#pragma unroll
      for (int j = 0; j < C; ++j) acc[r][j] *= old;
    }
    for (int x1 = 0; x1 < here; x1 += AHEAD) {
      if (x1) ask(x1);
#pragma unroll
      for (int x = 0; x < AHEAD; ++x)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const float g = __shfl_sync(0xffffffffu, f[r], (x1 + x) & 31);
#pragma unroll
          for (int j = 0; j < C; ++j) acc[r][j] += x1 + x >= here || g == 0.f ? 0.f : v[x][r][j] * g;        // a part without weights has no sums
        }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    T* const to = row(r);
    if (!to) continue;
    T o[C];
#pragma unroll
    for (int j = 0; j < C; ++j) o[j] = from_f32<T>(l[r] == 0.f ? 0.f : acc[r][j] / l[r]);
    if constexpr (C == 4) *reinterpret_cast<uint2*>(to + lane * C) = *reinterpret_cast<const uint2*>(o);
    else *reinterpret_cast<uint32_t*>(to + lane * C) = *reinterpret_cast<const uint32_t*>(o);
  }
}

// Zeros for the rows of entries none of whose tokens sees a key, or counts, sixteen rows of an entry at a time, dealt out over the blocks.  (With shared
// pages the last launch writes all rows.)
template <typename T, int D, int THREADS>
NXD_DEVICE void finish_idle(const PagedAttn& p, int thread) {
  const int chunks = (p.tile_rows + 15) / 16;
  for (long i = blockIdx.x; i < (long)p.B * p.row_tiles * chunks; i += gridDim.x) {
    const int e = (int)(i / chunks);
    if (entry_tiles(p, e) > 0) continue;
    const int b = e / p.row_tiles, row0 = e % p.row_tiles * p.tile_rows + (int)(i % chunks) * 16;
    const int rows = min(min(16, p.tile_rows), p.W * p.G - row0);
    for (int x = thread; x < rows * p.Hkv * (D / 8); x += THREADS) {
      const int c = x % (D / 8), y = x / (D / 8), head = y % p.Hkv, row = row0 + y / p.Hkv;
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + b * p.o_sb + row / p.G * p.o_sw + (long)(head * p.G + row % p.G) * p.o_sh + c * 8) =
          make_uint4(0, 0, 0, 0);
    }
  }
}

template <typename T> NXD_DEVICE uint32_t pack16(float lo, float hi);
template <> NXD_DEVICE uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> NXD_DEVICE uint32_t pack16<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <typename T> NXD_DEVICE void unpack16(uint32_t v, float& lo, float& hi);
template <> NXD_DEVICE void unpack16<__nv_bfloat16>(uint32_t v, float& lo, float& hi) { lo = __uint_as_float(v << 16); hi = __uint_as_float(v & 0xffff0000u); }
template <> NXD_DEVICE void unpack16<__half>(uint32_t v, float& lo, float& hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  lo = f.x;
  hi = f.y;
}

}  // namespace paged
}  // namespace nxd
