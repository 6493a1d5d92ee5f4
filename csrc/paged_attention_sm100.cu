// Attention of many query rows over a paged key/value cache on the tensor memory: drafted windows, portions of prompts, and the rows of a whole
// batch over the pages that all of it shares.  The work is dealt out as paged.cuh says, in tiles of 128 keys and of 128 query rows, or pairs of
// them.
//
// A block has two streams, half a step out of phase, so that one's softmax runs under the other's products:
//   PAIR     up to 256 rows: stream t has row tile t, both walk the same key tiles
//   else     up to 128 rows: both have the same row tile, stream t the key tiles of its parity; their sums are joined when they leave
// TMEM (512 columns): scores of stream 0 / 1, sums of stream 0 / 1, 128 columns each.
//   warps 0-3, 4-7  softmax  : thread = query row of stream 0 / 1; rows and pages that a row does not see are -inf; P over the scores
//   warps 8-11  rows         : query rows into shared memory (from wherever tokens and heads lie), sums out of TMEM to the output or to a part
//   warp 12     keys, values : pages by TMA, boxes of the largest power of two that divides a page; a hole, and all behind the last key, is a box
//                              outside the map, which arrives as zeros
//   warp 13     products     : S = Q Kᵀ and O += P V, issued by one elected lane
// Every wait gives up after two seconds (a wait that long is an error in here): the block then runs to its end without waiting, and its rows are NaN.
#include <cuda.h>

#include <algorithm>
#include <string>

#include "attention_sm100.cuh"
#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace nxd {

CUtensorMap make_tmap_bf16_heads(const void* ptr, const uint64_t (&dims)[4], const uint64_t (&strides)[3], uint32_t box_cols, uint32_t box_rows);

namespace {

using namespace paged;
using namespace fa;

constexpr int kRowsThreads = 512;
constexpr int kRows = 128, kKeyTile = 128;
constexpr int kSlots = 4;                        // key and value tiles in flight or in use
constexpr int kHoles = 8;                        // key tiles whose holes are remembered: more than are between the loads and the slower softmax
constexpr uint32_t kOutStage = 32 * 128;         // an output warp's 32 rows x 128 bytes on their way to memory
template <int D> constexpr uint32_t kTileBytes = 128 * D * 2;
constexpr uint32_t kHalfTile = 128 * 64 * 2;     // one [128 x 64] box
template <int D> constexpr uint32_t tiles_smem() { return (2 + kSlots) * kTileBytes<D> + 4 * kOutStage + 2048 /*row sums*/ + 1024 /*align*/ + 512 /*barriers*/; }

NXD_DEVICE void give_up_wait(uint32_t bar, uint32_t parity, uint32_t gave_up) {
  uint32_t done, tries = 0;
  uint64_t t0 = 0;
  while (true) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return;
    if ((++tries & 63u) == 0) {
      uint32_t over;
      uint64_t t;
      asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(over) : "r"(gave_up) : "memory");
      if (over) return;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
      if (t0 == 0) t0 = t;
      else if (t - t0 > 2000000000ull) {
        asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(gave_up), "r"(1u) : "memory");
        return;
      }
    }
  }
}

// P = 2^(s * scale - max) of 32 columns, packed to T in their first half; `sum` grows by it.  MAX: the maximum of the whole row beside it, NaN
// where there is one.
template <typename T, bool MAX>
NXD_DEVICE void exps(uint32_t (&r)[4][32], int c, uint64_t scale, uint64_t shift, uint64_t& sum, float& mx) {
  float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    if constexpr (MAX) {
#pragma unroll
      for (int k = 0; k < 4; ++k) m4[k] = max3_nan(m4[k], __uint_as_float(r[k][i]), __uint_as_float(r[k][i + 1]));
    }
    const uint64_t x = fma2(pack2u(r[c][i], r[c][i + 1]), scale, shift);
    float p0, p1;
    unpack2(x, p0, p1);
    p0 = ex2(p0);
    p1 = ex2(p1);
    sum = add2(sum, pack2(p0, p1));
    r[c][i >> 1] = pack16<T>(p0, p1);
  }
  if constexpr (MAX) mx = max3_nan(m4[0], m4[1], max3_nan(m4[2], m4[3], m4[3]));
}

// A share's next piece: key tiles [j0, j0 + n) of one pair; stream t has n_t of them
struct Item { int e, head, j0, n, n0, n1; bool begins, ends; };

template <bool PAIR, bool SHARED>
NXD_DEVICE Item make_item(const PagedAttn& p, const Walk& w, long left) {
  Item it;
  it.e = w.e; it.head = w.head; it.j0 = w.tile;
  it.n = (int)min((long)(w.tiles - w.tile), left);
  it.begins = w.tile == 0;
  it.ends = w.tile + it.n == w.tiles;
  if constexpr (PAIR) {
    // tiles of the pair that the first row tile sees, and whether there are rows in the second
    int first, second;
    if constexpr (SHARED) {
      first = w.tiles;
      second = w.e * p.pre_tile_rows + kRows < p.B * p.W * p.G ? w.tiles : 0;
    } else {
      const int b = w.e / p.row_tiles, r0 = w.e % p.row_tiles * p.tile_rows;
      first = row_key_tiles(p, b, r0, r0 + kRows);
      second = (r0 + kRows) / p.G < new_tokens(p, b) ? w.tiles : 0;
    }
    it.n0 = max(0, min(it.n, first - it.j0));
    it.n1 = max(0, min(it.n, second - it.j0));
  } else {
    it.n0 = (it.n + 1) / 2;
    it.n1 = it.n / 2;
  }
  return it;
}

// Where a role is in the block's share: all of them walk it on their own
template <bool PAIR, bool SHARED>
struct Share {
  Walk w;
  long left;
  NXD_DEVICE Item next(const PagedAttn& p) {       // n = 0: no more
    if (left <= 0) return Item{};
    const Item it = make_item<PAIR, SHARED>(p, w, left);
    left -= it.n;
    if (left > 0) next_pair<SHARED>(p, w);
    return it;
  }
};

template <typename T, int D, bool PAIR, bool SHARED>
__global__ void __launch_bounds__(kRowsThreads, 1)
paged_tiles_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const PagedAttn p, int box) {
  constexpr uint32_t TILE = kTileBytes<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = smem_base, sKV = smem_base + 2 * TILE, sO = sKV + kSlots * TILE, sStat = sO + 4 * kOutStage;
  const uint32_t bars = sStat + 2048;
  // per stream or row tile: qf[2] qe[2] s[2] p[2] of[2] oe[2] lf[2] le[2] | ring: kvf[] kve[] | tmem slot, gave up | holes[]
  const uint32_t bar_qf = bars, bar_qe = bars + 16, bar_s = bars + 32, bar_p = bars + 48, bar_of = bars + 64, bar_oe = bars + 80, bar_lf = bars + 96,
                 bar_le = bars + 112, bar_kvf = bars + 128, bar_kve = bar_kvf + 8 * kSlots, tmem_slot = bar_kve + 8 * kSlots, gave_up = tmem_slot + 4,
                 holes = gave_up + 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto wait = [&](uint32_t bar, uint32_t parity) { give_up_wait(bar, parity, gave_up); };

  if (warp == 12 && lane == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_qf + 8 * i, 128); mbar_init(bar_qe + 8 * i, 1); mbar_init(bar_s + 8 * i, 1);
      mbar_init(bar_p + 8 * i, 128); mbar_init(bar_of + 8 * i, 1); mbar_init(bar_oe + 8 * i, 128);
      mbar_init(bar_lf + 8 * i, 128); mbar_init(bar_le + 8 * i, 128);
    }
    for (int i = 0; i < kSlots; ++i) { mbar_init(bar_kvf + 8 * i, 1); mbar_init(bar_kve + 8 * i, 1); }
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(gave_up), "r"(0u) : "memory");
    fence_barrier_init();
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == 13) {
    tcgen05_alloc(tmem_slot, 512);
    tcgen05_relinquish();
  }
  pdl_wait();
  const Place at = find_place<kRowsThreads, SHARED>(p, gridDim.x, blockIdx.x);
  Share<PAIR, SHARED> share;
  share.left = min(at.per, at.total - blockIdx.x * at.per);
  share.w = Walk{at.e, 0, 0, 1};
  if (share.left > 0) {
    share.w.tiles = walk_tiles<SHARED>(p, at.e);
    share.w.head = (int)(at.tile / share.w.tiles);
    share.w.tile = (int)(at.tile % share.w.tiles);
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  pdl_trigger();                                   // behind the allocation; blocks of the merge wait for this grid
  uint32_t tmem_base;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
  const uint32_t tmem_S = tmem_base, tmem_O = tmem_base + 256;
  const int row_tiles = SHARED ? 1 : p.row_tiles, tile_rows = SHARED ? p.pre_tile_rows : p.tile_rows;
  const int all_rows = SHARED ? p.B * p.W * p.G : p.W * p.G;
  auto first_row = [&](const Item& it) { return SHARED ? it.e * tile_rows : it.e % row_tiles * tile_rows; };
  auto keys_of = [&](const Item& it) { return SHARED ? p.shared : all_keys(p, it.e / row_tiles); };
  auto key_at = [&](int j) { return (SHARED ? 0 : p.shared) + j * kKeyTile; };
  // sequence and token of a row, and whether it counts
  auto row_token = [&](const Item& it, int row, int& b, int& w) {
    const int t = row / p.G;
    b = SHARED ? t / p.W : it.e / row_tiles;
    w = SHARED ? t - b * p.W : t;
    return row < all_rows && w < new_tokens(p, b);
  };
  // ring position of step j's keys of stream t, counted from the item's first; the values are the next
  auto ring_at = [&](int t, int j) { return PAIR ? 2 * j : 2 * (2 * j + t); };

  // registers: 128 a thread at launch, 2 x 168 + 88 + 88 = 4 x 128 from here on
  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 12) {
      // lane = box of a tile
      int slot = 0, tile = 0;
      uint32_t ph = 0;
      const int boxes = kKeyTile / box;
      for (Item it = share.next(p); it.n > 0; it = share.next(p)) {
        const int n = keys_of(it), b = it.e / row_tiles;
        const int* table = SHARED ? p.shared_pages : p.table + b * p.table_sb;
        for (int j = 0; j < it.n; ++j, ++tile) {
          const int key = key_at(it.j0 + j) + lane * box;
          int page = -1;
          const bool inside = lane < boxes && key < n;
          if (inside) page = table[key / p.ps];
          if ((unsigned)page >= (unsigned)p.pages) page = -1;
          const unsigned hole = __ballot_sync(0xffffffffu, inside && page < 0);
          const int row = key % p.ps;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            wait(bar_kve + 8 * slot, ph ^ 1);
            if (lane == 0) {
              if (kv == 0) asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(holes + (tile % kHoles) * 4), "r"(hole) : "memory");
              mbar_expect_tx(bar_kvf + 8 * slot, TILE);
            }
            __syncwarp();
            if (lane < boxes) {
              // x, row in the page, head, page; a page of -1 is outside the map
              const uint32_t dst = sKV + slot * TILE + lane * box * 128;
#pragma unroll
              for (int h = 0; h < D / 64; ++h) tma_load_4d(dst + h * kHalfTile, kv ? &tv : &tk, bar_kvf + 8 * slot, h * 64, page < 0 ? 0 : row, it.head, page);
            }
            if (++slot == kSlots) { slot = 0; ph ^= 1; }
          }
        }
      }
      uint32_t over;
      asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(over) : "r"(gave_up) : "memory");
      if (over) {                                  // nothing of this block is on its way when it ends
        asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(gave_up), "r"(0u) : "memory");
        for (int i = 0; i < kSlots; ++i) wait(bar_kvf + 8 * ((slot + i) % kSlots), (slot + i) / kSlots ? ph : ph ^ 1);
        asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(gave_up), "r"(1u) : "memory");
      }
    } else if (warp == 13) {
      // all 32 lanes run this loop; the helpers elect one lane
      constexpr uint32_t kTypes = sizeof(T) == 2 && std::is_same<T, __half>::value ? (1u << 7) | (1u << 10) : 0u;
      constexpr uint32_t idesc_s = make_idesc(false, false, kRows, kKeyTile) & ~kTypes;
      constexpr uint32_t idesc_o = make_idesc(false, true, kRows, D) & ~kTypes;
      uint32_t steps = 0, q_items = 0, o_items = 0;                  // bit t: parity of stream t's (PAIR: row tile t's) count
      auto issue_s = [&](int t, int q, int pos, bool first, bool last, bool last_k) {
        const int slot = pos % kSlots;
        if (first) wait(bar_qf + 8 * q, (q_items >> q) & 1);
        wait(bar_kvf + 8 * slot, (uint32_t)((pos / kSlots) & 1));
        tcgen05_fence_after();
        const uint64_t a = make_smem_desc(sQ + q * TILE, 16, 1024), b = make_smem_desc(sKV + slot * TILE, 16, 1024);
        if constexpr (D == 128) mma_ss8<kHalfTile / 16, 2, kHalfTile / 16, 2>(tmem_S + t * 128, a, b, idesc_s, 0u, bar_s + 8 * t);
        else mma_ss4<2, 2>(tmem_S + t * 128, a, b, idesc_s, 0u, bar_s + 8 * t);
        if (last_k) tcgen05_commit_e(bar_kve + 8 * slot);
        if (last) { tcgen05_commit_e(bar_qe + 8 * q); q_items ^= 1u << q; }      // the row tile's last scores
      };
      Item it = share.next(p);
      int pos0 = 0, il = 0;                        // ring position of the item's first keys, number of the item
      // PAIR: row tile t belongs to stream t.  Otherwise item il's rows lie in tile il & 1, which both streams read: the item's last scores are
      // those of its last key tile.
      auto scores = [&](int t, int j, const Item& i, int base, int number) {
        const int nt = t ? i.n1 : i.n0;
        const bool last = PAIR ? j + 1 == nt : 2 * j + t + 1 == i.n;
        issue_s(t, PAIR ? t : number & 1, base + ring_at(t, j), j == 0, last, !PAIR || t == 1 || j >= i.n1);
      };
      for (int t = 0; t < 2; ++t)
        if ((t ? it.n1 : it.n0) > 0) scores(t, 0, it, 0, 0);
      for (; it.n > 0; ++il) {
        Item nx{};
        const int pos1 = pos0 + 2 * it.n, steps_n = max(it.n0, it.n1);
        bool asked = false;
        for (int j = 0; j < steps_n; ++j) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int nt = t ? it.n1 : it.n0;
            if (j < nt) {
              const int pos = pos0 + ring_at(t, j) + 1, slot = pos % kSlots;
              const uint32_t ph = (steps >> t) & 1;
              steps ^= 1u << t;
              wait(bar_kvf + 8 * slot, (uint32_t)((pos / kSlots) & 1));
              if (j == 0) { wait(bar_oe + 8 * t, ((o_items >> t) & 1) ^ 1); o_items ^= 1u << t; }   // the item before left O
              const uint32_t v_s = sKV + slot * TILE;
              wait(bar_p + 8 * t, ph);
              tcgen05_fence_after();
#pragma unroll
              for (int h = 0; h < 2; ++h)
                mma_ts4<16, 128>(tmem_O + t * 128, tmem_S + t * 128 + h * 32, make_smem_desc(v_s + h * 8192, kHalfTile, 1024), idesc_o, (j | h) ? 1u : 0u);
              if (!PAIR || t == 1 || j >= it.n1) tcgen05_commit_e(bar_kve + 8 * slot);
              if (j == nt - 1) tcgen05_commit_e(bar_of + 8 * t);
            }
            if (j + 1 < nt) {                      // scores over P of this step: behind its product in pipe order
              scores(t, j + 1, it, pos0, il);
            } else if (j == (PAIR && nt ? nt : steps_n) - 1) {
              // first scores of the next item: this stream's last product has been issued (streams that share their rows: stream 0's, too, so that
              // the item's last scores, which give the rows back, are the last to be issued)
              if (!asked) { nx = share.next(p); asked = true; }
              if ((t ? nx.n1 : nx.n0) > 0) scores(t, 0, nx, pos1, il + 1);
            }
          }
        }
        it = nx;
        pos0 = pos1;
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    const int quarter = warp & 3, own = quarter * 32 + lane;
    const uint32_t tO = tmem_O + ((uint32_t)(quarter * 32) << 16), stage = sO + quarter * kOutStage;
    uint32_t ph = 0, q_loads = 0;                  // bit t: parity of stream t's items, of row tile t's loads
    // thread = row: 16 bytes of it at a time, into the place that a 128-byte swizzle gives them
    auto load_q = [&](const Item& it, int q, int tile) {
      int b, w;
      const int row = first_row(it) + tile * kRows + own;
      const bool live = row_token(it, row, b, w);
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) +
                                                        (live ? b * p.q_sb + w * p.q_sw + (long)(it.head * p.G + row % p.G) * p.q_sh : 0));
      wait(bar_qe + 8 * q, ((q_loads >> q) & 1) ^ 1);
      q_loads ^= 1u << q;
      const uint32_t dst = sQ + q * TILE + own * 128;
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        uint4 x[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) x[c] = live ? src[h * 8 + c] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < 8; ++c)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + h * kHalfTile + ((c ^ (own & 7)) << 4)), "r"(x[c].x), "r"(x[c].y), "r"(x[c].z),
                       "r"(x[c].w) : "memory");
      }
      fence_async_smem();
      mbar_arrive(bar_qf + 8 * q);
    };
    Item it = share.next(p);
    if (it.n > 0)
      for (int t = 0; t < (PAIR ? 2 : 1); ++t)
        if (!PAIR || (t ? it.n1 : it.n0) > 0) load_q(it, t, t);
    for (int il = 0; it.n > 0; ++il) {
      const Item nx = share.next(p);
      // the next item's rows before this one's sums: the products wait for those rows before they have issued the last of this item's
      if (nx.n > 0) {
        if (!PAIR) load_q(nx, (il + 1) & 1, 0);
        else
          for (int t = 0; t < 2; ++t)
            if ((t ? nx.n1 : nx.n0) > 0) load_q(nx, t, t);
      }
      const bool merge = !PAIR && it.n1 > 0, direct = !SHARED && p.shared == 0 && it.begins && it.ends;
      const long slot = part_slot<SHARED>(p, (long)it.e * p.Hkv + it.head, blockIdx.x, it.begins) * tile_rows;
#pragma unroll 1
      for (int t = 0; t < (PAIR ? 2 : 1); ++t) {
        const int r0 = t * kRows + quarter * 32;   // the warp's rows of the item's
        const int row = first_row(it) + r0 + lane;
        int b, w;
        const bool live = row_token(it, row, b, w);
        const bool none = (t ? it.n1 : it.n0) == 0;
        float m = -INFINITY, l = 0.f, f0 = 1.f, f1 = 0.f;
        if (!none) {
          wait(bar_of + 8 * t, (ph >> t) & 1);
          wait(bar_lf + 8 * t, (ph >> t) & 1);
          ph ^= 1u << t;
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(m), "=f"(l) : "r"(sStat + t * 1024 + own * 8) : "memory");
          mbar_arrive(bar_le + 8 * t);
          if (merge) {
            wait(bar_of + 8, (ph >> 1) & 1);
            wait(bar_lf + 8, (ph >> 1) & 1);
            ph ^= 2u;
            float m1, l1;
            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(m1), "=f"(l1) : "r"(sStat + 1024 + own * 8) : "memory");
            mbar_arrive(bar_le + 8);
            const float mm = fmaxf(m, m1);
            f0 = m == -INFINITY ? 0.f : exp2f(m - mm);
            f1 = m1 == -INFINITY ? 0.f : exp2f(m1 - mm);
            l = l * f0 + l1 * f1;
            m = mm;
          }
          tcgen05_fence_after();
          uint32_t over;
          asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(over) : "r"(gave_up) : "memory");
          if (over) l = __int_as_float(0x7fffffff);
        }
        if (!direct && live) {
          float* const ml = (SHARED ? p.pre_ml : p.part_ml) + (slot + r0 + lane) * 2;
          *reinterpret_cast<float2*>(ml) = make_float2(m, l);
        }
        // where this lane's row goes: -1 nowhere, -2 zeros
        long to = -1;
        if (direct ? row < all_rows : live && !none) {
          if (direct) to = b * p.o_sb + w * p.o_sw + (long)(it.head * p.G + row % p.G) * p.o_sh;
          else to = (slot + r0 + lane) * D;
        }
        const float inv = !direct ? 1.f : !live || l == 0.f ? 0.f : 1.f / l;
        f0 *= inv;
        f1 *= inv;
        if (!none) {
          // The rows leave through the warp's stage, 128 bytes of each at a time
          constexpr int COLS = 32;                           // sums of a stage: 128 bytes
#pragma unroll 1
          for (int c = 0; c < D / COLS; ++c) {
            uint32_t r[32];
            tcgen05_ld_32x32(tO + t * 128 + c * COLS, r);
            if (merge) {
              uint32_t r1[32];
              tcgen05_ld_32x32(tO + 128 + c * COLS, r1);
              tcgen05_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f0 + __uint_as_float(r1[i]) * f1);
            } else {
              tcgen05_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f0);
            }
            if (direct && inv == 0.f) {                      // a row that sees nothing, or does not count, whatever the products left
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = 0u;
            }
            if (c == D / COLS - 1) {                         // the next item's first product may overwrite O
              tcgen05_fence_before();
              mbar_arrive(bar_oe + 8 * t);
              if (merge) mbar_arrive(bar_oe + 8);
            }
            __syncwarp();                                    // what was in the stage has been read
            if (direct) {
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = pack16<T>(__uint_as_float(r[v * 8 + 2 * i]), __uint_as_float(r[v * 8 + 2 * i + 1]));
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 + ((v ^ ((lane >> 1) & 3)) << 4)), "r"(o[0]), "r"(o[1]), "r"(o[2]),
                             "r"(o[3]) : "memory");
              }
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 4; ++i) {                  // rows 8 i + lane / 4
                const int rr = 8 * i + (lane >> 2);
                uint4 o;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(o.x), "=r"(o.y), "=r"(o.z), "=r"(o.w)
                             : "r"(stage + rr * 64 + (((lane & 3) ^ ((rr >> 1) & 3)) << 4)) : "memory");
                const long dst = __shfl_sync(0xffffffffu, to, rr);
                if (dst >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + dst + c * COLS + (lane & 3) * 8) = o;
              }
            } else {
#pragma unroll
              for (int v = 0; v < 8; ++v)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((v ^ (lane & 7)) << 4)), "r"(r[4 * v]), "r"(r[4 * v + 1]),
                             "r"(r[4 * v + 2]), "r"(r[4 * v + 3]) : "memory");
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 8; ++i) {                  // rows 4 i + lane / 8
                const int rr = 4 * i + (lane >> 3);
                uint4 o;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(o.x), "=r"(o.y), "=r"(o.z), "=r"(o.w)
                             : "r"(stage + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4)) : "memory");
                const long dst = __shfl_sync(0xffffffffu, to, rr);
                if (dst >= 0) *reinterpret_cast<uint4*>((SHARED ? p.pre_o : p.part_o) + dst + c * COLS + (lane & 7) * 4) = o;
              }
            }
          }
        } else if (direct && to >= 0) {                      // rows that do not count
          for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + to + c) = make_uint4(0, 0, 0, 0);
        }
      }
      it = nx;
    }
    if (!SHARED && p.shared == 0)
      for (int e = blockIdx.x; e < p.B * p.row_tiles; e += gridDim.x)
        if (entry_tiles(p, e) == 0) finish_idle<T, D, 128>(p, e, threadIdx.x - 256);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    const int t = warp >= 4;                       // stream of this warpgroup
    const int quarter = warp & 3, own = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem_S + t * 128 + lane_base, tO = tmem_O + t * 128 + lane_base;
    const uint32_t my_s = bar_s + 8 * t, my_p = bar_p + 8 * t;
    const float sl2 = p.scale_log2;
    const uint64_t sl2_2 = pack2(sl2, sl2);
    int g = 0, items = 0, pos0 = 0, tile0 = 0;
    for (Item it = share.next(p); it.n > 0; pos0 += 2 * it.n, tile0 += it.n, it = share.next(p)) {
      const int nt = t ? it.n1 : it.n0;
      if (nt == 0) continue;
      int b, w;
      const int row = first_row(it) + (PAIR ? t * kRows : 0) + own, n = keys_of(it);
      const bool live = row_token(it, row, b, w);
      // keys that this row sees (one that does not count: all, whatever comes of it), and the fewest of the warp's rows
      const int sees = live ? min(visible_keys(p, b, w), n) : 0x7fffffff;
      const int sees_lo = __reduce_min_sync(0xffffffffu, sees);
      float m_ref = -INFINITY, l = 0.f;
      for (int j = 0; j < nt; ++j, ++g) {
        const int jt = PAIR ? j : 2 * j + t, key0 = key_at(it.j0 + jt), pos = pos0 + ring_at(t, j);
        wait(my_s, (uint32_t)(g & 1));
        tcgen05_fence_after();
        uint32_t hole;                             // written before the keys' barrier, which the products waited for
        asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(hole) : "r"(holes + ((tile0 + jt) % kHoles) * 4) : "memory");
        uint32_t sr[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tcgen05_ld_32x32(tS + c * 32, sr[c]);
        tcgen05_wait_ld();
        const int lim = sees - 1 - key0, lim_lo = sees_lo - 1 - key0;            // last column that is seen
        if (lim_lo < 127) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (lim_lo < c * 32 + 31) fwd_mask(sr[c], lim - c * 32);
        }
        if (hole) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (hole >> ((c * 32 + i) / box) & 1) sr[c][i] = 0xff800000u;
        }
        if (j == 0) {
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; i += 2)
#pragma unroll
            for (int c = 0; c < 4; ++c) m4[c] = max3(m4[c], __uint_as_float(sr[c][i]), __uint_as_float(sr[c][i + 1]));
          m_ref = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]);
        }
        float base = m_ref == -INFINITY ? 0.f : m_ref;       // a row that has seen nothing yet
        uint64_t shift = pack2(-base * sl2, -base * sl2), sum[4] = {0ull, 0ull, 0ull, 0ull};
        float mx, unused;
        exps<T, true>(sr, 0, sl2_2, shift, sum[0], mx);
        const bool need = (mx - base) * sl2 > 8.f || (m_ref == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xffffffffu, need)) {
          const float f = !need ? 1.f : m_ref == -INFINITY ? 0.f : ex2((m_ref - mx) * sl2);
          if (need) m_ref = base = mx;
          l *= f;
          shift = pack2(-base * sl2, -base * sl2);
          if (j > 0) {                             // PV of the step before is done (these scores came after it): O is quiescent
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t r[16];
              tcgen05_ld_32x16(tO + c * 16, r);
              tcgen05_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
              tcgen05_st_32x16(tO + c * 16, r);
            }
          }
          tcgen05_ld_32x32(tS, sr[0]);
          tcgen05_wait_ld();
          if (lim_lo < 31) fwd_mask(sr[0], lim);
          if (hole) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (hole >> (i / box) & 1) sr[0][i] = 0xff800000u;
          }
          sum[0] = 0ull;
          exps<T, false>(sr, 0, sl2_2, shift, sum[0], unused);
        }
        if (!(mx < INFINITY)) l = __int_as_float(0x7fffffff);        // NaN or +inf among the scores: a row of NaN
        tcgen05_st_32x16p(tS, sr[0]);
#pragma unroll
        for (int c = 1; c < 4; ++c) {
          exps<T, false>(sr, c, sl2_2, shift, sum[c], unused);
          tcgen05_st_32x16p(tS + c * 16, sr[c]);
        }
        if (key0 + kKeyTile > n) {
          // behind the last key: the rest of its page may hold anything, and 0 times NaN is NaN
          wait(bar_kvf + 8 * ((pos + 1) % kSlots), (uint32_t)(((pos + 1) / kSlots) & 1));
          if (key0 + own >= n) {
            const uint32_t dst = sKV + (pos + 1) % kSlots * TILE + own * 128;
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + (c >> 3) * kHalfTile + (c & 7) * 16), "r"(0u) : "memory");
          }
          fence_async_smem();
        }
        tcgen05_wait_st();
        tcgen05_fence_before();
        mbar_arrive(my_p);
        float l4[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) { float x, y; unpack2(sum[c], x, y); l4[c] = x + y; }
        l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
      }
      // ---- maximum (in units of the exponent) and row sum to the output warps
      wait(bar_le + 8 * t, (uint32_t)((items & 1) ^ 1));
      ++items;
      asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(sStat + t * 1024 + own * 8), "f"(m_ref * sl2), "f"(l) : "memory");
      mbar_arrive(bar_lf + 8 * t);
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 13) tcgen05_dealloc(tmem_base, 512);
}

template <typename T, int D, bool PAIR, bool SHARED>
void launch_tiles(const PagedAttn& p, int grid, cudaStream_t st) {
  // boxes of the largest power of two that divides a page
  const int box = std::min(p.ps & -p.ps, kKeyTile);
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)p.ps, (uint64_t)p.Hkv, (uint64_t)p.pages};
  // (the stride of a dimension of one is anything)
  auto step = [&](long stride, long n) { return (uint64_t)(n == 1 ? D : stride); };
  const uint64_t ks[3] = {step(p.k_sr, p.ps), step(p.k_sh, p.Hkv), step(p.k_sp, p.pages)}, vs[3] = {step(p.v_sr, p.ps), step(p.v_sh, p.Hkv), step(p.v_sp, p.pages)};
  const CUtensorMap tk = make_tmap_bf16_heads(p.k, dims, ks, 64, box), tv = make_tmap_bf16_heads(p.v, dims, vs, 64, box);
  NXD_ALLOW_SMEM((paged_tiles_kernel<T, D, PAIR, SHARED>), tiles_smem<D>());
  launch_dependent(paged_tiles_kernel<T, D, PAIR, SHARED>, grid, kRowsThreads, tiles_smem<D>(), st, tk, tv, p, box);
}

}  // namespace

void paged_tiles(const PagedAttn& p, int grid, bool over_shared, int D, int dt, cudaStream_t st) {
  const bool pair = (over_shared ? p.pre_tile_rows : p.tile_rows) == 2 * kRows;
#define NXD_TILES(T, Dv)                                                                                                     \
  do {                                                                                                                       \
    if (over_shared) { if (pair) launch_tiles<T, Dv, true, true>(p, grid, st); else launch_tiles<T, Dv, false, true>(p, grid, st); } \
    else { if (pair) launch_tiles<T, Dv, true, false>(p, grid, st); else launch_tiles<T, Dv, false, false>(p, grid, st); }     \
  } while (0)
  if (dt == kBF16) { if (D == 128) NXD_TILES(__nv_bfloat16, 128); else NXD_TILES(__nv_bfloat16, 64); }
  else { if (D == 128) NXD_TILES(__half, 128); else NXD_TILES(__half, 64); }
#undef NXD_TILES
}

}  // namespace nxd
