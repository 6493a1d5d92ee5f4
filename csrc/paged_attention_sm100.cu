// Attention of many query rows over a paged key/value cache on the tensor memory: drafted windows, portions of prompts, and the rows of a whole
// batch over the pages that all of it shares.  The work is dealt out as paged.cuh says.
//
// A block has two streams, half a step out of phase, so that one's softmax runs under the other's products:
//   PAIR     up to 256 rows: stream t has row tile t, both walk the same tiles of 128 keys; bound by products and exponentials
//   else     up to 128 rows: both have the same row tile, stream t the tiles of 64 keys of its parity; their sums are joined when they leave.  Bound by
//            HBM: small tiles, because each stream holds two of them while it works, and what is left of the ring is what is on its way
// TMEM (512 columns): scores of stream 0 / 1, sums of stream 0 / 1, 128 columns each.
//   warps 0-3, 4-7  softmax  : thread = query row of stream 0 / 1; rows and pages that a row does not see are -inf; P over the scores
//   warps 8-11  rows         : query rows into shared memory (from wherever tokens and heads lie), sums out of TMEM to the output or to a part
//   warp 12     keys, values : pages by TMA, boxes of the largest power of two that divides a page; a hole, and all behind the last key, is a box
//                              outside the map, which arrives as zeros
//   warp 13     products     : S = Q Kᵀ and O += P V, issued by one elected lane
//   warp 14     pieces       : the block's share cut into pieces of pairs, handed to the others two at a time
//   warp 15     failures     : rows of NaN where a wait ran out
// The row warps, which wait for all that the others do, give a wait up after two seconds (one that long is an error in here), and so do the others then.
// What a thread hands on from there is worth nothing; at the end copies and products in flight are waited for, and the block's rows become NaN.
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
constexpr int kRows = 128;
constexpr int kHoles = 32;                       // key tiles whose holes are remembered: more than are between the loads and the slower softmax
constexpr uint32_t kOutStage = 32 * 128;         // an output warp's 32 rows x 128 bytes on their way to memory

// Keys of a tile, tiles of the ring (keys and values each one), bytes.  ROWS: query rows of a row tile that may be there.  The products read 128
// all the same: with ROWS = 64 the others are whatever lies behind them, and so are their results.
template <int D, bool PAIR, int ROWS>
struct Cut {
  static constexpr int KEYS = PAIR ? 128 : 64;
  static constexpr uint32_t Q_TILE = ROWS * D * 2, Q_HALF = ROWS * 128, TILE = KEYS * D * 2, HALF = KEYS * 128;
  static constexpr uint32_t STAGE = PAIR ? 4 * kOutStage : 0, FIXED = 2 * Q_TILE + STAGE + 2048 /*row sums*/ + 1024 /*align*/ + 1024 /*barriers*/;
  static constexpr int SLOTS = PAIR ? 128 * 1024 / TILE : std::min(16u, (226 * 1024 - FIXED) / TILE);
  static constexpr uint32_t SMEM = FIXED + SLOTS * TILE;
};

constexpr uint32_t kLimit = 4;                   // behind the word that says that a block has given up: after how many ns
// → whether the phase has ended.  CLOCK: at most that long, and the word (WORD) says so to the others; otherwise until the word says so.
template <bool CLOCK, bool WORD>
NXD_DEVICE bool bounded_wait(uint32_t bar, uint32_t parity, uint32_t gave_up) {
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
    if (done) return true;
    if ((++tries & 63u) == 0) {
      if constexpr (WORD) {
        uint32_t over;
        asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(over) : "r"(gave_up) : "memory");
        if (over) return false;
      }
      if constexpr (CLOCK) {
        uint32_t limit;
        uint64_t t;
        asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(limit) : "r"(gave_up + kLimit) : "memory");
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
        if (t0 == 0) t0 = t;
        else if (t - t0 > limit) {
          if constexpr (WORD) asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(gave_up), "r"(1u) : "memory");
          return false;
        }
      }
    }
  }
}

// P = 2^(s * scale - max) of 32 columns, packed to T in their first half; `sum` grows by it.  MAX: the maximum of the whole row beside it, NaN
// where there is one.
template <typename T, int Q, bool MAX>
NXD_DEVICE void exps(uint32_t (&r)[Q][32], int c, uint64_t scale, uint64_t shift, uint64_t& sum, float& mx) {
  float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    if constexpr (MAX) {
#pragma unroll
      for (int k = 0; k < Q; ++k) m4[k] = max3_nan(m4[k], __uint_as_float(r[k][i]), __uint_as_float(r[k][i + 1]));
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

// A piece of a block's share: key tiles [j0, j0 + n) of one pair; stream t has n_t of them.  `keys`: of the pair's sequence.
struct alignas(16) Item { int e, head, j0, n, n0, n1, keys, ends; };      // ends: bit 0, the pair begins in it; bit 1, it ends

template <bool PAIR, bool SHARED>
NXD_DEVICE Item make_item(const PagedAttn& p, const Walk& w, long left) {
  Item it;
  it.e = w.e; it.head = w.head; it.j0 = w.tile;
  it.n = whole<SHARED>(p, w.tiles) ? w.tiles : (int)min((long)(w.tiles - w.tile), left);
  it.ends = (w.tile == 0) | (w.tile + it.n == w.tiles ? 2 : 0);
  it.keys = SHARED ? p.shared : all_keys(p, w.e / p.row_tiles);
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

// Where block's share begins, and how many tiles it has
template <bool SHARED>
NXD_DEVICE long begin_share(const PagedAttn& p, const Place& at, Walk& w) {
  long left = min(at.per, at.total - blockIdx.x * at.per);
  w = Walk{at.e, 0, 0, 1};
  if (left > 0) {
    w.tiles = walk_tiles<SHARED>(p, at.e);
    w.head = (int)(at.tile / w.tiles);
    w.tile = (int)(at.tile % w.tiles);
    if (w.tile > 0 && whole<SHARED>(p, w.tiles)) {         // the block in front has it
      left -= w.tiles - w.tile;
      if (left > 0) next_pair<SHARED>(p, w);
    }
  }
  return left;
}

// PAIR: a step of two row tiles and 128 keys takes 2.2 us: exponentials 1.05, products 1.05 (heads of 128 numbers), which overlap little.  2 x 1000 tokens (a
// quarter padding) behind 6000 keys, 48 heads of 64 on 8: 158 us, 470 TFLOP/s.  Otherwise: two tiles of 64 keys in 1.7 us, 5 TB/s over the GPU; windows of 5
// tokens of 8 sequences to 6000 keys, 64 heads on 8: 43 us, of which 7 are the start and 5 the launch that joins parts.
template <typename T, int D, bool PAIR, int ROWS, bool SHARED>
__global__ void __launch_bounds__(kRowsThreads, 1)
paged_tiles_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const PagedAttn p, int box) {
  using C = Cut<D, PAIR, ROWS>;
  constexpr int KEYS = C::KEYS, SLOTS = C::SLOTS;
  constexpr uint32_t TILE = C::TILE;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = smem_base, sKV = smem_base + 2 * C::Q_TILE, sO = sKV + SLOTS * TILE, sStat = sO + C::STAGE;
  const uint32_t bars = sStat + 2048;
  // per stream or row tile: qf[2] qe[2] s[2] p[2] of[2] oe[2] lf[2] le[2] | pieces: full[2] empty[2] | ring: kvf[] kve[] | tmem slot, products done |
  // gave up, limit, ring's end (slot, lap) | pieces[2] | holes[]
  const uint32_t bar_qf = bars, bar_qe = bars + 16, bar_s = bars + 32, bar_p = bars + 48, bar_of = bars + 64, bar_oe = bars + 80, bar_lf = bars + 96,
                 bar_le = bars + 112, bar_nf = bars + 128, bar_ne = bars + 144, bar_kvf = bars + 160, bar_kve = bar_kvf + 8 * SLOTS,
                 tmem_slot = bar_kve + 8 * SLOTS, bar_end = tmem_slot + 8, gave_up = tmem_slot + 16, last_key = tmem_slot + 24, pieces = tmem_slot + 32, holes = pieces + 64;
  static_assert(160 + 16 * SLOTS + 32 + 64 + 4 * kHoles <= 1024, "barriers");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto wait = [&](uint32_t bar, uint32_t parity) { return bounded_wait<false, true>(bar, parity, gave_up); };
  auto clocked_wait = [&](uint32_t bar, uint32_t parity) { bounded_wait<true, true>(bar, parity, gave_up); };
  // Whoever is told of something by a thread that gave up before sees this, too: the word is written first
  auto failed = [&] {
    uint32_t over;
    asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(over) : "r"(gave_up) : "memory");
    return over;
  };

  if (warp == 12 && lane == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_qf + 8 * i, 128); mbar_init(bar_qe + 8 * i, 1); mbar_init(bar_s + 8 * i, 1);
      mbar_init(bar_p + 8 * i, 128); mbar_init(bar_of + 8 * i, 1); mbar_init(bar_oe + 8 * i, 128);
      mbar_init(bar_lf + 8 * i, 128); mbar_init(bar_le + 8 * i, 128);
      mbar_init(bar_nf + 8 * i, 1); mbar_init(bar_ne + 8 * i, 14);       // readers: softmax, row, key and product warps
    }
    for (int i = 0; i < SLOTS; ++i) { mbar_init(bar_kvf + 8 * i, 1); mbar_init(bar_kve + 8 * i, 1); }
    mbar_init(bar_end, 1);
    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(gave_up), "r"(0u), "r"(abs(p.wait_ns)) : "memory");
    fence_barrier_init();
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == 13) {
    tcgen05_alloc(tmem_slot, 512);
    tcgen05_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  uint32_t tmem_base;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
  const uint32_t tmem_S = tmem_base, tmem_O = tmem_base + 256;
  const int row_tiles = SHARED ? 1 : p.row_tiles, tile_rows = SHARED ? p.pre_tile_rows : p.tile_rows;
  const int all_rows = SHARED ? p.B * p.W * p.G : p.W * p.G;
  auto first_row = [&](const Item& it) { return SHARED ? it.e * tile_rows : it.e % row_tiles * tile_rows; };
  auto key_at = [&](int j) { return (SHARED ? 0 : p.shared) + j * KEYS; };
  // a warp's next piece; n = 0: no more
  int piece = 0;
  auto next_item = [&](auto... clock) {
    const int st = piece & 1;
    bounded_wait<sizeof...(clock) != 0, true>(bar_nf + 8 * st, (uint32_t)((piece >> 1) & 1), gave_up);
    ++piece;
    Item it;
    const uint32_t at = pieces + st * 32;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(it.e), "=r"(it.head), "=r"(it.j0), "=r"(it.n) : "r"(at) : "memory");
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(it.n0), "=r"(it.n1), "=r"(it.keys), "=r"(it.ends) : "r"(at + 16) : "memory");
    const uint32_t over = failed();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_ne + 8 * st);
    if (over) it.n = it.n0 = it.n1 = 0;            // pieces may not be what they should
    return it;
  };
  // sequence and token of a row, and whether it counts
  auto row_token = [&](const Item& it, int row, int& b, int& w) {
    const int t = row / p.G;
    b = SHARED ? t / p.W : it.e / row_tiles;
    w = SHARED ? t - b * p.W : t;
    return row < all_rows && w < new_tokens(p, b);
  };
  // row `own` of a row tile, whole: 16 bytes at a time into the places that a 128-byte swizzle gives them
  auto load_q = [&](const Item& it, int q, int tile, int own) {
    int b, w;
    const int row = first_row(it) + tile * kRows + own;
    const bool live = row_token(it, row, b, w);
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) +
                                                      (live ? b * p.q_sb + w * p.q_sw + (long)(it.head * p.G + row % p.G) * p.q_sh : 0));
    const uint32_t dst = sQ + q * C::Q_TILE + own * 128;
    if (ROWS == kRows || own < ROWS) {
      uint4 x[D / 8];
#pragma unroll
      for (int c = 0; c < D / 8; ++c) x[c] = live ? src[c] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (c >> 3) * C::Q_HALF + (((c & 7) ^ (own & 7)) << 4)), "r"(x[c].x), "r"(x[c].y),
                     "r"(x[c].z), "r"(x[c].w) : "memory");
    }
    fence_async_smem();
    mbar_arrive(bar_qf + 8 * q);
  };
  // ring position of step j's keys of stream t, counted from the item's first; the values are the next
  auto ring_at = [&](int t, int j) { return PAIR ? 2 * j : 2 * (2 * j + t); };

  // registers: 128 a thread at launch, 2 x 168 + 88 + 88 = 4 x 128 from here on
  Place at;
  const bool late = !SHARED && p.shared > 0;       // the launch in front has waited for what is read here, and writes none of it (paged.cuh)
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (!late) pdl_wait();
    pdl_trigger();                                 // behind the allocation; the last launch waits for this grid
    at = find_place<256, SHARED, 256>(p, gridDim.x, blockIdx.x);
  }
  if (warp >= 12) {
    if (warp == 12) {
      // lane = box of a tile; pages are looked up for 32 boxes at a time, one round ahead of those that are asked for
      int slot = 0, tile = 0;
      uint32_t ph = 0;
      bool ok = true;
      const int boxes = KEYS / box, round = 32 / boxes;
      for (Item it = p.wait_ns < 0 ? Item{} : next_item(); it.n > 0; it = next_item()) {
        const int n = it.keys;
        const int* table = p.table + (SHARED ? 0 : it.e / row_tiles * p.table_sb);
        auto look_up = [&](int j) {
          const int at = j + lane / boxes, key = key_at(it.j0 + at) + lane % boxes * box;
          const int i = key / p.ps;
          return at >= it.n || key >= n ? -1 : i < p.shared_cols ? p.shared_pages[i] : table[i];
        };
        int found = look_up(0), next = look_up(round);
        for (int j = 0; j < it.n; ++j, ++tile) {
          const int in_round = j % round;
          if (in_round == 0 && j > 0) { found = next; next = look_up(j + round); }
          const int key = key_at(it.j0 + j) + lane * box;
          int page = __shfl_sync(0xffffffffu, found, (in_round * boxes + lane) & 31);
          if ((unsigned)page >= (unsigned)p.pages) page = -1;
          const unsigned hole = __ballot_sync(0xffffffffu, lane < boxes && key < n && page < 0);
          const int row = key % p.ps;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            ok &= wait(bar_kve + 8 * slot, ph ^ 1);
            if (lane == 0 && ok) {
              if (kv == 0) asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(holes + (tile % kHoles) * 4), "r"(hole) : "memory");
              mbar_expect_tx(bar_kvf + 8 * slot, TILE);
            }
            __syncwarp();
            if (lane < boxes && ok) {
              // x, row in the page, head, page; a page of -1 is outside the map
              const uint32_t dst = sKV + slot * TILE + lane * box * 128;
#pragma unroll
              for (int h = 0; h < D / 64; ++h) tma_load_4d(dst + h * C::HALF, kv ? &tv : &tk, bar_kvf + 8 * slot, h * 64, page < 0 ? 0 : row, it.head, page);
            }
            if (++slot == SLOTS) { slot = 0; ph ^= 1; }
          }
        }
      }
      if (lane == 0) asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(last_key), "r"(slot), "r"(ph) : "memory");
      asm volatile("bar.arrive 2, 224;" ::: "memory");     // warp 15 waits for this
    } else if (warp == 13) {
      // all 32 lanes run this loop; the helpers elect one lane
      constexpr uint32_t kTypes = sizeof(T) == 2 && std::is_same<T, __half>::value ? (1u << 7) | (1u << 10) : 0u;
      constexpr uint32_t idesc_s = make_idesc(false, false, kRows, KEYS) & ~kTypes;
      constexpr uint32_t idesc_o = make_idesc(false, true, kRows, D) & ~kTypes;
      uint32_t steps = 0, q_items = 0, o_items = 0;                  // bit t: parity of stream t's (PAIR: row tile t's) count
      auto issue_s = [&](int t, int q, int pos, bool first, bool last, bool last_k) {
        const int slot = pos % SLOTS;
        if (first) wait(bar_qf + 8 * q, (q_items >> q) & 1);
        wait(bar_kvf + 8 * slot, (uint32_t)((pos / SLOTS) & 1));
        tcgen05_fence_after();
        const uint64_t a = make_smem_desc(sQ + q * C::Q_TILE, 16, 1024), b = make_smem_desc(sKV + slot * TILE, 16, 1024);
        if constexpr (D == 128) mma_ss8<C::Q_HALF / 16, 2, C::HALF / 16, 2>(tmem_S + t * 128, a, b, idesc_s, 0u, bar_s + 8 * t);
        else mma_ss4<2, 2>(tmem_S + t * 128, a, b, idesc_s, 0u, bar_s + 8 * t);
        if (last_k) tcgen05_commit_e(bar_kve + 8 * slot);
        if (last) { tcgen05_commit_e(bar_qe + 8 * q); q_items ^= 1u << q; }      // the row tile's last scores
      };
      Item it = next_item();
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
              const int pos = pos0 + ring_at(t, j) + 1, slot = pos % SLOTS;
              const uint32_t ph = (steps >> t) & 1;
              steps ^= 1u << t;
              wait(bar_kvf + 8 * slot, (uint32_t)((pos / SLOTS) & 1));
              if (j == 0) { wait(bar_oe + 8 * t, ((o_items >> t) & 1) ^ 1); o_items ^= 1u << t; }   // the item before left O
              const uint32_t v_s = sKV + slot * TILE;
              wait(bar_p + 8 * t, ph);
              tcgen05_fence_after();
#pragma unroll
              for (int h = 0; h < KEYS / 64; ++h)
                mma_ts4<16, 128>(tmem_O + t * 128, tmem_S + t * 128 + h * 32, make_smem_desc(v_s + h * 8192, C::HALF, 1024), idesc_o, (j | h) ? 1u : 0u);
              if (!PAIR || t == 1 || j >= it.n1) tcgen05_commit_e(bar_kve + 8 * slot);
              if (j == nt - 1) tcgen05_commit_e(bar_of + 8 * t);
            }
            if (j + 1 < nt) {                      // scores over P of this step: behind its product in pipe order
              scores(t, j + 1, it, pos0, il);
            } else if (j == (PAIR && nt ? nt : steps_n) - 1) {
              // first scores of the next item: this stream's last product has been issued (streams that share their rows: stream 0's, too, so that
              // the item's last scores, which give the rows back, are the last to be issued)
              if (!asked) { nx = next_item(); asked = true; }
              if ((t ? nx.n1 : nx.n0) > 0) scores(t, 0, nx, pos1, il + 1);
            }
          }
        }
        it = nx;
        pos0 = pos1;
      }
      tcgen05_commit_e(bar_end);
      asm volatile("bar.arrive 2, 224;" ::: "memory");     // warp 15 waits for this
    }
    if (warp == 14) {
      Walk w;
      long left = begin_share<SHARED>(p, at, w);
      bool more = true;
      for (int i = 0; more; ++i) {
        more = left > 0;
        Item it{};
        if (more) {
          it = make_item<PAIR, SHARED>(p, w, left);
          left -= it.n;
          if (left > 0) next_pair<SHARED>(p, w);
        }
        const uint32_t st = i & 1, dst = pieces + st * 32;
        wait(bar_ne + 8 * st, (uint32_t)(((i >> 1) & 1) ^ 1));
        if (lane == 0) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(it.e), "r"(it.head), "r"(it.j0), "r"(it.n) : "memory");
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + 16), "r"(it.n0), "r"(it.n1), "r"(it.keys), "r"(it.ends) : "memory");
          mbar_arrive(bar_nf + 8 * st);
        }
      }
    }
    if (warp == 15) {
      asm volatile("bar.sync 2, 224;" ::: "memory");       // keys have been asked for, products issued, rows have left
      bounded_wait<true, false>(bar_end, 0, gave_up);      // nothing of this block is being multiplied, or told of that, when it ends
      Walk w;
      long left = 0;
      if (failed()) {                              // nor is anything on its way
        int slot;
        uint32_t ph;
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(slot), "=r"(ph) : "r"(last_key) : "memory");
        for (int i = 0; i < SLOTS; ++i) bounded_wait<true, false>(bar_kvf + 8 * ((slot + i) % SLOTS), (slot + i) / SLOTS ? ph : ph ^ 1, gave_up);
        left = begin_share<SHARED>(p, at, w);
      }
      while (left > 0) {                           // and its rows are NaN, or parts that make them NaN
        const Item it = make_item<PAIR, SHARED>(p, w, left);
        left -= it.n;
        if (left > 0) next_pair<SHARED>(p, w);
        const long slot = part_slot<SHARED>(p, (long)it.e * p.Hkv + it.head, blockIdx.x, it.ends & 1) * tile_rows;
#pragma unroll 1
        for (int r = lane; r < tile_rows; r += 32) {
          const int row = first_row(it) + r;
          int b, t;
          const bool live = row_token(it, row, b, t);
          if (!SHARED && p.shared == 0 && it.ends == 3) {
            const uint32_t x = live ? 0x7fff7fffu : 0u;
            T* const to = reinterpret_cast<T*>(p.out) + b * p.o_sb + t * p.o_sw + (long)(it.head * p.G + row % p.G) * p.o_sh;
            if (row < all_rows)
              for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(to + c) = make_uint4(x, x, x, x);
          } else if (live) {
            *reinterpret_cast<float2*>((SHARED ? p.pre_ml : p.part_ml) + (slot + r) * 2) = make_float2(0.f, __int_as_float(0x7fffffff));
          }
        }
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    const int quarter = warp & 3, own = quarter * 32 + lane;
    const uint32_t tO = tmem_O + ((uint32_t)(quarter * 32) << 16), stage = sO + quarter * kOutStage;
    uint32_t ph = 0, q_loads = 0;                  // bit t: parity of stream t's items, of row tile t's loads
    auto load_rows = [&](const Item& it, int q, int tile) {
      clocked_wait(bar_qe + 8 * q, ((q_loads >> q) & 1) ^ 1);
      q_loads ^= 1u << q;
      load_q(it, q, tile, own);
    };
    Item it = next_item(true);
    if (it.n > 0)
      for (int t = 0; t < (PAIR ? 2 : 1); ++t)
        if (!PAIR || (t ? it.n1 : it.n0) > 0) load_rows(it, t, t);
    for (int il = 0; it.n > 0; ++il) {
      const Item nx = next_item(true);
      // the next item's rows before this one's sums: the products wait for those rows before they have issued the last of this item's
      if (nx.n > 0) {
        if (!PAIR) load_rows(nx, (il + 1) & 1, 0);
        else
          for (int t = 0; t < 2; ++t)
            if ((t ? nx.n1 : nx.n0) > 0) load_rows(nx, t, t);
      }
      const bool merge = !PAIR && it.n1 > 0, direct = !SHARED && p.shared == 0 && it.ends == 3;
      const long slot = part_slot<SHARED>(p, (long)it.e * p.Hkv + it.head, blockIdx.x, it.ends & 1) * tile_rows;
#pragma unroll 1
      for (int t = 0; t < (PAIR ? 2 : 1); ++t) {
        const int r0 = t * kRows + quarter * 32;   // the warp's rows of the item's
        const int row = first_row(it) + r0 + lane;
        int b, w;
        const bool live = row_token(it, row, b, w);
        const bool none = (t ? it.n1 : it.n0) == 0;
        float m = -INFINITY, l = 0.f, f0 = 1.f, f1 = 0.f;
        if (!none) {
          clocked_wait(bar_of + 8 * t, (ph >> t) & 1);
          clocked_wait(bar_lf + 8 * t, (ph >> t) & 1);
          ph ^= 1u << t;
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(m), "=f"(l) : "r"(sStat + t * 1024 + own * 8) : "memory");
          mbar_arrive(bar_le + 8 * t);
          if (merge) {
            clocked_wait(bar_of + 8, (ph >> 1) & 1);
            clocked_wait(bar_lf + 8, (ph >> 1) & 1);
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
        if (!none && !__any_sync(0xffffffffu, to >= 0)) {
          tcgen05_fence_before();
          mbar_arrive(bar_oe + 8 * t);
          if (merge) mbar_arrive(bar_oe + 8);
        } else if (!none) {
          // PAIR: the rows leave through the warp's stage, 128 bytes of each at a time
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
            if constexpr (!PAIR) {
              if (to >= 0 && direct) {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                  uint32_t o[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i) o[i] = pack16<T>(__uint_as_float(r[v * 8 + 2 * i]), __uint_as_float(r[v * 8 + 2 * i + 1]));
                  *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + to + c * COLS + v * 8) = make_uint4(o[0], o[1], o[2], o[3]);
                }
              } else if (to >= 0) {
                uint4* dst = reinterpret_cast<uint4*>((SHARED ? p.pre_o : p.part_o) + to + c * COLS);
#pragma unroll
                for (int v = 0; v < 8; ++v) dst[v] = make_uint4(r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
              }
              continue;
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
    if (!SHARED && p.shared == 0) finish_idle<T, D, 128>(p, threadIdx.x - 256);
    asm volatile("bar.arrive 2, 224;" ::: "memory");       // warp 15 waits for this
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    const int t = warp >= 4;                       // stream of this warpgroup
    const int quarter = warp & 3, own = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem_S + t * 128 + lane_base, tO = tmem_O + t * 128 + lane_base;
    const uint32_t my_s = bar_s + 8 * t, my_p = bar_p + 8 * t;
    constexpr int Q = KEYS / 32;
    const float sl2 = p.scale_log2;
    const uint64_t sl2_2 = pack2(sl2, sl2);
    int g = 0, items = 0, pos0 = 0, tile0 = 0;
    // A piece of one step in front of the first works on whatever there is and leaves nothing behind (its weights go over the sums, which the first
    // product does not add to): a step's 10 KB of instructions come from memory, a part by each warp, while the place is found and the first keys
    // come.  Without it the first step took 3 to 5 us.
    const int part_of_step = warp;
    bool dry = true;
    int shared_keys = 0;                           // SHARED: in place of the item's keys, which are loaded whether a row sees them or not
    Item it{};
    it.n0 = it.n1 = 1;
    while (true) {
      const int nt = t ? it.n1 : it.n0;
      if (nt > 0) {
        int b = 0, w = 0;
        const int row = first_row(it) + (PAIR ? t * kRows : 0) + own, n = SHARED ? shared_keys : it.keys;
        const bool live = !dry && row_token(it, row, b, w);
        // keys that this row sees (one that does not count: all, whatever comes of it), and the fewest of the warp's rows
        const int sees = live ? min(visible_keys(p, b, w), n) : 0x7fffffff;
        const int sees_lo = __reduce_min_sync(0xffffffffu, sees);
        const bool rows_here = dry || __any_sync(0xffffffffu, live);             // otherwise the warp lets the scores be what they are
        float m_ref = -INFINITY, l = 0.f;
        for (int j = 0; j < nt; ++j) {
          const int jt = PAIR ? j : 2 * j + t, key0 = key_at(it.j0 + jt), pos = pos0 + ring_at(t, j);
          if (!dry) wait(my_s, (uint32_t)(g++ & 1));
          tcgen05_fence_after();
          if (rows_here) {
            const uint32_t tP = dry ? tO : tS;
            uint32_t hole;                             // written before the keys' barrier, which the products waited for
            asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(hole) : "r"(holes + ((tile0 + jt) % kHoles) * 4) : "memory");
            const int lim = sees - 1 - key0;           // last column that this row sees
            if (sees_lo - key0 < KEYS || (hole != 0 && !dry)) {
              // what is not seen becomes -inf where the scores lie, sixteen columns at a time: seldom, and few instructions to have at hand
              const int from = hole ? 0 : max(0, sees_lo - key0) >> 4;
#pragma unroll 1
              for (int c = from; c < KEYS / 16; ++c) {
                uint32_t r[16];
                tcgen05_ld_32x16(tS + c * 16, r);
                tcgen05_wait_ld();
                const int end = hole >> (c * 16 / box) & 1 ? -1 : lim - c * 16;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  if (i > end) r[i] = 0xff800000u;
                tcgen05_st_32x16(tS + c * 16, r);
              }
              tcgen05_wait_st();
            }
            uint32_t sr[Q][32];
#pragma unroll
            for (int c = 0; c < Q; ++c) tcgen05_ld_32x32(tS + c * 32, sr[c]);
            tcgen05_wait_ld();
            float base = m_ref == -INFINITY ? 0.f : m_ref;       // a row that has seen nothing yet: its first quarter is done again below
            uint64_t shift = pack2(-base * sl2, -base * sl2), sum[Q] = {};
            float mx, unused;
            mx = -INFINITY;
            if (!dry || part_of_step == 0) exps<T, Q, true>(sr, 0, sl2_2, shift, sum[0], mx);
            const bool need = dry ? part_of_step == 4 : (mx - base) * sl2 > 8.f || (m_ref == -INFINITY && mx > -INFINITY);
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
              sum[0] = 0ull;
              exps<T, Q, false>(sr, 0, sl2_2, shift, sum[0], unused);
            }
            if (!(mx < INFINITY)) l = __int_as_float(0x7fffffff);        // NaN or +inf among the scores: a row of NaN
            tcgen05_st_32x16p(tP, sr[0]);
#pragma unroll
            for (int c = 1; c < Q; ++c) {
              if (dry && part_of_step != c) continue;
              exps<T, Q, false>(sr, c, sl2_2, shift, sum[c], unused);
              tcgen05_st_32x16p(tP + c * 16, sr[c]);
            }
            float part = 0.f;
#pragma unroll
            for (int c = 0; c < Q; ++c) { float x, y; unpack2(sum[c], x, y); part += x + y; }
            l += part;
          }
          if (!dry && key0 + KEYS > n) {
            // behind the last key: the rest of its page may hold anything, and 0 times NaN is NaN
            wait(bar_kvf + 8 * ((pos + 1) % SLOTS), (uint32_t)(((pos + 1) / SLOTS) & 1));
            if (own < KEYS && key0 + own >= n) {
              const uint32_t dst = sKV + (pos + 1) % SLOTS * TILE + own * 128;
#pragma unroll
              for (int c = 0; c < D / 8; ++c)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + (c >> 3) * C::HALF + (c & 7) * 16), "r"(0u) : "memory");
            }
            fence_async_smem();
          }
          tcgen05_wait_st();
          tcgen05_fence_before();
          if (!dry) mbar_arrive(my_p);
        }
        // ---- maximum (in units of the exponent) and row sum to the output warps
        if (!dry) {
          wait(bar_le + 8 * t, (uint32_t)((items & 1) ^ 1));
          ++items;
          asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(sStat + t * 1024 + own * 8), "f"(m_ref * sl2), "f"(l) : "memory");
          mbar_arrive(bar_lf + 8 * t);
        }
      }
      if (!dry) { pos0 += 2 * it.n; tile0 += it.n; }
      if (dry) {
        if (!late) pdl_wait();
        pdl_trigger();
        if constexpr (SHARED) shared_keys = seen_of_shared(p, lane);
      }
      dry = false;
      it = next_item();
      if (it.n == 0) break;
    }
  }
  if (late) pdl_wait();
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 13) tcgen05_dealloc(tmem_base, 512);
}

template <typename T, int D, bool PAIR, int ROWS, bool SHARED>
void launch_tiles(const PagedAttn& p, int grid, cudaStream_t st) {
  using C = Cut<D, PAIR, ROWS>;
  // boxes of the largest power of two that divides a page
  const int box = std::min(p.ps & -p.ps, C::KEYS);
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)p.ps, (uint64_t)p.Hkv, (uint64_t)p.pages};
  // (the stride of a dimension of one is anything)
  auto step = [&](long stride, long n) { return (uint64_t)(n == 1 ? D : stride); };
  const uint64_t ks[3] = {step(p.k_sr, p.ps), step(p.k_sh, p.Hkv), step(p.k_sp, p.pages)}, vs[3] = {step(p.v_sr, p.ps), step(p.v_sh, p.Hkv), step(p.v_sp, p.pages)};
  const CUtensorMap tk = make_tmap_bf16_heads(p.k, dims, ks, 64, box), tv = make_tmap_bf16_heads(p.v, dims, vs, 64, box);
  constexpr uint32_t smem = C::SMEM;
  NXD_ALLOW_SMEM((paged_tiles_kernel<T, D, PAIR, ROWS, SHARED>), smem);
  launch_dependent(paged_tiles_kernel<T, D, PAIR, ROWS, SHARED>, grid, kRowsThreads, smem, st, tk, tv, p, box);
}
template <typename T, int D, bool SHARED>
void launch_rows(const PagedAttn& p, int rows, int grid, cudaStream_t st) {
  if (rows == 64) launch_tiles<T, D, false, 64, SHARED>(p, grid, st);
  else if (rows == kRows) launch_tiles<T, D, false, kRows, SHARED>(p, grid, st);
  else launch_tiles<T, D, true, kRows, SHARED>(p, grid, st);
}

}  // namespace

void paged_tiles(const PagedAttn& p, int grid, bool over_shared, int D, int dt, cudaStream_t st) {
  const int rows = over_shared ? p.pre_tile_rows : p.tile_rows;
#define NXD_TILES(T, Dv) do { if (over_shared) launch_rows<T, Dv, true>(p, rows, grid, st); else launch_rows<T, Dv, false>(p, rows, grid, st); } while (0)
  if (dt == kBF16) { if (D == 128) NXD_TILES(__nv_bfloat16, 128); else NXD_TILES(__nv_bfloat16, 64); }
  else { if (D == 128) NXD_TILES(__half, 128); else NXD_TILES(__half, 64); }
#undef NXD_TILES
}

}  // namespace nxd
