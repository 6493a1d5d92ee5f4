// A key/value cache in pages (k and v [pages, page_size, Hkv, D], a table of pages per sequence): appending with the position rotation on
// the way, and attention of a few query rows over it.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"

namespace nxd {

namespace {

// ---------------------------------------------------------------------------------------------------------------- append
// x' = (a cos − b sin, b cos + a sin), a and b the halves of a head, angle by the token's position: q to q_out, k into its page, v as it is
// beside it.  Bound by HBM: every number is read and written once; a thread turns 16 bytes of each half.
template <typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(
    const T* q, const T* k, const T* v, const long* positions, const long* lens, const float* cos_t, const float* sin_t, T* q_out, T* kc, T* vc,
    const int* table, int B, int W, int H, int Hkv, int half, int rows, int cols, int ps, int pages, long table_sb, long q_sb, long q_sw, long q_sh,
    long k_sb, long k_sw, long k_sh, long v_sb, long v_sw, long v_sh, long o_sb, long o_sw, long kc_sp, long kc_sr, long kc_sh, long vc_sp, long vc_sr,
    long vc_sh, long items) {
  constexpr int N = Pack16<T>::N;
  pdl_trigger();
  pdl_wait();
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= items) return;
  const int per_head = half / N, heads = H + 2 * Hkv;
  const int c = (int)(i % per_head) * N;
  const long j = i / per_head;
  const int h = (int)(j % heads);
  const long t = j / heads;
  const int b = (int)(t % B), w = (int)(t / B);            // tokens of all sequences beside one another, as projections leave them
  const long first = positions[b];
  const long m = lens ? lens[b] : W, pos = first + w;
  const bool live = first >= 0 && w < m && pos < rows;
  Pack16<T> lo, hi;
  if (h < H) {
    T* dst = q_out + b * o_sb + w * o_sw + (long)h * (2 * half) + c;
    if (!live) {
#pragma unroll
      for (int e = 0; e < N; ++e) { lo.set(e, 0.f); hi.set(e, 0.f); }
      lo.store(dst);
      hi.store(dst + half);
      return;
    }
    const T* src = q + b * q_sb + w * q_sw + h * q_sh + c;
    lo.load(src);
    hi.load(src + half);
    const float *cs = cos_t + pos * half + c, *sn = sin_t + pos * half + c;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = lo.f(e), y = hi.f(e);
      lo.set(e, x * cs[e] - y * sn[e]);
      hi.set(e, y * cs[e] + x * sn[e]);
    }
    lo.store(dst);
    hi.store(dst + half);
    return;
  }
  if (!live || pos / ps >= cols) return;
  const int page = table[b * table_sb + pos / ps], row = (int)(pos % ps);
  if (page < 0 || page >= pages) return;
  if (h < H + Hkv) {
    const T* src = k + b * k_sb + w * k_sw + (h - H) * k_sh + c;
    T* dst = kc + page * kc_sp + row * kc_sr + (h - H) * kc_sh + c;
    lo.load(src);
    hi.load(src + half);
    const float *cs = cos_t + pos * half + c, *sn = sin_t + pos * half + c;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = lo.f(e), y = hi.f(e);
      lo.set(e, x * cs[e] - y * sn[e]);
      hi.set(e, y * cs[e] + x * sn[e]);
    }
    lo.store(dst);
    hi.store(dst + half);
  } else {
    const T* src = v + b * v_sb + w * v_sw + (h - H - Hkv) * v_sh + c;
    T* dst = vc + page * vc_sp + row * vc_sr + (h - H - Hkv) * vc_sh + c;
    lo.load(src);
    hi.load(src + half);
    lo.store(dst);
    hi.store(dst + half);
  }
}

// ------------------------------------------------------------------------------------------------------- attention, few rows
constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kKeys = 16;                                  // keys of a warp's tile
constexpr int kTileKeys = kWarps * kKeys;                  // keys of a block's tile
constexpr int kStages = 3;
constexpr int kMinTiles = 4;                               // a block's share of a launch is no less: 256 keys
template <int D> constexpr int kPitch = D + 4;             // of the rows in which warps leave their sums: no bank twice
template <int D> constexpr int rows_smem() { return kWarps * kStages * 2 * kKeys * D * 2 + kWarps * 8 * kPitch<D> * 4; }

NXD_DEVICE void cp_async16(uint32_t dst, const void* src, bool live) {    // not live: 16 zero bytes, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
NXD_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> NXD_DEVICE void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
NXD_DEVICE void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
NXD_DEVICE void ldmatrix_x4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
NXD_DEVICE uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <typename T> NXD_DEVICE void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> NXD_DEVICE void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> NXD_DEVICE void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// A pair is a (sequence, key/value head, block of query rows); its tiles are those of the sequence's keys behind the shared pages.  All tiles
// of a launch, pair after pair, are dealt out evenly: block c takes `per` of them from c * per on, wherever that lies.  Each block finds its
// place from the positions alone, so that nothing about lengths has to be known on the host.
NXD_DEVICE int own_tiles(const PagedAttn& p, int b) {
  const int n = paged_keys(p, b) - p.shared;
  return n > 0 ? (n + kTileKeys - 1) / kTileKeys : 0;
}

// Sum of a launch's tiles, and where `at` lies in them: sequence and tile within it (128 threads, all of them call).  b = B: behind the last.
struct Place { int b; long tile; };
NXD_DEVICE long find_place(const PagedAttn& p, int grid, long& per, int block, Place& out) {
  __shared__ long sums[kWarps];
  __shared__ long found[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (p.B + kThreads - 1) / kThreads, b0 = min(p.B, (int)threadIdx.x * each), b1 = min(p.B, b0 + each);
  long mine = 0;
  for (int b = b0; b < b1; ++b) mine += own_tiles(p, b);
  long scan = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long x = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += x;
  }
  if (lane == 31) sums[warp] = scan;
  if (threadIdx.x == 0) { found[0] = p.B; found[1] = 0; }
  __syncthreads();
  long before = scan - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  const long pairs = (long)p.Hkv * p.row_blocks;
  total *= pairs;
  per = max((long)kMinTiles, (total + grid - 1) / grid);
  long left = block * per - before * pairs;
  if (left >= 0 && left < mine * pairs) {
    for (int b = b0; b < b1; ++b) {
      const long t = own_tiles(p, b) * pairs;
      if (left < t) { found[0] = b; found[1] = left; break; }
      left -= t;
    }
  }
  __syncthreads();
  out.b = (int)found[0];
  out.tile = found[1];
  return total;
}

// Where a block reads next: keys of one pair
struct Cursor { int b, pair, tile, tiles, n; };

NXD_DEVICE void next_tile(const PagedAttn& p, Cursor& c) {
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.pair < p.Hkv * p.row_blocks) return;
  c.pair = 0;
  do {
    ++c.b;
    c.tiles = c.b < p.B ? own_tiles(p, c.b) : 1;
  } while (c.tiles == 0);
  c.n = c.b < p.B ? paged_keys(p, c.b) : 0;
}

// Sum over the shared pages' parts of one row, relative to their joint maximum: columns c0 .. c0 + C of the row
template <int D, int C>
NXD_DEVICE void add_shared(const PagedAttn& p, int b, int kvh, int row, int c0, float& m, float& l, float (&acc)[C]) {
  const long at = (long)kvh * p.pre_rows + (long)b * p.W * p.G + row, step = (long)p.Hkv * p.pre_rows;
  for (int s = 0; s < p.pre_splits; ++s) {
    const float2 ml = reinterpret_cast<const float2*>(p.pre_ml)[at + s * step];
    const float* o = p.pre_o + (at + s * step) * D + c0;
    const float mn = fmaxf(m, ml.x);
    const float f = m == -INFINITY ? 0.f : exp2f(m - mn), g = ml.x == -INFINITY ? 0.f : exp2f(ml.x - mn);
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = acc[i] * f + (g != 0.f ? o[i] * g : 0.f);
    l = l * f + ml.y * g;
    m = mn;
  }
}

// One block per share of the tiles; SHARED: one per (key/value head and block of rows of the whole batch, stretch of the shared pages).
// Bound by HBM: 4 D bytes per key and key/value head.  A warp walks 16-key tiles of its own through its own ring of cp.async stages, which runs
// ahead over the ends of pairs.  Scores Sᵀ = K Qᵀ and sums Oᵀ += Vᵀ Pᵀ by mma.sync with the keys, then the head's columns, as the 16 rows of the
// instruction and 8 R query rows as its columns, so that a group of up to 8 heads wastes nothing; the accumulator of Sᵀ becomes the operand Pᵀ by an
// 8 x 8 transposition in registers.  Probabilities are rounded to the cache's type for the second product: half a step of 2^-8 (2^-11) each, which average out over
// the keys; row sums are those of the unrounded ones.
template <typename T, int D, int R, bool SHARED>
__global__ void __launch_bounds__(kThreads, 2) paged_rows_kernel(const PagedAttn p) {
  constexpr int CH = D / 8, KS = D / 16, PITCH = kPitch<D>;
  constexpr int STAGE = 2 * kKeys * D * 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sm_m[kWarps][8 * R], sm_l[kWarps][8 * R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hq = lane >> 2, quad = lane & 3;
  pdl_trigger();                                           // the merge's blocks may take their places; they wait for this grid
  pdl_wait();
  const int tokens = SHARED ? p.B * p.W : p.W, rows = tokens * p.G, pairs = p.Hkv * p.row_blocks;
  Cursor cur;
  long left;                                               // tiles of this block
  if constexpr (SHARED) {
    const int tiles = (p.shared + kTileKeys - 1) / kTileKeys;
    const int per = (tiles + gridDim.y - 1) / gridDim.y, t0 = blockIdx.y * per;
    cur = Cursor{0, (int)blockIdx.x, t0, min(tiles, t0 + per), p.shared};
    left = cur.tiles - t0;
  } else {
    long per;
    Place at;
    const long total = find_place(p, gridDim.x, per, blockIdx.x, at);
    left = min(per, total - blockIdx.x * per);
    if (left <= 0) return;
    cur.b = at.b;
    cur.tiles = own_tiles(p, at.b);
    cur.pair = (int)(at.tile / cur.tiles);
    cur.tile = (int)(at.tile % cur.tiles);
    cur.n = paged_keys(p, at.b);
  }
  const T* const kc = reinterpret_cast<const T*>(p.k);
  const T* const vc = reinterpret_cast<const T*>(p.v);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (kStages * STAGE);
  float* const sm_o = reinterpret_cast<float*>(smem + kWarps * kStages * STAGE);       // [warp][8 rows][PITCH]

  // page of this warp's 16 keys at a cursor: -1 where there is none
  auto page_at = [&](const Cursor& c) {
    const int key = (SHARED ? 0 : p.shared) + c.tile * kTileKeys + warp * kKeys;
    if (key >= c.n) return -1;
    const int page = SHARED ? p.shared_pages[key / p.ps] : p.table[c.b * p.table_sb + key / p.ps];
    return (unsigned)page < (unsigned)p.pages ? page : -1;
  };
  // CH lanes copy one row, 16-byte chunk c of row r lands at chunk (c ^ (r & 7)): both ways of reading are conflict-free
  auto load_tile = [&](const Cursor& c, int page, int stage) {
    constexpr int PASS = 32 / CH;
    const int key = (SHARED ? 0 : p.shared) + c.tile * kTileKeys + warp * kKeys, kvh = c.pair / p.row_blocks;
    const int row0 = key % p.ps, cc = lane % CH;
    const long at = page < 0 ? 0 : page;
    const T* kb = kc + at * p.k_sp + kvh * p.k_sh + cc * 8;
    const T* vb = vc + at * p.v_sp + kvh * p.v_sh + cc * 8;
    const uint32_t dst = ring + stage * STAGE;
#pragma unroll
    for (int i = 0; i < kKeys / PASS; ++i) {
      const int r = i * PASS + lane / CH;
      const bool live = page >= 0 && key + r < c.n;
      const uint32_t off = r * (D * 2) + ((cc ^ (r & 7)) << 4);
      cp_async16(dst + off, kb + (row0 + r) * p.k_sr, live);
      cp_async16(dst + kKeys * D * 2 + off, vb + (row0 + r) * p.v_sr, live);
    }
  };

  Cursor ahead = cur;
  long asked = 0;
  int page = left > 0 ? page_at(ahead) : -1;
  // pages of tiles that have been asked for, stage by stage: the products skip holes
  uint32_t holes = 0;                                      // bit s: the tile in stage s is a hole
  auto ask = [&](int stage) {
    if (asked < left) {
      load_tile(ahead, page, stage);
      holes = (holes & ~(1u << stage)) | (page < 0 ? 1u << stage : 0u);
      if (++asked < left) {
        if constexpr (SHARED) ++ahead.tile; else next_tile(p, ahead);
        page = page_at(ahead);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) ask(s);

  uint32_t qf[R][KS][2];
  float m[R][2], l[R][2], o[R][KS][4];
  int lim[R][2], lim_all = 0;                              // first key that a row does not see; that none of the live rows has before it
  bool whole = false;                                      // the pair begins in this block
  auto row_token = [&](int row, int& b, int& w) {          // of the pair's row
    const int t = row / p.G;
    b = SHARED ? t / p.W : cur.b;
    w = SHARED ? t % p.W : t;
  };
  auto begin = [&]() {
    const int kvh = cur.pair / p.row_blocks, r0 = (cur.pair % p.row_blocks) * 8 * R;
    whole = SHARED || cur.tile == 0;
    lim_all = SHARED ? 0 : (int)min(p.positions[cur.b] + r0 / p.G + 1, (long)cur.n);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      int b, w;
      const int row = r0 + i * 8 + hq;
      row_token(row, b, w);
      const bool live = row < rows && w < paged_new_tokens(p, b);
      const T* qp = reinterpret_cast<const T*>(p.q) + (live ? b * p.q_sb + w * p.q_sw + (long)(kvh * p.G + row % p.G) * p.q_sh : 0) + quad * 2;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qf[i][k][0] = live ? *reinterpret_cast<const uint32_t*>(qp + k * 16) : 0u;
        qf[i][k][1] = live ? *reinterpret_cast<const uint32_t*>(qp + k * 16 + 8) : 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][k][e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = r0 + i * 8 + quad * 2 + e;
        row_token(r, b, w);
        const bool on = r < rows && w < paged_new_tokens(p, b);
        lim[i][e] = on ? (int)min(p.positions[b] + w + 1, (long)cur.n) : 0;
        m[i][e] = -INFINITY;
        l[i][e] = 0.f;
      }
    }
  };

  // the four warps' sums of the pair, to the output or to a part
  auto finish = [&](bool last) {
    const int kvh = cur.pair / p.row_blocks, r0 = (cur.pair % p.row_blocks) * 8 * R;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], s);
    if (hq == 0)
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) { sm_m[warp][i * 8 + quad * 2 + e] = m[i][e]; sm_l[warp][i * 8 + quad * 2 + e] = l[i][e]; }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i) __syncthreads();
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) sm_o[(warp * 8 + quad * 2 + (e & 1)) * PITCH + k * 16 + hq + (e >> 1) * 8] = o[i][k][e];
      __syncthreads();
      constexpr int PER = kThreads / D;                    // rows at a time
#pragma unroll
      for (int x = 0; x < 8 / PER; ++x) {
        const int rr = x * PER + (int)threadIdx.x / D, col = threadIdx.x % D, row = r0 + i * 8 + rr, rs = i * 8 + rr;
        if (row >= rows) break;
        float mn = fmaxf(fmaxf(sm_m[0][rs], sm_m[1][rs]), fmaxf(sm_m[2][rs], sm_m[3][rs])), ls = 0.f, acc[1] = {0.f};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float c = mn == -INFINITY ? 0.f : exp2f(sm_m[w][rs] - mn);
          acc[0] += sm_o[(w * 8 + rr) * PITCH + col] * c;
          ls += sm_l[w][rs] * c;
        }
        if constexpr (SHARED) {
          const long at = ((long)blockIdx.y * p.Hkv + kvh) * p.pre_rows + row;
          p.pre_o[at * D + col] = acc[0];
          if (col == 0) { p.pre_ml[at * 2] = mn; p.pre_ml[at * 2 + 1] = ls; }
        } else if (whole && last) {
          if (p.pre_splits) add_shared<D>(p, cur.b, kvh, row, col, mn, ls, acc);
          int b, w;
          row_token(row, b, w);
          const bool live = w < paged_new_tokens(p, b) && !(ls == 0.f);
          reinterpret_cast<T*>(p.out)[b * p.o_sb + w * p.o_sw + (long)(kvh * p.G + row % p.G) * p.o_sh + col] = from_f32<T>(live ? acc[0] / ls : 0.f);
        } else {
          const long at = (long)(blockIdx.x * 2 + (whole ? 1 : 0)) * (8 * R) + rs;
          p.part_o[at * D + col] = acc[0];
          if (col == 0) { p.part_ml[at * 2] = mn; p.part_ml[at * 2 + 1] = ls; }
        }
      }
    }
    __syncthreads();                                       // the sums have been read
  };

  if (left > 0) begin();
  else if constexpr (SHARED) { cur.n = 0; begin(); finish(true); return; }    // a stretch behind the shared keys
  for (long t = 0; t < left; ++t) {
    const int stage = (int)(t % kStages);
    cp_async_wait<kStages - 2>();
    __syncwarp();                                          // tile t of all lanes is there; all lanes are done with tile t - 1
    const bool hole = holes >> stage & 1;
    ask((int)((t + kStages - 1) % kStages));
    const int key = (SHARED ? 0 : p.shared) + cur.tile * kTileKeys + warp * kKeys;
    if (!hole) {
      const uint32_t ks = ring + stage * STAGE, vs = ks + kKeys * D * 2;
      float s[R][4];
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        // matrices: keys 0-7 / columns 16 k.., keys 8-15 / 16 k.., keys 0-7 / 16 k + 8.., keys 8-15 / 16 k + 8..
        const int r = (((lane >> 3) & 1) << 3) + (lane & 7), c = k * 2 + (lane >> 4);
        uint32_t a[4];
        ldmatrix_x4(a, ks + r * (D * 2) + ((c ^ (r & 7)) << 4));
#pragma unroll
        for (int i = 0; i < R; ++i) mma16816<T>(s[i], a, qf[i][k][0], qf[i][k][1]);
      }
      const bool masked = key + kKeys > lim_all;
      uint32_t pf[R][2];
#pragma unroll
      for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {                      // key hq + 8 (e / 2), row 2 quad + e % 2
          s[i][e] *= p.scale_log2;
          if (masked && key + hq + (e >> 1) * 8 >= lim[i][e & 1]) s[i][e] = -INFINITY;
        }
        float mx[2], f[2];
        bool grew = false;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(s[i][e], s[i][e + 2]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
          grew = grew || mx[e] > m[i][e];
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mn = fmaxf(m[i][e], mx[e]);
            f[e] = mx[e] > m[i][e] ? exp2f(m[i][e] - mn) : 1.f;       // m = -inf: 0
            m[i][e] = mn;
            l[i][e] *= f[e];
          }
#pragma unroll
          for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][k][e] *= f[e & 1];
        }
        float pr[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pr[e] = exp2f(s[i][e] - (m[i][e & 1] == -INFINITY ? 0.f : m[i][e & 1]));
          l[i][e & 1] += pr[e];
        }
        pf[i][0] = transpose8x8(pack16<T>(pr[0], pr[1]));
        pf[i][1] = transpose8x8(pack16<T>(pr[2], pr[3]));
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        // matrices of V, transposed: columns 16 k.. / keys 0-7, 16 k + 8.. / keys 0-7, 16 k.. / keys 8-15, 16 k + 8.. / keys 8-15
        const int r = ((lane >> 4) << 3) + (lane & 7), c = k * 2 + ((lane >> 3) & 1);
        uint32_t a[4];
        ldmatrix_x4t(a, vs + r * (D * 2) + ((c ^ (r & 7)) << 4));
#pragma unroll
        for (int i = 0; i < R; ++i) mma16816<T>(o[i][k], a, pf[i][0], pf[i][1]);
      }
    }
    const bool end = cur.tile + 1 == cur.tiles;
    if (end || t + 1 == left) {
      finish(end);
      if (t + 1 < left) {
        next_tile(p, cur);
        begin();
      }
    } else {
      ++cur.tile;
    }
  }
}

// Rows whose pair several blocks walked, or that see no key of their own: a warp joins the parts of one row.
template <typename T, int D, int R>
__global__ void __launch_bounds__(kThreads) paged_merge_kernel(const PagedAttn p, int grid) {
  constexpr int C = D / 32;
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / (p.Hkv * p.row_blocks), pair = blockIdx.x % (p.Hkv * p.row_blocks);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // tiles of the sequences before this one, and of all
  __shared__ long sums[2][kWarps];
  long before = 0, total = 0;
  for (int i = threadIdx.x; i < p.B; i += kThreads) {
    const int t = own_tiles(p, i);
    total += t;
    if (i < b) before += t;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (lane == 0) { sums[0][warp] = before; sums[1][warp] = total; }
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) { before += sums[0][w]; total += sums[1][w]; }
  const long pairs = (long)p.Hkv * p.row_blocks;
  const long per = max((long)kMinTiles, (total * pairs + grid - 1) / grid);
  const int tiles = own_tiles(p, b);
  const long t0 = before * pairs + (long)pair * tiles;
  const int c0 = (int)(t0 / per), c1 = tiles ? (int)((t0 + tiles - 1) / per) : c0;
  if (tiles && c0 == c1) return;                           // one block had the whole pair
  const int rs = blockIdx.y * kWarps + warp, row = (pair % p.row_blocks) * 8 * R + rs, kvh = pair / p.row_blocks;
  if (row >= p.W * p.G) return;
  const int w = row / p.G, c = lane * C;
  float m = -INFINITY, l = 0.f, acc[C];
#pragma unroll
  for (int i = 0; i < C; ++i) acc[i] = 0.f;
  if (tiles) {
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
    auto slot = [&](int x) { return (long)(2 * (c0 + x) + (x == 0)) * (8 * R) + rs; };
    const int n = c1 - c0 + 1;
    for (int x = lane; x < n; x += 32) m = fmaxf(m, ml[slot(x)].x);
    m = warp_max(m);
    for (int x0 = 0; x0 < n; x0 += 32) {
      const float2 a = x0 + lane < n ? ml[slot(x0 + lane)] : make_float2(-INFINITY, 0.f);
      const float f = a.x == -INFINITY ? 0.f : exp2f(a.x - m);
      l += warp_sum(a.y * f);
      const int here = min(32, n - x0);
#pragma unroll 8
      for (int x = 0; x < here; ++x) {
        const float g = __shfl_sync(0xffffffffu, f, x);
        const float* src = p.part_o + slot(x0 + x) * D + c;
        float v[C];
        if constexpr (C == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
        else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
#pragma unroll
        for (int i = 0; i < C; ++i) acc[i] += v[i] * g;
      }
    }
  }
  const bool live = w < paged_new_tokens(p, b);
  if (live && p.pre_splits) add_shared<D>(p, b, kvh, row, c, m, l, acc);
  T* dst = reinterpret_cast<T*>(p.out) + b * p.o_sb + w * p.o_sw + (long)(kvh * p.G + row % p.G) * p.o_sh + c;
#pragma unroll
  for (int i = 0; i < C; ++i) dst[i] = from_f32<T>(live && !(l == 0.f) ? acc[i] / l : 0.f);
}

template <typename T, int D, int R>
void launch_rows(const PagedAttn& p, int grid, cudaStream_t st) {
  if (p.pre_splits) {
    PagedAttn s = p;
    s.row_blocks = (p.B * p.W * p.G + 8 * R - 1) / (8 * R);
    NXD_ALLOW_SMEM((paged_rows_kernel<T, D, R, true>), rows_smem<D>());
    launch_dependent(paged_rows_kernel<T, D, R, true>, dim3(p.Hkv * s.row_blocks, p.pre_splits), kThreads, rows_smem<D>(), st, s);
  }
  NXD_ALLOW_SMEM((paged_rows_kernel<T, D, R, false>), rows_smem<D>());
  launch_dependent(paged_rows_kernel<T, D, R, false>, grid, kThreads, rows_smem<D>(), st, p);
  launch_dependent(paged_merge_kernel<T, D, R>, dim3(p.B * p.Hkv * p.row_blocks, 2 * R), kThreads, 0, st, p, grid);
}

}  // namespace

int device_sm_count();

// Blocks of the few-row kernel, rows of a block, stretches of the shared pages
PagedPlan paged_plan(int B, int W, int G, int Hkv, int shared) {
  PagedPlan plan;
  plan.row_tiles = W * G > 8 ? 2 : 1;
  plan.grid = 2 * device_sm_count();
  plan.pre_rows = (int)(((long)B * W * G + 15) / 16 * 16);
  plan.pre_splits = 0;
  if (shared > 0) {
    const long pairs = (long)Hkv * (((long)B * W * G + 8 * plan.row_tiles - 1) / (8 * plan.row_tiles));
    plan.pre_splits = (int)std::max(1l, std::min({(2l * plan.grid + pairs - 1) / pairs, (shared + 255l) / 256, 64l}));
  }
  return plan;
}

void paged_attention(PagedAttn p, const PagedPlan& plan, int D, int dt, cudaStream_t st) {
  p.row_blocks = (p.W * p.G + 8 * plan.row_tiles - 1) / (8 * plan.row_tiles);
  p.pre_splits = plan.pre_splits;
  p.pre_rows = plan.pre_rows;
#define NXD_PAGED(T, Dv) do { if (plan.row_tiles == 1) launch_rows<T, Dv, 1>(p, plan.grid, st); else launch_rows<T, Dv, 2>(p, plan.grid, st); } while (0)
  if (dt == kBF16) { if (D == 128) NXD_PAGED(__nv_bfloat16, 128); else NXD_PAGED(__nv_bfloat16, 64); }
  else { if (D == 128) NXD_PAGED(__half, 128); else NXD_PAGED(__half, 64); }
#undef NXD_PAGED
}

void paged_append(const void* q, const void* k, const void* v, const long* positions, const long* lens, const float* cos_t, const float* sin_t,
                  void* q_out, void* kc, void* vc, const int* table, int B, int W, int H, int Hkv, int D, int rows, int cols, int ps, int pages,
                  long table_sb, const long (*s)[3], long o_sb, long o_sw, const long (*cs)[3], int dt, cudaStream_t st) {
  const int half = D / 2;
  const long items = (long)B * W * (H + 2 * Hkv) * (half / (dt == kF32 ? 4 : 8));
  if (items == 0) return;
#define NXD_APPEND(T)                                                                                                                              \
  launch_dependent(paged_append_kernel<T>, (unsigned)((items + 255) / 256), 256, 0, st, (const T*)q, (const T*)k, (const T*)v, positions, lens,      \
                   cos_t, sin_t, (T*)q_out, (T*)kc, (T*)vc, table, B, W, H, Hkv, half, rows, cols, ps, pages, table_sb, s[0][0], s[0][1], s[0][2],   \
                   s[1][0], s[1][1], s[1][2], s[2][0], s[2][1], s[2][2], o_sb, o_sw, cs[0][0], cs[0][1], cs[0][2], cs[1][0], cs[1][1], cs[1][2], items)
  if (dt == kBF16) NXD_APPEND(__nv_bfloat16);
  else if (dt == kF16) NXD_APPEND(__half);
  else NXD_APPEND(float);
#undef NXD_APPEND
}

}  // namespace nxd
