// A key/value cache in pages (k and v [pages, page_size, Hkv, D], a table of pages per sequence): appending with the position rotation on
// the way, and attention of a few query rows over it.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace nxd {

int device_sm_count();

namespace {

// ---------------------------------------------------------------------------------------------------------------- append
// x' = (a cos − b sin, b cos + a sin), a and b the halves of a head, angle by the token's position: q to q_out, k into its page, v as it is
// beside it.  Bound by HBM: every number is read and written once.  A thread has 16 bytes of each half of one head, a block as many as it can of one
// token, whose position, page, cosines and sines its threads share in L1.  4 x 2000 tokens, 64 heads on 8: 49 us, 5.0 TB/s (threads that go through
// heads with their cosines and sines in registers: 99, too few of them at a time); one token 2.6.
struct AppendArgs {
  const void *q, *k, *v;
  const long *positions, *lens;
  const float *cos_t, *sin_t;
  void *q_out, *kc, *vc;
  const int* table;
  int* lost;                                               // becomes 1 where a token that counts has no place; null: nobody asks
  int B, W, H, Hkv, half, rows, cols, ps, pages, parts;    // parts: blocks of a token
  long table_sb, q_sb, q_sw, q_sh, k_sb, k_sw, k_sh, v_sb, v_sw, v_sh, o_sb, o_sw, kc_sp, kc_sr, kc_sh, vc_sp, vc_sr, vc_sh;
};
constexpr int kAppendThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs p) {
  constexpr int N = Pack16<T>::N;
  pdl_trigger();
  const unsigned t = blockIdx.x / p.parts, item = blockIdx.x % p.parts * kAppendThreads + threadIdx.x, chunks = p.half / N;
  const int h = (int)(item / chunks), c = (int)(item % chunks) * N;
  const int w = (int)(t / p.B), b = (int)(t % p.B);        // tokens of all sequences beside one another, as projections leave them
  pdl_wait();
  if (h >= p.H + 2 * p.Hkv) return;
  const long first = p.positions[b], m = p.lens ? p.lens[b] : p.W, pos = first + w;
  const bool live = first >= 0 && first < p.rows && w < m && pos < p.rows, query = h < p.H, key = h < p.H + p.Hkv;
  T* const q_out = (T*)p.q_out + b * p.o_sb + w * p.o_sw + (long)h * (2 * p.half) + c;
  Pack16<T> lo, hi;
  if (!live) {
    if (p.lost && item == 0 && first >= 0 && w < m) *p.lost = 1;       // behind the rotation tables
    if (query) {
#pragma unroll
      for (int e = 0; e < N; ++e) { lo.set(e, 0.f); hi.set(e, 0.f); }
      lo.store(q_out);
      hi.store(q_out + p.half);
    }
    return;
  }
  const T* const src = (query ? (const T*)p.q + b * p.q_sb + w * p.q_sw + h * p.q_sh
                        : key ? (const T*)p.k + b * p.k_sb + w * p.k_sw + (h - p.H) * p.k_sh
                              : (const T*)p.v + b * p.v_sb + w * p.v_sw + (h - p.H - p.Hkv) * p.v_sh) + c;
  lo.load(src);
  hi.load(src + p.half);
  T* dst = q_out;
  if (!query) {
    const int column = (int)pos / p.ps, row = (int)pos - column * p.ps;            // positions with a place in the tables fit
    const int page = column < p.cols ? p.table[b * p.table_sb + column] : -1;
    if (page < 0 || page >= p.pages) {
      if (p.lost) *p.lost = 1;
      return;
    }
    dst = key ? (T*)p.kc + page * p.kc_sp + row * p.kc_sr + (h - p.H) * p.kc_sh + c
              : (T*)p.vc + page * p.vc_sp + row * p.vc_sr + (h - p.H - p.Hkv) * p.vc_sh + c;
  }
  if (key) {
    const float *cs = p.cos_t + pos * p.half + c, *sn = p.sin_t + pos * p.half + c;
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const float4 co = *reinterpret_cast<const float4*>(cs + e), si = *reinterpret_cast<const float4*>(sn + e);
      const float cf[4] = {co.x, co.y, co.z, co.w}, sf[4] = {si.x, si.y, si.z, si.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = lo.f(e + i), y = hi.f(e + i);
        lo.set(e + i, x * cf[i] - y * sf[i]);
        hi.set(e + i, y * cf[i] + x * sf[i]);
      }
    }
  }
  lo.store(dst);
  hi.store(dst + p.half);
}

// ------------------------------------------------------------------------------------------------------- attention, few rows
using namespace paged;

constexpr int kKeys = 16;                                  // keys of a warp's tile
constexpr int kTileKeys = kWarps * kKeys;                  // keys of a block's tile
constexpr float kNone = -1e30f;                            // the maximum of a row that has seen no key: below every score, and finite
constexpr int kCluster8 = 8;                               // blocks of a cluster at most
template <int D> constexpr int kPitch = D + 4;             // of the rows in which warps leave their sums: no bank twice
template <int D> constexpr int kSums = kWarps * 8 * kPitch<D> * 4;          // bytes of them
// two blocks an SM, three stages of 8 KB a warp: three blocks with two took 28.7 us for 26.7 (64 sequences of 300 to 600 keys, 8 heads), 74 for 66 (16 to 8192)
constexpr int kStages = 3;
template <int D> constexpr int rows_smem(bool cluster) { return kWarps * kStages * 2 * kKeys * D * 2 + (cluster ? 0 : kSums<D>); }

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
NXD_DEVICE float remote(const float* at, int rank) {       // the same place in another block's shared memory
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(at), rank)) : "memory");
  return v;
}

// How a block gets its work (paged.cuh): dealt out; one pair for the blocks of a cluster, which take its tiles in turn and join their sums in shared
// memory; dealt out over the shared pages, with the rows of the whole batch (8 R at most), all of whose results are parts
enum Deal { kDealt, kCluster, kShared };

// Bound by HBM: 4 D bytes per key and key/value head.  A warp walks 16-key tiles of its own through its own ring of cp.async stages, which runs
// ahead over the ends of pairs.  Scores Sᵀ = K Qᵀ and sums Oᵀ += Vᵀ Pᵀ by mma.sync with the keys, then the head's columns, as the 16 rows of the
// instruction and 8 R query rows as its columns, so that a group of up to 8 heads wastes nothing; the accumulator of Sᵀ becomes the operand Pᵀ by an
// 8 x 8 transposition in registers.  The second product takes probabilities as two numbers of the cache's type, the rounded one and what that left, 2^-16
// (2^-22) of them at most: memory is what bounds this kernel, and a product more costs nothing where it does (us, one / two: one token of 16 sequences
// to 8192 keys, 32 heads on 8, 72 / 73, the call; of 6 to 2500, 40 single heads, 43 / 43; 16 rows to 1000 keys, 32 pairs of 4, 31 / 31; one sequence to
// 4000 keys, 16 rows of 8 heads, 20.5 / 21.3).  The first of these alone: 66 us, 6.0 TB/s; the second 40; one sequence to 300: 6.7.
template <typename T, int D, int R, Deal DEAL>
__global__ void __launch_bounds__(kThreads, 2) paged_rows_kernel(const PagedAttn p) {
  constexpr bool SHARED = DEAL == kShared;
  constexpr int CH = D / 8, KS = D / 16, PITCH = kPitch<D>;
  constexpr int STAGE = 2 * kKeys * D * 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sm_m[kWarps][8 * R], sm_l[kWarps][8 * R], sm_bm[8 * R], sm_bl[8 * R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hq = lane >> 2, quad = lane & 3;
  const int rows = SHARED ? p.B * p.W * p.G : p.W * p.G;
  const bool late = !SHARED && p.shared > 0;               // the launch over the shared pages is in front (paged.cuh)
  if (!late) pdl_wait();
  int shared_keys = 0;
  auto keys_of = [&](int e) { return SHARED ? shared_keys : e < p.B ? all_keys(p, e) : 0; };
  pdl_trigger();                                           // the last launch's blocks may take their places; they wait for this grid
  // Pages of this warp's keys in 32 tiles of a pair from tile t0 on, one a lane: -1 where there is none
  const int step = DEAL == kCluster ? p.cluster : 1;
  auto fetch_pages = [&](int e, int t0) {
    const unsigned i = ((SHARED ? 0u : (unsigned)p.shared) + (unsigned)(t0 + lane * step) * kTileKeys + warp * kKeys) / (unsigned)p.ps;
    if (i >= (unsigned)(SHARED ? p.shared_cols : p.cols)) return -1;
    const int page = i < (unsigned)p.shared_cols ? p.shared_pages[i] : p.table[e * p.table_sb + i];
    return (unsigned)page < (unsigned)p.pages ? page : -1;
  };
  struct { Walk w; int n; } cur;
  long left;                                               // tiles of this block
  int pages = -1, next_page = 0;
  if constexpr (DEAL == kCluster) {
    const int pair = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster;
    pages = fetch_pages(pair / p.Hkv, rank);               // beside the positions: it needs none of them
    cur.w = Walk{pair / p.Hkv, pair % p.Hkv, rank, entry_tiles(p, pair / p.Hkv)};
    cur.n = keys_of(cur.w.e);
    left = cur.w.tiles > rank ? (cur.w.tiles - rank + step - 1) / step : 0;
  } else {
    const Place at = find_place<kThreads, SHARED>(p, gridDim.x, blockIdx.x);
    left = min(at.per, at.total - blockIdx.x * at.per);
    if (left > 0) {
      cur.w.e = at.e;
      cur.w.tiles = walk_tiles<SHARED>(p, at.e);
      cur.w.head = (int)(at.tile / cur.w.tiles);
      cur.w.tile = (int)(at.tile % cur.w.tiles);
      pages = fetch_pages(at.e, cur.w.tile);
      if constexpr (SHARED) shared_keys = seen_of_shared(p, lane);       // beside the pages
      cur.n = keys_of(at.e);
    }
  }
  const T* const kc = reinterpret_cast<const T*>(p.k);
  const T* const vc = reinterpret_cast<const T*>(p.v);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (kStages * STAGE);
  // sums of the warps [warp][8 rows][PITCH] and of a cluster's block [8 R][D]: a cluster's lie over the ring, which has been read by then
  float* const sm_o = reinterpret_cast<float*>(smem + (DEAL == kCluster ? 0 : kWarps * kStages * STAGE));
  float* const sm_b = reinterpret_cast<float*>(smem + kSums<D>);

  // CH lanes copy one row, 16-byte chunk c of row r lands at chunk (c ^ (r & 7)): both ways of reading are conflict-free
  auto load_tile = [&](const Walk& c, int n, int page, int stage) {
    constexpr int PASS = 32 / CH;
    const int key = (SHARED ? 0 : p.shared) + c.tile * kTileKeys + warp * kKeys;
    const int row0 = key % p.ps, cc = lane % CH;
    const long at = page < 0 ? 0 : page;
    const T* kb = kc + at * p.k_sp + c.head * p.k_sh + cc * 8;
    const T* vb = vc + at * p.v_sp + c.head * p.v_sh + cc * 8;
    const uint32_t dst = ring + stage * STAGE;
#pragma unroll
    for (int i = 0; i < kKeys / PASS; ++i) {
      const int r = i * PASS + lane / CH;
      const bool live = page >= 0 && key + r < n;
      const uint32_t off = r * (D * 2) + ((cc ^ (r & 7)) << 4);
      cp_async16(dst + off, kb + (row0 + r) * p.k_sr, live);
      cp_async16(dst + kKeys * D * 2 + off, vb + (row0 + r) * p.v_sr, live);
    }
  };

  auto ahead = cur;
  long asked = 0;
  uint32_t holes = 0;                                      // bit s: none of the warp's keys in stage s is there
  auto ask = [&](int stage) {
    if (asked < left) {
      if (next_page == 32) { pages = fetch_pages(ahead.w.e, ahead.w.tile); next_page = 0; }
      const int page = __shfl_sync(0xffffffffu, pages, next_page++);
      load_tile(ahead.w, ahead.n, page, stage);
      holes = (holes & ~(1u << stage)) | (page < 0 ? 1u << stage : 0u);
      if (++asked < left) {
        ahead.w.tile += step;
        if (DEAL != kCluster && ahead.w.tile == ahead.w.tiles) {
          next_pair<SHARED>(p, ahead.w);
          if (ahead.w.head == 0) ahead.n = keys_of(ahead.w.e);
          next_page = 32;
        }
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
    b = SHARED ? t / p.W : cur.w.e;
    w = SHARED ? t % p.W : t;
  };
  auto begin = [&]() {
    const int kvh = cur.w.head;
    whole = DEAL == kCluster || cur.w.tile == 0;
    lim_all = SHARED ? 0 : min(visible_keys(p, cur.w.e, 0), cur.n);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      int b, w;
      const int row = i * 8 + hq;
      row_token(row, b, w);
      const bool live = row < rows && w < new_tokens(p, b);
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
        const int r = i * 8 + quad * 2 + e;
        row_token(r, b, w);
        lim[i][e] = r < rows && w < new_tokens(p, b) ? min(visible_keys(p, b, w), cur.n) : 0;
        m[i][e] = kNone;
        l[i][e] = 0.f;
      }
    }
  };

  // the four warps' sums of the pair, to the output or to a part
  auto finish = [&](bool last) {
    const int kvh = cur.w.head;
    const bool direct = !SHARED && p.shared == 0 && whole && last;
    if (DEAL == kCluster) __syncthreads();
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
        for (int e = 0; e < 2; ++e) { sm_m[warp][i * 8 + quad * 2 + e] = m[i][e] == kNone ? -INFINITY : m[i][e]; sm_l[warp][i * 8 + quad * 2 + e] = l[i][e]; }
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
        const int rr = x * PER + (int)threadIdx.x / D, col = threadIdx.x % D, row = i * 8 + rr;
        if (row >= rows) break;
        float mn = fmaxf(fmaxf(sm_m[0][row], sm_m[1][row]), fmaxf(sm_m[2][row], sm_m[3][row])), ls = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float c = mn == -INFINITY ? 0.f : exp2f(sm_m[w][row] - mn);
          acc += sm_o[(w * 8 + rr) * PITCH + col] * c;
          ls += sm_l[w][row] * c;
        }
        if (DEAL == kCluster && p.cluster > 1) {
          sm_b[row * D + col] = acc;
          if (col == 0) { sm_bm[row] = mn; sm_bl[row] = ls; }
        } else if (direct) {
          int b, w;
          row_token(row, b, w);
          const bool live = w < new_tokens(p, b) && !(ls == 0.f);
          reinterpret_cast<T*>(p.out)[b * p.o_sb + w * p.o_sw + (long)(kvh * p.G + row % p.G) * p.o_sh + col] = from_f32<T>(live ? acc / ls : 0.f);
        } else {
          const long slot = part_slot<SHARED>(p, (long)cur.w.e * p.Hkv + kvh, blockIdx.x, whole) * (8 * R) + row;
          (SHARED ? p.pre_o : p.part_o)[slot * D + col] = acc;
          if (col == 0) *reinterpret_cast<float2*>((SHARED ? p.pre_ml : p.part_ml) + slot * 2) = make_float2(mn, ls);
        }
      }
    }
    __syncthreads();                                       // the sums have been read
  };

  if (DEAL == kCluster || left > 0) begin();
  for (long t = 0; t < left; ++t) {
    const int stage = (int)(t % kStages);
    cp_async_wait<kStages - 2>();
    __syncwarp();                                          // tile t of all lanes is there; all lanes are done with tile t - 1
    const bool hole = holes >> stage & 1;
    ask((int)((t + kStages - 1) % kStages));
    const int key = (SHARED ? 0 : p.shared) + cur.w.tile * kTileKeys + warp * kKeys;
    if (!hole) {
      const uint32_t ks = ring + stage * STAGE, vs = ks + kKeys * D * 2;
      float s[R][4], s1[R][4];                             // two chains of products: a warp waits for one most of its time
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = s1[i][e] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        // matrices: keys 0-7 / columns 16 k.., keys 8-15 / 16 k.., keys 0-7 / 16 k + 8.., keys 8-15 / 16 k + 8..
        const int r = (((lane >> 3) & 1) << 3) + (lane & 7), c = k * 2 + (lane >> 4);
        uint32_t a[4];
        ldmatrix_x4(a, ks + r * (D * 2) + ((c ^ (r & 7)) << 4));
#pragma unroll
        for (int i = 0; i < R; ++i) mma16816<T>(k & 1 ? s1[i] : s[i], a, qf[i][k][0], qf[i][k][1]);
      }
      const bool masked = key + kKeys > lim_all;
      uint32_t pf[R][2], pl[R][2];                         // weights to the type, and what that left of them
#pragma unroll
      for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] += s1[i][e];
#pragma unroll
        for (int e = 0; e < 4; ++e)                        // key hq + 8 (e / 2), row 2 quad + e % 2
          if (masked && key + hq + (e >> 1) * 8 >= lim[i][e & 1]) s[i][e] = -INFINITY;
        // Weights relative to a maximum that is at most 2^8 behind: it is looked for among the eight lanes of a row when one of them finds it passed
        float x[4];
        bool passed = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = fmaf(s[i][e], p.scale_log2, -m[i][e & 1]);
          passed = passed || x[e] > 8.f;
        }
        if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(s[i][e], s[i][e + 2]) * p.scale_log2;
#pragma unroll
            for (int y = 4; y < 32; y <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, y));
            const float mn = fmaxf(m[i][e], mx), f = exp2f(m[i][e] - mn);      // none before: 0
            m[i][e] = mn;
            l[i][e] *= f;
#pragma unroll
            for (int k = 0; k < KS; ++k) { o[i][k][e] *= f; o[i][k][e + 2] *= f; }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = fmaf(s[i][e], p.scale_log2, -m[i][e & 1]);
        }
        float pr[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pr[e] = exp2f(x[e]);
          l[i][e & 1] += pr[e];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t hi = pack16<T>(pr[2 * e], pr[2 * e + 1]);
          float h0, h1;
          unpack16<T>(hi, h0, h1);
          pf[i][e] = transpose8x8(hi);
          pl[i][e] = transpose8x8(pack16<T>(pr[2 * e] - h0, pr[2 * e + 1] - h1));
        }
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        // matrices of V, transposed: columns 16 k.. / keys 0-7, 16 k + 8.. / keys 0-7, 16 k.. / keys 8-15, 16 k + 8.. / keys 8-15
        const int r = ((lane >> 4) << 3) + (lane & 7), c = k * 2 + ((lane >> 3) & 1);
        uint32_t a[4];
        ldmatrix_x4t(a, vs + r * (D * 2) + ((c ^ (r & 7)) << 4));
#pragma unroll
        for (int i = 0; i < R; ++i) {
          mma16816<T>(o[i][k], a, pf[i][0], pf[i][1]);
          mma16816<T>(o[i][k], a, pl[i][0], pl[i][1]);
        }
      }
    }
    const bool end = cur.w.tile + 1 == cur.w.tiles;
    if (DEAL != kCluster && (end || t + 1 == left)) {
      finish(end);
      if (t + 1 < left) {
        next_pair<SHARED>(p, cur.w);
        if (cur.w.head == 0) cur.n = keys_of(cur.w.e);
        begin();
      }
    } else {
      cur.w.tile += step;
    }
  }
  if constexpr (DEAL == kCluster) {
    finish(true);
    if (p.cluster > 1) {
      cluster_sync_all();
      constexpr int PER = kThreads / D;
      const int rank = blockIdx.x % p.cluster, col = threadIdx.x % D;
      for (int row = rank * PER + (int)threadIdx.x / D; row < rows; row += p.cluster * PER) {
        float mb[kCluster8], lb[kCluster8], ob[kCluster8], mn = -INFINITY, ls = 0.f, acc = 0.f;
#pragma unroll
        for (int x = 0; x < kCluster8; ++x) {
          const int from = x < p.cluster ? x : 0;
          mb[x] = x < p.cluster ? remote(sm_bm + row, from) : -INFINITY;
          lb[x] = remote(sm_bl + row, from);
          ob[x] = remote(sm_b + row * D + col, from);
          mn = fmaxf(mn, mb[x]);
        }
#pragma unroll
        for (int x = 0; x < kCluster8; ++x) {
          if (x >= p.cluster) break;
          const float c = mn == -INFINITY ? 0.f : exp2f(mb[x] - mn);
          acc += ob[x] * c;
          ls += lb[x] * c;
        }
        if (p.shared) {
          const long slot = part_slot<false>(p, (long)cur.w.e * p.Hkv + cur.w.head, 0, true) * (8 * R) + row;
          p.part_o[slot * D + col] = acc;
          if (col == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(mn, ls);
          continue;
        }
        int b, w;
        row_token(row, b, w);
        const bool live = w < new_tokens(p, b) && !(ls == 0.f);
        reinterpret_cast<T*>(p.out)[b * p.o_sb + w * p.o_sw + (long)(cur.w.head * p.G + row % p.G) * p.o_sh + col] = from_f32<T>(live ? acc / ls : 0.f);
      }
      cluster_sync_all();                                  // nobody reads a block's sums any more
    }
  }
  if (DEAL == kDealt && p.shared == 0) finish_idle<T, D, kThreads>(p, threadIdx.x);
  if (late) pdl_wait();
}

// Pairs that are cut: block (c − 1, ·) has the one that is cut first in front of block c's share, and a warp of it joins the parts of ROWS rows at a time.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kThreads) paged_merge_kernel(const PagedAttn p, int grid) {
  const int block = blockIdx.x + 1;
  const Place at = find_place<kThreads, false>(p, grid, block);        // the kernel before this one waited for all that positions come from
  pdl_trigger();
  pdl_wait();
  if (at.e >= p.B * p.row_tiles) return;
  const int tiles = entry_tiles(p, at.e), head = (int)(at.tile / tiles);
  const long off = at.tile % tiles, t0 = block * at.per - off;
  if (off == 0 || off > at.per || whole<false>(p, tiles)) return;      // not cut here, or before, or not at all
  const int b = at.e / p.row_tiles, n = (int)((t0 + tiles - 1) / at.per) - (block - 1) + 1;
  const int row0 = at.e % p.row_tiles * p.tile_rows, rows = min(p.tile_rows, p.W * p.G - row0), m = new_tokens(p, b);
  for (int r0 = (blockIdx.y * kWarps + (threadIdx.x >> 5)) * ROWS; r0 < rows; r0 += gridDim.y * kWarps * ROWS) {
    bool live[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) live[r] = r0 + r < rows && (row0 + r0 + r) / p.G < m;
    join_parts<T, D, ROWS>(p, n, live, [&](int x, int r) { return part_slot<false>(p, 0, block - 1 + x, x == 0) * p.tile_rows + r0 + r; },
                           [&](int r) {
                             const int row = row0 + r0 + r, w = row / p.G;
                             return r0 + r < rows ? reinterpret_cast<T*>(p.out) + b * p.o_sb + w * p.o_sw + (long)(head * p.G + row % p.G) * p.o_sh : nullptr;
                           });
  }
}

// With shared pages: every row's parts over the shared pages and over its own.  Block (entry, ·), a warp per row and key/value head.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(const PagedAttn p, int grid) {
  __shared__ long sums[2][kWarps];
  const int e = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, entries = p.B * p.row_tiles;
  const int b = e / p.row_tiles, row0 = e % p.row_tiles * p.tile_rows, rows = min(p.tile_rows, p.W * p.G - row0);
  const int item = blockIdx.y * kWarps + warp, head = item / rows, rs = item % rows, row = row0 + rs, w = row / p.G;
  // parts over its own pages: a cluster leaves one, a launch that is dealt out as many as the pair was cut into
  int own = 1, b0 = 0;
  if (p.cluster == 0) {
    int before = 0, all = 0;
    for (int i = threadIdx.x; i < entries; i += kThreads) {
      const int t = entry_tiles(p, i);
      all += t;
      if (i < e) before += t;
    }
    const int w0 = __reduce_add_sync(0xffffffffu, before), w1 = __reduce_add_sync(0xffffffffu, all);
    if (lane == 0) { sums[0][warp] = w0; sums[1][warp] = w1; }
    __syncthreads();
    long first = 0, total = 0;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) { first += sums[0][x]; total += sums[1][x]; }
    const long per = max((long)p.min_tiles, (total * p.Hkv + grid - 1) / grid);
    const int tiles = entry_tiles(p, e);
    const long t0 = first * p.Hkv + (long)head * tiles;
    b0 = (int)(t0 / per);
    own = tiles == 0 ? 0 : whole<false>(p, tiles) ? 1 : (int)((t0 + tiles - 1) / per) - b0 + 1;
  }
  const bool live = item < rows * p.Hkv && w < new_tokens(p, b);
  const long r = (long)b * p.W * p.G + row, pre = r / p.pre_tile_rows * p.Hkv + head, s0 = pre * p.pre_tiles;
  const int c0 = (int)(s0 / p.pre_per), over = (int)((s0 + p.pre_tiles - 1) / p.pre_per) - c0 + 1, at = (int)(r % p.pre_tile_rows);
  pdl_trigger();
  pdl_wait();
  if (item >= rows * p.Hkv) return;
  const bool counts[1] = {live};
  join_parts<T, D, 1>(p, live ? over + own : 0, counts,
                      [&](int x, int) {
                        return x < over ? p.slots + part_slot<true>(p, pre, c0 + x, x == 0) * p.pre_tile_rows + at
                                        : part_slot<false>(p, (long)e * p.Hkv + head, b0 + x - over, x == over) * p.tile_rows + rs;
                      },
                      [&](int) { return reinterpret_cast<T*>(p.out) + b * p.o_sb + w * p.o_sw + (long)(head * p.G + row % p.G) * p.o_sh; });
}

template <typename T, int D, int R, Deal DEAL>
void launch_rows(const PagedAttn& p, int grid, cudaStream_t st) {
  constexpr int smem = rows_smem<D>(DEAL == kCluster);
  static_assert(DEAL != kCluster || kSums<D> + 8 * R * D * 4 <= smem, "a cluster's sums lie over the ring");
  NXD_ALLOW_SMEM((paged_rows_kernel<T, D, R, DEAL>), smem);
  if (DEAL != kCluster || p.cluster == 1) return launch_dependent(paged_rows_kernel<T, D, R, DEAL>, grid, kThreads, smem, st, p);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid; cfg.blockDim = kThreads; cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 2;
  NXD_CUDA_CHECK(cudaLaunchKernelEx(&cfg, paged_rows_kernel<T, D, R, DEAL>, p));
}
// T: of what comes out; dt: of queries and caches
template <typename T, int D>
int launch(const PagedAttn& p, const PagedPlan& plan, int dt, int out_dt, cudaStream_t st) {
  if (p.shared) {
    if (plan.pre_tiles) paged_tiles(p, plan.pre_grid, true, D, dt, out_dt, st);
    else if (p.pre_tile_rows == 8) launch_rows<T, D, 1, kShared>(p, plan.pre_grid, st);
    else launch_rows<T, D, 2, kShared>(p, plan.pre_grid, st);
  }
  if (p.cluster && p.tile_rows == 8) launch_rows<T, D, 1, kCluster>(p, plan.grid, st);
  else if (p.cluster) launch_rows<T, D, 2, kCluster>(p, plan.grid, st);
  else if (plan.tiles) paged_tiles(p, plan.grid, false, D, dt, out_dt, st);
  else if (p.tile_rows == 8) launch_rows<T, D, 1, kDealt>(p, plan.grid, st);
  else launch_rows<T, D, 2, kDealt>(p, plan.grid, st);
  const int rows = std::min(p.tile_rows, p.W * p.G);
  if (p.shared)
    launch_dependent(paged_join_kernel<T, D>, dim3(p.B * p.row_tiles, (rows * p.Hkv + kWarps - 1) / kWarps), kThreads, 0, st, p, plan.grid);
  else if (!p.cluster && plan.grid > 1) {
    // a warp joins four rows at once where there are many, whose loads are in flight together; eight blocks of y, or what follows has waves (us, 2 x 1000
    // tokens of 48 heads of 64 behind 6000 keys, a block for 8 rows each / this: 166 / 156; 2 x 1000 tokens, 32 heads, to 2000 keys 112 / 102; 463
    // tokens, 64 heads, to 489 keys 54 / 45).  Few rows have more parts each, and warps enough.
    auto merge = [&](auto kernel, int each) {
      launch_dependent(kernel, dim3(plan.grid - 1, std::min((rows + each * kWarps - 1) / (each * kWarps), 8)), kThreads, 0, st, p, plan.grid);
    };
    if (rows > 64) merge(paged_merge_kernel<T, D, 4>, 4);
    else merge(paged_merge_kernel<T, D, 1>, 1);
  }
  return p.shared ? 3 : !p.cluster && plan.grid > 1 ? 2 : 1;
}

}  // namespace

// Up to 16 query rows of a sequence and key/value head (8 where there are many long tables, below) go to the kernel above, more to tiles of 64, 128 or 256
// rows on the tensor memory.  Lengths are the tables': nothing about positions is known here.
PagedPlan paged_plan(PagedAttn& p) {
  PagedPlan plan{};
  const int sms = device_sm_count();
  // rows, the most that go to the few-row kernel → whether there are more; rows of a tile
  auto cut = [](long rows, int few, int& tile_rows) {
    tile_rows = rows <= few ? (rows <= 8 ? 8 : 16) : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
    return rows > few;
  };
  const long rows = (long)p.W * p.G, all = rows * p.B;
  // Portions of prompts, whose own rows fill the row tiles, gain nothing from the batch's: the shared pages are the first of their own
  // (nor is there room for them where the join, a warp for each row and head, would have more than 65535 blocks of one sequence).
  p.shared = rows <= 128 && rows * p.Hkv <= 65535l * kWarps ? p.shared_cols * p.ps : 0;
  // Nine to sixteen rows of long sequences, enough of them to fill the GPU, are the tensor memory's, too: there the few-row kernel is bound by its
  // instructions (us, few rows / tiles: 16 sequences to 3000 keys, 16 rows, 8 heads, 50 / 45; 4 to 8000 50 / 34; 8 to 4000 38 / 35; but 1 to 2000
  // 11 / 18, 32 to 1000 33 / 43).
  const long pairs = (long)p.B * p.Hkv, cap = (long)p.cols * p.ps - p.shared;
  plan.tiles = cut(rows, cap > 2048 && pairs * cap > 131072 ? 8 : 16, p.tile_rows);
  // Row tiles of 256 read keys half as often, but they have to fill the GPU (us, 256 / 128 rows: 33 tokens, 48 heads on 8, 21 / 17; 300, 8 on 8, 27 / 22;
  // 4 x 64, 32 on 8, to 3000 keys 47 / 40; but 500, 32 on 8, to 6000 72 / 80, 1000 to 1000 46 / 83).
  if (p.tile_rows == 256 && (rows + 255) / 256 * pairs * 5 < 2 * sms) p.tile_rows = 128;
  p.row_tiles = (int)((rows + p.tile_rows - 1) / p.tile_rows);
  auto tile_keys = [](int tile_rows) { return tile_rows == 256 ? 128 : kTileKeys; };
  p.tile_keys = tile_keys(p.tile_rows);
  p.min_tiles = plan.tiles ? 1 : 256 / p.tile_keys;
  // A cut writes and reads the sums of all rows once more for each part, and a last launch has work: short pairs are not cut (us, cut / not: 463 tokens,
  // 64 heads on 8, 45 / 37; 1000, 32 on 8, 56 / 46; 2 x 1000 to 2000 keys 104 / 90; 283, 8 on 8, 22 / 20).  Windows' sums are small: 16 x 6 tokens,
  // 32 heads on 8, to 900 keys, 12 tiles at most not cut / 4: 32 / 28.
  p.whole_tiles = !plan.tiles ? 0 : p.tile_rows == 64 ? 4 : 12;
  plan.grid = plan.tiles ? sms : 2 * sms;
  // A cluster per pair, as many blocks in it as the GPU takes at once, has neither a search for places nor a second launch (us, dealt out / cluster:
  // 1 sequence of 1000 keys, 8 heads, 19 / 9.8; 64 of 300 to 600, 8 heads, 36 / 28; 16 of 4096 to 8192, 8 heads, 72 / 68), but the longest
  // sequence lasts as long as its own blocks take, at 47 GB/s each: 2048 keys, 22 us, at most.
  if (!plan.tiles) {
    int size = 1;
    while (size < kCluster8 && ((cap > 256l * size && pairs * size * 2 <= 2 * sms) || cap > 2048l * size)) size *= 2;
    if (cap <= 2048l * size && pairs * size < (1l << 30)) {
      p.cluster = size;
      plan.grid = (int)(pairs * size);
    }
  }
  plan.slots = (p.shared ? (long)p.B * p.row_tiles * p.Hkv + (p.cluster ? 0 : plan.grid) : p.cluster ? 0l : 2l * plan.grid) * p.tile_rows;
  p.slots = plan.slots;
  if (p.shared) {
    plan.pre_tiles = cut(all, 16, p.pre_tile_rows);
    // Row tiles of 256 where there is work for all: fewer than two of their tiles for an SM are better cut finer (us, 256 / 128 rows: 57 rows of 48
    // heads over 464 keys 33 / 29, 56 of 32 over 960 41 / 32, 32 x 4 over 2048 38 / 36; but 32 x 5 of 64 heads over 4096 73 / 90).
    if (p.pre_tile_rows == 256 && (all + 255) / 256 * p.Hkv * ((p.shared + 127) / 128) <= 2 * sms) p.pre_tile_rows = 128;
    p.pre_row_tiles = (int)((all + p.pre_tile_rows - 1) / p.pre_tile_rows);
    const int keys = tile_keys(p.pre_tile_rows);
    p.pre_tiles = (p.shared + keys - 1) / keys;
    // Small ones on three fifths of the GPU, so that the launch over the rows' own pages has the rest, but no more than 384 keys a block for that (8 rows
    // of 32 heads over 4096 keys: 19 us with 86 blocks, 24 with 128; 43 of 64 heads over 368: 25 with 384 keys a block, 22 with 128).
    const long total = (long)p.pre_row_tiles * p.Hkv * p.pre_tiles, most = plan.pre_tiles ? sms : 2 * sms;
    p.pre_per = (int)std::max((total + most - 1) / most, std::min(384l / keys, (5 * total + 3 * most - 1) / (3 * most)));
    plan.pre_grid = (int)((total + p.pre_per - 1) / p.pre_per);
    plan.pre_slots = ((long)p.pre_row_tiles * p.Hkv + plan.pre_grid) * p.pre_tile_rows;
  }
  return plan;
}

int paged_attention(const PagedAttn& p, const PagedPlan& plan, int D, int dt, cudaStream_t st) {
  if (dt == kBF16) return D == 128 ? launch<__nv_bfloat16, 128>(p, plan, dt, dt, st) : launch<__nv_bfloat16, 64>(p, plan, dt, dt, st);
  return D == 128 ? launch<__half, 128>(p, plan, dt, dt, st) : launch<__half, 64>(p, plan, dt, dt, st);
}

int paged_attention_half(const PagedAttn& p, const PagedPlan& plan, int D, int out_dt, cudaStream_t st) {
  if (!plan.tiles || p.shared) nxd_throw("paged_attention_half: not for tiles", __FILE__, __LINE__);
  if (out_dt == kBF16) return D == 128 ? launch<__nv_bfloat16, 128>(p, plan, kF16, out_dt, st) : launch<__nv_bfloat16, 64>(p, plan, kF16, out_dt, st);
  return D == 128 ? launch<__half, 128>(p, plan, kF16, out_dt, st) : launch<__half, 64>(p, plan, kF16, out_dt, st);
}

void paged_append(const void* q, const void* k, const void* v, const long* positions, const long* lens, const float* cos_t, const float* sin_t,
                  void* q_out, void* kc, void* vc, const int* table, int* lost, int B, int W, int H, int Hkv, int D, int rows, int cols, int ps,
                  int pages, long table_sb, const long (*s)[3], long o_sb, long o_sw, const long (*cs)[3], int dt, cudaStream_t st) {
  const int half = D / 2;
  const long tokens = (long)B * W, items = (long)(H + 2 * Hkv) * (half / (dt == kF32 ? 4 : 8)), parts = (items + kAppendThreads - 1) / kAppendThreads;
  if (tokens == 0) return;
  if (tokens * parts >= (1l << 31)) nxd_throw("paged_append: too many tokens", __FILE__, __LINE__);
  const AppendArgs a{q, k, v, positions, lens, cos_t, sin_t, q_out, kc, vc, table, lost, B, W, H, Hkv, half, rows, cols, ps, pages, (int)parts,
                     table_sb, s[0][0], s[0][1], s[0][2], s[1][0], s[1][1], s[1][2], s[2][0], s[2][1], s[2][2], o_sb, o_sw,
                     cs[0][0], cs[0][1], cs[0][2], cs[1][0], cs[1][1], cs[1][2]};
  const unsigned grid = (unsigned)(tokens * parts);
  if (dt == kBF16) launch_dependent(paged_append_kernel<__nv_bfloat16>, grid, kAppendThreads, 0, st, a);
  else if (dt == kF16) launch_dependent(paged_append_kernel<__half>, grid, kAppendThreads, 0, st, a);
  else launch_dependent(paged_append_kernel<float>, grid, kAppendThreads, 0, st, a);
}

}  // namespace nxd
