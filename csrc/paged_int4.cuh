// What the attention kernels over a cache in 4 bits share (Int4Attn: kernels.h; how work is dealt out: paged.cuh).
#pragma once
#include <algorithm>
#include <cfloat>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace nxd {
namespace int4 {

using namespace paged;

constexpr int kKeys = 16;                                  // keys of a warp's part of a tile
constexpr float kNone = -1e30f;                            // the reference of a row that has seen no key
constexpr int kCluster8 = 8;                               // blocks of a cluster at most
constexpr int kStages = 3;
template <int D> constexpr int kPitch = D + 4;             // of rows of sums
template <int D> constexpr int kStage = 2 * kKeys * (D / 2) + 2 * kKeys * 16;        // bytes of a warp's part: codes of keys and values, steps of both, 16 bytes a key
template <int D> constexpr int kQPitch = D * 2 + 16;       // bytes of a query row: ldmatrix meets no bank twice
template <int D, int R> constexpr int kQueries = 8 * R * (kQPitch<D> + 16 + 8);        // of 8 R rows: numbers, sums of their groups, units and limits

template <int BYTES> NXD_DEVICE void cp_async(uint32_t dst, const void* src, bool live) {      // not live: zero bytes, nothing is read
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(live ? BYTES : 0), "n"(BYTES) : "memory");
}
template <int BYTES> NXD_DEVICE void cp_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
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
NXD_DEVICE void ldmatrix_x2t(uint32_t (&r)[2], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}
NXD_DEVICE uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
NXD_DEVICE void stmatrix_x2t(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
NXD_DEVICE void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
NXD_DEVICE void mma1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(b0));
}
NXD_DEVICE uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
NXD_DEVICE uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
NXD_DEVICE float remote(const float* at, int rank) {       // the same place in another block's shared memory
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(at), rank)) : "memory");
  return v;
}
NXD_DEVICE __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
NXD_DEVICE uint32_t as_u32(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
NXD_DEVICE uint32_t pack_half(float lo, float hi) { return as_u32(__floats2half2_rn(lo, hi)); }
// Codes 0 to 3 of either half of a word as halves: the denormals c 2^-24, those of 1 and 3 times 16.  The last by a difference, which is exact and leaves the pipe of
// logic, the one that these kernels fill, one of five instructions less.
struct Codes { uint32_t c0, c1, c2, c3; };
NXD_DEVICE Codes codes_of(uint32_t w) {
  const uint32_t up = __byte_perm(w, 0, 0x4341), c2 = up & 0x000f000fu;
  return {w & 0x000f000fu, w & 0x00f000f0u, c2, as_u32(__hsub2(as_half2(up), as_half2(c2)))};
}
// 16-byte chunk c of row r of a tile of codes lies at chunk c ^ (…): ldmatrix meets no bank twice
template <int D> NXD_DEVICE uint32_t chunk_at(int r, int c) { return r * (D / 2) + ((c ^ (D == 128 ? (r >> 1) & 3 : (r >> 2) & 1)) << 4); }


// Where block's share of all key tiles begins (paged.cuh), found by one warp: entry and tile within the entry's pairs, and how many tiles it has
struct Share { int e, tile, tiles; };
NXD_DEVICE Share find_share(const Int4Attn& p, int grid, int block, int lane) {
  const int entries = p.B * p.row_tiles, each = (entries + 31) / 32, e0 = min(entries, lane * each), e1 = min(entries, e0 + each);
  long mine = 0;
  for (int e = e0; e < e1; ++e) mine += entry_tiles(p, e);
  long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  const long total = __shfl_sync(0xffffffffu, upto, 31) * p.Hkv, per = max((long)p.min_tiles, (total + grid - 1) / grid);
  long left = block * per - (upto - mine) * p.Hkv;
  Share s{entries, 0, 0};
  const bool here = left >= 0 && left < mine * p.Hkv;
  if (here)
    for (int e = e0; e < e1; ++e) {
      const long t = (long)entry_tiles(p, e) * p.Hkv;
      if (left < t) {
        s = Share{e, (int)left, (int)min(per, total - block * per)};
        break;
      }
      left -= t;
    }
  const unsigned who = __ballot_sync(0xffffffffu, here);
  const int from = who ? __ffs(who) - 1 : 0;
  s.e = __shfl_sync(0xffffffffu, s.e, from);
  s.tile = __shfl_sync(0xffffffffu, s.tile, from);
  s.tiles = __shfl_sync(0xffffffffu, s.tiles, from);
  return s;
}

// keys that some row of an entry sees
NXD_DEVICE int keys_of(const Int4Attn& p, int e) {
  if (e >= p.B * p.row_tiles) return 0;
  const int b = e / p.row_tiles, row0 = e % p.row_tiles * p.tile_rows, m = new_tokens(p, b);
  return row0 / p.G < m ? visible_keys(p, b, min(m, (row0 + p.tile_rows + p.G - 1) / p.G) - 1) : 0;
}

// Zeros for the rows of entries none of whose tokens sees a key, or counts, 16 rows of an entry at a time, a warp each
template <typename T, int D, int WARPS>
NXD_DEVICE void finish_idle_warps(const Int4Attn& p, int warp, int lane) {
  const int chunks = (p.tile_rows + 15) / 16;
  for (long i = blockIdx.x + (long)gridDim.x * warp; i < (long)p.B * p.row_tiles * chunks; i += (long)gridDim.x * WARPS) {
    const int e = (int)(i / chunks);
    if (entry_tiles(p, e) > 0) continue;
    const int b = e / p.row_tiles, row0 = e % p.row_tiles * p.tile_rows + (int)(i % chunks) * 16;
    const int rows = min(min(16, p.tile_rows - (int)(i % chunks) * 16), p.W * p.G - row0);
    for (int x = lane; x < rows * p.Hkv * (D / 8); x += 32) {
      const int c = x % (D / 8), y = x / (D / 8), head = y % p.Hkv, row = row0 + y / p.Hkv;
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + b * p.o_sb + row / p.G * p.o_sw + (long)(head * p.G + row % p.G) * p.o_sh + c * 8) =
          make_uint4(0, 0, 0, 0);
    }
  }
}

// A warp's ring of cp.async stages: 16 keys of every tile of its block's share, asked for in order, over the ends of pairs.  A lane copies 16 bytes of codes of one or two
// keys and of their values (rows row and row + PASS of 16, chunk lane % CH), and one row of steps: half a warp has the keys', half the values'.  Places are in
// units of what is copied.
template <int D, int WARPS, bool CLUSTER>
struct Ring {
  static constexpr int NG = D / 32, CH = D / 32, PASS = 32 / CH, STAGE = kStage<D>, TILE = WARPS * kKeys;
  static constexpr int V_AT = kKeys * (D / 2), KS_AT = 2 * V_AT, VS_AT = KS_AT + kKeys * 16;
  static constexpr uint32_t kHole = 0xffffffffu;
  const Int4Attn& p;
  Walk* pair;                                              // this warp's, in shared memory: the pair that is asked for
  const int warp, lane;
  const uint32_t ring, dst0, dst1, k_mine, v_mine, s_mine;
  uint32_t kc = kHole, vc = 0, ks = 0, vs = 0;             // where the warp's keys in 32 tiles lie, a tile a lane; no page there: kHole
  int asked = 0, next_page = 32, tile, last, n;            // tiles that have been asked for, the next one's lane; the pair's next tile, tiles, keys
  const int tiles, step;                                   // of the block
  uint32_t holes = 0;                                      // bit i: there is no page for the warp's keys of the tile that was asked for i before the last one

  NXD_DEVICE Ring(const Int4Attn& p_, Walk* pair_, const Walk& first, int tiles_, int step_, uint32_t ring_, int warp_, int lane_)
      : p(p_), pair(pair_), warp(warp_), lane(lane_), ring(ring_), dst0(ring_ + chunk_at<D>(lane_ / CH, lane_ % CH)),
        dst1(ring_ + chunk_at<D>((PASS + lane_ / CH) % 16, lane_ % CH)), k_mine(lane_ / CH * (uint32_t)p_.k_sr + lane_ % CH),
        v_mine(lane_ / CH * (uint32_t)p_.v_sr + lane_ % CH), s_mine(lane_ < 16 ? lane_ * (uint32_t)p_.ks_sr : (lane_ - 16) * (uint32_t)p_.vs_sr),
        tile(first.tile), last(first.tiles), n(tiles_ > 0 ? keys_of(p_, first.e) : 0), tiles(tiles_), step(step_) {
    if (lane == 0) *pair = first;
    __syncwarp();
  }
  NXD_DEVICE void fetch() {
    const Walk w = *pair;
    const unsigned key = (unsigned)(tile + lane * step) * TILE + warp * kKeys, i = key / (unsigned)p.ps, row = key - i * (unsigned)p.ps;
    kc = kHole;
    vc = ks = vs = 0;
    if (i >= (unsigned)p.cols) return;
    const int page = i < (unsigned)p.shared_cols ? p.shared_pages[i] : p.table[w.e / p.row_tiles * p.table_sb + i];
    if ((unsigned)page >= (unsigned)p.pages) return;
    const uint32_t u = page, h = w.head;
    kc = u * (uint32_t)p.k_sp + row * (uint32_t)p.k_sr + h * (uint32_t)p.k_sh;
    vc = u * (uint32_t)p.v_sp + row * (uint32_t)p.v_sr + h * (uint32_t)p.v_sh;
    ks = u * (uint32_t)p.ks_sp + row * (uint32_t)p.ks_sr + h * (uint32_t)p.ks_sh;
    vs = u * (uint32_t)p.vs_sp + row * (uint32_t)p.vs_sr + h * (uint32_t)p.vs_sh;
  }
  NXD_DEVICE void ask(int stage) {
    if (asked < tiles) {
      if (!CLUSTER && tile == last) {
        __syncwarp();
        Walk w = *pair;
        next_pair<false>(p, w);
        tile = 0;
        last = w.tiles;
        n = keys_of(p, w.e);
        __syncwarp();
        if (lane == 0) *pair = w;
        __syncwarp();
        next_page = 32;
      }
      if (next_page == 32) { fetch(); next_page = 0; }
      const uint32_t k = __shfl_sync(0xffffffffu, kc, next_page), v = __shfl_sync(0xffffffffu, vc, next_page);
      const uint32_t sk = __shfl_sync(0xffffffffu, ks, next_page), sv = __shfl_sync(0xffffffffu, vs, next_page);
      ++next_page;
      const bool there = k != kHole;
      const int row = lane / CH, seen = there ? n - (tile * TILE + warp * kKeys) : 0;          // keys that anybody sees
      const uint8_t* const kp = reinterpret_cast<const uint8_t*>(p.k);
      const uint8_t* const vp = reinterpret_cast<const uint8_t*>(p.v);
      const uint8_t* const sp = reinterpret_cast<const uint8_t*>(lane < 16 ? p.ks : p.vs);
      const uint32_t to = stage * STAGE, ka = k + k_mine, va = v + v_mine, sa = (lane < 16 ? sk : sv) + s_mine;
      const uint32_t kb = ka + PASS * (uint32_t)p.k_sr, vb = va + PASS * (uint32_t)p.v_sr;
      if (seen >= kKeys) {                                 // all of them
        cp_async<16>(dst0 + to, kp + (uint64_t)ka * 16);
        cp_async<16>(dst0 + to + V_AT, vp + (uint64_t)va * 16);
        if constexpr (PASS < 16) {
          cp_async<16>(dst1 + to, kp + (uint64_t)kb * 16);
          cp_async<16>(dst1 + to + V_AT, vp + (uint64_t)vb * 16);
        }
        cp_async<NG * 4>(ring + to + KS_AT + lane * 16, sp + (uint64_t)sa * (NG * 4));
      } else {                                             // the others are zeros; addresses of what is not read stay inside all the same
        cp_async<16>(dst0 + to, kp + (uint64_t)(row < seen ? ka : 0u) * 16, row < seen);
        cp_async<16>(dst0 + to + V_AT, vp + (uint64_t)(row < seen ? va : 0u) * 16, row < seen);
        if constexpr (PASS < 16) {
          cp_async<16>(dst1 + to, kp + (uint64_t)(PASS + row < seen ? kb : 0u) * 16, PASS + row < seen);
          cp_async<16>(dst1 + to + V_AT, vp + (uint64_t)(PASS + row < seen ? vb : 0u) * 16, PASS + row < seen);
        }
        cp_async<NG * 4>(ring + to + KS_AT + lane * 16, sp + (uint64_t)((lane & 15) < seen ? sa : 0u) * (NG * 4), (lane & 15) < seen);
      }
      holes = holes * 2 + !there;
      ++asked;
      tile += step;
    } else {
      holes *= 2;
    }
    cp_async_commit();
  }
  template <int STAGES> NXD_DEVICE bool hole() const { return holes >> (STAGES - 2) & 1; }         // of the tile that comes next, before another one is asked for

};

// A warp makes a row of queries ready: number d of a group at (d % 4) 8 + d / 4, so that four 8 x 8 matrices of a group are the operands of its two products; odd
// numbers, which meet codes that lie one place up, a sixteenth.  The row is multiplied by a power of two that brings its largest number to 2^14; unit: what
// brings scores back (codes are 2^-24 of themselves), not 0, which would make NaN of the -inf of what nobody sees.
// sums: of the groups, 2^-5 of them, as two halves each, the rounded ones, then what that left.
template <typename T, int D>
NXD_DEVICE void ready_query(const T* row, bool live, uint32_t to, uint32_t sums, float* unit, float scale_log2, int lane) {
  constexpr int N = D / 32, NG = D / 32;                   // numbers of a lane, groups
  const T* const qp = row + lane * N;
  float x[N], most = 0.f, sum = 0.f;
  if constexpr (N == 4) {
    const uint2 u = live ? *reinterpret_cast<const uint2*>(qp) : make_uint2(0, 0);
    unpack16<T>(u.x, x[0], x[1]);
    unpack16<T>(u.y, x[2], x[3]);
  } else {
    unpack16<T>(live ? *reinterpret_cast<const uint32_t*>(qp) : 0u, x[0], x[1]);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) most = fmaxf(most, fabsf(x[k]));
  most = warp_max(most);
  const int e = min(max((int)(__float_as_uint(most) >> 23), 20), 244);
  const float up = __uint_as_float((uint32_t)(268 - e) << 23);
  to += lane * N / 32 * 64;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int d = lane * N % 32 + k;
    x[k] *= up;
    sum += x[k];
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + ((d & 3) * 8 + (d >> 2)) * 2), "h"(__half_as_ushort(__float2half_rn(d & 1 ? x[k] * 0.0625f : x[k]))) : "memory");
  }
#pragma unroll
  for (int k = 1; k < 32 / N; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
  sum *= 0.03125f;
  if (lane % (32 / N) == 0) {
    const __half hi = __float2half_rn(sum);
    const uint32_t at = sums + lane / (32 / N) * 2;
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(__half_as_ushort(hi)) : "memory");
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(at + NG * 2), "h"(__half_as_ushort(__float2half_rn(sum - __half2float(hi)))) : "memory");
    if constexpr (NG == 2) asm volatile("st.shared.u32 [%0], %1;" ::"r"(sums + 8 + lane / (32 / N) * 4), "r"(0u) : "memory");
  }
  if (lane == 0) *unit = fmaxf(__uint_as_float((uint32_t)(e + 10) << 23) * scale_log2, FLT_MIN);
}

template <typename K>
inline void launch_cluster(K kernel, const Int4Attn& p, int grid, int threads, int smem, int cluster, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid; cfg.blockDim = threads; cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
  NXD_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
}

// A cluster's blocks have left their sums [rows][D], maxima and weights of a pair in shared memory: joined, times `factor`, to the output, rows in turn
template <typename T, int D, int THREADS>
NXD_DEVICE void join_cluster(const Int4Attn& p, const Walk& w0, int row0, int rows, const float* sm_b, const float* sm_bm, const float* sm_bl, float factor) {
  cluster_sync_all();
  constexpr int PER = THREADS / D;
  const int rank = blockIdx.x % p.cluster, col = threadIdx.x % D, b = w0.e / p.row_tiles, count = new_tokens(p, b);
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
      const float c = mb[x] == -INFINITY ? 0.f : exp2f(mb[x] - mn);
      acc += ob[x] * c;
      ls += lb[x] * c;
    }
    const int w = (row0 + row) / p.G;
    const bool live = w < count && !(ls == 0.f);
    reinterpret_cast<T*>(p.out)[b * p.o_sb + w * p.o_sw + (long)(w0.head * p.G + (row0 + row) % p.G) * p.o_sh + col] = from_f32<T>(live ? factor * acc / ls : 0.f);
  }
  cluster_sync_all();                                      // nobody reads a block's sums any more
}

}  // namespace int4

void int4_tiles(const Int4Attn& p, int grid, int D, int dt, cudaStream_t st);       // more than eight rows of a pair (paged_int4_tiles.cu)

}  // namespace nxd
