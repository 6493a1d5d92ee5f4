// A key/value cache in pages that is held in 4 bits: 32 numbers of a token's head are m + s c, m and s in half precision, c of 0 to 15 (kernels.h: Int4Pages).
// Appending with the position rotation on the way, reading tokens back, and attention of query rows over the codes.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace nxd {

int device_sm_count();

namespace {

using namespace paged;

// ---------------------------------------------------------------------------------------------------------------- append
constexpr int kAppendThreads = 128;

NXD_DEVICE float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
NXD_DEVICE float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

template <typename T> struct Eight {                       // eight numbers beside one another
  static constexpr int PACKS = 8 / Pack16<T>::N;
  Pack16<T> p[PACKS];
  NXD_DEVICE void load(const T* at) {
#pragma unroll
    for (int i = 0; i < PACKS; ++i) p[i].load(at + i * Pack16<T>::N);
  }
  NXD_DEVICE void store(T* at) const {
#pragma unroll
    for (int i = 0; i < PACKS; ++i) p[i].store(at + i * Pack16<T>::N);
  }
  NXD_DEVICE float f(int i) const { return p[i / Pack16<T>::N].f(i % Pack16<T>::N); }
  NXD_DEVICE void set(int i, float x) { p[i / Pack16<T>::N].set(i % Pack16<T>::N, x); }
};

// A thread has eight numbers of one head, which lie beside one another, and reads the eight that turn with them where those lie elsewhere; four threads
// have the 32 numbers that share m and s.  Bound by HBM.  Keys turn as a c - b s with what the rounding of b s left put back, one rounding in
// all; a code whose quotient is nearer than 2^-15 to a border is found again from the products in 64 bits, so that codes are those of exact numbers.
template <typename T>
__global__ void __launch_bounds__(kAppendThreads) int4_append_kernel(const Int4Append p) {
  pdl_trigger();
  const unsigned t = blockIdx.x / p.parts, item = blockIdx.x % p.parts * kAppendThreads + threadIdx.x, chunks = p.D / 8;
  const int h = (int)(item / chunks), c = (int)(item % chunks) * 8;
  const int w = (int)(t / p.B), b = (int)(t % p.B);        // tokens of all sequences beside one another, as projections leave them
  pdl_wait();
  if (h >= p.H + 2 * p.Hkv) return;
  const long slot = p.slots[(long)b * p.W + w], first = p.positions[b], pos = first + w;
  const bool has = slot >= 0 && slot < p.tokens, inside = first > -(1l << 40) && first < p.rows && pos >= 0 && pos < p.rows;
  const bool live = has && inside, query = h < p.H, key = !query && h < p.H + p.Hkv;
  if (!live) {
    if (p.lost && item == 0 && has) *p.lost = 1;
    if (query) {
      Eight<T> zero;
#pragma unroll
      for (int i = 0; i < 8; ++i) zero.set(i, 0.f);
      zero.store((T*)p.q_out + b * p.o_sb + w * p.o_sw + (long)h * p.D + c);
    }
    return;
  }
  const T* const src = query ? (const T*)p.q + b * p.q_sb + w * p.q_sw + h * p.q_sh
                       : key ? (const T*)p.k + b * p.k_sb + w * p.k_sw + (h - p.H) * p.k_sh
                             : (const T*)p.v + b * p.v_sb + w * p.v_sw + (h - p.H - p.Hkv) * p.v_sh;
  Eight<T> mine, other;
  mine.load(src + c);
  // x = a co + b si, for each of the eight numbers: what turns with it, with the sine's sign
  float x[8], co[8], si[8], turned[8];
  const bool turns = (query || key) && c < 2 * p.half;
#pragma unroll
  for (int i = 0; i < 8; ++i) { co[i] = 1.f; si[i] = 0.f; x[i] = mine.f(i); turned[i] = 0.f; }
  if (turns && p.pairs) {
    const float4 cv = *reinterpret_cast<const float4*>(p.cos_t + pos * p.half + c / 2), sv = *reinterpret_cast<const float4*>(p.sin_t + pos * p.half + c / 2);
    const float cf[4] = {cv.x, cv.y, cv.z, cv.w}, sf[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      turned[i] = x[i ^ 1];
      co[i] = cf[i / 2];
      si[i] = i & 1 ? sf[i / 2] : -sf[i / 2];
    }
  } else if (turns) {
    const bool low = c < p.half;
    const int at = low ? c : c - p.half;
    other.load(src + (low ? c + p.half : at));
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 cv = *reinterpret_cast<const float4*>(p.cos_t + pos * p.half + at + i), sv = *reinterpret_cast<const float4*>(p.sin_t + pos * p.half + at + i);
      const float cf[4] = {cv.x, cv.y, cv.z, cv.w}, sf[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        turned[i + j] = other.f(i + j);
        co[i + j] = cf[j];
        si[i + j] = low ? -sf[j] : sf[j];
      }
    }
  }
  if (query) {
#pragma unroll
    for (int i = 0; i < 8; ++i) mine.set(i, turns ? x[i] * co[i] + turned[i] * si[i] : x[i]);
    mine.store((T*)p.q_out + b * p.o_sb + w * p.o_sw + (long)h * p.D + c);
    return;
  }
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float e = __fmul_rn(turned[i], si[i]);
    y[i] = turns ? __fadd_rn(__fmaf_rn(x[i], co[i], e), __fmaf_rn(turned[i], si[i], -e)) : x[i];
  }
  float lo = y[0], hi = y[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) { lo = min_nan(lo, y[i]); hi = max_nan(hi, y[i]); }
  const unsigned four = 0xfu << (threadIdx.x & 28);        // the threads of the 32 numbers: all of one head
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(four, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(four, hi, o));
  }
  const __half m16 = __float2half_rn(lo);
  const float m = __half2float(m16);
  const __half s16 = __float2half_rn(__fdiv_rn(__fsub_rn(hi, m), 15.f));
  const float s = __half2float(s16), inv = s > 0.f && s <= 65504.f ? 1.f / s : 0.f;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = inv == 0.f ? 0.f : (y[i] - m) * inv;
    float r = rintf(q);
    if (fabsf(q - r) > 0.5f - 0x1p-15f) {                  // a border, from numbers that are exact
      const double exact = turns ? (double)x[i] * co[i] + (double)turned[i] * si[i] : (double)x[i], at = floorf(q);
      const double above = (exact - m) - (at + 0.5) * s;
      r = (float)(above > 0 || (above == 0 && ((int)at & 1)) ? at + 1 : at);
    }
    codes |= (uint32_t)fminf(fmaxf(r, 0.f), 15.f) << (4 * i);
  }
  const Int4Pages& to = key ? p.kp : p.vp;
  const int head = h - p.H - (key ? 0 : p.Hkv), page = (int)slot / p.ps, row = (int)slot - page * p.ps;
  *reinterpret_cast<uint32_t*>(to.codes + page * to.c_sp + row * to.c_sr + head * to.c_sh + c / 2) = codes;
  uint16_t* const steps = to.steps + page * to.s_sp + row * to.s_sr + head * to.s_sh + c / 32;
  if (c % 32 == 0) *steps = __half_as_ushort(s16);
  if (c % 32 == 8) steps[p.D / 32] = __half_as_ushort(m16);
}

// ---------------------------------------------------------------------------------------------------------------- gather
constexpr int kGatherThreads = 256;
// Tokens at slots as numbers of T: a thread has eight of them.  Bound by HBM.
template <typename T>
__global__ void __launch_bounds__(kGatherThreads) int4_gather_kernel(const Int4Pages kp, const Int4Pages vp, const int* slots, T* k, T* v, long items, int Hkv, int D,
                                                                    int ps, long tokens) {
  pdl_trigger();
  pdl_wait();
  const long i = (long)blockIdx.x * kGatherThreads + threadIdx.x;
  if (i >= items) return;
  const bool key = blockIdx.y == 0;
  const unsigned chunks = D / 8, per = Hkv * chunks;
  const long t = i / per;
  const unsigned x = (unsigned)(i - t * per), head = x / chunks, c = x % chunks * 8;
  const long slot = slots[t];
  Eight<T> out;
  if (slot >= 0 && slot < tokens) {
    const Int4Pages& from = key ? kp : vp;
    const int page = (int)slot / ps, row = (int)slot - page * ps;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(from.codes + page * from.c_sp + row * from.c_sr + head * from.c_sh + c / 2);
    const uint16_t* const steps = from.steps + page * from.s_sp + row * from.s_sr + head * from.s_sh + c / 32;
    const float s = __half2float(__ushort_as_half(steps[0])), m = __half2float(__ushort_as_half(steps[D / 32]));
#pragma unroll
    for (int j = 0; j < 8; ++j) out.set(j, fmaf((float)(codes >> (4 * j) & 15), s, m));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) out.set(j, 0.f);
  }
  out.store((key ? k : v) + i * 8);
}

// ------------------------------------------------------------------------------------------------------- attention, few rows
constexpr int kKeys = 16;                                  // keys of a warp's tile
constexpr int kTileKeys = kWarps * kKeys;                  // keys of a block's tile
constexpr float kNone = -1e30f;                            // the reference of a row that has seen no key
constexpr int kCluster8 = 8;                               // blocks of a cluster at most
constexpr int kStages = 3;
template <int D> constexpr int kPitch = D + 4;             // of the rows in which warps leave their sums: no bank twice
template <int D> constexpr int kStage = 2 * kKeys * (D / 2) + 2 * kKeys * 16;        // bytes: codes of keys and values, steps of both, 16 bytes a key
template <int D> constexpr int kSums = kWarps * 8 * kPitch<D> * 4;
// a cluster's sums lie over the ring, which has been read by then; otherwise the ring runs on while sums are written
template <int D, int R, bool CLUSTER> constexpr int rows_smem = CLUSTER ? std::max(kWarps * kStages * kStage<D>, kSums<D> + 8 * R * D * 4)
                                                                        : kWarps * kStages * kStage<D> + kSums<D>;

template <int BYTES> NXD_DEVICE void cp_async(uint32_t dst, const void* src, bool live) {      // not live: zero bytes, nothing is read
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(live ? BYTES : 0), "n"(BYTES) : "memory");
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
// 16-byte chunk c of row r of a tile of codes lies at chunk c ^ (…): ldmatrix meets no bank twice
template <int D> NXD_DEVICE uint32_t chunk_at(int r, int c) { return r * (D / 2) + ((c ^ (D == 128 ? (r >> 1) & 3 : (r >> 2) & 1)) << 4); }

// Scores Sᵀ = K Qᵀ and sums Oᵀ += Vᵀ Pᵀ by mma.sync of half precision, with the keys, then the head's numbers, as the 16 rows of the instruction and 8 R
// query rows as its columns; a warp walks 16-key tiles of its own through its own ring of cp.async stages, which runs ahead over the ends of pairs.
//
// Codes enter the products as they lie: four bits at the bottom of a half are the denormal c 2^-24, one place up 16 times that, so a mask makes two numbers
// ready, and what is over is put right in the queries, or in the sums when they leave.  With c of group g, steps s and m (both exact):
//   q . k = sum_g s_g (q_g . c_g) + sum_g m_g (sum of q_g)       the second a product of its own, with the sums of q as two halves each
//   o     = sum_j (p_j s_jg) c_j  + sum_j p_j m_jg               the weights times s of 16 keys as operands; the second again a product of its own
// Queries are multiplied by a power of two that brings the row's largest to 2^14.  Weights p are relative to a reference M, at most 2^15 and with s at
// most 2^15 (`room` below), so that they are halves of all their bits: 11 of each product's.  Where the output is in half precision too, weights
// are two halves, the rounded one and what that left (22 bits).
// TWO: so for T = half.
template <typename T, int D, int R, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, R == 1 ? 4 : 2) int4_rows_kernel(const Int4Attn p) {
  constexpr bool TWO = sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value;
  constexpr int NG = D / 32, CH = D / 32, PITCH = kPitch<D>, STAGE = kStage<D>;
  constexpr int V_AT = kKeys * (D / 2), KS_AT = 2 * V_AT, VS_AT = KS_AT + kKeys * 16;
  constexpr uint32_t LOW = 0x000f000fu, HIGH = 0x00f000f0u;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sm_m[kWarps][8 * R], sm_l[kWarps][8 * R], sm_bm[8 * R], sm_bl[8 * R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hq = lane >> 2, quad = lane & 3;
  pdl_wait();
  pdl_trigger();                                           // the last launch's blocks may take their places; they wait for this grid
  // keys that some row of an entry sees
  auto keys_of = [&](int e) {
    if (e >= p.B * p.row_tiles) return 0;
    const int b = e / p.row_tiles, row0 = e % p.row_tiles * p.tile_rows, m = new_tokens(p, b);
    return row0 / p.G < m ? visible_keys(p, b, min(m, (row0 + p.tile_rows + p.G - 1) / p.G) - 1) : 0;
  };
  // Pages of this warp's keys in 32 tiles of a pair from tile t0 on, one a lane: -1 where there is none
  const int step = CLUSTER ? p.cluster : 1;
  auto fetch_pages = [&](int e, int t0) {
    const unsigned i = ((unsigned)(t0 + lane * step) * kTileKeys + warp * kKeys) / (unsigned)p.ps;
    if (i >= (unsigned)p.cols) return -1;
    const int page = i < (unsigned)p.shared_cols ? p.shared_pages[i] : p.table[e / p.row_tiles * p.table_sb + i];
    return (unsigned)page < (unsigned)p.pages ? page : -1;
  };
  struct { Walk w; int n; } cur;
  long left = 0;                                           // tiles of this block
  int pages = -1, next_page = 0;
  if constexpr (CLUSTER) {
    const int pair = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster;
    pages = fetch_pages(pair / p.Hkv, rank);               // beside the positions: it needs none of them
    cur.w = Walk{pair / p.Hkv, pair % p.Hkv, rank, entry_tiles(p, pair / p.Hkv)};
    cur.n = keys_of(cur.w.e);
    left = cur.w.tiles > rank ? (cur.w.tiles - rank + step - 1) / step : 0;
  } else {
    const Place at = find_place<kThreads, false>(p, gridDim.x, blockIdx.x);
    left = min(at.per, at.total - blockIdx.x * at.per);
    if (left > 0) {
      cur.w.e = at.e;
      cur.w.tiles = entry_tiles(p, at.e);
      cur.w.head = (int)(at.tile / cur.w.tiles);
      cur.w.tile = (int)(at.tile % cur.w.tiles);
      pages = fetch_pages(at.e, cur.w.tile);
      cur.n = keys_of(at.e);
    }
  }
  const uint8_t* const kc = reinterpret_cast<const uint8_t*>(p.k);
  const uint8_t* const vc = reinterpret_cast<const uint8_t*>(p.v);
  const uint16_t* const ksc = reinterpret_cast<const uint16_t*>(p.ks);
  const uint16_t* const vsc = reinterpret_cast<const uint16_t*>(p.vs);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (kStages * STAGE);
  // sums of the warps [warp][8 rows][PITCH] and of a cluster's block [8 R][D]
  float* const sm_o = reinterpret_cast<float*>(smem + (CLUSTER ? 0 : kWarps * kStages * STAGE));
  float* const sm_b = reinterpret_cast<float*>(smem + kSums<D>);

  auto load_tile = [&](const Walk& c, int n, int page, int stage) {
    constexpr int PASS = 32 / CH;
    const int key = c.tile * kTileKeys + warp * kKeys, row0 = key % p.ps, cc = lane % CH;
    const long at = page < 0 ? 0 : page;
    const uint8_t* kb = kc + at * p.k_sp + c.head * p.k_sh + cc * 16;
    const uint8_t* vb = vc + at * p.v_sp + c.head * p.v_sh + cc * 16;
    const uint32_t dst = ring + stage * STAGE;
#pragma unroll
    for (int i = 0; i < kKeys / PASS; ++i) {
      const int r = i * PASS + lane / CH;
      const bool live = page >= 0 && key + r < n;
      cp_async<16>(dst + chunk_at<D>(r, cc), kb + (row0 + r) * p.k_sr, live);
      cp_async<16>(dst + V_AT + chunk_at<D>(r, cc), vb + (row0 + r) * p.v_sr, live);
    }
    const int r = lane & 15;                               // steps: half a warp has the keys', half the values'
    const uint16_t* sb = lane < 16 ? ksc + at * p.ks_sp + c.head * p.ks_sh + (row0 + r) * p.ks_sr : vsc + at * p.vs_sp + c.head * p.vs_sh + (row0 + r) * p.vs_sr;
    cp_async<NG * 4>(dst + KS_AT + lane * 16, sb, page >= 0 && key + r < n);
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
        if (!CLUSTER && ahead.w.tile == ahead.w.tiles) {
          next_pair<false>(p, ahead.w);
          if (ahead.w.head == 0) ahead.n = keys_of(ahead.w.e);
          next_page = 32;
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) ask(s);

  uint32_t qf[R][NG][4], qs[R];                            // queries of group g: two steps of 16 numbers; sums of queries
  float m[R][2], l[R][2], o[R][2 * NG][4], om[R][4], unit[R][2];
  int lim[R][2], lim_all = 0;                              // first key that a row does not see; that none of the live rows has before it
  float room = 15.f;                                       // weights relative to M may be at most 2^room: 15 less what the largest s needs
  float s_most = 1.f;                                      // 2^(15 - room)
  bool whole = false;                                      // the pair begins in this block
  int row0 = 0, rows = 0;                                  // of the entry
  auto begin = [&]() {
    const int kvh = cur.w.head, b = cur.w.e / p.row_tiles, count = new_tokens(p, b);
    row0 = cur.w.e % p.row_tiles * p.tile_rows;
    rows = min(8 * R, p.W * p.G - row0);
    whole = CLUSTER || cur.w.tile == 0;
    lim_all = min(visible_keys(p, b, row0 / p.G), cur.n);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int row = i * 8 + hq, w = (row0 + row) / p.G;
      const bool live = row < rows && w < count;
      const T* const qp = reinterpret_cast<const T*>(p.q) + (live ? b * p.q_sb + w * p.q_sw + (long)(kvh * p.G + (row0 + row) % p.G) * p.q_sh : 0) + quad * 8;
      uint4 raw[NG];
      float most = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        raw[g] = live ? *reinterpret_cast<const uint4*>(qp + g * 32) : make_uint4(0, 0, 0, 0);
        const uint32_t u[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float lo, hi;
          unpack16<T>(u[x], lo, hi);
          most = fmaxf(most, fmaxf(fabsf(lo), fabsf(hi)));
        }
      }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int e = min(max((int)(__float_as_uint(most) >> 23), 20), 244);
      const float up = __uint_as_float((uint32_t)(268 - e) << 23);                       // the largest to 2^14 … 2^15
      const float down = __uint_as_float((uint32_t)(e + 10) << 23) * p.scale_log2;             // 2^24 / up: codes are 2^-24 of themselves
      float sums[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float x[8];
        const uint32_t u[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
        sums[g] = 0.f;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          unpack16<T>(u[y], x[2 * y], x[2 * y + 1]);
          x[2 * y] *= up;
          x[2 * y + 1] *= up;
          sums[g] += x[2 * y] + x[2 * y + 1];
        }
        qf[i][g][0] = pack_half(x[0], x[4]);
        qf[i][g][1] = pack_half(x[1] * 0.0625f, x[5] * 0.0625f);
        qf[i][g][2] = pack_half(x[2], x[6]);
        qf[i][g][3] = pack_half(x[3] * 0.0625f, x[7] * 0.0625f);
        sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
        sums[g] = (sums[g] + __shfl_xor_sync(0xffffffffu, sums[g], 2)) * 0.03125f;         // below 2^15
      }
      // columns 2 quad, 2 quad + 1 of the product with m: its halves of groups (2 quad, 2 quad + 1) % NG, first the rounded ones, then what that left
      const int pair = NG == 4 ? quad & 1 : 0, part = NG == 4 ? quad >> 1 : quad;
      const float a = pair ? sums[NG - 2] : sums[0], c = pair ? sums[NG - 1] : sums[1];
      const __half ah = __float2half_rn(a), ch = __float2half_rn(c);
      qs[i] = part == 0 ? as_u32(__halves2half2(ah, ch)) : part == 1 ? pack_half(a - __half2float(ah), c - __half2float(ch)) : 0u;
#pragma unroll
      for (int k = 0; k < 2 * NG; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][k][x] = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) om[i][x] = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = i * 8 + quad * 2 + x, w2 = (row0 + r) / p.G;
        unit[i][x] = __shfl_sync(0xffffffffu, down, (quad * 2 + x) * 4);
        lim[i][x] = r < rows && w2 < count ? min(visible_keys(p, b, w2), cur.n) : 0;
        m[i][x] = kNone;
        l[i][x] = 0.f;
      }
    }
  };

  // the four warps' sums of the pair, to the output or to a part
  auto finish = [&](bool last) {
    const int kvh = cur.w.head, b = cur.w.e / p.row_tiles, count = new_tokens(p, b);
    const bool direct = whole && last;
    if (CLUSTER) __syncthreads();                          // all of the ring has been read
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
      for (int g = 0; g < NG; ++g) {
        // what m adds to group g stands in row NG + g of its product
        const float m0 = __shfl_sync(0xffffffffu, om[i][0], (NG + g) * 4 + quad), m1 = __shfl_sync(0xffffffffu, om[i][1], (NG + g) * 4 + quad);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sm_o[(warp * 8 + quad * 2 + (e & 1)) * PITCH + g * 32 + hq * 4 + k * 2 + (e >> 1)] = fmaf(o[i][2 * g + k][e], e >> 1 ? 0x1p20f : 0x1p24f, e & 1 ? m1 : m0);
      }
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
        if (CLUSTER && p.cluster > 1) {
          sm_b[row * D + col] = acc;
          if (col == 0) { sm_bm[row] = mn; sm_bl[row] = ls; }
        } else if (direct) {
          const int w = (row0 + row) / p.G;
          const bool live = w < count && !(ls == 0.f);
          reinterpret_cast<T*>(p.out)[b * p.o_sb + w * p.o_sw + (long)(kvh * p.G + (row0 + row) % p.G) * p.o_sh + col] = from_f32<T>(live ? acc / ls : 0.f);
        } else {
          const long slot = part_slot<false>(p, (long)cur.w.e * p.Hkv + kvh, blockIdx.x, whole) * p.tile_rows + row;
          p.part_o[slot * D + col] = acc;
          if (col == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(mn, ls);
        }
      }
    }
    __syncthreads();                                       // the sums have been read
  };

  if (CLUSTER || left > 0) begin();
  for (long t = 0; t < left; ++t) {
    const int stage = (int)(t % kStages);
    cp_async_wait<kStages - 2>();
    __syncwarp();                                          // tile t of all lanes is there; all lanes are done with tile t - 1
    const bool hole = holes >> stage & 1;
    ask((int)((t + kStages - 1) % kStages));
    const int key = cur.w.tile * kTileKeys + warp * kKeys;
    if (!hole) {
      const uint32_t at = ring + stage * STAGE;
      // scores: keys hq and hq + 8, rows 2 quad and 2 quad + 1
      float s[R][4];
      const uint32_t km = at + KS_AT + hq * 16 + NG * 2 + (NG == 4 ? (quad & 1) * 4 : 0);
      const uint32_t m0 = lds32(km), m1 = lds32(km + 8 * 16);
#pragma unroll
      for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
        mma1688(s[i], m0, m1, qs[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] *= 0x1p-19f;   // sums of q were divided by 2^5, codes by 2^24
      }
      float ks0[NG], ks1[NG];
      {
        const uint2 a = lds64(at + KS_AT + hq * 16), b = lds64(at + KS_AT + (hq + 8) * 16);
        const uint32_t u[2] = {a.x, a.y}, v[2] = {b.x, b.y};
#pragma unroll
        for (int g = 0; g < NG; g += 2) {
          const float2 x = __half22float2(as_half2(u[g / 2])), y = __half22float2(as_half2(v[g / 2]));
          ks0[g] = x.x; ks0[g + 1] = x.y;
          ks1[g] = y.x; ks1[g + 1] = y.y;
        }
      }
      const int rr = (((lane >> 3) & 1) << 3) + (lane & 7), rc = lane >> 4;
#pragma unroll
      for (int g = 0; g < NG; g += 2) {
        uint32_t a[4];                                     // keys hq, hq + 8 of group g, of group g + 1: eight codes each
        ldmatrix_x4(a, at + chunk_at<D>(rr, g + rc));
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t k0 = a[2 * x], k1 = a[2 * x + 1], k2 = k0 >> 8, k3 = k1 >> 8;
#pragma unroll
          for (int i = 0; i < R; ++i) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816(d, k0 & LOW, k1 & LOW, k0 & HIGH, k1 & HIGH, qf[i][g + x][0], qf[i][g + x][1]);
            mma16816(d, k2 & LOW, k3 & LOW, k2 & HIGH, k3 & HIGH, qf[i][g + x][2], qf[i][g + x][3]);
            s[i][0] = fmaf(d[0], ks0[g + x], s[i][0]);
            s[i][1] = fmaf(d[1], ks0[g + x], s[i][1]);
            s[i][2] = fmaf(d[2], ks1[g + x], s[i][2]);
            s[i][3] = fmaf(d[3], ks1[g + x], s[i][3]);
          }
        }
      }
      // steps of the values of keys 2 quad, 2 quad + 1, and of those + 8, two of one group beside one another
      uint32_t vs[NG][2];
      float s_max = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint2 a = lds64(at + VS_AT + (2 * quad + 8 * x) * 16), b = lds64(at + VS_AT + (2 * quad + 1 + 8 * x) * 16);
        const uint32_t u[2] = {a.x, a.y}, v[2] = {b.x, b.y};
#pragma unroll
        for (int g = 0; g < NG; ++g) vs[g][x] = __byte_perm(u[g / 2], v[g / 2], g & 1 ? 0x7632 : 0x5410);
      }
      {
        __half2 x = __hmax2(as_half2(vs[0][0]), as_half2(vs[0][1]));
#pragma unroll
        for (int g = 1; g < NG; ++g) x = __hmax2(x, __hmax2(as_half2(vs[g][0]), as_half2(vs[g][1])));
        const float2 f = __half22float2(x);
        s_max = fmaxf(f.x, f.y);
      }
      const bool masked = key + kKeys > lim_all;
      uint32_t ph[R][2], pl[R][2];
      bool passed = s_max > s_most;
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] *= unit[i][e & 1];
          if (masked && key + hq + (e >> 1) * 8 >= lim[i][e & 1]) s[i][e] = -INFINITY;
          passed = passed || s[i][e] - m[i][e & 1] > room;
        }
      // a weight, or a weight times s, would pass 2^15: another reference, 2^3 away from that
      if (__any_sync(0xffffffffu, passed)) {
        const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(s_max));
        if (__uint_as_float(most) > s_most) {
          const int e = min((int)(most >> 23) - 127 + 1, 16);
          s_most = __uint_as_float((uint32_t)(e + 127) << 23);
          room = 15.f - e;
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(s[i][e], s[i][e + 2]);
#pragma unroll
            for (int y = 4; y < 32; y <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, y));
            const float mn = fmaxf(m[i][e], mx - (room - 3.f)), f = exp2f(m[i][e] - mn);      // none before: 0
            m[i][e] = mn;
            l[i][e] *= f;
            om[i][e] *= f;
            om[i][e + 2] *= f;
#pragma unroll
            for (int k = 0; k < 2 * NG; ++k) { o[i][k][e] *= f; o[i][k][e + 2] *= f; }
          }
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float pr[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pr[e] = exp2f(s[i][e] - m[i][e & 1]);
          l[i][e & 1] += pr[e];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t hi = pack_half(pr[2 * e], pr[2 * e + 1]);
          ph[i][e] = transpose8x8(hi);
          if constexpr (TWO) {
            const float2 f = __half22float2(as_half2(hi));
            pl[i][e] = transpose8x8(pack_half(pr[2 * e] - f.x, pr[2 * e + 1] - f.y));
          }
        }
      }
      {
        uint32_t a[2];                                     // row x of the product: the x-th number of the steps, s of all groups, then m
        ldmatrix_x2t(a, at + VS_AT + (lane & 15) * 16);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          mma16816(om[i], a[0], 0u, a[1], 0u, ph[i][0], ph[i][1]);
          if constexpr (TWO) mma16816(om[i], a[0], 0u, a[1], 0u, pl[i][0], pl[i][1]);
        }
      }
#pragma unroll
      for (int g = 0; g < NG; g += 2) {
        uint32_t a[4];                                     // keys 2 quad.. and 8 + 2 quad.. of group g, of group g + 1: four codes of either key
        ldmatrix_x4t(a, at + V_AT + chunk_at<D>(rr, g + rc));
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t v0 = a[2 * x], v1 = a[2 * x + 1], v2 = v0 >> 8, v3 = v1 >> 8;
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const __half2 s0 = as_half2(vs[g + x][0]), s1 = as_half2(vs[g + x][1]);
            const __half2 w0 = __hmul2(as_half2(ph[i][0]), s0), w1 = __hmul2(as_half2(ph[i][1]), s1);
            mma16816(o[i][2 * (g + x)], v0 & LOW, v0 & HIGH, v1 & LOW, v1 & HIGH, as_u32(w0), as_u32(w1));
            mma16816(o[i][2 * (g + x) + 1], v2 & LOW, v2 & HIGH, v3 & LOW, v3 & HIGH, as_u32(w0), as_u32(w1));
            if constexpr (TWO) {
              const __half2 y0 = __hfma2(as_half2(pl[i][0]), s0, __hfma2(as_half2(ph[i][0]), s0, __hneg2(w0)));
              const __half2 y1 = __hfma2(as_half2(pl[i][1]), s1, __hfma2(as_half2(ph[i][1]), s1, __hneg2(w1)));
              mma16816(o[i][2 * (g + x)], v0 & LOW, v0 & HIGH, v1 & LOW, v1 & HIGH, as_u32(y0), as_u32(y1));
              mma16816(o[i][2 * (g + x) + 1], v2 & LOW, v2 & HIGH, v3 & LOW, v3 & HIGH, as_u32(y0), as_u32(y1));
            }
          }
        }
      }
    }
    const bool end = cur.w.tile + 1 == cur.w.tiles;
    if (!CLUSTER && (end || t + 1 == left)) {
      finish(end);
      if (t + 1 < left) {
        next_pair<false>(p, cur.w);
        if (cur.w.head == 0) cur.n = keys_of(cur.w.e);
        begin();
      }
    } else {
      cur.w.tile += step;
    }
  }
  if constexpr (CLUSTER) {
    finish(true);
    if (p.cluster > 1) {
      cluster_sync_all();
      constexpr int PER = kThreads / D;
      const int rank = blockIdx.x % p.cluster, col = threadIdx.x % D, b = cur.w.e / p.row_tiles, count = new_tokens(p, b);
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
        const int w = (row0 + row) / p.G;
        const bool live = w < count && !(ls == 0.f);
        reinterpret_cast<T*>(p.out)[b * p.o_sb + w * p.o_sw + (long)(cur.w.head * p.G + (row0 + row) % p.G) * p.o_sh + col] = from_f32<T>(live ? acc / ls : 0.f);
      }
      cluster_sync_all();                                  // nobody reads a block's sums any more
    }
  } else {
    finish_idle<T, D, kThreads>(p, threadIdx.x);
  }
}

template <typename T, int D, int R, bool CLUSTER>
void launch_rows(const Int4Attn& p, int grid, cudaStream_t st) {
  constexpr int smem = rows_smem<D, R, CLUSTER>;
  NXD_ALLOW_SMEM((int4_rows_kernel<T, D, R, CLUSTER>), smem);
  if (!CLUSTER || p.cluster == 1) return launch_dependent(int4_rows_kernel<T, D, R, CLUSTER>, grid, kThreads, smem, st, p);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid; cfg.blockDim = kThreads; cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 2;
  NXD_CUDA_CHECK(cudaLaunchKernelEx(&cfg, int4_rows_kernel<T, D, R, CLUSTER>, p));
}
template <typename T, int D>
int launch(const Int4Attn& p, const PagedPlan& plan, cudaStream_t st) {
  if (p.cluster && p.tile_rows == 8) launch_rows<T, D, 1, true>(p, plan.grid, st);
  else if (p.cluster) launch_rows<T, D, 2, true>(p, plan.grid, st);
  else if (p.tile_rows == 8) launch_rows<T, D, 1, false>(p, plan.grid, st);
  else launch_rows<T, D, 2, false>(p, plan.grid, st);
  if (p.cluster || plan.grid <= 1) return 1;
  const int rows = std::min(p.tile_rows, p.W * p.G);
  launch_dependent(paged_merge_kernel<T, D, 1>, dim3(plan.grid - 1, (rows + kWarps - 1) / kWarps), kThreads, 0, st, static_cast<const PagedAttn&>(p), plan.grid);
  return 2;
}

}  // namespace

PagedPlan int4_plan(Int4Attn& p) {
  PagedPlan plan{};
  const int sms = device_sm_count();
  const long rows = (long)p.W * p.G;
  p.tile_rows = rows <= 8 ? 8 : 16;
  p.row_tiles = (int)((rows + p.tile_rows - 1) / p.tile_rows);
  p.tile_keys = kTileKeys;
  p.min_tiles = 256 / kTileKeys;
  p.whole_tiles = 0;
  p.shared = 0;
  const int each = p.tile_rows == 8 ? 4 : 2;               // blocks of an SM
  const long pairs = (long)p.B * p.row_tiles * p.Hkv, cap = (long)p.cols * p.ps;
  plan.grid = each * sms;
  int size = 1;
  while (size < kCluster8 && ((cap > 256l * size && pairs * size * 2 <= (long)each * sms) || cap > 4096l * size)) size *= 2;
  if (cap <= 4096l * size && pairs * size < (1l << 30)) {
    p.cluster = size;
    plan.grid = (int)(pairs * size);
  }
  plan.slots = p.cluster ? 0l : 2l * plan.grid * p.tile_rows;
  p.slots = plan.slots;
  return plan;
}

int int4_attention(const Int4Attn& p, const PagedPlan& plan, int D, int dt, cudaStream_t st) {
  if (dt == kBF16) return D == 128 ? launch<__nv_bfloat16, 128>(p, plan, st) : launch<__nv_bfloat16, 64>(p, plan, st);
  return D == 128 ? launch<__half, 128>(p, plan, st) : launch<__half, 64>(p, plan, st);
}

void int4_append(Int4Append p, int dt, cudaStream_t st) {
  const long tokens = (long)p.B * p.W, items = (long)(p.H + 2 * p.Hkv) * (p.D / 8);
  p.parts = (int)((items + kAppendThreads - 1) / kAppendThreads);
  if (tokens == 0) return;
  if (tokens * p.parts >= (1l << 31)) nxd_throw("int4_append: too many tokens", __FILE__, __LINE__);
  const unsigned grid = (unsigned)(tokens * p.parts);
  if (dt == kBF16) launch_dependent(int4_append_kernel<__nv_bfloat16>, grid, kAppendThreads, 0, st, p);
  else if (dt == kF16) launch_dependent(int4_append_kernel<__half>, grid, kAppendThreads, 0, st, p);
  else launch_dependent(int4_append_kernel<float>, grid, kAppendThreads, 0, st, p);
}

void int4_gather(const Int4Pages& kp, const Int4Pages& vp, const int* slots, void* k, void* v, long n, int Hkv, int D, int ps, long tokens, int dt, cudaStream_t st) {
  const long items = n * Hkv * (D / 8), blocks = (items + kGatherThreads - 1) / kGatherThreads;
  if (items == 0) return;
  if (blocks >= (1l << 31)) nxd_throw("int4_gather: too many tokens", __FILE__, __LINE__);
  const dim3 grid((unsigned)blocks, 2);
  auto go = [&](auto* k, auto* v, auto kernel) { launch_dependent(kernel, grid, kGatherThreads, 0, st, kp, vp, slots, k, v, items, Hkv, D, ps, tokens); };
  if (dt == kBF16) go((__nv_bfloat16*)k, (__nv_bfloat16*)v, int4_gather_kernel<__nv_bfloat16>);
  else if (dt == kF16) go((__half*)k, (__half*)v, int4_gather_kernel<__half>);
  else go((float*)k, (float*)v, int4_gather_kernel<float>);
}

}  // namespace nxd
