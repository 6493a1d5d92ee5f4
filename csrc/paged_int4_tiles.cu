// Attention of nine and more query rows of a (sequence, key/value head) over a cache in pages of 4 bits.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged_int4.cuh"

namespace nxd {
namespace {

using namespace int4;

constexpr int kTileWarps = 8, kTileThreads = kTileWarps * 32;
constexpr int kTileKeys = kTileWarps * kKeys;
constexpr float kRoom = 15.f;                              // weights are at most 2^15: halves
constexpr int kWeightPitch = kTileKeys * 2 + 16;           // bytes of a row of weights: ldmatrix and stmatrix meet no bank twice
// Where the output is in half precision too, weights are two halves, the rounded one and what that left; with 40 rows there is room for two stages then
template <typename T> constexpr int kHalves = std::is_same<T, __half>::value ? 2 : 1;
template <typename T, int R> constexpr int kTileStages = kHalves<T> == 2 && R == 5 ? 2 : 3;
template <typename T, int D, int R> constexpr int kRing = kTileWarps * kTileStages<T, R> * kStage<D>;
template <int D> constexpr int kParts = kTileWarps / (D / 32);                         // warps that have the same 32 columns of the sums, for other keys
// two tiles' weights; at a pair's end the sums of all parts but the first lie over them
template <typename T, int D, int R> constexpr int kWeights = 8 * R * std::max(2 * kHalves<T> * kWeightPitch, (kParts<D> - 1) * kPitch<D> * 4);
// a cluster's sums lie over the ring, which has been read by then
template <typename T, int D, int R> constexpr int tiles_smem = kQueries<D, R> + kWeights<T, D, R> + std::max(kRing<T, D, R>, 8 * R * D * 4);

// Scores Sᵀ = K Qᵀ and sums Oᵀ += Vᵀ Pᵀ by mma.sync of half precision, with the keys, then the head's numbers, as the 16 rows of the instruction and query rows
// as its columns, 8 R of them in a row tile.  A block walks tiles of 128 keys: in the first product each of its eight warps has 16 keys, in the second 32 columns of the
// sums (a group of the steps) for half of the keys (heads of 64: a quarter), so that no code is made a number twice; weights go from the one to the other
// through shared memory, with one barrier a tile.  Each warp asks for its own 16 keys by cp.async, two tiles ahead, over the ends of pairs.
//
// Codes enter the first product as they lie: four bits at the bottom of a half are the denormal c 2^-24, one place up 16 times that, so a mask makes two
// numbers ready, and what is over is put right in the queries.  With c of group g, steps s and m (all exact, the sums of q as two halves each):
//   q . k = sum_g s_g (q_g . c_g) + sum_g m_g (sum of q_g)       the second a product of its own
// Queries are multiplied by a power of two that brings the row's largest to 2^14.  For the second product values are made half their size, c / 2 s + m / 2 rounded once
// to half precision (2^-11 of them; half, so that none is too large), and meet weights rounded to halves: relative to a reference of the row, at most 2^15
// below which they have all their bits down to 2^-29 of it.
//
// Bound by the products, which hold the tensor pipe for 8 cycles each, and by what feeds them from shared memory: with 40 rows 3600 cycles an SM for 128 keys, 4350 with weights in two
// halves (windows of 5 tokens, 64 heads on 8, 8 sequences to 6000 keys: 58 us in bf16, 67 in half precision).
template <typename T, int D, int R, bool CLUSTER>
__global__ void __launch_bounds__(kTileThreads, 2) int4_tiles_kernel(const Int4Attn p) {
  constexpr int NG = D / 32, PITCH = kPitch<D>, STAGES = kTileStages<T, R>, HALVES = kHalves<T>, STAGE = kStage<D>, PARTS = kParts<D>;
  constexpr int V_AT = kKeys * (D / 2), KS_AT = 2 * V_AT, VS_AT = KS_AT + kKeys * 16;
  constexpr uint32_t LOW = 0x000f000fu, HIGH = 0x00f000f0u;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sm_l[kTileWarps][8 * R], sm_top[kTileWarps][8 * R], sm_bm[8 * R], sm_bl[8 * R];
  __shared__ Walk sm_ahead[kTileWarps];
  __shared__ Share sm_share;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hq = lane >> 2, quad = lane & 3;
  pdl_wait();
  pdl_trigger();                                           // the last launch's blocks may take their places; they wait for this grid
  const int step = CLUSTER ? p.cluster : 1;
  int tiles_left = 0;                                      // tiles of this block
  Walk cur{};                                              // the pair in work
  if constexpr (CLUSTER) {
    const int pair = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster;
    cur = Walk{pair / p.Hkv, pair % p.Hkv, rank, entry_tiles(p, pair / p.Hkv)};
    tiles_left = cur.tiles > rank ? (cur.tiles - rank + step - 1) / step : 0;
  } else {
    if (warp == 0) {
      const Share s = find_share(p, gridDim.x, blockIdx.x, lane);
      if (lane == 0) sm_share = s;
    }
    __syncthreads();
    const Share s = sm_share;
    tiles_left = s.tiles;
    if (tiles_left > 0) {
      cur.e = s.e;
      cur.tiles = entry_tiles(p, s.e);
      cur.head = s.tile / cur.tiles;
      cur.tile = s.tile % cur.tiles;
    }
  }
  const uint32_t sm_q = (uint32_t)__cvta_generic_to_shared(smem), sm_qs = sm_q + 8 * R * kQPitch<D>, sm_p = sm_q + kQueries<D, R>;
  float* const sm_unit = reinterpret_cast<float*>(smem + 8 * R * (kQPitch<D> + 16));
  int* const sm_lim = reinterpret_cast<int*>(sm_unit + 8 * R);
  float* const sm_o = reinterpret_cast<float*>(smem + kQueries<D, R>);          // sums of all parts but the first [part - 1][8 R][PITCH]
  float* const sm_b = reinterpret_cast<float*>(smem + kQueries<D, R> + kWeights<T, D, R>);        // a cluster's: the block's sums [8 R][D]
  const uint32_t ring0 = sm_p + kWeights<T, D, R>;
  Ring<D, kTileWarps, CLUSTER> ring(p, sm_ahead + warp, cur, tiles_left, step, ring0 + warp * (STAGES * STAGE), warp, lane);
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) ring.ask(s);

  // this warp's columns of the sums, and which keys it has for them; number k of a lane's four columns is 32 group + 4 hq + k
  const int group = warp % NG, part = warp / NG;
  float m[R][2], l[R][2], o[R][2][4];
  uint32_t qs[R];                                          // sums of queries
  int lim_all = 0;                                         // first key that some live row does not see
  bool whole = false;                                      // the pair begins in this block
  int row0 = 0, rows = 0;                                  // of the entry
  auto begin = [&] {
    const int b = cur.e / p.row_tiles, count = new_tokens(p, b), n = keys_of(p, cur.e);
    row0 = cur.e % p.row_tiles * p.tile_rows;
    rows = min(8 * R, p.W * p.G - row0);
    whole = CLUSTER || cur.tile == 0;
    lim_all = min(visible_keys(p, b, row0 / p.G), n);
    for (int r = warp; r < 8 * R; r += kTileWarps) {
      const int w = (row0 + r) / p.G;
      const bool live = r < rows && w < count;
      ready_query<T, D>(reinterpret_cast<const T*>(p.q) + (live ? b * p.q_sb + w * p.q_sw + (long)(cur.head * p.G + (row0 + r) % p.G) * p.q_sh : 0), live,
                        sm_q + r * kQPitch<D>, sm_qs + r * 16, sm_unit + r, p.scale_log2, lane);
      if (lane == 0) sm_lim[r] = live ? min(visible_keys(p, b, w), n) : 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R; ++i) {
      qs[i] = lds32(sm_qs + (i * 8 + hq) * 16 + quad * 4);
#pragma unroll
      for (int x = 0; x < 4; ++x) o[i][0][x] = o[i][1][x] = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        m[i][x] = kNone;
        l[i][x] = 0.f;
      }
    }
  };

  // the block's sums of the pair, to the output or to a part
  auto finish = [&](bool last) {
    const int kvh = cur.head, b = cur.e / p.row_tiles, count = new_tokens(p, b);
    const bool direct = whole && last;
    __syncthreads();                                       // nobody reads weights any more
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], s);
        if (hq == 0) sm_l[warp][i * 8 + quad * 2 + e] = l[i][e];
        if (part > 0)
          *reinterpret_cast<float4*>(sm_o + ((part - 1) * 8 * R + i * 8 + quad * 2 + e) * PITCH + group * 32 + hq * 4) =
              make_float4(o[i][0][e], o[i][0][e + 2], o[i][1][e], o[i][1][e + 2]);
      }
    __syncthreads();                                       // and all of the ring has been read (a cluster's)
    if (part > 0) return;
    const long slot = part_slot<false>(p, (long)cur.e * p.Hkv + kvh, blockIdx.x, whole) * p.tile_rows;
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = i * 8 + quad * 2 + e, col = group * 32 + hq * 4;
        if (row >= rows) continue;
        float4 x = make_float4(o[i][0][e], o[i][0][e + 2], o[i][1][e], o[i][1][e + 2]);
#pragma unroll
        for (int k = 0; k < PARTS - 1; ++k) {
          const float4 y = *reinterpret_cast<const float4*>(sm_o + (k * 8 * R + row) * PITCH + col);
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        float ls = 0.f;
#pragma unroll
        for (int w = 0; w < kTileWarps; ++w) ls += sm_l[w][row];
        const float top = m[i][e] == kNone ? -INFINITY : m[i][e];
        if (CLUSTER && p.cluster > 1) {
          *reinterpret_cast<float4*>(sm_b + row * D + col) = x;
          if (col == 0) { sm_bm[row] = top; sm_bl[row] = ls; }
        } else if (direct) {
          const int w = (row0 + row) / p.G;
          const float inv = w < count && !(ls == 0.f) ? 2.f / ls : 0.f;                    // values were halved
          const bool none = w >= count || ls == 0.f;
          *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + b * p.o_sb + w * p.o_sw + (long)(kvh * p.G + (row0 + row) % p.G) * p.o_sh + col) =
              none ? make_uint2(0, 0) : make_uint2(pack16<T>(x.x * inv, x.y * inv), pack16<T>(x.z * inv, x.w * inv));
        } else {
          *reinterpret_cast<float4*>(p.part_o + (slot + row) * D + col) = x;
          if (col == 0) *reinterpret_cast<float2*>(p.part_ml + (slot + row) * 2) = make_float2(top, ls);
        }
      }
  };

  if (CLUSTER || tiles_left > 0) begin();
  int stage = 0, ask_stage = STAGES - 1;
  for (int t = 0; t < tiles_left; ++t) {
    cp_async_wait<STAGES - 2>();
    __syncwarp();                                          // tile t of all lanes is there
    const uint32_t at = ring.ring + stage * STAGE, weights = sm_p + (t & 1) * (8 * R * HALVES * kWeightPitch);
    // scores: keys hq and hq + 8, rows 2 quad and 2 quad + 1
    float s[R][4];
    {
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
      const uint2 a0 = lds64(at + KS_AT + hq * 16), b0 = lds64(at + KS_AT + (hq + 8) * 16);
      const uint32_t ua[2] = {a0.x, a0.y}, ub[2] = {b0.x, b0.y};
#pragma unroll
      for (int g = 0; g < NG; g += 2) {
        const float2 k0s = __half22float2(as_half2(ua[g / 2])), k1s = __half22float2(as_half2(ub[g / 2]));
        uint32_t a[4];                                     // keys hq, hq + 8 of group g, of group g + 1: eight codes each
        ldmatrix_x4(a, at + chunk_at<D>((((lane >> 3) & 1) << 3) + (lane & 7), g + (lane >> 4)));
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const Codes k0 = codes_of(a[2 * x]), k1 = codes_of(a[2 * x + 1]);
          const float f0 = x ? k0s.y : k0s.x, f1 = x ? k1s.y : k1s.x;
#pragma unroll
          for (int i = 0; i < R; ++i) {
            uint32_t q[4];
            ldmatrix_x4(q, sm_q + (i * 8 + (lane & 7)) * kQPitch<D> + (g + x) * 64 + (lane >> 3) * 16);
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816(d, k0.c0, k1.c0, k0.c1, k1.c1, q[0], q[1]);
            mma16816(d, k0.c2, k1.c2, k0.c3, k1.c3, q[2], q[3]);
            s[i][0] = fmaf(d[0], f0, s[i][0]);
            s[i][1] = fmaf(d[1], f0, s[i][1]);
            s[i][2] = fmaf(d[2], f1, s[i][2]);
            s[i][3] = fmaf(d[3], f1, s[i][3]);
          }
        }
      }
    }
    const int key = cur.tile * kTileKeys + warp * kKeys;
    const bool hole = ring.template hole<STAGES>();
    if (hole || key + kKeys > lim_all) {
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (hole || key + hq + (e >> 1) * 8 >= sm_lim[i * 8 + quad * 2 + (e & 1)]) s[i][e] = -INFINITY;
    }
    // to exponents, in place; l: the rows' sums of weights if nobody's weight passes the room
    const float* const units = sm_unit + quad * 2;
    bool passed = false;
    float more[R][2];
    const uint32_t to = weights + (lane & 7) * kWeightPitch + (warp * kKeys + (lane >> 3 & 1) * 8) * 2;
    auto weigh = [&] {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float p0 = exp2f(s[i][0]), p1 = exp2f(s[i][1]), p2 = exp2f(s[i][2]), p3 = exp2f(s[i][3]);
        more[i][0] = p0 + p2;
        more[i][1] = p1 + p3;
        const uint32_t h0 = pack_half(p0, p1), h1 = pack_half(p2, p3);
        stmatrix_x2t(to + i * 8 * kWeightPitch, h0, h1);
        if constexpr (HALVES == 2) {
          const float2 f0 = __half22float2(as_half2(h0)), f1 = __half22float2(as_half2(h1));
          stmatrix_x2t(to + (R + i) * 8 * kWeightPitch, pack_half(p0 - f0.x, p1 - f0.y), pack_half(p2 - f1.x, p3 - f1.y));
        }
      }
    };
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float2 u = *reinterpret_cast<const float2*>(units + i * 8);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool none = m[i][e] == kNone;                // a row without a reference takes one from the first key that it sees
        const float base = none ? 0.f : m[i][e], room = none ? -3e38f : kRoom, f = e ? u.y : u.x;
        s[i][e] = fmaf(s[i][e], f, -base);
        s[i][e + 2] = fmaf(s[i][e + 2], f, -base);
        passed = passed || s[i][e] > room || s[i][e + 2] > room;
      }
    }
    weigh();
    // Behind the barrier all weights of the tile are there, and nobody reads the last one's weights and values any more.  Where a weight passes the room, the block
    // takes another reference, 2^3 away from that, and weighs again.
    if (__syncthreads_or(passed)) {
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(s[i][e], s[i][e + 2]) + (m[i][e] == kNone ? 0.f : m[i][e]);
#pragma unroll
          for (int y = 4; y < 32; y <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, y));
          if (hq == 0) sm_top[warp][i * 8 + quad * 2 + e] = mx;
        }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = sm_top[hq][i * 8 + quad * 2 + e];
#pragma unroll
          for (int y = 4; y < 32; y <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, y));
          const bool none = m[i][e] == kNone;
          if (none && mx == -INFINITY) continue;           // none yet
          const float mn = fmaxf(m[i][e], mx - (kRoom - 3.f)), by = (none ? 0.f : m[i][e]) - mn, f = none ? 0.f : exp2f(by);
          m[i][e] = mn;
          l[i][e] *= f;
          s[i][e] += by;
          s[i][e + 2] += by;
#pragma unroll
          for (int k = 0; k < 2; ++k) { o[i][k][e] *= f; o[i][k][e + 2] *= f; }
        }
      weigh();
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < R; ++i) { l[i][0] += more[i][0]; l[i][1] += more[i][1]; }
    ring.ask(ask_stage);
    ask_stage = ask_stage + 1 == STAGES ? 0 : ask_stage + 1;
    // sums: 16 keys of two warps' parts at a time
#pragma unroll
    for (int j = 0; j < NG; j += 2) {
      const int w = part * NG + j + (lane >> 4);           // whose keys this lane's addresses are
      const uint32_t from = ring0 + w * (STAGES * STAGE) + stage * STAGE;
      uint32_t a[4], st[4];                                // of either part's keys 2 quad.. and 8 + 2 quad..: four codes of a key; number hq of the steps
      ldmatrix_x4t(a, from + V_AT + chunk_at<D>(lane & 15, group));
      ldmatrix_x4t(st, from + VS_AT + (lane & 15) * 16);
      uint32_t v[2][2][4];                                 // [part][keys 2 quad.. or 8 + 2 quad..][column]
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const __half2 s2 = as_half2(__shfl_sync(0xffffffffu, st[x], group * 4 + quad));
        const __half2 m2 = __hmul2(as_half2(__shfl_sync(0xffffffffu, st[x], (NG + group) * 4 + quad)), __float2half2_rn(0.5f));
        const __half2 half2x = __float2half2_rn(0.5f);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t c = y ? a[x] >> 8 : a[x];
          // 1024 + c and 64 + c, halved
          const __half2 c0 = __hfma2(as_half2((c & LOW) | 0x64006400u), half2x, __float2half2_rn(-512.f));
          const __half2 c1 = __hfma2(as_half2((c & HIGH) | 0x54005400u), half2x, __float2half2_rn(-32.f));
          v[x >> 1][x & 1][2 * y] = as_u32(__hfma2(c0, s2, m2));
          v[x >> 1][x & 1][2 * y + 1] = as_u32(__hfma2(c1, s2, m2));
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          uint32_t q[4];
          ldmatrix_x4(q, weights + ((h * R + i) * 8 + (lane & 7)) * kWeightPitch + ((part * NG + j) * kKeys + (lane >> 3) * 8) * 2);
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int k = 0; k < 2; ++k) mma16816(o[i][k], v[x][0][2 * k], v[x][0][2 * k + 1], v[x][1][2 * k], v[x][1][2 * k + 1], q[2 * x], q[2 * x + 1]);
        }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    cur.tile += step;
    if (!CLUSTER && (cur.tile == cur.tiles || t + 1 == tiles_left)) {
      finish(cur.tile == cur.tiles);
      if (t + 1 < tiles_left) {
        next_pair<false>(p, cur);
        begin();
      }
    }
  }
  if constexpr (CLUSTER) {
    finish(true);
    if (p.cluster > 1) join_cluster<T, D, kTileThreads>(p, cur, row0, rows, sm_b, sm_bm, sm_bl, 2.f);
  } else {
    finish_idle_warps<T, D, kTileWarps>(p, warp, lane);
  }
}

template <typename T, int D, int R>
void launch_tiles(const Int4Attn& p, int grid, cudaStream_t st) {
  constexpr int smem = tiles_smem<T, D, R>;
  if (p.cluster) {
    NXD_ALLOW_SMEM((int4_tiles_kernel<T, D, R, true>), smem);
    launch_cluster(int4_tiles_kernel<T, D, R, true>, p, grid, kTileThreads, smem, p.cluster, st);
  } else {
    NXD_ALLOW_SMEM((int4_tiles_kernel<T, D, R, false>), smem);
    launch_cluster(int4_tiles_kernel<T, D, R, false>, p, grid, kTileThreads, smem, 1, st);
  }
}
template <typename T, int D>
void launch(const Int4Attn& p, int grid, cudaStream_t st) {
  if (p.tile_rows == 16) launch_tiles<T, D, 2>(p, grid, st);
  else if (p.tile_rows == 24) launch_tiles<T, D, 3>(p, grid, st);
  else if (p.tile_rows == 32) launch_tiles<T, D, 4>(p, grid, st);
  else launch_tiles<T, D, 5>(p, grid, st);
}

}  // namespace

void int4_tiles(const Int4Attn& p, int grid, int D, int dt, cudaStream_t st) {
  if (dt == kBF16) { if (D == 128) launch<__nv_bfloat16, 128>(p, grid, st); else launch<__nv_bfloat16, 64>(p, grid, st); }
  else { if (D == 128) launch<__half, 128>(p, grid, st); else launch<__half, 64>(p, grid, st); }
}

}  // namespace nxd
