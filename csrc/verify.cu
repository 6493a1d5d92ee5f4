// Drafted tokens against the target's probabilities, from given random numbers:
//   token i is taken while u_i q_i(x_i) < p_i(x_i);  where the first one is refused, n, the next token comes from max(p_n − q_n, 0), behind the last
//   from p_K: the first v with w(0) + … + w(v) > s (w(0) + … + w(V − 1)).
// Everything is compared and summed in 64 bits: a border between two of V tokens lies within eps of a drawn number with probability V eps, which
// sums in 32 bits would make a per cent.
#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "sm100_ptx.cuh"

namespace nxd {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kParts = 32 / kWarps;                        // sums that a warp keeps: one for each lane of a block's search

// N numbers of p and of q (0 where there is none, or behind the row's end)
template <typename T, int N>
struct Pair {
  Pack16<T> a, b;
  NXD_DEVICE void load(const T* p, const T* q, int v, int V, bool packets) {
    if (packets && v < V) {
      a.load(p + v);
      if (q) b.load(q + v);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        a.v[i] = v + i < V ? p[v + i] : from_f32<T>(0.f);
        b.v[i] = q && v + i < V ? q[v + i] : from_f32<T>(0.f);
      }
    }
    if (!q)
#pragma unroll
      for (int i = 0; i < N; ++i) b.v[i] = from_f32<T>(0.f);
  }
  NXD_DEVICE double weight(int i) const {
    const double d = (double)a.f(i) - (double)fmaxf(b.f(i), 0.f);      // negative and NaN: 0, on the draft's side here
    return d > 0 ? d : 0;                                              // and on the target's
  }
};

NXD_DEVICE double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

NXD_DEVICE double remote_double(const double* at, int rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(mapa_shared(smem_u32(at), rank)) : "memory");
  return v;
}

// One cluster per sequence: each block sums a stretch of the vocabulary in 32 parts; where the drawn share of the sum lies is found from the sums,
// and a warp walks the one part that has it again (out of L2).  Bound by HBM, one row of p and one of q, and by its chain: the drafted tokens, their
// probabilities, the walk, the exchange of sums, the second walk.  Blocks of 256 threads, so that all of a batch of 64 are there at once: with 512
// they came in two to four rounds and 64 x 7 drafts over 100352 tokens took 24 to 47 us, so 16 (one sequence over 32000: 7).
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) verify_kernel(const long* tokens, const T* draft, const T* target, const float* accept, const float* sample,
                                                          long* out, long* accepted, int K, int V, long d_sb, long d_sk, long t_sb, long t_sk) {
  constexpr int N = Pack16<T>::N, STEP = 32 * N, AHEAD = 16 / N;      // a warp's steps of 32 x 16 bytes, of which so many are asked for at once
  __shared__ double sums[32];
  __shared__ double block_sum;
  __shared__ int refused, bonus;
  const int rank = (int)cluster_ctarank(), size = (int)gridDim.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  if (warp == 0) {
    int n = K;
    bool plain = true;                                     // the next token comes from p alone
    for (int i0 = 0; i0 < K && n == K; i0 += 32) {
      const int i = i0 + lane;
      bool ok = true, none = false;
      if (i < K) {
        const long x = tokens[(long)b * K + i];
        none = x < 0 || x >= V;                            // no token was drafted here
        ok = !none && (double)accept[(long)b * K + i] * (double)fmaxf(to_f32<T>(draft[b * d_sb + i * d_sk + x]), 0.f) < (double)to_f32<T>(target[b * t_sb + i * t_sk + x]);
      }
      const unsigned bad = __ballot_sync(0xffffffffu, !ok), ends = __ballot_sync(0xffffffffu, none);
      if (bad) {
        n = i0 + __ffs(bad) - 1;
        plain = ends >> (n - i0) & 1;
      }
    }
    if (lane == 0) { refused = n; bonus = plain; }
  }
  __syncthreads();
  const int n = refused;
  const T* const p = target + b * t_sb + n * t_sk;
  const T* q = bonus ? nullptr : draft + b * d_sb + n * d_sk;
  const bool packets = (uintptr_t)p % 16 == 0 && (uintptr_t)q % 16 == 0 && V % N == 0;
  // steps of STEP numbers: `per` to a part, the same number for every part of the cluster
  const int steps = (V + STEP - 1) / STEP, all = size * 32, per = (steps + all - 1) / all;
  auto first_step = [&](int part) { return min((long)steps, (long)(rank * 32 + part) * per); };
  // sum of this block's weights, by parts; q null: of p alone
  auto add_up = [&](const T* q) {
#pragma unroll 1
    for (int i = 0; i < kParts; ++i) {
      const int part = warp * kParts + i, s1 = (int)first_step(part + 1);
      double sum = 0;
      auto walk = [&](int s, auto whole) {                 // AHEAD steps
        constexpr bool all_there = decltype(whole)::value;
        Pair<T, N> x[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) x[a].load(p, q, s + a < s1 ? (s + a) * STEP + lane * N : V, V, packets);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          if (!all_there && s + a >= s1) break;            // conversions to 64 bits are slow: none for what is not there
#pragma unroll
          for (int j = 0; j < N; ++j) sum += x[a].weight(j);
        }
      };
      int s = (int)first_step(part);
      for (; s + AHEAD <= s1; s += AHEAD) walk(s, std::true_type{});
      if (s < s1) walk(s, std::false_type{});
      sum = warp_sum64(sum);
      if (lane == 0) sums[part] = sum;
    }
    __syncthreads();
    if (warp == 0) {
      const double x = warp_sum64(sums[lane]);
      if (lane == 0) block_sum = x;
    }
    cluster_sync_all();
    return lane < size ? remote_double(&block_sum, lane) : 0.;
  };
  double of_block = add_up(q), total = warp_sum64(of_block);           // lane = block
  if (q && !(total > 0)) {                                 // nothing is left of p - q: from p itself
    cluster_sync_all();                                    // every block has read the sums
    q = nullptr;
    of_block = add_up(q);
    total = warp_sum64(of_block);
  }
  if (warp == 0) {
    const double want = (double)sample[b] * total;
    // the block, then the part, in which the running sum passes `want`; if roundings leave none, the last that has anything
    auto find = [&](double x, double before, double& start) {          // lane = place; start: the sum before the place found
      double scan = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += y;
      }
      const unsigned some = __ballot_sync(0xffffffffu, x > 0), past = __ballot_sync(0xffffffffu, x > 0 && before + scan > want);
      const int at = past ? __ffs(past) - 1 : 31 - __clz(some);
      if (at >= 0) start = before + __shfl_sync(0xffffffffu, scan - x, at);
      return at;
    };
    double base = 0, start = 0;
    const int mine = find(of_block, 0., base);
    if (mine == rank) {
      const int at = find(sums[lane], base, start);
      const int f0 = (int)first_step(at), f1 = (int)first_step(at + 1);
      long chosen = -1, last = -1;
      for (int s = f0; s < f1 && chosen < 0; s += AHEAD) {
        Pair<T, N> x[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) x[i].load(p, q, s + i < f1 ? (s + i) * STEP + lane * N : V, V, packets);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          if (s + i >= f1) break;
          double part = 0;
#pragma unroll
          for (int j = 0; j < N; ++j) part += x[i].weight(j);
          double scan = part;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += y;
          }
          double run = start + (scan - part);
          int hit = -1, tail = -1;
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const double w = x[i].weight(j);
            run += w;
            if (w > 0) tail = j;
            if (hit < 0 && w > 0 && run > want) hit = j;
          }
          const int v = (s + i) * STEP;
          const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), tails = __ballot_sync(0xffffffffu, tail >= 0);
          const int first = __ffs(hits) - 1, end = 31 - __clz(tails);
          if (chosen < 0 && hits) chosen = v + first * N + __shfl_sync(0xffffffffu, hit, first);
          if (tails) last = v + end * N + __shfl_sync(0xffffffffu, tail, end);
          start += __shfl_sync(0xffffffffu, scan, 31);
        }
      }
      if (lane == 0) out[(long)b * (K + 1) + n] = chosen >= 0 ? chosen : last;
    }
    if (rank == 0) {
      if (mine < 0 && lane == 0) out[(long)b * (K + 1) + n] = -1;      // a row without probabilities
      for (int i = lane; i <= K; i += 32)
        if (i != n) out[(long)b * (K + 1) + i] = i < n ? tokens[(long)b * K + i] : -1;
      if (lane == 0) accepted[b] = n;
    }
  }
  cluster_sync_all();                                      // nobody reads a block's sums any more
}

}  // namespace

int device_sm_count();

void verify_drafts(const long* tokens, const void* draft, const void* target, const float* accept, const float* sample, long* out, long* accepted,
                   int B, int K, int V, const long* draft_s, const long* target_s, int dt, cudaStream_t st) {
  if (B == 0) return;
  // two blocks per SM and more, and no block with less than a step for every second warp
  int size = 1;
  while (size < 8 && (long)B * size < 2 * device_sm_count() && V / (2 * size) >= 2048) size *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(size, B);
  cfg.blockDim = kThreads;
  cfg.stream = st;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = size;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
#define NXD_VERIFY(T)                                                                                                                          \
  NXD_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_kernel<T>, tokens, (const T*)draft, (const T*)target, accept, sample, out, accepted, K, V,        \
                                    draft_s[0], draft_s[1], target_s[0], target_s[1]))
  if (dt == kF32) NXD_VERIFY(float);
  else if (dt == kBF16) NXD_VERIFY(__nv_bfloat16);
  else NXD_VERIFY(__half);
#undef NXD_VERIFY
}

}  // namespace nxd
