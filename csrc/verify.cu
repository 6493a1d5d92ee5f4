// Drafted tokens against the target's probabilities, from given random numbers:
//   token i is taken while u_i q_i(x_i) < p_i(x_i);  where the first one is refused, n, the next token comes from max(p_n − q_n, 0), behind the last
//   from p_K: the first v with w(0) + … + w(v) > s (w(0) + … + w(V − 1)).
// Everything is compared and summed in 64 bits: a border between two of V tokens lies within eps of a drawn number with probability V eps, which
// sums in 32 bits would make a per cent.
#include <algorithm>
#include <string>

#include "common.cuh"
#include "kernels.h"
#include "sm100_ptx.cuh"

namespace nxd {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;

template <typename T, int N>
NXD_DEVICE void load_weights(const T* p, const T* q, int v, int V, bool packets, double (&w)[N], double& plain) {
  float a[N], b[N];
  if (packets) {
    Pack16<T> x;
    x.load(p + v);
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = x.f(i);
    if (q) x.load(q + v);
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = q ? x.f(i) : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      a[i] = v + i < V ? to_f32<T>(p[v + i]) : 0.f;
      b[i] = q && v + i < V ? to_f32<T>(q[v + i]) : 0.f;
    }
  }
  plain = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double x = (double)a[i], d = x - (double)b[i];
    w[i] = d > 0 ? d : 0;                                  // NaN: 0
    plain += x > 0 ? x : 0;
  }
}

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

// One cluster per sequence: each block sums a stretch of the vocabulary, each warp a stretch of the block's; where the drawn share of the sum lies
// is found from the sums, and the one warp that has it walks its stretch again (out of L2).  Bound by HBM: one row of p and one of q; one
// sequence alone by its chain of drafted tokens, their probabilities, the walk and the exchange.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(const long* tokens, const T* draft, const T* target, const float* accept, const float* sample,
                                                          long* out, long* accepted, int K, int V, long d_sb, long d_sk, long t_sb, long t_sk) {
  constexpr int N = Pack16<T>::N, STEP = 32 * N;
  __shared__ double sums[2][kWarps];                       // of max(p − q, 0) and of p
  __shared__ double block_sums[2];
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
        ok = !none && (double)accept[(long)b * K + i] * (double)to_f32<T>(draft[b * d_sb + i * d_sk + x]) < (double)to_f32<T>(target[b * t_sb + i * t_sk + x]);
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
  const T* const q = bonus ? nullptr : draft + b * d_sb + n * d_sk;
  const bool packets = (uintptr_t)p % 16 == 0 && (uintptr_t)q % 16 == 0 && V % N == 0;
  // steps of STEP numbers, the same number for every warp of the cluster
  const int steps = (V + STEP - 1) / STEP, per = (steps + size * kWarps - 1) / (size * kWarps), s0 = (rank * kWarps + warp) * per, s1 = min(steps, s0 + per);
  double sum = 0, sum_p = 0;
#pragma unroll 4
  for (int s = s0; s < s1; ++s) {
    const int v = s * STEP + lane * N;
    if (v < V) {
      double w[N], all;
      load_weights<T, N>(p, q, v, V, packets, w, all);
#pragma unroll
      for (int i = 0; i < N; ++i) sum += w[i];
      sum_p += all;
    }
  }
  sum = warp_sum64(sum);
  sum_p = warp_sum64(sum_p);
  if (lane == 0) { sums[0][warp] = sum; sums[1][warp] = sum_p; }
  __syncthreads();
  if (threadIdx.x < 2) {
    double x = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) x += sums[threadIdx.x][w];
    block_sums[threadIdx.x] = x;
  }
  cluster_sync_all();
  if (warp == 0) {
    double total[2] = {0, 0};
    for (int r = 0; r < size; ++r) {
      total[0] += remote_double(&block_sums[0], r);
      total[1] += remote_double(&block_sums[1], r);
    }
    const int which = total[0] > 0 ? 0 : 1;                // nothing left of p - q: from p itself
    const double want = (double)sample[b] * total[which];
    // the block, then the warp, in which the running sum passes `want`; if roundings leave none, the last that has anything
    double before = 0, base = 0;
    int mine = -1;
    for (int r = 0; r < size; ++r) {
      const double x = remote_double(&block_sums[which], r);
      if (x > 0) { mine = r; base = before; }
      before += x;
      if (x > 0 && before > want) break;
    }
    if (mine == rank) {
      int at = -1;
      double start = base;
      before = base;
      for (int w = 0; w < kWarps; ++w) {
        const double x = sums[which][w];
        if (x > 0) { at = w; start = before; }
        before += x;
        if (x > 0 && before > want) break;
      }
      const T* const qq = which ? nullptr : q;
      const int f0 = (rank * kWarps + at) * per, f1 = min(steps, f0 + per);
      long chosen = -1, last = -1;
      for (int s = f0; s < f1 && chosen < 0; ++s) {
        const int v = s * STEP + lane * N;
        double w[N], all, part = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = 0;
        if (v < V) load_weights<T, N>(p, qq, v, V, packets, w, all);
        int hit = -1, tail = -1;
#pragma unroll
        for (int i = 0; i < N; ++i) part += w[i];
        double scan = part;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double x = __shfl_up_sync(0xffffffffu, scan, o);
          if (lane >= o) scan += x;
        }
        double run = start + (scan - part);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          run += w[i];
          if (w[i] > 0) tail = v + i;
          if (hit < 0 && w[i] > 0 && run > want) hit = v + i;
        }
        const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), tails = __ballot_sync(0xffffffffu, tail >= 0);
        if (hits) chosen = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
        else if (tails) last = __shfl_sync(0xffffffffu, tail, 31 - __clz(tails));
        start += __shfl_sync(0xffffffffu, scan, 31);
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
  // about two blocks per SM in all, and no block with less than a step for every second warp
  int size = 1;
  while (size < 8 && (long)B * size < device_sm_count() && V / (2 * size) >= 4096) size *= 2;
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
