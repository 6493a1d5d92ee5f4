// Page tables of a batch and the slots of its new tokens from the lengths of its requests.
//
// A row wants ceil(length / page_size) columns and holds some; what is missing is taken from a ring of free pages, in the order of the rows, and what
// a row gives back goes to the ring's end.  So row b's first page stands at the sum of what the rows before it take, and what it gives back goes behind
// what they give back: two prefix sums over the rows, which every block finds for itself from the rows' numbers (a thread has rows beside one another, one
// scan over the block's sums).  Then blocks write tables, slots and the ring, each for rows of its own.  Pages are taken from the ring as it was, so no block
// reads a place of it that another one writes.
//
// Small batches are bound by the launch and a chain of four loads (a row's numbers, the ring's beginning, the ring, the slot): 16 rows 3.7 us, 338 rows of 72 columns 4.3.
// Large ones that are not changed in place move both copies of tables and ring, 0.64 of the copy rate at 2000 rows of 2000 columns with 4 million pages, 15.2 us; that every
// block goes over all rows' numbers for itself costs 5 us at 4096 rows and most of 70 at 30000, where a launch before this one that does would be better.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "sm100_ptx.cuh"

namespace nxd {

int device_sm_count();

namespace {

constexpr int kThreads = 512;

// What a block knows of one of its rows
struct Row {
  long first;                // of its new tokens
  long at, back;             // where its pages are taken from and given back to, counted from the ring's beginning
  int had, take, give, count;
};

// What a row wants before anybody knows whether there is as much: columns, pages that are missing, pages that it gives back, and tokens that count
struct Wish { int had, take, give, count; long first; bool long_; };
NXD_DEVICE Wish wish(const PageTables& p, int b) {
  Wish w;
  w.first = p.positions[b];
  const long m = p.lens ? p.lens[b] : p.W;
  w.count = w.first < 0 ? 0 : (int)(m < 0 ? 0 : m > p.W ? p.W : m);
  w.first = min(w.first, 1l << 40);
  const long length = p.lengths ? p.lengths[b] : w.count > 0 ? w.first + w.count : -1;
  w.long_ = length > (long)p.cols * p.ps;                  // that is below 2^31: what is divided has 32 bits (of 64 bits: 30000 rows 85 us for 71)
  const int want = w.long_ ? p.cols : length > 0 ? (int)(((unsigned)length + (unsigned)p.ps - 1) / (unsigned)p.ps) : 0;
  w.had = max(p.shared, min(p.held[b], p.cols));
  w.take = w.long_ ? 0 : max(0, want - w.had);
  w.give = length == 0 || (p.trim && length > 0) ? max(0, w.had - max(p.shared, want)) : 0;
  return w;
}

// IN_PLACE: one cluster, all of whose blocks have read the rows' numbers before the first of them writes; otherwise outputs are other tensors
template <bool IN_PLACE>
__global__ void __launch_bounds__(kThreads) page_tables_kernel(const PageTables p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ long sums[kThreads / 32][2], totals[3];
  Row* const rows = reinterpret_cast<Row*>(smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b0 = blockIdx.x * p.rows, b1 = min(p.B, b0 + p.rows);
  const int each = (p.B + kThreads - 1) / kThreads, r0 = min(p.B, (int)threadIdx.x * each), r1 = min(p.B, r0 + each);
  pdl_trigger();
  pdl_wait();
  const long head = p.span[0], tail = p.span[1];
  long take = 0, give = 0;
  bool few = false;
  for (int b = r0; b < r1; ++b) {
    const Wish w = wish(p, b);
    take += w.take;
    give += w.give;
    few |= w.long_;
  }
  long st = take, sg = give;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long x = __shfl_up_sync(0xffffffffu, st, o), y = __shfl_up_sync(0xffffffffu, sg, o);
    if (lane >= o) { st += x; sg += y; }
  }
  if (lane == 31) { sums[warp][0] = st; sums[warp][1] = sg; }
  if (threadIdx.x == 0) totals[0] = totals[1] = totals[2] = 0;
  __syncthreads();
  st -= take;
  sg -= give;
  for (int w = 0; w < warp; ++w) { st += sums[w][0]; sg += sums[w][1]; }
  // what the rows before this thread's take and give back; the last row that finds enough says how many are taken in all
  long taken = -1;
  for (int b = r0; b < r1; ++b) {
    const Wish w = wish(p, b);
    const bool fits = st + w.take <= tail - head;
    if (w.take && !fits) few = true;
    if (fits) taken = st + w.take;
    if (b >= b0 && b < b1) rows[b - b0] = Row{w.first, head + st, tail + sg, w.had, fits ? w.take : 0, w.give, w.count};
    st += w.take;
    sg += w.give;
  }
  if (taken >= 0) atomicMax((unsigned long long*)&totals[0], (unsigned long long)taken);       // not negative: their order is the numbers'
  if (r1 == p.B && r0 < r1) totals[1] = sg;
  __syncthreads();
  if constexpr (IN_PLACE) cluster_sync_all();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
    p.span_out[0] = head + totals[0];
    p.span_out[1] = tail + totals[1];
  }
  if (few && p.few) *p.few = 1;
  const long P = p.P;
  auto place = [&](long i) { return (unsigned)((unsigned long)i % (unsigned long)P); };       // in the ring, whatever the counts are
  const int n = b1 - b0, part = blockIdx.y * kThreads + threadIdx.x, stride = gridDim.y * kThreads;
  if (blockIdx.y == 0)
    for (int i = threadIdx.x; i < n; i += kThreads) p.held_out[b0 + i] = rows[i].had + rows[i].take - rows[i].give;
  auto column = [&](const Row& r, int c, int old) {        // what a column holds from now on, and to the ring what it gives back
    if (c >= r.had && c < r.had + r.take) return p.free[place(r.at + c - r.had)];
    if (c < r.had && c >= r.had - r.give) {
      p.free_out[place(r.back + c - (r.had - r.give))] = old;
      return -1;
    }
    return old;
  };
  auto old = [&](int i, int c) { return p.table + (b0 + i) * p.table_sb + c; };
  auto now = [&](int i, int c) { return p.table_out + (b0 + i) * p.out_sb + c; };
  if constexpr (IN_PLACE) {
    // columns that change, four threads a row, and a warp a row for those that are left
    constexpr int FEW = 4;
    for (int i = threadIdx.x / FEW; i < n; i += kThreads / FEW) {
      const Row& r = rows[i];
      const int c = r.had - r.give + (int)threadIdx.x % FEW;
      if (c < r.had + r.take) *now(i, c) = column(r, c, *old(i, c));
    }
    for (int i = warp; i < n; i += kThreads / 32) {
      const Row& r = rows[i];
      for (int c = r.had - r.give + FEW + lane; c < r.had + r.take; c += 32) *now(i, c) = column(r, c, *old(i, c));
    }
  } else {
    // four columns at a time where rows are whole packets; threads beside one another have a row, as many rows at a time as there are threads for, and four of those
    const bool fours = p.cols % 4 == 0 && p.table_sb % 4 == 0 && ((uintptr_t)p.table | (uintptr_t)p.table_out) % 16 == 0;
    constexpr int ROWS = 4;
    const int packs = fours ? p.cols / 4 : p.cols, bits = packs > kThreads / 2 ? 9 : packs > 1 ? 32 - __clz(packs - 1) : 0;           // 2^bits threads a row
    const int rows_at = kThreads >> bits, first = (blockIdx.y << bits) + (threadIdx.x & ((1 << bits) - 1)), apart = gridDim.y << bits;
    static_assert(kThreads == 1 << 9);
    for (int i0 = threadIdx.x >> bits; i0 < n; i0 += rows_at * ROWS)
      for (int pack = first; pack < packs; pack += apart) {
        if (fours) {
          const int c = pack * 4;
          int4 x[ROWS];
#pragma unroll
          for (int y = 0; y < ROWS; ++y)
            if (i0 + y * rows_at < n) x[y] = *reinterpret_cast<const int4*>(old(i0 + y * rows_at, c));
#pragma unroll
          for (int y = 0; y < ROWS; ++y) {
            const int i = i0 + y * rows_at;
            if (i >= n) break;
            const Row& r = rows[i];
            if (!(c + 4 <= r.had - r.give || c >= r.had + r.take)) x[y] = make_int4(column(r, c, x[y].x), column(r, c + 1, x[y].y), column(r, c + 2, x[y].z), column(r, c + 3, x[y].w));
            *reinterpret_cast<int4*>(now(i, c)) = x[y];
          }
        } else {
          int x[ROWS];
#pragma unroll
          for (int y = 0; y < ROWS; ++y)
            if (i0 + y * rows_at < n) x[y] = *old(i0 + y * rows_at, pack);
#pragma unroll
          for (int y = 0; y < ROWS; ++y)
            if (i0 + y * rows_at < n) *now(i0 + y * rows_at, pack) = column(rows[i0 + y * rows_at], pack, x[y]);
        }
      }
    // the rest of the ring, as it was: all places but those that pages were given back to
    const unsigned given = (unsigned)min((long)totals[1], P), tail_at = place(tail), all = gridDim.x * gridDim.y * kThreads;
    auto kept = [&](unsigned i) { return (i >= tail_at ? i - tail_at : i - tail_at + (unsigned)P) >= given; };
    const unsigned me = (blockIdx.y * gridDim.x + blockIdx.x) * kThreads + threadIdx.x, whole = (((uintptr_t)p.free | (uintptr_t)p.free_out) % 16 == 0) ? (unsigned)P / 4 : 0;
    constexpr int PACKS = 4;
    for (unsigned i0 = me; i0 < whole; i0 += all * PACKS) {
      int4 x[PACKS];
#pragma unroll
      for (int y = 0; y < PACKS; ++y)
        if (i0 + y * all < whole) x[y] = reinterpret_cast<const int4*>(p.free)[i0 + y * all];
#pragma unroll
      for (int y = 0; y < PACKS; ++y) {
        const unsigned i = i0 + y * all;
        if (i >= whole) break;
        if (given == 0 || (kept(4 * i) && kept(4 * i + 1) && kept(4 * i + 2) && kept(4 * i + 3))) reinterpret_cast<int4*>(p.free_out)[i] = x[y];
        else {
          if (kept(4 * i)) p.free_out[4 * i] = x[y].x;
          if (kept(4 * i + 1)) p.free_out[4 * i + 1] = x[y].y;
          if (kept(4 * i + 2)) p.free_out[4 * i + 2] = x[y].z;
          if (kept(4 * i + 3)) p.free_out[4 * i + 3] = x[y].w;
        }
      }
    }
    for (unsigned i = whole * 4 + me; i < (unsigned)P; i += all)
      if (kept(i)) p.free_out[i] = p.free[i];
  }
  bool lost = false;
  for (unsigned x = part; x < (unsigned)n * p.W; x += stride) {          // fewer than 2^31
    const int i = (int)(x / p.W), w = (int)(x - (unsigned)i * p.W);
    const Row r = rows[i];
    int slot = -1;
    if (w < r.count) {
      const long pos = r.first + w;
      const int c = pos < (long)p.cols * p.ps ? (int)((unsigned)pos / (unsigned)p.ps) : p.cols;
      if (c >= p.shared && c < r.had + r.take - r.give) {
        const int page = c < r.had ? p.table[(b0 + i) * p.table_sb + c] : p.free[place(r.at + c - r.had)];
        if (page >= 0 && page < P) slot = page * p.ps + (int)((unsigned)pos - (unsigned)c * p.ps);
      }
      lost |= slot < 0;
    }
    p.slots[(long)(b0 + i) * p.W + w] = slot;
  }
  if (lost && p.few) *p.few = 1;
}

}  // namespace

void page_tables(PageTables p, bool in_place, cudaStream_t st) {
  if (p.B == 0) {
    if (!in_place) {
      NXD_CUDA_CHECK(cudaMemcpyAsync(p.free_out, p.free, p.P * sizeof(int), cudaMemcpyDeviceToDevice, st));
      NXD_CUDA_CHECK(cudaMemcpyAsync(p.span_out, p.span, 2 * sizeof(long), cudaMemcpyDeviceToDevice, st));
    }
    return;
  }
  const int sms = device_sm_count();
  if (in_place) {
    int size = 1;
    while (size < 8 && (p.B > 64 * size || (long)p.B * p.W > 2048l * size)) size *= 2;
    p.rows = (p.B + size - 1) / size;
    const int smem = p.rows * (int)sizeof(Row);
    NXD_ALLOW_SMEM(page_tables_kernel<true>, kMaxPageRows / 8 * (int)sizeof(Row));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = size; cfg.blockDim = kThreads; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = size;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    NXD_CUDA_CHECK(cudaLaunchKernelEx(&cfg, page_tables_kernel<true>, p));
    return;
  }
  // about two blocks an SM, rows whole or in parts
  const long work = (long)p.B * (p.cols + p.W);
  const long blocks = std::max(1l, std::min(2l * sms, (work + 2 * kThreads - 1) / (2 * kThreads)));
  int gx = (int)std::max(std::min((long)p.B, blocks), (p.B + 511l) / 512);
  p.rows = (p.B + gx - 1) / gx;
  gx = (p.B + p.rows - 1) / p.rows;
  const int gy = (int)std::max(1l, blocks / gx);
  launch_dependent(page_tables_kernel<false>, dim3(gx, gy), kThreads, p.rows * sizeof(Row), st, p);
}

}  // namespace nxd
