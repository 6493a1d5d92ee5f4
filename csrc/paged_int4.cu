// A key/value cache in pages that is held in 4 bits: 32 numbers of a token's head are m + s c, m and s in half precision, c of 0 to 15 (kernels.h: Int4Pages).
// Appending with the position rotation on the way, reading tokens back, and attention of query rows over the codes.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged_int4.cuh"

namespace nxd {

int device_sm_count();

namespace {

using namespace int4;

// ---------------------------------------------------------------------------------------------------------------- append
constexpr int kAppendThreads = 128;
// From here on queries go by a launch of their own, which takes fewer registers, so that more of its threads wait for memory at a time (us, one launch / two: 1 token of 32
// heads 4.1 / 5.4, 4 x 500 tokens of 64 heads on 8 alike, 4 x 2000 100 / 95).
constexpr long kSplitTokens = 2000;

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

// How the numbers of a head turn: halves of the whole head, neighbours, or halves of a part of it
enum Turn { kHalves, kPairs, kPart };

// m and s of 32 numbers that four threads have, from the least and the largest of them, which are off by `off` at most; from exact ones where that leaves two halves
template <typename F>
NXD_DEVICE void steps_of(float lo, float hi, float off, unsigned four, F exact, __half& m16, __half& s16) {
  constexpr float k15 = 1.f / 15.f;
  m16 = __float2half_rn(lo + off);
  const float range = hi - __half2float(m16), more = off + fminf(range, 0x1p17f) * 0x1p-22f;          // its own roundings and the product's
  s16 = __float2half_rn((range + more) * k15);
  const bool doubt = __half_as_ushort(m16) != __half_as_ushort(__float2half_rn(lo - off)) || __half_as_ushort(s16) != __half_as_ushort(__float2half_rn((range - more) * k15));
  if (doubt) {                                             // never where a NaN is: its halves are alike
    double a = exact(0), b = a;
#pragma unroll
    for (int i = 1; i < 8; ++i) { const double x = exact(i); a = fmin(a, x); b = fmax(b, x); }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      a = fmin(a, __shfl_xor_sync(four, a, o));
      b = fmax(b, __shfl_xor_sync(four, b, o));
    }
    // by way of 32 bits, as torch rounds numbers of 64 to halves (a value that the first rounding puts on a border differs)
    m16 = __float2half_rn((float)a);
    s16 = __float2half_rn((float)((b - (double)__half2float(m16)) / 15.));
  }
}

// A thread has CH times eight numbers of one head, half a head apart, so that with kHalves all that turns together is its own (kPart reads the eight that turn with
// its own once more); four threads have the 32 numbers that share m and s.  Keys turn as a c - b s with what the rounding of b s left put back, one rounding in all; a
// code whose quotient is near a border, and steps that are, are found again from the products in 64 bits, so that codes are those of exact numbers.  Queries
// are bound by HBM (4 x 2000 tokens of 64 heads, a quarter padding: 40 us, 0.75 of the copy rate), keys and values by their arithmetic: 8 heads of those tokens 25 us,
// where memory would take 7; a call for single tokens by its launch, 4 us.
enum Role { kAll, kQuery, kCache };                     // whose numbers a launch has: everybody's, queries', or keys' and values'
template <typename T, int D0, Turn TURN, int CH, Role ROLE>
__global__ void __launch_bounds__(kAppendThreads, ROLE == kQuery ? 12 : 8) int4_append_kernel(const Int4Append p) {
  const int D = D0 ? D0 : p.D;
  pdl_trigger();
  const unsigned t = blockIdx.x, item = blockIdx.y * kAppendThreads + threadIdx.x, chunks = D / (8 * CH);
  const int h = (int)(item / chunks) + (ROLE == kCache ? p.H : 0), c0 = (int)(item % chunks) * 8;
  const int w = (int)(t / (unsigned)p.B), b = (int)(t - (unsigned)w * p.B);        // tokens of all sequences beside one another, as projections leave them
  pdl_wait();
  if (h >= (ROLE == kQuery ? p.H : p.H + 2 * p.Hkv)) return;
  const bool query = ROLE == kQuery || (ROLE == kAll && h < p.H), key = !query && h < p.H + p.Hkv;
  const T* const src = query ? (const T*)p.q + b * p.q_sb + w * p.q_sw + h * p.q_sh
                       : key ? (const T*)p.k + b * p.k_sb + w * p.k_sw + (h - p.H) * p.k_sh
                             : (const T*)p.v + b * p.v_sb + w * p.v_sw + (h - p.H - p.Hkv) * p.v_sh;
  Eight<T> x[CH], other[CH];                               // the numbers, and with kPart those that turn with them
#pragma unroll
  for (int j = 0; j < CH; ++j) x[j].load(src + c0 + j * (D / 2));       // whether the token counts or not: beside its slot and position
  const long slot = p.slots[(long)b * p.W + w], first = p.positions[b], pos = first + w;
  const bool has = slot >= 0 && slot < p.tokens, inside = first > -(1l << 40) && first < p.rows && pos >= 0 && pos < p.rows;
  const bool live = has && inside;
  if (!live) {
    if (ROLE != kCache && p.lost && item == 0 && has) *p.lost = 1;
    if (query) {
      Eight<T> zero;
#pragma unroll
      for (int i = 0; i < 8; ++i) zero.set(i, 0.f);
#pragma unroll
      for (int j = 0; j < CH; ++j) zero.store((T*)p.q_out + b * p.o_sb + w * p.o_sw + (long)h * D + c0 + j * (D / 2));
    }
    return;
  }
  // y = x co + (what turns with it) si, the sine's sign taken where it is used: with kHalves both halves have the same angles
  constexpr int ANGLES = TURN == kHalves ? 1 : CH;
  float co[ANGLES][8], si[ANGLES][8];
  bool turns[CH];
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int c = c0 + j * (D / 2);
    turns[j] = (query || key) && (TURN == kHalves || c < 2 * p.half);
    if (!turns[j] || j >= ANGLES) continue;
    const int at = TURN == kPairs ? c / 2 : TURN == kHalves || c < p.half ? c : c - p.half;
    if constexpr (TURN == kPart) other[j].load(src + (c < p.half ? c + p.half : at));
#pragma unroll
    for (int i = 0; i < (TURN == kPairs ? 4 : 8); i += 4) {
      const float4 cv = *reinterpret_cast<const float4*>(p.cos_t + pos * p.half + at + i), sv = *reinterpret_cast<const float4*>(p.sin_t + pos * p.half + at + i);
      co[j][i] = cv.x; co[j][i + 1] = cv.y; co[j][i + 2] = cv.z; co[j][i + 3] = cv.w;
      si[j][i] = sv.x; si[j][i + 1] = sv.y; si[j][i + 2] = sv.z; si[j][i + 3] = sv.w;
    }
  }
  auto turned = [&](int j, int i) { return TURN == kPairs ? x[j].f(i ^ 1) : TURN == kHalves ? x[CH - 1 - j].f(i) : other[j].f(i); };
  auto cosine = [&](int j, int i) { return co[j % ANGLES][TURN == kPairs ? i / 2 : i]; };
  auto sine = [&](int j, int i) {
    const float f = si[j % ANGLES][TURN == kPairs ? i / 2 : i];
    const bool low = TURN == kPairs ? !(i & 1) : TURN == kHalves ? j == 0 : c0 + j * (D / 2) < p.half;
    return low ? -f : f;
  };
  if (query) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      Eight<T> y = x[j];
      if (turns[j])
#pragma unroll
        for (int i = 0; i < 8; ++i) y.set(i, x[j].f(i) * cosine(j, i) + turned(j, i) * sine(j, i));
      y.store((T*)p.q_out + b * p.o_sb + w * p.o_sw + (long)h * D + c0 + j * (D / 2));
    }
    return;
  }
  const Int4Pages& to = key ? p.kp : p.vp;
  const int head = h - p.H - (key ? 0 : p.Hkv), page = (int)slot / p.ps, row = (int)slot - page * p.ps;
  uint8_t* const codes_to = to.codes + page * to.c_sp + row * to.c_sr + head * to.c_sh;
  uint16_t* const steps_to = to.steps + page * to.s_sp + row * to.s_sr + head * to.s_sh;
  const unsigned four = 0xfu << (threadIdx.x & 28);        // the threads of the 32 numbers: all of one head
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = x[j].f(i);
      if (turns[j]) {
        const float z = turned(j, i), f = sine(j, i), e = __fmul_rn(z, f);
        y[i] = __fadd_rn(__fmaf_rn(y[i], cosine(j, i), e), __fmaf_rn(z, f, -e));
      }
    }
    const int c = c0 + j * (D / 2);
    auto exact = [&](int i) {                              // seldom: from memory once more
      const int at = c + i;
      const double own = to_f32<T>(src[at]);
      if (!turns[j]) return own;
      const bool low = TURN == kPairs ? !(i & 1) : at < p.half;
      const int with = TURN == kPairs ? at ^ 1 : low ? at + p.half : at - p.half, angle = TURN == kPairs ? at / 2 : low ? at : at - p.half;
      const double turn = (double)to_f32<T>(src[with]) * p.sin_t[pos * p.half + angle], keep = own * p.cos_t[pos * p.half + angle];
      return low ? keep - turn : keep + turn;
    };
    float lo = y[0], hi = y[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) { lo = min_nan(lo, y[i]); hi = max_nan(hi, y[i]); }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      lo = min_nan(lo, __shfl_xor_sync(four, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(four, hi, o));
    }
    __half m16, s16;
    const float size = fmaxf(fabsf(lo), fabsf(hi));
    steps_of(lo, hi, fminf(size, 0x1p17f) * (key ? 0x1.8p-23f : 0.f), four, exact, m16, s16);       // one bound for all four threads: they meet in there
    const float m = __half2float(m16), s = __half2float(s16), inv = s > 0.f && s <= 65504.f ? (1.f / 15.f) / s : 0.f;
    // quotients as shares of 15, held between 0 and 1 (NaN: 0); with 2^23 and a half of that added their last bits are the codes
    constexpr float kBits = 0x1.8p23f;
    uint32_t codes = 0;
    float worst = 0.f;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      const float q = __saturatef((y[i] - m) * inv), r = fmaf(q, 15.f, kBits);
      worst = fmaxf(worst, fabsf(fmaf(q, 15.f, kBits - r)));
      codes = codes * 16 + __float_as_uint(r);
    }
    codes -= 0x4b400000u * 0x11111111u;
    // quotients are off by 15 * 2^-22, what the numbers are off by aside
    const float border = 0.5f - 0x1p-17f - 0x1p-18f * size * inv;
    if (worst > border) {                                  // those near a border from numbers that are exact
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = __saturatef((y[i] - m) * inv), r = fmaf(q, 15.f, kBits);
        if (!(fabsf(fmaf(q, 15.f, kBits - r)) > border)) continue;
        const double d = exact(i) - m;
        const int at = min(14, max(0, (int)floor(d / s))); // the border is at + 1 / 2, whichever way the quotient was rounded
        const double above = d - (at + 0.5) * s;
        codes = (codes & ~(15u << (4 * i))) | (uint32_t)(above > 0 || (above == 0 && (at & 1)) ? at + 1 : at) << (4 * i);
      }
    }
    *reinterpret_cast<uint32_t*>(codes_to + c / 2) = codes;
    if (c % 32 == 0) steps_to[c / 32] = __half_as_ushort(s16);
    if (c % 32 == 8) steps_to[D / 32 + c / 32] = __half_as_ushort(m16);
  }
}

// ---------------------------------------------------------------------------------------------------------------- gather
constexpr int kGatherThreads = 128;
// Tokens at slots as numbers of T: a block has the keys or the values of TOKENS tokens (with many heads a part of them, with few as many times TOKENS as there are threads for), a
// thread eight numbers of TOKENS tokens at a time, which are asked for together.  Where all blocks are on the GPU at once anyway, one token is quicker (us, one / four: 1 token
// of 32 heads 1.6 / 1.7, 240 of 8 heads of 64 1.9 / 2.5, 500 of 8 heads 2.8 / 3.0; but 2000 5.3 / 5.0, 8000 17.0 / 12.6, 8000 of 32 heads 67 / 47).  Bound by the start of its
// blocks and two dependent loads each: 8000 tokens of 8 heads at 0.52 of the copy rate.
template <typename T, int D0, int TOKENS>
__global__ void __launch_bounds__(kGatherThreads) int4_gather_kernel(const Int4Pages kp, const Int4Pages vp, const int* slots, T* k, T* v, long n, int Hkv, int D1, int ps, long tokens, int abreast) {
  const int D = D0 ? D0 : D1, items = Hkv * (D / 8);
  pdl_trigger();
  pdl_wait();
  const bool key = blockIdx.z == 0;
  const Int4Pages& from = key ? kp : vp;
  const int mine = abreast > 1 ? (int)(threadIdx.x / (unsigned)items) : 0;       // which of the tokens
  const long t0 = (long)blockIdx.x * TOKENS * abreast + mine;
  if (mine >= abreast || t0 >= n) return;
  auto here = [&](int t) { return t0 + t * abreast < n; };
  const uint8_t* codes[TOKENS];
  const uint16_t* steps[TOKENS];
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    const int slot = here(t) ? slots[t0 + t * abreast] : -1;
    const bool there = slot >= 0 && slot < tokens;
    const int page = there ? slot / ps : 0, row = there ? slot - page * ps : 0;
    codes[t] = there ? from.codes + page * from.c_sp + row * from.c_sr : nullptr;
    steps[t] = from.steps + page * from.s_sp + row * from.s_sr;
  }
  T* const to = (key ? k : v) + t0 * Hkv * D;
  for (int i = blockIdx.y * kGatherThreads + threadIdx.x - mine * items; i < items; i += gridDim.y * kGatherThreads) {
    const int head = i / (D / 8), c = (i - head * (D / 8)) * 8;
    uint32_t word[TOKENS];
    uint16_t s16[TOKENS], m16[TOKENS];
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
      word[t] = 0;
      s16[t] = m16[t] = 0;
      if (codes[t]) {
        word[t] = *reinterpret_cast<const uint32_t*>(codes[t] + head * from.c_sh + c / 2);
        const uint16_t* const st = steps[t] + head * from.s_sh + c / 32;
        s16[t] = st[0];
        m16[t] = st[D / 32];
      }
    }
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
      if (!here(t)) break;
      const float s = __half2float(__ushort_as_half(s16[t])), m = __half2float(__ushort_as_half(m16[t]));
      Eight<T> out;                                        // without a slot: zeros
#pragma unroll
      for (int j = 0; j < 8; ++j) out.set(j, fmaf(__uint_as_float(0x4b000000u | (word[t] >> (4 * j) & 15)) - 0x1p23f, s, m));
      out.store(to + ((long)t * abreast * items + i) * 8);
    }
  }
}

// ----------------------------------------------------------------------------------------------- numbers for portions of prompts
constexpr int kUnpackThreads = 128, kUnpackEach = 4;       // packets of a thread at a time
// Pages of all sequences as halves, for the attention of many rows (paged_attention_sm100.cu), which the unpacked numbers serve many times: half of m + s c rounded
// once, so that a group whose ends are halves has none that is infinite; the units of the queries and the sums of the weights have the other factor.  Block (column of a
// sequence, head, keys or values), a thread 16 bytes at a time.  Keys that nobody sees are left as they are.  Bound by the start of its many small blocks:
// 2 sequences of 6000 keys, 8 heads of 64, 10 us, 25 MB written (16 numbers a thread: 12).
template <int D>
__global__ void __launch_bounds__(kUnpackThreads) int4_unpack_kernel(const Int4Attn p, __half* k, __half* v, int* table) {
  constexpr int C = D / 8;
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / p.cols, col = blockIdx.x % p.cols, head = blockIdx.y;
  const bool key = blockIdx.z == 0;
  int page = col < p.shared_cols ? p.shared_pages[col] : p.table[b * p.table_sb + col];
  if ((unsigned)page >= (unsigned)p.pages) page = -1;
  if (head == 0 && key && threadIdx.x == 0) table[blockIdx.x] = page < 0 ? -1 : (int)blockIdx.x;
  const int items = page < 0 ? 0 : min(p.ps, all_keys(p, b) - col * p.ps) * C;
  const uint8_t* const codes = key ? reinterpret_cast<const uint8_t*>(p.k) + (page * p.k_sp + head * p.k_sh) * 16 : reinterpret_cast<const uint8_t*>(p.v) + (page * p.v_sp + head * p.v_sh) * 16;
  const __half* const steps = key ? reinterpret_cast<const __half*>(p.ks) + (page * p.ks_sp + head * p.ks_sh) * (D / 16) : reinterpret_cast<const __half*>(p.vs) + (page * p.vs_sp + head * p.vs_sh) * (D / 16);
  const long c_sr = (key ? p.k_sr : p.v_sr) * 16, s_sr = (key ? p.ks_sr : p.vs_sr) * (D / 16);
  __half* const to = (key ? k : v) + ((long)blockIdx.x * p.Hkv + head) * p.ps * D;
  for (int i0 = threadIdx.x; i0 < items; i0 += kUnpackThreads * kUnpackEach) {
    uint32_t word[kUnpackEach];
    __half s[kUnpackEach], m[kUnpackEach];
#pragma unroll
    for (int y = 0; y < kUnpackEach; ++y) {
      const int i = i0 + y * kUnpackThreads, row = i / C, c = i % C;
      if (i < items) {
        word[y] = *reinterpret_cast<const uint32_t*>(codes + row * c_sr + c * 4);
        s[y] = steps[row * s_sr + c / 4];
        m[y] = steps[row * s_sr + D / 32 + c / 4];
      }
    }
#pragma unroll
    for (int y = 0; y < kUnpackEach; ++y) {
      const int i = i0 + y * kUnpackThreads;
      if (i >= items) break;
      const __half2 half2x = __float2half2_rn(0.5f), s2 = __half2half2(s[y]), m2 = __hmul2(__half2half2(m[y]), half2x);
      uint32_t o[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t two = word[y] >> (8 * x);           // numbers 2 x and 2 x + 1
        o[x] = as_u32(__hfma2(__hfma2(as_half2((two & 0xfu) | (two & 0xf0u) << 12 | 0x64006400u), half2x, __float2half2_rn(-512.f)), s2, m2));
      }
      *reinterpret_cast<uint4*>(to + (long)i * 8) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// Queries as halves: a row is multiplied by a power of two that brings its largest number to 2^14; the row's unit takes that back, and that keys are halved.  A thread has
// eight numbers.  2 x 1000 tokens of 48 heads of 64: 6 us, 25 MB.
template <int D>
__global__ void __launch_bounds__(128) int4_queries_kernel(const __nv_bfloat16* q, __half* out, float* units, unsigned rows, unsigned W, unsigned H, long q_sb, long q_sw,
                                                           long q_sh) {
  constexpr unsigned C = D / 8;
  pdl_trigger();
  pdl_wait();
  const unsigned r = (blockIdx.x * 128 + threadIdx.x) / C, c = threadIdx.x % C;
  const unsigned mask = (C == 16 ? 0xffffu : 0xffu) << (threadIdx.x % 32 / C * C);       // a row's threads
  if (r >= rows) return;
  const unsigned h = r % H, t = r / H, w = t % W, b = t / W;
  Eight<__nv_bfloat16> x;
  x.load(q + b * q_sb + w * q_sw + h * q_sh + c * 8);
  float most = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(x.f(k)));
#pragma unroll
  for (int k = 1; k < (int)C; k <<= 1) most = fmaxf(most, __shfl_xor_sync(mask, most, k));
  const int e = min(max((int)(__float_as_uint(most) >> 23), 20), 244);
  const float up = __uint_as_float((uint32_t)(268 - e) << 23);
  uint32_t o[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) o[k] = pack_half(x.f(2 * k) * up, x.f(2 * k + 1) * up);
  reinterpret_cast<uint4*>(out)[(size_t)r * C + c] = make_uint4(o[0], o[1], o[2], o[3]);
  if (c == 0) units[r] = __uint_as_float((uint32_t)(e - 13) << 23);
}

// ------------------------------------------------------------------------------------------------------- attention, up to eight rows
constexpr int kRowWarps = 8;                               // two blocks an SM; the warps have a pair's keys in turn
template <int D> constexpr int kRing = kRowWarps * kStages * kStage<D>;
template <int D> constexpr int kSums = kRowWarps * 8 * kPitch<D> * 4;        // sums of the warps
// a cluster's sums lie over the ring, which has been read by then; otherwise the ring runs on while sums are written
template <int D, bool CLUSTER> constexpr int rows_smem = kQueries<D, 1> + (CLUSTER ? std::max(kRing<D>, kSums<D> + 8 * D * 4) : kRing<D> + kSums<D>);

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
//
// Bound by how few warps hide one another's latencies: some 220 instructions of a warp for 16 keys, 18 of them products of 8 cycles each, from four warps a scheduler (127
// registers), which issue in 53 of 100 cycles and wait for fixed latencies most; the pipes of logic and of products are busy for 40 and 21 of 100.  1030 cycles an SM for 128
// keys where memory would take 650 (16 sequences of 8192 keys, 8 heads: 37 us, 3.4 TB/s; copies alone take 26).
template <typename T, int D, bool CLUSTER>
__global__ void __launch_bounds__(kRowWarps * 32, 2) int4_rows_kernel(const Int4Attn p) {
  constexpr bool TWO = std::is_same<T, __half>::value;     // weights as two halves
  constexpr int NG = D / 32, PITCH = kPitch<D>, WARPS = kRowWarps, THREADS = WARPS * 32, STAGE = kStage<D>, TILE = WARPS * kKeys;
  constexpr int V_AT = kKeys * (D / 2), KS_AT = 2 * V_AT, VS_AT = KS_AT + kKeys * 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sm_m[WARPS][8], sm_l[WARPS][8], sm_bm[8], sm_bl[8];
  __shared__ Walk sm_ahead[WARPS];
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
  const uint32_t sm_q = (uint32_t)__cvta_generic_to_shared(smem), sm_qs = sm_q + 8 * kQPitch<D>, ring0 = sm_q + kQueries<D, 1>;
  float* const sm_unit = reinterpret_cast<float*>(smem + 8 * (kQPitch<D> + 16));
  int* const sm_lim = reinterpret_cast<int*>(sm_unit + 8);
  // sums of the warps [warp][8 rows][PITCH] and of a cluster's block [8][D]
  float* const sm_o = reinterpret_cast<float*>(smem + kQueries<D, 1> + (CLUSTER ? 0 : kRing<D>));
  float* const sm_b = reinterpret_cast<float*>(smem + kQueries<D, 1> + kSums<D>);
  Ring<D, WARPS, CLUSTER> ring(p, sm_ahead + warp, cur, tiles_left, step, ring0 + warp * (kStages * STAGE), warp, lane);
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) ring.ask(s);

  uint32_t qf[NG][4], qs;                                  // queries of group g: two steps of 16 numbers; sums of queries
  float m[2], l[2], o[2 * NG][4], om[4], unit[2];          // of rows 2 quad and 2 quad + 1
  int lim[2], lim_all = 0;                                 // first key that a row does not see; that none of the live rows has before it
  float room = 15.f;                                       // weights relative to M may be at most 2^room: 15 less what the largest s needs
  __half2 s_most2 = __half2half2(__ushort_as_half(0x3c00));                              // 2^(15 - room), twice
  bool whole = false;                                      // the pair begins in this block
  int row0 = 0, rows = 0;                                  // of the entry
  auto begin = [&] {
    const int b = cur.e / p.row_tiles, count = new_tokens(p, b), n = keys_of(p, cur.e);
    row0 = cur.e % p.row_tiles * p.tile_rows;
    rows = min(8, p.W * p.G - row0);
    whole = CLUSTER || cur.tile == 0;
    lim_all = min(visible_keys(p, b, row0 / p.G), n);
    {                                                      // a row a warp
      const int w = (row0 + warp) / p.G;
      const bool live = warp < rows && w < count;
      ready_query<T, D>(reinterpret_cast<const T*>(p.q) + (live ? b * p.q_sb + w * p.q_sw + (long)(cur.head * p.G + (row0 + warp) % p.G) * p.q_sh : 0), live,
                        sm_q + warp * kQPitch<D>, sm_qs + warp * 16, sm_unit + warp, p.scale_log2, lane);
      if (lane == 0) sm_lim[warp] = live ? min(visible_keys(p, b, w), n) : 0;
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < NG; ++g) ldmatrix_x4(qf[g], sm_q + (lane & 7) * kQPitch<D> + g * 64 + (lane >> 3) * 16);
    qs = lds32(sm_qs + hq * 16 + quad * 4);
#pragma unroll
    for (int k = 0; k < 2 * NG; ++k)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[k][x] = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) om[x] = 0.f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      unit[x] = sm_unit[quad * 2 + x];
      lim[x] = sm_lim[quad * 2 + x];
      m[x] = kNone;
      l[x] = 0.f;
    }
  };

  // the warps' sums of the pair, to the output or to a part
  auto finish = [&](bool last) {
    const int kvh = cur.head, b = cur.e / p.row_tiles, count = new_tokens(p, b);
    const bool direct = whole && last;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], s);
      if (hq == 0) sm_m[warp][quad * 2 + e] = m[e] == kNone ? -INFINITY : m[e];
    }
    __syncthreads();                                       // all of the ring has been read (a cluster's), and what was read of the last pair's sums
    // every warp's sums relative to the block's maximum
    float f[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = quad * 2 + e;
      float mn = sm_m[hq][row];
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, s));
      f[e] = mn == -INFINITY || m[e] == kNone ? 0.f : exp2f(m[e] - mn);
      if (hq == 0) {
        sm_l[warp][row] = l[e] * f[e];
        if (warp == 0) sm_bm[row] = mn;
      }
    }
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // what m adds to group g stands in row NG + g of its product
        const float m0 = __shfl_sync(0xffffffffu, om[e], (NG + g) * 4 + quad) * f[e], f24 = f[e] * 0x1p24f, f20 = f[e] * 0x1p20f;
        *reinterpret_cast<float4*>(sm_o + (warp * 8 + quad * 2 + e) * PITCH + g * 32 + hq * 4) =
            make_float4(fmaf(o[2 * g][e], f24, m0), fmaf(o[2 * g][e + 2], f20, m0), fmaf(o[2 * g + 1][e], f24, m0), fmaf(o[2 * g + 1][e + 2], f20, m0));
      }
    __syncthreads();
    constexpr int PER = THREADS / D;                       // rows at a time
#pragma unroll
    for (int x = 0; x < 8 / PER; ++x) {
      const int row = x * PER + (int)threadIdx.x / D, col = threadIdx.x % D;
      if (row >= rows) break;
      float acc = 0.f, ls = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        acc += sm_o[(w * 8 + row) * PITCH + col];
        ls += sm_l[w][row];
      }
      if (CLUSTER && p.cluster > 1) {
        sm_b[row * D + col] = acc;
        if (col == 0) sm_bl[row] = ls;
      } else if (direct) {
        const int w = (row0 + row) / p.G;
        const bool live = w < count && !(ls == 0.f);
        reinterpret_cast<T*>(p.out)[b * p.o_sb + w * p.o_sw + (long)(kvh * p.G + (row0 + row) % p.G) * p.o_sh + col] = from_f32<T>(live ? acc / ls : 0.f);
      } else {
        const long slot = part_slot<false>(p, (long)cur.e * p.Hkv + kvh, blockIdx.x, whole) * p.tile_rows + row;
        p.part_o[slot * D + col] = acc;
        if (col == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(sm_bm[row], ls);
      }
    }
  };

  // 16 keys from `key` on, which lie in shared memory at `at`
  auto tile = [&](const uint32_t at, const int key) {
    const int rr = lane & 15, rc = lane >> 4;              // whose 16 bytes of codes this lane has ldmatrix read: row, group
    // scores: keys hq and hq + 8, rows 2 quad and 2 quad + 1
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    const uint32_t km = at + KS_AT + hq * 16 + NG * 2 + (NG == 4 ? (quad & 1) * 4 : 0);
    mma1688(s, lds32(km), lds32(km + 8 * 16), qs);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] *= 0x1p-19f;          // sums of q were divided by 2^5, codes by 2^24
    const uint2 a0 = lds64(at + KS_AT + hq * 16), b0 = lds64(at + KS_AT + (hq + 8) * 16);
    const uint32_t ua[2] = {a0.x, a0.y}, ub[2] = {b0.x, b0.y};
#pragma unroll
    for (int g = 0; g < NG; g += 2) {
      const float2 s0 = __half22float2(as_half2(ua[g / 2])), s1 = __half22float2(as_half2(ub[g / 2]));
      uint32_t a[4];                                       // keys hq, hq + 8 of group g, of group g + 1: eight codes each
      ldmatrix_x4(a, at + chunk_at<D>(rr, g + rc));
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const Codes k0 = codes_of(a[2 * x]), k1 = codes_of(a[2 * x + 1]);
        const float f0 = x ? s0.y : s0.x, f1 = x ? s1.y : s1.x;
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        mma16816(d, k0.c0, k1.c0, k0.c1, k1.c1, qf[g + x][0], qf[g + x][1]);
        mma16816(d, k0.c2, k1.c2, k0.c3, k1.c3, qf[g + x][2], qf[g + x][3]);
        s[0] = fmaf(d[0], f0, s[0]);
        s[1] = fmaf(d[1], f0, s[1]);
        s[2] = fmaf(d[2], f1, s[2]);
        s[3] = fmaf(d[3], f1, s[3]);
      }
    }
    // steps of the values: row x of the operand is the x-th number of the steps (s of all groups, then m) of keys 2 quad, 2 quad + 1, and of those + 8
    uint32_t va[2];
    const uint32_t vs_at = at + VS_AT + rr * 16;
    ldmatrix_x2t(va, vs_at);
    const uint32_t mine = lds32(vs_at + (NG == 4 ? rc * 4 : 0));        // two s of one key
    bool passed = !__hble2(as_half2(mine), s_most2);
    if (key + kKeys > lim_all) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (key + hq + (e >> 1) * 8 >= lim[e & 1]) s[e] = -INFINITY;
    }
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = fmaf(s[e], unit[e & 1], -m[e & 1]);
    passed = passed || fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) > room;
    // a weight, or a weight times s, would pass 2^15: another reference, 2^3 away from that
    if (__any_sync(0xffffffffu, passed)) {
      // the largest s, as a half's bits (NaN: as it comes), and the power of two above it
      const uint32_t most = __reduce_max_sync(0xffffffffu, max(mine & 0xffffu, mine >> 16));
      if (most > (as_u32(s_most2) & 0xffffu)) {
        const int e = min((int)(most >> 10) - 15 + 1, 16);
        s_most2 = e < 16 ? __half2half2(__ushort_as_half((unsigned short)((e + 15) << 10))) : __half2half2(__ushort_as_half(0x7bff));
        room = 15.f - e;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(s[e], s[e + 2]) * unit[e];
#pragma unroll
        for (int y = 4; y < 32; y <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, y));
        const float mn = fmaxf(m[e], mx - (room - 3.f)), f = exp2f(m[e] - mn);      // none before: 0
        m[e] = mn;
        l[e] *= f;
        om[e] *= f;
        om[e + 2] *= f;
#pragma unroll
        for (int k = 0; k < 2 * NG; ++k) { o[k][e] *= f; o[k][e + 2] *= f; }
        x[e] = fmaf(s[e], unit[e], -mn);
        x[e + 2] = fmaf(s[e + 2], unit[e], -mn);
      }
    }
    uint32_t ph[2], pl[2] = {0u, 0u};                      // weights as the second product's operand: rounded, and what that left
    {
      float pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pr[e] = exp2f(x[e]);
        l[e & 1] += pr[e];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t hi = pack_half(pr[2 * e], pr[2 * e + 1]);
        ph[e] = transpose8x8(hi);
        if constexpr (TWO) {
          const float2 f = __half22float2(as_half2(hi));
          pl[e] = transpose8x8(pack_half(pr[2 * e] - f.x, pr[2 * e + 1] - f.y));
        }
      }
    }
    // A product adds to what it is given by cutting off, always towards zero, and the two sums are a hundred times their difference where keys are many: results in half
    // precision would show it (26,000 keys: 0.00033 against 64 bits for 0.0002), so that their products begin at zero and are added here.
    auto weigh = [&](float (&sum)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const __half2 (&w)[2], const __half2 (&left)[2]) {
      if constexpr (TWO) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        mma16816(d, a0, a1, a2, a3, as_u32(w[0]), as_u32(w[1]));
        mma16816(d, a0, a1, a2, a3, as_u32(left[0]), as_u32(left[1]));
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += d[e];
      } else {
        mma16816(sum, a0, a1, a2, a3, as_u32(w[0]), as_u32(w[1]));
      }
    };
    const __half2 p2[2] = {as_half2(ph[0]), as_half2(ph[1])}, left2[2] = {as_half2(pl[0]), as_half2(pl[1])};
    weigh(om, va[0], 0u, va[1], 0u, p2, left2);
#pragma unroll
    for (int g = 0; g < NG; g += 2) {
      uint32_t a[4];                                       // keys 2 quad.. and 8 + 2 quad.. of group g, of group g + 1: four codes of either key
      ldmatrix_x4t(a, at + V_AT + chunk_at<D>(rr, g + rc));
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const Codes v0 = codes_of(a[2 * y]), v1 = codes_of(a[2 * y + 1]);
        __half2 w[2], left[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const __half2 s = as_half2(__shfl_sync(0xffffffffu, va[k], (g + y) * 4 + quad));
          w[k] = __hmul2(p2[k], s);
          if constexpr (TWO) left[k] = __hfma2(left2[k], s, __hfma2(p2[k], s, __hneg2(w[k])));          // what the roundings of the weight and of its product with s left
        }
        weigh(o[2 * (g + y)], v0.c0, v0.c1, v1.c0, v1.c1, w, left);
        weigh(o[2 * (g + y) + 1], v0.c2, v0.c3, v1.c2, v1.c3, w, left);
      }
    }
  };

  if (CLUSTER || tiles_left > 0) begin();
  int stage = 0, ask_stage = kStages - 1;
  for (int t = 0; t < tiles_left; ++t) {
    cp_async_wait<kStages - 2>();
    __syncwarp();                                          // tile t of all lanes is there; all lanes are done with tile t - 1
    const bool hole = ring.template hole<kStages>();
    ring.ask(ask_stage);
    ask_stage = ask_stage + 1 == kStages ? 0 : ask_stage + 1;
    if (!hole) tile(ring.ring + stage * STAGE, cur.tile * TILE + warp * kKeys);
    stage = stage + 1 == kStages ? 0 : stage + 1;
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
    if (p.cluster > 1) join_cluster<T, D, THREADS>(p, cur, row0, rows, sm_b, sm_bm, sm_bl, 1.f);
  } else {
    finish_idle_warps<T, D, WARPS>(p, warp, lane);
  }
}

// Joins the parts of pairs that are cut: block (x, r) row r of pair x, or, where there are fewer blocks than pairs (CUTS), of the pair that is cut first in front
// of block x + 1's share; each warp has a quarter of the parts.  Bound by its start and two dependent loads, 5 us.
template <typename T, int D, bool CUTS>
__global__ void __launch_bounds__(kThreads) int4_merge_kernel(const Int4Attn p, int grid, float factor) {
  constexpr int C = D / 32, AHEAD = 8;
  __shared__ float sums[kWarps][D], ms[kWarps], ls[kWarps];
  __shared__ long before[2][kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.y;
  // the kernel before this one waited for all that positions come from
  int e, head, first;                                                  // first: block that has the pair's first part
  long t0, per;                                                        // the pair's first tile of all, tiles of a block
  if constexpr (CUTS) {
    const Place at = find_place<kThreads, false>(p, grid, blockIdx.x + 1);
    e = at.e;
    if (e >= p.B * p.row_tiles) return pdl_wait();
    const int tiles = entry_tiles(p, e);
    head = (int)(at.tile / tiles);
    const long off = at.tile % tiles;
    per = at.per;
    t0 = (blockIdx.x + 1) * per - off;
    if (off == 0 || off > per) return pdl_wait();                      // not cut here, or before
    first = blockIdx.x;
  } else {
    e = blockIdx.x / p.Hkv;
    head = blockIdx.x % p.Hkv;
    int ahead = 0, all = 0;
    for (int i = threadIdx.x; i < p.B * p.row_tiles; i += kThreads) {
      const int t = entry_tiles(p, i);
      all += t;
      if (i < e) ahead += t;
    }
    ahead = __reduce_add_sync(0xffffffffu, ahead);
    all = __reduce_add_sync(0xffffffffu, all);
    if (lane == 0) { before[0][warp] = ahead; before[1][warp] = all; }
    __syncthreads();
    long total = 0;
    t0 = 0;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) { t0 += before[0][x]; total += before[1][x]; }
    total *= p.Hkv;
    per = max((long)p.min_tiles, (total + grid - 1) / grid);
    const int tiles = entry_tiles(p, e);
    t0 = t0 * p.Hkv + (long)head * tiles;
    first = (int)(t0 / per);
    if (tiles == 0 || (t0 + tiles - 1) / per == first) return pdl_wait();          // not cut
  }
  pdl_wait();
  pdl_trigger();                                           // not before: blocks of the next launch would stand where the first one's should
  const int tiles = entry_tiles(p, e), b = e / p.row_tiles, n = (int)((t0 + tiles - 1) / per) - first + 1;
  const int row = e % p.row_tiles * p.tile_rows + r, w = row / p.G;
  if (row >= p.W * p.G) return;
  float m = -INFINITY, l = 0.f, acc[C] = {};
  const int mine = (n - warp + kWarps - 1) / kWarps;                   // parts warp, warp + 4, ...
  auto slot = [&](int x) { return part_slot<false>(p, 0, first + warp + kWarps * x, warp + x == 0) * p.tile_rows + r; };
  for (int x0 = 0; x0 < mine; x0 += 32) {
    const int here = min(32, mine - x0);
    const float2 a = lane < here ? reinterpret_cast<const float2*>(p.part_ml)[slot(x0 + lane)] : make_float2(-INFINITY, 0.f);
    float v[AHEAD][C];
    auto ask = [&](int x1) {
#pragma unroll
      for (int x = 0; x < AHEAD; ++x)
        if (x1 + x < here) {
          const float* src = p.part_o + slot(x0 + x1 + x) * D + lane * C;
          if constexpr (C == 4) *reinterpret_cast<float4*>(v[x]) = *reinterpret_cast<const float4*>(src);
          else *reinterpret_cast<float2*>(v[x]) = *reinterpret_cast<const float2*>(src);
        }
    };
    ask(0);
    const float mn = fmaxf(m, warp_max(a.x)), old = m == -INFINITY ? 0.f : exp2f(m - mn), f = a.x == -INFINITY ? 0.f : exp2f(a.x - mn);
    l = l * old + warp_sum(a.y * f);
    m = mn;
#pragma unroll
    for (int j = 0; j < C; ++j) acc[j] *= old;
    for (int x1 = 0; x1 < here; x1 += AHEAD) {
      if (x1) ask(x1);
#pragma unroll
      for (int x = 0; x < AHEAD; ++x) {
        const float g = __shfl_sync(0xffffffffu, f, (x1 + x) & 31);
#pragma unroll
        for (int j = 0; j < C; ++j) acc[j] += x1 + x >= here || g == 0.f ? 0.f : v[x][j] * g;        // a part without weights has no sums
      }
    }
  }
#pragma unroll
  for (int j = 0; j < C; ++j) sums[warp][lane * C + j] = acc[j];
  if (lane == 0) { ms[warp] = m; ls[warp] = l; }
  __syncthreads();
  if (threadIdx.x >= D) return;
  float mn = -INFINITY, total = 0.f, o = 0.f;
#pragma unroll
  for (int x = 0; x < kWarps; ++x) mn = fmaxf(mn, ms[x]);
#pragma unroll
  for (int x = 0; x < kWarps; ++x) {
    const float f = mn == -INFINITY ? 0.f : exp2f(ms[x] - mn);
    total += ls[x] * f;
    o += sums[x][threadIdx.x] * f;
  }
  const bool live = w < new_tokens(p, b) && !(total == 0.f);
  reinterpret_cast<T*>(p.out)[b * p.o_sb + w * p.o_sw + (long)(head * p.G + row % p.G) * p.o_sh + threadIdx.x] = from_f32<T>(live ? factor * o / total : 0.f);
}

template <typename T, int D, bool CLUSTER>
void launch_rows(const Int4Attn& p, int grid, cudaStream_t st) {
  constexpr int smem = rows_smem<D, CLUSTER>;
  NXD_ALLOW_SMEM((int4_rows_kernel<T, D, CLUSTER>), smem);
  launch_cluster(int4_rows_kernel<T, D, CLUSTER>, p, grid, kRowWarps * 32, smem, CLUSTER ? p.cluster : 1, st);
}
template <typename T, int D>
int launch(const Int4Attn& p, const PagedPlan& plan, int dt, cudaStream_t st) {
  if (p.tile_rows > 8) int4_tiles(p, plan.grid, D, dt, st);
  else if (p.cluster) launch_rows<T, D, true>(p, plan.grid, st);
  else launch_rows<T, D, false>(p, plan.grid, st);
  if (p.cluster || plan.grid <= 1) return 1;
  const int rows = std::min(p.tile_rows, p.W * p.G);
  const long pairs = (long)p.B * p.row_tiles * p.Hkv;
  const float factor = p.tile_rows > 8 ? 2.f : 1.f;        // the tiles' values are halved
  if (pairs < plan.grid) launch_dependent(int4_merge_kernel<T, D, false>, dim3((unsigned)pairs, rows), kThreads, 0, st, p, plan.grid, factor);
  else launch_dependent(int4_merge_kernel<T, D, true>, dim3(plan.grid - 1, rows), kThreads, 0, st, p, plan.grid, factor);
  return 2;
}

}  // namespace

PagedPlan int4_plan(Int4Attn& p, int D, int dt) {
  PagedPlan plan{};
  const int sms = device_sm_count();
  const long rows = (long)p.W * p.G;
  // more than eight rows in row tiles of up to 40, alike
  p.row_tiles = rows <= 8 ? 1 : (int)((rows + 39) / 40);
  p.tile_rows = rows <= 8 ? 8 : std::max(16, (int)((rows + 8l * p.row_tiles - 1) / (8l * p.row_tiles)) * 8);
  p.row_tiles = (int)((rows + p.tile_rows - 1) / p.tile_rows);
  p.tile_keys = 128;
  p.min_tiles = 1;
  p.whole_tiles = 0;
  p.shared = 0;
  const int each = 2;                                      // blocks of an SM
  const long heads = (long)p.B * p.Hkv, pairs = heads * p.row_tiles, cap = (long)p.cols * p.ps;
  // Every row tile reads and unpacks the keys for itself, 0.115 us for 1000 keys of a head over the GPU; unpacking them once to half precision for the tensor memory
  // takes 0.19 us for 1000 and 18 us in all (us, row tiles / unpacked: 8 sequences to 6000 keys, 8 heads, 64 rows 81 / 93, 96 rows 134 / 96; 2 to 3000, 8
  // heads, 128 rows 30 / 36, 256 rows 54 / 40; 1 to 1000, 40 heads, 200 rows 26 / 31; 2 x 1000 tokens to 6000, 48 heads of 64 on 8, 504 / 169).
  // Results in half precision would show that keys, values and weights are rounded to halves there (0.0004 against 64 bits, where rounding the result costs 0.00021; row tiles
  // 0.00028), those in bf16 hardly do (0.00169 and 0.00168, where rounding the result costs 0.00166; with keys of six times that size 0.00177 and 0.00167).
  // A head whose table alone would take more than 1 GB of memory (2 million tokens of 128 numbers) is not unpacked.
  plan.tiles = dt == kBF16 && cap <= (1l << 28) / D && (23l * p.row_tiles - 38) * heads * cap > 3600000;
  if (plan.tiles) return plan;
  plan.grid = each * sms;
  // A cluster per pair, as many blocks in it as the GPU takes at once, has neither a search for places nor a second launch, but the longest sequence lasts as long as
  // its own blocks take (us, dealt out / cluster: 1 sequence of 300 keys, 8 heads, 11.1 / 6.2; 16 to 8192 keys, 8 heads, 41.7 / 38.2; 6 to 2500, 40
  // heads, 30.5 / 25.1; but 1 of 100000, 8 heads, 36.5 / 49.6): 4096 keys a block at most.
  int size = 1;
  while (size < kCluster8 && ((cap > 512l * size && pairs * size * 2 <= (long)each * sms) || cap > 4096l * size)) size *= 2;
  if (cap <= 4096l * size && pairs * size < (1l << 30)) {
    p.cluster = size;
    plan.grid = (int)(pairs * size);
  }
  plan.slots = p.cluster ? 0l : 2l * plan.grid * p.tile_rows;
  p.slots = plan.slots;
  return plan;
}

int int4_attention(const Int4Attn& p, const PagedPlan& plan, int D, int dt, cudaStream_t st) {
  if (dt == kBF16) return D == 128 ? launch<__nv_bfloat16, 128>(p, plan, dt, st) : launch<__nv_bfloat16, 64>(p, plan, dt, st);
  return D == 128 ? launch<__half, 128>(p, plan, dt, st) : launch<__half, 64>(p, plan, dt, st);
}

void int4_unpack(const Int4Attn& p, void* k, void* v, int* table, int D, cudaStream_t st) {
  const long blocks = (long)p.B * p.cols;
  if (blocks == 0) return;
  if (blocks >= (1l << 31) || p.Hkv > 65535) nxd_throw("int4_unpack: too many keys", __FILE__, __LINE__);
  const dim3 grid((unsigned)blocks, p.Hkv, 2);
  if (D == 128) launch_dependent(int4_unpack_kernel<128>, grid, kUnpackThreads, 0, st, p, (__half*)k, (__half*)v, table);
  else launch_dependent(int4_unpack_kernel<64>, grid, kUnpackThreads, 0, st, p, (__half*)k, (__half*)v, table);
}
void int4_queries(const void* q, void* out, float* units, int B, int W, int H, int D, long q_sb, long q_sw, long q_sh, cudaStream_t st) {
  const long rows = (long)B * W * H;
  if (rows == 0) return;
  if (rows * (D / 8) >= (1l << 31)) nxd_throw("int4_queries: too many rows", __FILE__, __LINE__);
  const unsigned grid = (unsigned)((rows * (D / 8) + 127) / 128);
  if (D == 128) launch_dependent(int4_queries_kernel<128>, grid, 128, 0, st, (const __nv_bfloat16*)q, (__half*)out, units, (unsigned)rows, W, H, q_sb, q_sw, q_sh);
  else launch_dependent(int4_queries_kernel<64>, grid, 128, 0, st, (const __nv_bfloat16*)q, (__half*)out, units, (unsigned)rows, W, H, q_sb, q_sw, q_sh);
}

int int4_append(const Int4Append& p, int dt, cudaStream_t st) {
  const bool two = p.D % 64 == 0;                          // eight numbers of each half: four threads have the same 32 in either
  const long tokens = (long)p.B * p.W;
  if (tokens == 0) return 0;
  int launches = 0;
  auto go = [&](auto kernel, int heads) {
    const long parts = ((long)heads * (p.D / (two ? 16 : 8)) + kAppendThreads - 1) / kAppendThreads;
    if (tokens >= (1l << 31) || parts > 65535) nxd_throw("int4_append: too many tokens or heads", __FILE__, __LINE__);
    launch_dependent(kernel, dim3((unsigned)tokens, (unsigned)parts), kAppendThreads, 0, st, p);
    ++launches;
  };
  auto split = [&](auto all, auto queries, auto cache) {
    if (tokens < kSplitTokens) return go(all, p.H + 2 * p.Hkv);
    go(queries, p.H);
    go(cache, 2 * p.Hkv);
  };
#define NXD_TURN(Dv, turn) split(int4_append_kernel<T, Dv, turn, 2, kAll>, int4_append_kernel<T, Dv, turn, 2, kQuery>, int4_append_kernel<T, Dv, turn, 2, kCache>)
  auto typed = [&](auto zero) {
    using T = decltype(zero);
    if (!two) return p.pairs ? go(int4_append_kernel<T, 0, kPairs, 1, kAll>, p.H + 2 * p.Hkv) : go(int4_append_kernel<T, 0, kPart, 1, kAll>, p.H + 2 * p.Hkv);
    if (p.pairs) return p.D == 128 ? NXD_TURN(128, kPairs) : NXD_TURN(0, kPairs);
    if (2 * p.half == p.D) return p.D == 128 ? NXD_TURN(128, kHalves) : NXD_TURN(0, kHalves);
    return p.D == 128 ? NXD_TURN(128, kPart) : NXD_TURN(0, kPart);
  };
#undef NXD_TURN
  if (dt == kBF16) typed(__nv_bfloat16());
  else if (dt == kF16) typed(__half());
  else typed(float());
  return launches;
}

void int4_gather(const Int4Pages& kp, const Int4Pages& vp, const int* slots, void* k, void* v, long n, int Hkv, int D, int ps, long tokens, int dt, cudaStream_t st) {
  if (n == 0) return;
  if (n >= (1l << 31)) nxd_throw("int4_gather: too many tokens", __FILE__, __LINE__);
  const int items = Hkv * (D / 8), abreast = std::max(1, kGatherThreads / items), parts = std::min(64, (items + kGatherThreads - 1) / kGatherThreads);
  const bool one = (n + abreast - 1) / abreast * parts * 2 <= 16l * device_sm_count();
  const int tokens_at = (one ? 1 : 4) * abreast;
  const dim3 grid((unsigned)((n + tokens_at - 1) / tokens_at), parts, 2);
  auto go = [&](auto* k, auto* v, auto kernel) { launch_dependent(kernel, grid, kGatherThreads, 0, st, kp, vp, slots, k, v, n, Hkv, D, ps, tokens, abreast); };
  auto typed = [&](auto zero) {
    using T = decltype(zero);
    if (one) D == 128 ? go((T*)k, (T*)v, int4_gather_kernel<T, 128, 1>) : go((T*)k, (T*)v, int4_gather_kernel<T, 0, 1>);
    else D == 128 ? go((T*)k, (T*)v, int4_gather_kernel<T, 128, 4>) : go((T*)k, (T*)v, int4_gather_kernel<T, 0, 4>);
  };
  if (dt == kBF16) typed(__nv_bfloat16());
  else if (dt == kF16) typed(__half());
  else typed(float());
}

}  // namespace nxd
