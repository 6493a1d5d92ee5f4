// Bindings of the paged key/value cache in 4 bits and of the page tables: checks of arguments, workspaces, launches.
#include <cmath>
#include <limits>

#include "paged_checks.h"

namespace {

struct Pool { const Tensor &k_codes, &k_steps, &v_codes, &v_steps; };

void check_pool(const Pool& p) {
  for (const auto& [codes, steps] : {std::pair<const Tensor&, const Tensor&>{p.k_codes, p.k_steps}, {p.v_codes, p.v_steps}}) {
    CHECK_ARG(codes.dim() == 4 && codes.scalar_type() == at::kByte && steps.dim() == 5 && steps.scalar_type() == at::kHalf,
              "pages are uint8 codes [pages, page size, heads, head size / 2] and float16 steps [pages, page size, heads, 2, head size / 32]");
    CHECK_ARG(codes.sizes().slice(0, 3) == steps.sizes().slice(0, 3) && codes.size(3) > 0 && codes.size(3) % 16 == 0 && steps.size(3) == 2 &&
              steps.size(4) * 16 == codes.size(3), "codes " + list(codes.sizes()) + " and steps " + list(steps.sizes()) + " do not match");
  }
  CHECK_ARG(p.k_codes.sizes() == p.v_codes.sizes(), "keys " + list(p.k_codes.sizes()) + " and values " + list(p.v_codes.sizes()) + " do not match");
  for (const Tensor* t : {&p.k_steps, &p.v_codes, &p.v_steps}) CHECK_ARG(t->device() == p.k_codes.device(), "all tensors are on one device");
  const int64_t ps = p.k_codes.size(1);
  CHECK_ARG(p.k_codes.size(0) > 0 && p.k_codes.size(2) > 0 && ps > 0 && ps % 16 == 0, "a page holds a multiple of 16 tokens, got " + std::to_string(ps));
  CHECK_ARG(p.k_codes.size(0) * ps < (1ll << 31), "a pool of too many tokens");
}
void check_queries(const Tensor& q, const Pool& p) {
  CHECK_ARG(q.dim() == 4, "queries are [batch, new tokens, heads, head size]");
  CHECK_ARG(q.size(2) > 0 && q.size(2) % p.k_codes.size(2) == 0,
            std::to_string(q.size(2)) + " query heads do not go with " + std::to_string(p.k_codes.size(2)) + " key heads");
  CHECK_ARG(q.size(3) == 2 * p.k_codes.size(3), "heads of " + std::to_string(q.size(3)) + " numbers, pages of " + std::to_string(2 * p.k_codes.size(3)));
  CHECK_ARG(q.device() == p.k_codes.device(), "queries and pages are on one device");
  CHECK_ARG(q.size(0) < (1 << 20) && q.size(1) < (1 << 24) && q.size(0) * q.size(1) * q.size(2) < (1ll << 30), "too many query rows: " + list(q.sizes()));
}
bool float_type(const Tensor& t) { return half_type(t) || t.scalar_type() == at::kFloat; }
// Places within a pool are counted in 32 bits: packets of 16 bytes of codes, rows of steps
bool places_ok(const Tensor& t, int64_t unit, int64_t behind) {
  int64_t last = behind;
  for (int64_t d = 0; d < 3; ++d) {
    if (t.size(d) <= 1) continue;
    if (t.stride(d) < 0 || t.stride(d) / unit > (1ll << 32) / (t.size(d) - 1)) return false;
    last += (t.size(d) - 1) * (t.stride(d) / unit);
  }
  return last < (1ll << 32) - 1;
}
// Codes in whole 16-byte packets, a row's steps beside one another and aligned to all of them where they are 8 or 16 bytes
bool pages_ok(const Tensor& codes, const Tensor& steps) {
  if (codes.dim() != 4 || steps.dim() != 5 || !packets(codes)) return false;
  const int64_t row = 2 * steps.size(4), bytes = row == 4 || row == 8 ? 2 * row : 2;
  bool ok = steps.stride(4) == 1 && steps.stride(3) == steps.size(4) && (uintptr_t)steps.data_ptr() % bytes == 0;
  if (steps.size(4) == 1) ok = steps.stride(3) == 1 && (uintptr_t)steps.data_ptr() % 2 == 0;
  for (int64_t d = 0; d < 3; ++d) ok = ok && (steps.size(d) <= 1 || steps.stride(d) * 2 % bytes == 0);
  return ok;
}
bool pool_ok(const Pool& p) { return pages_ok(p.k_codes, p.k_steps) && pages_ok(p.v_codes, p.v_steps); }

nxd::Int4Pages pages_of(const Tensor& codes, const Tensor& steps) {
  return {codes.data_ptr<uint8_t>(), reinterpret_cast<uint16_t*>(steps.data_ptr()), codes.stride(0), codes.stride(1), codes.stride(2),
          steps.stride(0), steps.stride(1), steps.stride(2)};
}
Tensor as_slots(const Tensor& t, int64_t B, int64_t W, const Tensor& like) {
  CHECK_ARG(t.dim() == 2 && t.size(0) == B && t.size(1) == W && t.device() == like.device() && at::isIntegralType(t.scalar_type(), false),
            "slots must be whole numbers [" + std::to_string(B) + ", " + std::to_string(W) + "] on the pages' device");
  return t.scalar_type() == at::kLong ? t.clamp(-1, std::numeric_limits<int>::max()).to(at::kInt).contiguous() : ints(t, at::kInt);
}
void check_flag(const c10::optional<Tensor>& t, const char* name, const Tensor& like) {
  CHECK_ARG(!t.has_value() || (t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == 1 && t->device() == like.device()),
            std::string(name) + " must be an int32 tensor of one number on the same device");
}

// Whether the kernels take these
bool int4_append_ok(const Tensor& q, const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs, const Tensor& cos_t, bool pairs) {
  return q.dim() == 4 && float_type(q) && cos_t.dim() == 2 && cos_t.size(1) % (pairs ? 4 : 8) == 0 && pool_ok({kc, ks, vc, vs});
}
bool int4_gather_ok(const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs, at::ScalarType type) {
  return (type == at::kFloat || type == at::kBFloat16 || type == at::kHalf) && pool_ok({kc, ks, vc, vs});
}
bool int4_attention_ok(const Tensor& q, const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs) {
  return q.dim() == 4 && half_type(q) && (q.size(3) == 64 || q.size(3) == 128) && pool_ok({kc, ks, vc, vs});
}

// None, here and below: not for the kernel
c10::optional<Tensor> int4_append(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& positions_, const Tensor& cos_, const Tensor& sin_,
                                  const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs, const Tensor& slots_, bool pairs,
                                  const c10::optional<Tensor>& lost) {
  const Pool pool{kc, ks, vc, vs};
  check_pool(pool);
  check_queries(q_, pool);
  const int64_t B = q_.size(0), W = q_.size(1), H = q_.size(2), D = q_.size(3), Hkv = kc.size(2);
  CHECK_ARG(k_.sizes() == v_.sizes() && k_.dim() == 4 && k_.size(0) == B && k_.size(1) == W && k_.size(2) == Hkv && k_.size(3) == D,
            "new keys and values must be " + list({B, W, Hkv, D}));
  CHECK_ARG(k_.scalar_type() == q_.scalar_type() && v_.scalar_type() == q_.scalar_type() && k_.device() == q_.device() && v_.device() == q_.device(),
            "queries, keys and values are of one type and on one device");
  CHECK_ARG(cos_.dim() == 2 && cos_.sizes() == sin_.sizes() && cos_.size(1) * 2 <= D && cos_.size(0) < (1ll << 31) && cos_.scalar_type() == at::kFloat &&
            sin_.scalar_type() == at::kFloat && cos_.device() == q_.device() && sin_.device() == q_.device(),
            "cos and sin must be float32 tables [positions, at most " + std::to_string(D / 2) + "] on the queries' device");
  CHECK_ARG(positions_.dim() == 1 && positions_.size(0) == B && positions_.device() == q_.device(), "positions must be [" + std::to_string(B) + "] on the queries' device");
  check_flag(lost, "lost", q_);
  if (!int4_append_ok(q_, kc, ks, vc, vs, cos_, pairs)) return c10::nullopt;
  CHECK_ARG(q_.is_cuda(), "the kernel's tensors are on a GPU");
  c10::cuda::CUDAGuard guard(q_.device());
  const Tensor positions = ints(positions_, at::kLong), slots = as_slots(slots_, B, W, q_);
  auto table = [](const Tensor& t) { return t.is_contiguous() && packets(t) ? t : t.clone(at::MemoryFormat::Contiguous); };
  const Tensor q = as_packets(q_), k = as_packets(k_), v = as_packets(v_), cos_t = table(cos_), sin_t = table(sin_);
  Tensor out = rows_out(q);
  if (B == 0 || W == 0) return out;
  nxd::Int4Append p{};
  p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr();
  p.positions = positions.data_ptr<long>();
  p.slots = slots.data_ptr<int>();
  p.cos_t = cos_t.data_ptr<float>(); p.sin_t = sin_t.data_ptr<float>();
  p.q_out = out.data_ptr();
  p.lost = lost.has_value() ? lost->data_ptr<int>() : nullptr;
  p.kp = pages_of(kc, ks); p.vp = pages_of(vc, vs);
  p.B = (int)B; p.W = (int)W; p.H = (int)H; p.Hkv = (int)Hkv; p.D = (int)D; p.half = (int)cos_t.size(1); p.rows = (int)cos_t.size(0); p.ps = (int)kc.size(1);
  p.tokens = kc.size(0) * kc.size(1);
  p.pairs = pairs;
  p.q_sb = q.stride(0); p.q_sw = q.stride(1); p.q_sh = q.stride(2);
  p.k_sb = k.stride(0); p.k_sw = k.stride(1); p.k_sh = k.stride(2);
  p.v_sb = v.stride(0); p.v_sw = v.stride(1); p.v_sh = v.stride(2);
  p.o_sb = out.stride(0); p.o_sw = out.stride(1);
  count_launches(nxd::int4_append(p, dt_code(q), stream()));
  return out;
}

c10::optional<std::vector<Tensor>> int4_gather(const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs, const Tensor& slots_, at::ScalarType type) {
  const Pool pool{kc, ks, vc, vs};
  check_pool(pool);
  CHECK_ARG(slots_.dim() == 2, "slots are [batch, tokens]");
  CHECK_ARG(at::isFloatingType(type), "numbers are read as floating-point ones");
  if (!int4_gather_ok(kc, ks, vc, vs, type)) return c10::nullopt;
  CHECK_ARG(kc.is_cuda(), "the kernel's tensors are on a GPU");
  c10::cuda::CUDAGuard guard(kc.device());
  const Tensor slots = as_slots(slots_, slots_.size(0), slots_.size(1), kc);
  const int64_t B = slots.size(0), W = slots.size(1), Hkv = kc.size(2), D = 2 * kc.size(3);
  Tensor k = empty_on({B, W, Hkv, D}, type, kc.device()), v = empty_on({B, W, Hkv, D}, type, kc.device());
  nxd::int4_gather(pages_of(kc, ks), pages_of(vc, vs), slots.data_ptr<int>(), k.data_ptr(), v.data_ptr(), B * W, (int)Hkv, (int)D, (int)kc.size(1),
                   kc.size(0) * kc.size(1), dt_code(k), stream());
  count_launches(k.numel() > 0);
  return std::vector<Tensor>{k, v};
}

// Bytes of unpacked keys and values at a time: sequences, then key/value heads, in turns where there are more (one head of one sequence may take more, int4_plan)
constexpr int64_t kUnpacked = 256ll << 20;

// Many rows of bf16: their sequences' pages are unpacked to halves, which the attention on the tensor memory reads
void attend_portion(const nxd::Int4Attn& p, const Tensor& q, int64_t D) {
  const int64_t head = (int64_t)p.cols * p.ps * D * 4, each = std::max<int64_t>(head, 1) * p.Hkv;                   // bytes of a head, of a sequence
  const int64_t seqs = std::min<int64_t>(p.B, std::max<int64_t>(1, kUnpacked / each));
  const int64_t heads = std::min<int64_t>(p.Hkv, std::max<int64_t>(1, kUnpacked / std::max<int64_t>(head, 1)));
  const int H = p.G * p.Hkv;
  const Tensor q16 = empty_on({p.B, p.W, H, D}, at::kHalf, q.device()), units = empty_on({p.B, p.W, H}, at::kFloat, q.device());
  nxd::int4_queries(q.data_ptr(), q16.data_ptr(), units.data_ptr<float>(), p.B, p.W, H, (int)D, p.q_sb, p.q_sw, p.q_sh, stream());
  count_launches(1);
  const int64_t pages = seqs * p.cols;
  const Tensor k16 = empty_on({pages, heads, p.ps, D}, at::kHalf, q.device()), v16 = empty_on({pages, heads, p.ps, D}, at::kHalf, q.device());
  const Tensor table = empty_on({seqs, p.cols}, at::kInt, q.device());
  for (int64_t b = 0; b < p.B; b += seqs)
    for (int64_t h = 0; h < p.Hkv; h += heads) {
      nxd::Int4Attn from = p;
      from.B = (int)std::min<int64_t>(seqs, p.B - b);
      from.Hkv = (int)std::min<int64_t>(heads, p.Hkv - h);
      from.positions = p.positions + b;
      from.lens = p.lens ? p.lens + b : nullptr;
      from.table = p.table + b * p.table_sb;
      from.k = (const uint8_t*)p.k + h * p.k_sh * 16; from.v = (const uint8_t*)p.v + h * p.v_sh * 16;
      from.ks = (const uint16_t*)p.ks + h * p.ks_sh * (D / 16); from.vs = (const uint16_t*)p.vs + h * p.vs_sh * (D / 16);
      nxd::int4_unpack(from, k16.data_ptr(), v16.data_ptr(), table.data_ptr<int>(), (int)D, stream());
      nxd::PagedAttn to = from;
      to.q = (const uint16_t*)q16.data_ptr() + b * q16.stride(0) + h * p.G * q16.stride(2);
      to.q_sb = q16.stride(0); to.q_sw = q16.stride(1); to.q_sh = q16.stride(2);
      to.k = k16.data_ptr(); to.v = v16.data_ptr();
      to.out = (uint16_t*)p.out + b * p.o_sb + h * p.G * p.o_sh;
      to.table = table.data_ptr<int>(); to.table_sb = p.cols;
      to.shared_pages = nullptr; to.shared_cols = 0;
      to.pages = (int)pages;
      to.k_sp = to.v_sp = (int64_t)from.Hkv * p.ps * D; to.k_sh = to.v_sh = p.ps * D; to.k_sr = to.v_sr = D;
      to.units = units.data_ptr<float>() + b * units.stride(0) + h * p.G;
      to.u_sb = units.stride(0); to.u_sw = units.stride(1);
      to.wait_ns = 2000000000;
      const nxd::PagedPlan plan = nxd::paged_plan(to);
      Tensor work;
      if (plan.slots > 0) work = empty_on({plan.slots * (D + 2)}, at::kFloat, q.device());
      to.part_o = to.pre_o = work.defined() ? work.data_ptr<float>() : nullptr;
      to.part_ml = to.pre_ml = to.part_o + plan.slots * D;
      count_launches(1 + nxd::paged_attention_half(to, plan, (int)D, nxd::kBF16, stream()));
    }
}

c10::optional<Tensor> int4_attention(const Tensor& q_, const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs, const Tensor& table_,
                                     const Tensor& positions_, const c10::optional<double>& scale_, const c10::optional<Tensor>& lens_,
                                     const c10::optional<Tensor>& shared_) {
  const Pool pool{kc, ks, vc, vs};
  check_pool(pool);
  check_queries(q_, pool);
  const int64_t B = q_.size(0), W = q_.size(1), H = q_.size(2), D = q_.size(3), Hkv = kc.size(2), ps = kc.size(1);
  const std::string rows = std::to_string(B);
  CHECK_ARG(table_.dim() == 2 && table_.size(0) == B && table_.device() == q_.device() && table_.size(1) * ps < (1ll << 31) &&
            table_.size(1) * ps * Hkv < (1ll << 38), "page_table must be [" + rows + ", pages of a sequence] on the queries' device, of fewer than 2^31 tokens");
  CHECK_ARG(positions_.dim() == 1 && positions_.size(0) == B && positions_.device() == q_.device(), "positions must be [" + rows + "] on the queries' device");
  CHECK_ARG(!lens_.has_value() || (lens_->dim() == 1 && lens_->size(0) == B && lens_->device() == q_.device()), "lens must be [" + rows + "] on the queries' device");
  CHECK_ARG(!shared_.has_value() || (shared_->dim() == 1 && shared_->device() == q_.device() && shared_->size(0) <= table_.size(1)),
            "shared_pages is a list of no more pages than page_table has, on the queries' device");
  const double scale = scale_.has_value() ? *scale_ : 1 / std::sqrt((double)D);
  CHECK_ARG(scale > 0 && scale < 1e30, "the scale of the scores is positive");
  if (!int4_attention_ok(q_, kc, ks, vc, vs)) return c10::nullopt;
  for (const Tensor* t : {&kc, &vc}) CHECK_ARG(places_ok(*t, 16, D / 32 - 1), "pages whose codes span 64 GB and more");
  for (const Tensor* t : {&ks, &vs}) CHECK_ARG(places_ok(*t, D / 16, 0), "pages whose steps span 2^32 rows and more");
  CHECK_ARG(q_.is_cuda(), "the kernels' tensors are on a GPU");
  c10::cuda::CUDAGuard guard(q_.device());
  const Tensor positions = ints(positions_, at::kLong), table = as_table(table_), q = as_packets(q_);
  const c10::optional<Tensor> lens = ints(lens_, at::kLong), shared = ints(shared_, at::kInt);
  Tensor out = rows_out(q);
  if (q.numel() == 0) return out;
  nxd::Int4Attn p{};
  p.q = q.data_ptr(); p.k = kc.data_ptr(); p.v = vc.data_ptr(); p.ks = ks.data_ptr(); p.vs = vs.data_ptr(); p.out = out.data_ptr();
  p.table = table.data_ptr<int>();
  p.shared_cols = shared.has_value() ? (int)shared->size(0) : 0;
  p.shared_pages = p.shared_cols ? shared->data_ptr<int>() : nullptr;
  p.positions = positions.data_ptr<long>();
  p.lens = lens.has_value() ? lens->data_ptr<long>() : nullptr;
  p.B = (int)B; p.W = (int)W; p.G = (int)(H / Hkv); p.Hkv = (int)Hkv; p.cols = (int)table.size(1); p.ps = (int)ps; p.pages = (int)kc.size(0);
  p.q_sb = q.stride(0); p.q_sw = q.stride(1); p.q_sh = q.stride(2);
  p.o_sb = out.stride(0); p.o_sw = out.stride(1); p.o_sh = out.stride(2);
  p.table_sb = table.stride(0);
  const int64_t row = D / 16;                       // halves of a token's steps
  p.k_sp = kc.stride(0) / 16; p.k_sr = kc.stride(1) / 16; p.k_sh = kc.stride(2) / 16;
  p.v_sp = vc.stride(0) / 16; p.v_sr = vc.stride(1) / 16; p.v_sh = vc.stride(2) / 16;
  p.ks_sp = ks.stride(0) / row; p.ks_sr = ks.stride(1) / row; p.ks_sh = ks.stride(2) / row;
  p.vs_sp = vs.stride(0) / row; p.vs_sr = vs.stride(1) / row; p.vs_sh = vs.stride(2) / row;
  p.scale_log2 = std::max((float)(scale * 1.4426950408889634), std::numeric_limits<float>::min());        // kernels count less as 0
  if (p.cols == 0) return out.zero_();               // nobody sees a key
  const nxd::PagedPlan plan = nxd::int4_plan(p, (int)D, dt_code(q));
  if (plan.tiles) {
    attend_portion(p, q, D);
    return out;
  }
  Tensor work;                                     // parts of pairs that are cut: sums and statistics
  if (plan.slots > 0) work = empty_on({plan.slots * (D + 2)}, at::kFloat, q.device());
  p.part_o = work.defined() ? work.data_ptr<float>() : nullptr;
  p.part_ml = p.part_o + plan.slots * D;
  count_launches(nxd::int4_attention(p, plan, (int)D, dt_code(q), stream()));
  return out;
}

std::vector<Tensor> assign_pages(const Tensor& table, const Tensor& held, const Tensor& free, const Tensor& span, const Tensor& positions_, int64_t W,
                                 int64_t ps, const c10::optional<Tensor>& lens_, const c10::optional<Tensor>& lengths_, int64_t shared, bool trim,
                                 const c10::optional<Tensor>& few, bool in_place) {
  CHECK_ARG(table.dim() == 2 && table.scalar_type() == at::kInt && (table.size(1) <= 1 || table.stride(1) == 1),
            "page_table must be an int32 tensor [batch, pages of a sequence]");
  const int64_t B = table.size(0), n = table.size(1);
  auto check = [&](const Tensor& t, const char* name, at::ScalarType type, int64_t size) {
    CHECK_ARG(t.scalar_type() == type && t.dim() == 1 && t.size(0) == size && t.is_contiguous() && t.device() == table.device(),
              std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor of " + std::to_string(size) + " numbers on the tables' device");
  };
  check(held, "held", at::kInt, B);
  check(span, "span", at::kLong, 2);
  CHECK_ARG(free.scalar_type() == at::kInt && free.dim() == 1 && free.size(0) > 0 && free.is_contiguous() && free.device() == table.device(),
            "free must be a contiguous int32 tensor with a place for every page of the pool");
  auto rows = [&](const Tensor& t, const char* name) {
    CHECK_ARG(t.dim() == 1 && t.size(0) == B && t.device() == table.device(), std::string(name) + " must be [" + std::to_string(B) + "] on the tables' device");
  };
  rows(positions_, "positions");
  if (lens_.has_value()) rows(*lens_, "lens");
  if (lengths_.has_value()) rows(*lengths_, "lengths");
  CHECK_ARG(!in_place || B <= 1 || table.stride(0) >= n, "rows of a page_table that is changed in place lie apart");
  const int64_t P = free.size(0);
  CHECK_ARG(W >= 0 && W < (1ll << 31) && ps > 0 && ps < (1ll << 31) && P < (1ll << 31) && n < (1ll << 30) && P * ps < (1ll << 31) && n * ps < (1ll << 31) &&
            B * std::max<int64_t>(W, 1) < (1ll << 31) && B < nxd::kMaxPageRows,
            "too many tokens: " + std::to_string(P) + " pages of " + std::to_string(ps) + ", " + std::to_string(B) + " rows of " + std::to_string(W) + " new tokens");
  CHECK_ARG(0 <= shared && shared <= n, "shared columns: " + std::to_string(shared) + " of " + std::to_string(n));
  check_flag(few, "short", table);
  CHECK_ARG(table.is_cuda(), "the kernel's tensors are on a GPU");
  c10::cuda::CUDAGuard guard(table.device());
  const Tensor positions = ints(positions_, at::kLong);
  const c10::optional<Tensor> lens = ints(lens_, at::kLong), lengths = ints(lengths_, at::kLong);
  const at::Device on = table.device();
  const Tensor table_out = in_place ? table : empty_on({B, n}, at::kInt, on), held_out = in_place ? held : empty_on({B}, at::kInt, on);
  const Tensor free_out = in_place ? free : empty_on({P}, at::kInt, on), span_out = in_place ? span : empty_on({2}, at::kLong, on);
  const Tensor slots = empty_on({B, W}, at::kInt, on);
  nxd::PageTables p{};
  p.table = table.data_ptr<int>(); p.held = held.data_ptr<int>(); p.free = free.data_ptr<int>(); p.span = span.data_ptr<long>();
  p.positions = positions.data_ptr<long>();
  p.lens = lens.has_value() ? lens->data_ptr<long>() : nullptr;
  p.lengths = lengths.has_value() ? lengths->data_ptr<long>() : nullptr;
  p.table_out = table_out.data_ptr<int>(); p.held_out = held_out.data_ptr<int>(); p.free_out = free_out.data_ptr<int>(); p.span_out = span_out.data_ptr<long>();
  p.slots = slots.data_ptr<int>();
  p.few = few.has_value() ? few->data_ptr<int>() : nullptr;
  p.B = (int)B; p.W = (int)W; p.cols = (int)n; p.ps = (int)ps; p.P = (int)P; p.shared = (int)shared; p.trim = trim;
  p.table_sb = table.stride(0); p.out_sb = table_out.stride(0);
  nxd::page_tables(p, in_place, stream());
  count_launches(B > 0);
  return {table_out, held_out, free_out, span_out, slots};
}

}  // namespace

void bind_paged_int4(pybind11::module_& m) {
  m.def("int4_append", &int4_append);
  m.def("int4_append_ok", &int4_append_ok);
  m.def("int4_gather", &int4_gather);
  m.def("int4_gather_ok", &int4_gather_ok);
  m.def("int4_attention", &int4_attention);
  m.def("int4_attention_ok", &int4_attention_ok);
  m.def("assign_pages", &assign_pages);
}
