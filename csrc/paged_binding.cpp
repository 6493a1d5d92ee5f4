// Bindings of the paged key/value cache and of the verification of drafted tokens: checks of arguments, workspaces, launches.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <limits>

#include "paged_checks.h"

namespace {

// q [B, W, H, D], caches [pages, page_size, Hkv, D], table [B, cols], positions [B], lens [B] or none
void check_cache(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& table, const Tensor& positions, const c10::optional<Tensor>& lens) {
  CHECK_ARG(q.dim() == 4 && kc.dim() == 4 && vc.dim() == 4, "queries are [batch, new tokens, heads, head size], caches [pages, page size, heads, head size]");
  CHECK_ARG(kc.sizes() == vc.sizes() && kc.size(3) == q.size(3) && kc.size(2) > 0 && q.size(2) > 0 && q.size(2) % kc.size(2) == 0,
            "heads do not match: queries " + list(q.sizes()) + ", keys " + list(kc.sizes()) + ", values " + list(vc.sizes()));
  CHECK_ARG(q.scalar_type() == kc.scalar_type() && q.scalar_type() == vc.scalar_type(), "queries and caches are of one type");
  CHECK_ARG(kc.device() == q.device() && vc.device() == q.device(), "queries and caches are on one device");
  CHECK_ARG(kc.size(0) > 0 && kc.size(1) > 0 && kc.size(0) < (1ll << 31) && kc.size(1) % 16 == 0,
            "a page holds a multiple of 16 tokens, got " + std::to_string(kc.size(1)));
  CHECK_ARG(table.dim() == 2 && table.size(0) == q.size(0) && table.scalar_type() == at::kInt && table.device() == q.device() &&
            (table.size(1) <= 1 || table.stride(1) == 1) && table.size(1) * kc.size(1) < (1ll << 31),
            "page_table must be an int32 tensor [" + std::to_string(q.size(0)) + ", pages of a sequence] on the queries' device");
  check_ints(positions, "positions", at::kLong, q.size(0), q);
  if (lens.has_value()) check_ints(*lens, "lens", at::kLong, q.size(0), q);
  CHECK_ARG(q.size(0) < (1 << 20) && q.size(1) < (1 << 24) && q.size(0) * q.size(1) * q.size(2) < (1ll << 30), "too many query rows: " + list(q.sizes()));
}

// Whether the append kernel takes these: 32- or 16-bit types, halves of heads and cache rows of whole 16-byte packets
bool paged_append_ok(const Tensor& q, const Tensor& kc, const Tensor& vc) {
  return q.dim() == 4 && kc.dim() == 4 && vc.dim() == 4 && (half_type(q) || q.scalar_type() == at::kFloat) &&
         q.size(3) * q.element_size() % 32 == 0 && packets(kc) && packets(vc);
}
// Whether the attention kernels take these: 16-bit types, heads of 64 or 128 numbers, cache rows of whole 16-byte packets
bool paged_attention_ok(const Tensor& q, const Tensor& kc, const Tensor& vc) {
  return q.dim() == 4 && kc.dim() == 4 && vc.dim() == 4 && half_type(q) && (q.size(3) == 64 || q.size(3) == 128) && packets(kc) && packets(vc);
}

// None: not for the kernel
c10::optional<Tensor> paged_append(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& positions_, const Tensor& cos_t, const Tensor& sin_t, Tensor kc,
                    Tensor vc, const Tensor& table_, const c10::optional<Tensor>& lens_, const c10::optional<Tensor>& lost) {
  const Tensor positions = ints(positions_, at::kLong), table = as_table(table_);
  const c10::optional<Tensor> lens = ints(lens_, at::kLong);
  check_cache(q_, kc, vc, table, positions, lens);
  if (!paged_append_ok(q_, kc, vc)) return c10::nullopt;
  CHECK_ARG(k_.sizes() == v_.sizes() && k_.dim() == 4 && k_.size(0) == q_.size(0) && k_.size(1) == q_.size(1) && k_.size(2) == kc.size(2) &&
            k_.size(3) == q_.size(3), "new keys and values must be " + list({q_.size(0), q_.size(1), kc.size(2), q_.size(3)}));
  CHECK_ARG(k_.scalar_type() == q_.scalar_type() && v_.scalar_type() == q_.scalar_type() && k_.device() == q_.device() && v_.device() == q_.device(),
            "queries, keys and values are of one type and on one device");
  CHECK_ARG(cos_t.dim() == 2 && cos_t.sizes() == sin_t.sizes() && cos_t.size(1) * 2 == q_.size(3) && cos_t.scalar_type() == at::kFloat &&
            sin_t.scalar_type() == at::kFloat && cos_t.is_contiguous() && sin_t.is_contiguous() && cos_t.device() == q_.device() && sin_t.device() == q_.device(),
            "cos and sin must be contiguous float32 tables [positions, " + std::to_string(q_.size(3) / 2) + "]");
  CHECK_ARG(!lost.has_value() || (lost->scalar_type() == at::kInt && lost->dim() == 1 && lost->size(0) == 1 && lost->device() == q_.device()),
            "lost must be an int32 tensor of one number on the queries' device");
  CHECK_ARG(q_.is_cuda(), "the kernel's tensors are on a GPU");
  c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = as_packets(q_), k = as_packets(k_), v = as_packets(v_), cos_p = as_packets(cos_t), sin_p = as_packets(sin_t);
  Tensor out = rows_out(q);
  if (q.size(0) == 0 || q.size(1) == 0) return out;
  const long s[3][3] = {{q.stride(0), q.stride(1), q.stride(2)}, {k.stride(0), k.stride(1), k.stride(2)}, {v.stride(0), v.stride(1), v.stride(2)}};
  const long cs[2][3] = {{kc.stride(0), kc.stride(1), kc.stride(2)}, {vc.stride(0), vc.stride(1), vc.stride(2)}};
  nxd::paged_append(q.data_ptr(), k.data_ptr(), v.data_ptr(), positions.data_ptr<long>(), lens.has_value() ? lens->data_ptr<long>() : nullptr,
                    cos_p.data_ptr<float>(), sin_p.data_ptr<float>(), out.data_ptr(), kc.data_ptr(), vc.data_ptr(), table.data_ptr<int>(),
                    lost.has_value() ? lost->data_ptr<int>() : nullptr, (int)q.size(0),
                    (int)q.size(1), (int)q.size(2), (int)kc.size(2), (int)q.size(3), (int)cos_t.size(0), (int)table.size(1), (int)kc.size(1),
                    (int)kc.size(0), table.stride(0), s, out.stride(0), out.stride(1), cs, dt_code(q), stream());
  count_launches(1);
  return out;
}

// Nanoseconds after which the tile kernel gives a wait up, so that its rows are NaN; negative: its keys are not loaded, so that waits do run out
std::atomic<int> wait_ns{2000000000};

// None: not for the kernels
c10::optional<Tensor> paged_attention(const Tensor& q_, const Tensor& kc, const Tensor& vc, const Tensor& table_, const Tensor& positions_,
                                      const c10::optional<double>& scale_, const c10::optional<Tensor>& lens_, const c10::optional<Tensor>& shared_pages_) {
  const Tensor positions = ints(positions_, at::kLong), table = as_table(table_);
  const c10::optional<Tensor> lens = ints(lens_, at::kLong), shared_pages = ints(shared_pages_, at::kInt);
  check_cache(q_, kc, vc, table, positions, lens);
  if (!paged_attention_ok(q_, kc, vc)) return c10::nullopt;
  CHECK_ARG(q_.is_cuda(), "the kernels' tensors are on a GPU");
  const int64_t ps = kc.size(1);
  int64_t shared = 0;                              // shared pages
  if (shared_pages.has_value()) {
    CHECK_ARG(shared_pages->dim() == 1, "shared_pages is a list of pages");
    check_ints(*shared_pages, "shared_pages", at::kInt, shared_pages->size(0), q_);
    shared = shared_pages->size(0);
    CHECK_ARG(shared_pages->size(0) <= table.size(1),
              "more shared pages than a sequence has: " + std::to_string(shared_pages->size(0)) + ", page_table of " + std::to_string(table.size(1)));
  }
  const double scale = scale_.has_value() ? *scale_ : 1 / std::sqrt((double)q_.size(3));
  CHECK_ARG(scale > 0 && scale < 1e30, "the scale of the scores is positive");
  c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = as_packets(q_);
  Tensor out = rows_out(q);
  if (q.numel() == 0) return out;
  const int64_t B = q.size(0), W = q.size(1), H = q.size(2), D = q.size(3), Hkv = kc.size(2);
  nxd::PagedAttn p{};
  p.q = q.data_ptr(); p.k = kc.data_ptr(); p.v = vc.data_ptr(); p.out = out.data_ptr();
  p.table = table.data_ptr<int>();
  p.shared_pages = shared ? shared_pages->data_ptr<int>() : nullptr;
  p.positions = positions.data_ptr<long>();
  p.lens = lens.has_value() ? lens->data_ptr<long>() : nullptr;
  p.B = (int)B; p.W = (int)W; p.G = (int)(H / Hkv); p.Hkv = (int)Hkv; p.cols = (int)table.size(1); p.ps = (int)ps; p.pages = (int)kc.size(0);
  p.shared_cols = (int)shared;
  p.q_sb = q.stride(0); p.q_sw = q.stride(1); p.q_sh = q.stride(2);
  p.o_sb = out.stride(0); p.o_sw = out.stride(1); p.o_sh = out.stride(2);
  p.table_sb = table.stride(0);
  p.k_sp = kc.stride(0); p.k_sr = kc.stride(1); p.k_sh = kc.stride(2);
  p.v_sp = vc.stride(0); p.v_sr = vc.stride(1); p.v_sh = vc.stride(2);
  const nxd::PagedPlan plan = nxd::paged_plan(p);
  // one workspace: parts of pairs that are cut, then parts over the shared pages, each sums and statistics
  Tensor work;
  if (plan.slots + plan.pre_slots > 0) work = at::empty({(plan.slots + plan.pre_slots) * (D + 2)}, q.options().dtype(at::kFloat));
  p.part_o = work.defined() ? work.data_ptr<float>() : nullptr;
  p.pre_o = p.part_o + plan.slots * D;             // join_parts counts on this order
  p.part_ml = p.pre_o + plan.pre_slots * D;
  p.pre_ml = p.part_ml + plan.slots * 2;
  p.wait_ns = wait_ns.load();
  p.scale_log2 = std::max((float)(scale * 1.4426950408889634), std::numeric_limits<float>::min());        // kernels count less as 0
  count_launches(nxd::paged_attention(p, plan, (int)D, dt_code(q), stream()));
  return out;
}

std::vector<Tensor> verify_drafts(const Tensor& tokens, const Tensor& draft_, const Tensor& target_, const Tensor& accept, const Tensor& sample) {
  CHECK_ARG(tokens.dim() == 2 && tokens.scalar_type() == at::kLong && tokens.is_contiguous(), "draft_tokens must be a contiguous int64 tensor [batch, drafts]");
  const int64_t B = tokens.size(0), K = tokens.size(1);
  CHECK_ARG(draft_.dim() == 3 && target_.dim() == 3 && draft_.size(0) == B && draft_.size(1) == K && target_.size(0) == B && target_.size(1) == K + 1 &&
            draft_.size(2) == target_.size(2) && target_.size(2) > 0 && target_.size(2) < (1 << 30),
            "probabilities must be [batch, drafts, vocabulary] of the draft and [batch, drafts + 1, vocabulary] of the target, got " + list(draft_.sizes()) + " and " +
            list(target_.sizes()));
  CHECK_ARG(draft_.scalar_type() == target_.scalar_type() && (half_type(draft_) || draft_.scalar_type() == at::kFloat),
            "probabilities are float32, bfloat16 or float16, both of one type");
  CHECK_ARG(accept.sizes() == tokens.sizes() && accept.scalar_type() == at::kFloat && accept.is_contiguous(),
            "accept_uniforms must be a contiguous float32 tensor [batch, drafts]");
  CHECK_ARG(sample.dim() == 1 && sample.size(0) == B && sample.scalar_type() == at::kFloat && sample.is_contiguous(),
            "sample_uniforms must be a contiguous float32 tensor [batch]");
  for (const Tensor& t : {tokens, draft_, target_, accept, sample}) CHECK_ARG(t.is_cuda() && t.device() == target_.device(), "all tensors are on one device");
  CHECK_ARG(B < 65536 && K < (1 << 20), "too many sequences or drafts");
  c10::cuda::CUDAGuard guard(target_.device());
  const Tensor draft = draft_.stride(2) == 1 ? draft_ : draft_.contiguous(), target = target_.stride(2) == 1 ? target_ : target_.contiguous();
  Tensor out = at::empty({B, K + 1}, tokens.options()), accepted = at::empty({B}, tokens.options());
  const long ds[2] = {draft.stride(0), draft.stride(1)}, ts[2] = {target.stride(0), target.stride(1)};
  nxd::verify_drafts(tokens.data_ptr<long>(), draft.data_ptr(), target.data_ptr(), accept.data_ptr<float>(), sample.data_ptr<float>(),
                     out.data_ptr<long>(), accepted.data_ptr<long>(), (int)B, (int)K, (int)target.size(2), ds, ts, dt_code(target), stream());
  count_launches(B > 0);
  return {out, accepted};
}

}  // namespace

void bind_paged(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("paged_append", &paged_append, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("positions"), py::arg("cos"), py::arg("sin"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("page_table"), py::arg("lens"), py::arg("lost") = py::none());
  m.def("paged_append_ok", &paged_append_ok);
  m.def("paged_attention", &paged_attention);
  m.def("paged_wait_ns", [](int ns) { return wait_ns.exchange(ns); });      // → what it was
  m.def("paged_attention_ok", &paged_attention_ok);
  m.def("verify_drafts", &verify_drafts);
}
