// The PyTorch side of decoding with several hypotheses: choosing tokens, and moving the states that belong to them.  As in
// torch_ops.cpp, ops.py keeps the public functions and each of them is one call into this module.
#include "torch_util.h"

#include <algorithm>

namespace lethe_torch {
namespace {

constexpr int64_t kMostBeams = 64, kMostGroup = 256, kMostSlots = 65536, kMostEntries = 4096;

void need_bool(const Tensor& t, const char* name) {
  if (t.defined() && t.scalar_type() != at::kBool) fail(std::string(name) + " must be a tensor of truth values");
}

// ---------------------------------------------------------------------------------------------
// Selection
// ---------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor, OptTensor> beam_select(const Tensor& logits, const Tensor& scores, const OptTensor& allowed_, const OptTensor& finished_,
                                                          const OptTensor& penalty_, std::optional<int64_t> k_, double temperature, std::optional<int64_t> eos) {
  return guarded([&]() -> std::tuple<Tensor, Tensor, Tensor, OptTensor> {
    need_cuda(logits);
    const Tensor allowed_in = opt(allowed_), finished_in = opt(finished_), penalty_in = opt(penalty_);
    need_device(logits, scores, allowed_in, finished_in, penalty_in);
    need_type(logits, "logits");
    need_float(scores, "scores");
    need_float(penalty_in, "penalty");
    need_bool(allowed_in, "allowed");
    need_bool(finished_in, "finished");
    need_shape(logits.dim() == 3, "logits [B, W, V]");
    const int64_t B = logits.size(0), W = logits.size(1), V = logits.size(2);
    const int64_t shape2[] = {B, W};
    const at::IntArrayRef beams(shape2);
    need_shape(scores.sizes() == beams && (!finished_in.defined() || finished_in.sizes() == beams) && (!penalty_in.defined() || penalty_in.sizes() == beams),
               "scores, finished, penalty [B, W] for logits [B, W, V]");
    const int64_t k = k_.value_or(W);
    if (W < 1 || W > kMostBeams || k < 1 || k > kMostBeams)
      fail("beam_select takes 1 to " + std::to_string(kMostBeams) + " beams and as many candidates (got " + std::to_string(W) + " and " + std::to_string(k) + ")");
    if (V < 1) fail("beam_select needs a vocabulary");
    if (!(temperature >= 1e-6 && temperature <= 1e6)) fail("temperature must be between 1e-6 and 1e6");
    if (finished_in.defined() && !eos) fail("finished beams need eos, the token that they go on with");
    if (eos && (*eos < 0 || *eos >= V)) fail("eos must be a token of the vocabulary");
    refuse_tangents({logits, scores, penalty_in});
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(logits.device());
    Parts all;
    const int64_t n = B * k, at_best = all.reserve(4 * n), at_parents = all.reserve(8 * n), at_tokens = all.reserve(8 * n), at_ended = all.reserve(eos ? n : 0);
    all.make(logits);
    const int64_t shape_out[] = {B, k};
    const Tensor best = all.part(at_best, shape_out, at::kFloat), parents = all.part(at_parents, shape_out, at::kLong), tokens = all.part(at_tokens, shape_out, at::kLong);
    const Tensor ended = eos ? all.part(at_ended, shape_out, at::kBool) : Tensor();
    const OptTensor ended_out = eos ? OptTensor(ended) : std::nullopt;
    if (B == 0) return {best, parents, tokens, ended_out};
    const Tensor x = lazy(logits) || !packed_from(logits, 2) ? as(logits, logits.scalar_type()) : logits;
    const Tensor s = as32(scores), pen = as32(penalty_in);
    const Tensor fin = finished_in.defined() ? as(finished_in, at::kBool) : finished_in;
    Tensor allowed;
    if (allowed_in.defined()) {
      const auto shape = logits.sizes();
      need_shape(allowed_in.dim() <= 3 && at::is_expandable_to(allowed_in.sizes(), shape), "allowed must go with logits [B, W, V]");
      const Tensor whole = lazy(allowed_in) ? as(allowed_in, at::kBool) : allowed_in;
      allowed = whole.expand(shape);
      if (!packed_from(allowed, 2)) allowed = whole.dim() >= 1 && whole.size(-1) == V ? whole.contiguous().expand(shape) : allowed.contiguous();
    }
    LetheGdnBeamArgs a;
    memset(&a, 0, sizeof(a));
    a.B = B; a.V = V; a.W = static_cast<int32_t>(W); a.k = static_cast<int32_t>(k);
    a.x_type = code(x.scalar_type());
    a.temperature = temperature;
    a.logits = ptr(x); a.logits_batch = step_of(x, 0); a.logits_beam = step_of(x, 1);
    if (allowed.defined()) {
      a.allowed = ptr<uint8_t>(allowed); a.allowed_batch = step_of(allowed, 0); a.allowed_beam = step_of(allowed, 1);
    }
    a.scores = ptr<float>(s); a.finished = ptr<uint8_t>(fin); a.penalty = ptr<float>(pen);
    a.eos = eos ? *eos : -1;
    a.out_scores = ptr<float>(best); a.parents = ptr<int64_t>(parents); a.tokens = ptr<int64_t>(tokens);
    a.out_finished = ptr<uint8_t>(ended);
    a.work_bytes = lethe_gdn_beam_work_bytes(B, a.W, V, a.k, a.x_type);
    const Tensor work = at::empty({static_cast<int64_t>(a.work_bytes)}, logits.options().dtype(at::kByte));
    a.work = ptr(work);
    check(lethe_gdn_beam_select(&a, stream_of(logits)));
    return {best, parents, tokens, ended_out};
  });
}

// ---------------------------------------------------------------------------------------------
// States
// ---------------------------------------------------------------------------------------------
// rows of tensors, each a sequence's: [rows, ...], or [B, W, ...] where there are groups
struct Rows {
  std::vector<LetheGdnStates> s;      // without tensors whose rows are empty
  std::vector<Tensor> moved;
};

void check_state(const Tensor& t, const Tensor& like) {
  need_cuda(t);
  need_device(like, t);
  if (t.layout() != at::kStrided || t._is_zerotensor()) fail("states are tensors with memory of their own (they are updated in place)");
  if (t.requires_grad()) fail("states are updated in place and cannot require a gradient");
  refuse_tangents({t});
}

Rows rows_of(const std::vector<Tensor>& states, const Tensor& like, int64_t B, int64_t W, bool grouped, const char* shapes) {
  Rows r;
  for (const Tensor& t : states) {
    check_state(t, like);
    const bool groups = grouped && t.dim() >= 2 && t.size(0) == B && t.size(1) == W && t.size(0) != B * W;
    need_shape(groups || (t.dim() >= 1 && t.size(0) == B * W), shapes);
    const int64_t from = groups ? 2 : 1, e = t.element_size();
    if (t.numel() == 0) continue;
    if (!packed_from(t, from)) fail("the row of a sequence must be contiguous in each of its states (they are updated in place)");
    LetheGdnStates s;
    s.data = t.data_ptr();
    s.row_bytes = e * t.numel() / (B * W);
    s.stride = W > 1 || !groups ? e * t.stride(from - 1) : 0;
    s.group_stride = groups ? e * t.stride(0) : s.stride * W;
    if (B * W == 1) s.stride = 0;
    if (B == 1) s.group_stride = 0;
    // whole rows, none in another's place
    const int64_t inner = std::max<int64_t>(W - 1, 0) * s.stride, outer = (B - 1) * s.group_stride;
    const bool apart = (W == 1 || s.stride >= s.row_bytes) && (B == 1 || s.group_stride >= s.row_bytes) &&
                       (W == 1 || B == 1 || s.group_stride >= inner + s.row_bytes || s.stride >= outer + s.row_bytes);
    if (!apart) fail("rows of a state overlap");
    r.s.push_back(s);
    r.moved.push_back(t);
  }
  // None of them in another's place either; rows of one buffer's slices may lie between each other's.
  std::vector<size_t> order(r.s.size());
  for (size_t i = 0; i < order.size(); ++i) order[i] = i;
  std::sort(order.begin(), order.end(), [&](size_t i, size_t j) { return r.s[i].data < r.s[j].data; });
  const auto end = [&](size_t i) { return static_cast<const char*>(r.s[i].data) + (W - 1) * r.s[i].stride + (B - 1) * r.s[i].group_stride + r.s[i].row_bytes; };
  for (size_t a = 0; a < order.size(); ++a)
    for (size_t b = a + 1; b < order.size(); ++b) {
      const LetheGdnStates &x = r.s[order[a]], &y = r.s[order[b]];
      if (static_cast<const char*>(y.data) >= end(order[a])) break;
      const bool even = (B == 1 || (x.group_stride == W * x.stride && y.group_stride == W * y.stride)) && x.stride == y.stride && x.stride > 0;
      const int64_t past = even ? (static_cast<const char*>(y.data) - static_cast<const char*>(x.data)) % x.stride : 0;
      if (!even || past < x.row_bytes || x.stride - past < y.row_bytes) fail("two of the states share memory");
    }
  return r;
}

// an index or a mark that lies in the memory of a state is read before any of that is written
Tensor apart(Tensor t, const Rows& r) {
  t = as(t, t.scalar_type());
  for (const Tensor& s : r.moved)
    if (spans(t, s)) return t.clone();
  return t;
}

void changed(const Rows& r) {
  for (const Tensor& t : r.moved)
    if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

void reorder_states(const std::vector<Tensor>& states, const Tensor& parents) {
  return guarded([&] {
    need_cuda(parents);
    need_index(parents, "parents");
    need_shape(parents.dim() == 2, "parents [B, W]");
    const int64_t B = parents.size(0), W = parents.size(1);
    if (W > kMostGroup) fail("reorder_states takes groups of up to " + std::to_string(kMostGroup) + " rows");
    at::NoGradGuard no_grad;
    if (B * W == 0) {
      for (const Tensor& t : states) check_state(t, parents);
      return;
    }
    const Rows r = rows_of(states, parents, B, W, true, "states [B W, ...] or [B, W, ...] for parents [B, W]");
    if (r.s.empty()) return;
    c10::cuda::CUDAGuard guard(parents.device());
    const Tensor p = apart(parents, r);
    check(lethe_gdn_reorder_states(r.s.data(), static_cast<int32_t>(r.s.size()), B, static_cast<int32_t>(W), ptr(p), p.scalar_type() == at::kLong,
                                   status_word(parents.device().index()), stream_of(parents)));
    changed(r);
  });
}

int64_t check_slots(const Tensor& live) {
  need_cuda(live);
  need_bool(live, "live");
  need_shape(live.dim() == 1, "live [slots]");
  if (live.size(0) < 1 || live.size(0) > kMostSlots) fail("a pool has 1 to " + std::to_string(kMostSlots) + " slots");
  return live.size(0);
}

std::pair<Tensor, Tensor> fork_states(const std::vector<Tensor>& states, const Tensor& live_in, const Tensor& source_in) {
  return guarded([&]() -> std::pair<Tensor, Tensor> {
    const int64_t S = check_slots(live_in);
    need_device(live_in, source_in);
    need_index(source_in, "source");
    need_shape(source_in.dim() == 1, "source [n]");
    const int64_t n = source_in.size(0);
    if (n > kMostEntries) fail("fork_states takes up to " + std::to_string(kMostEntries) + " entries");
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(live_in.device());
    const Rows r = rows_of(states, live_in, 1, S, false, "states [slots, ...] for live [slots]");
    const Tensor live = apart(live_in, r), source = apart(source_in, r);
    if (n == 0) return {at::empty({n}, live.options().dtype(at::kLong)), live.clone()};
    Parts all;
    const int64_t at_target = all.reserve(8 * n), at_after = all.reserve(S);
    all.make(live);
    const Tensor target = all.part(at_target, {n}, at::kLong), after = all.part(at_after, {S}, at::kBool);
    check(lethe_gdn_fork_states(r.s.data(), static_cast<int32_t>(r.s.size()), S, ptr<uint8_t>(live), ptr(source), source.scalar_type() == at::kLong, n,
                                ptr<int64_t>(target), ptr<uint8_t>(after), status_word(live.device().index()), stream_of(live)));
    changed(r);
    return {target, after};
  });
}

std::pair<Tensor, Tensor> compact_states(const std::vector<Tensor>& states, const Tensor& live_in) {
  return guarded([&]() -> std::pair<Tensor, Tensor> {
    const int64_t S = check_slots(live_in);
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(live_in.device());
    const Rows r = rows_of(states, live_in, 1, S, false, "states [slots, ...] for live [slots]");
    const Tensor live = apart(live_in, r);
    Parts all;
    const int64_t at_place = all.reserve(8 * S), at_count = all.reserve(8);
    all.make(live);
    const Tensor place = all.part(at_place, {S}, at::kLong), count = all.part(at_count, {}, at::kLong);
    check(lethe_gdn_compact_states(r.s.data(), static_cast<int32_t>(r.s.size()), S, ptr<uint8_t>(live), ptr<int64_t>(place), ptr<int64_t>(count),
                                   status_word(live.device().index()), stream_of(live)));
    changed(r);
    return {place, count};
  });
}

}  // namespace

void bind_beam(pybind11::module_& m) {
  using pybind11::arg;
  m.def("beam_select", &beam_select, arg("logits"), arg("scores"), arg("allowed"), arg("finished"), arg("penalty"), arg("k"), arg("temperature"), arg("eos"));
  m.def("reorder_states", &reorder_states);
  m.def("fork_states", &fork_states);
  m.def("compact_states", &compact_states);
}

}  // namespace lethe_torch
