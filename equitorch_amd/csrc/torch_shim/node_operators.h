// Autograd nodes of the operators on invariant node features over the C ABI: embedding of node kinds, attention among the nodes of
// a structure, gated feed-forward block.  Operands are checked by the Python layer, which also holds the same launches
// through ctypes for when this extension is not there; a backward under gradient mode hands over to a Python callable.
#pragma once

#include <functional>

#include "cgtp.h"

namespace {

// A Python callable for gradients of higher order, kept under a number until its last holder goes.
struct Fallback {
  int64_t id = -1;
  std::shared_ptr<void> guard;
  void set(py::object fn) {
    static int64_t next = (int64_t)1 << 40;            // apart from the numbers of edge handles
    const int64_t mine = next++;
    edge_fallbacks()[mine] = std::move(fn);
    id = mine;
    guard = std::shared_ptr<void>(nullptr, [mine](void*) {
      if (!Py_IsInitialized()) return;
      py::gil_scoped_acquire gil;
      edge_fallbacks().erase(mine);
    });
  }
};
// Keeps a callable for as long as a node may ask for it, whatever becomes of the plan.
struct FallbackHolder : torch::CustomClassHolder {
  Fallback fallback;
  explicit FallbackHolder(const Fallback& f) : fallback(f) {}
};
// fn(grad_out, inputs, need, *more) -> gradients, into the first places of `places`.
template <typename... More>
variable_list call_fallback(int64_t id, const at::Tensor& g, const variable_list& inputs, const std::vector<bool>& need, size_t places,
                            More... more) {
  py::gil_scoped_acquire gil;
  const auto it = edge_fallbacks().find(id);
  TORCH_CHECK(it != edge_fallbacks().end(), "cgtp: no tensor expression for a gradient of higher order");
  py::list in, wanted;
  for (const auto& t : inputs) in.append(t.defined() ? py::cast(t) : py::none());
  for (bool n : need) wanted.append(n);
  const py::tuple r = it->second(g, in, wanted, more...);
  variable_list out(places);
  for (size_t i = 0; i < inputs.size(); ++i)
    if (!r[i].is_none()) out[i] = r[i].cast<at::Tensor>();
  return out;
}

int32_t code_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CGTP_F32;
    case at::kDouble: return CGTP_F64;
    case at::kBFloat16: return CGTP_BF16;
    default: return CGTP_F16;
  }
}
at::Tensor bytes_on(const at::Tensor& like, int64_t n) { return at::empty({n}, like.options().dtype(at::kByte)); }
void* mutable_ptr(const at::Tensor& t) { return const_cast<void*>(ptr_or_null(t)); }

// ---- embedding ------------------------------------------------------------------------------------------------------
struct EmbedGrad;
struct Embed : torch::autograd::Function<Embed> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& kind, const at::Tensor& table, double scale) {
    c10::hip::HIPGuardMasqueradingAsCUDA guard(table.device());
    auto shape = kind.sizes().vec();
    shape.push_back(table.size(1));
    at::Tensor out = at::empty(shape, table.options());
    check_status(cgtp_embed_forward(kind.data_ptr<int64_t>(), table.data_ptr(), out.data_ptr(), kind.numel(), table.size(0),
                                    (int)table.size(1), scale, code_of(table), current_stream(table)), "cgtp_embed_forward");
    ctx->save_for_backward({kind});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["kinds"] = table.size(0);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g);
};
// The gradient is linear in grad_out; its own gradient is the lookup again.
struct EmbedGrad : torch::autograd::Function<EmbedGrad> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& kind, const at::Tensor& grad_out, int64_t kinds, double scale) {
    c10::hip::HIPGuardMasqueradingAsCUDA guard(grad_out.device());
    const at::Tensor g = grad_out.contiguous();
    const int64_t n = kind.numel(), c = g.size(-1);
    at::Tensor out = at::empty({kinds, c}, g.options());
    const at::Tensor ws = bytes_on(g, cgtp_embed_workspace_bytes(n, kinds, (int)c, code_of(g)));
    check_status(cgtp_embed_backward(kind.data_ptr<int64_t>(), g.data_ptr(), out.data_ptr(), ws.data_ptr(), n, kinds, (int)c, scale,
                                     code_of(g), current_stream(g)), "cgtp_embed_backward");
    ctx->save_for_backward({kind});
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return {at::Tensor(), Embed::apply(ctx->get_saved_variables()[0], g[0].contiguous(), ctx->saved_data["scale"].toDouble()),
            at::Tensor(), at::Tensor()};
  }
};
inline variable_list Embed::backward(AutogradContext* ctx, variable_list g) {
  return {at::Tensor(), EmbedGrad::apply(ctx->get_saved_variables()[0], g[0], ctx->saved_data["kinds"].toInt(),
                                         ctx->saved_data["scale"].toDouble()), at::Tensor()};
}

// ---- gated feed-forward block -----------------------------------------------------------------------------------------
cgtp_gff_args gff_args(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t act) {
  cgtp_gff_args a{};
  a.x = x.data_ptr();
  a.w_gate = wg.data_ptr();
  a.w_up = wu.data_ptr();
  a.w_down = wd.data_ptr();
  a.n_rows = x.size(0);
  a.c_in = (int32_t)x.size(1);
  a.hidden = (int32_t)wg.size(1);
  a.c_out = (int32_t)wd.size(1);
  a.activation = (int32_t)act;
  a.dtype = code_of(x);
  return a;
}

// keep: (gate, up, mid) one after the other for a backward, else mid alone.
at::Tensor gff_forward(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t act, bool keep,
                       at::Tensor* kept) {
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  cgtp_gff_args a = gff_args(x, wg, wu, wd, act);
  at::Tensor out = at::empty({a.n_rows, a.c_out}, x.options());
  const int64_t width = (a.hidden + 7) / 8 * 8;
  *kept = at::empty({keep ? 3 : 1, a.n_rows, width}, x.options());
  char* p = (char*)kept->data_ptr();
  const int64_t each = a.n_rows * width * x.element_size();
  if (keep) {
    a.gate = p;
    a.up = p + each;
    p += 2 * each;
  }
  a.mid = p;
  a.out = out.data_ptr();
  at::Tensor ws;
  if (const int64_t n = cgtp_gff_workspace_bytes(&a, 0)) {
    ws = bytes_on(x, n);
    a.workspace = ws.data_ptr();
  }
  check_status(cgtp_gff_forward(&a, current_stream(x)), "cgtp_gff_forward");
  return out;
}

struct Gff : torch::autograd::Function<Gff> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd,
                            int64_t act, int64_t fallback) {
    at::Tensor kept;
    at::Tensor out = gff_forward(x, wg, wu, wd, act, true, &kept);
    ctx->save_for_backward({x, wg, wu, wd, kept});
    ctx->saved_data["act"] = act;
    ctx->saved_data["fallback"] = fallback;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const variable_list s = ctx->get_saved_variables();
    std::vector<bool> need;
    for (size_t i = 0; i < 4; ++i) need.push_back(ctx->needs_input_grad(i));
    if (at::GradMode::is_enabled())
      return call_fallback(ctx->saved_data["fallback"].toInt(), grad[0], {s[0], s[1], s[2], s[3]}, need, 6);
    const at::Tensor &x = s[0], &kept = s[4];
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    cgtp_gff_args a = gff_args(x, s[1], s[2], s[3], ctx->saved_data["act"].toInt());
    const at::Tensor g = grad[0].contiguous();
    variable_list out(6);
    for (size_t i = 0; i < 4; ++i)
      if (need[i]) out[i] = at::empty(s[i].sizes(), s[i].options());
    const int64_t width = kept.size(2);
    const at::Tensor mids = at::empty({2, a.n_rows, width}, x.options());
    const int64_t each = a.n_rows * width * x.element_size();
    char *p = (char*)kept.data_ptr(), *q = (char*)mids.data_ptr();
    a.gate = p;
    a.up = p + each;
    a.mid = p + 2 * each;
    a.grad_gate = q;
    a.grad_up = q + each;
    a.grad_out = g.data_ptr();
    a.grad_x = mutable_ptr(out[0]);
    a.grad_w_gate = mutable_ptr(out[1]);
    a.grad_w_up = mutable_ptr(out[2]);
    a.grad_w_down = mutable_ptr(out[3]);
    at::Tensor ws;
    if (const int64_t n = cgtp_gff_workspace_bytes(&a, 1)) {
      ws = bytes_on(x, n);
      a.workspace = ws.data_ptr();
    }
    check_status(cgtp_gff_backward(&a, current_stream(x)), "cgtp_gff_backward");
    return out;
  }
};

// ---- attention among the nodes of a structure ---------------------------------------------------------------------------
// The kernels' tables of a plan for one number of heads.
struct AttnHandle {
  at::Tensor q_items, q_joins, k_items, k_joins;
  int64_t q_slots, k_slots, wide_q, wide_k, stream;      // stream: what the tables were allocated on
  Fallback fallback;
  void set_fallback(py::object fn) { fallback.set(std::move(fn)); }
};

// The tables are read on the current stream: where that is not the stream of their memory, the memory is not handed out again
// before what is queued here is done, whatever becomes of the plan.
void record_tables(const AttnHandle& h, const at::Tensor& like) {
  const auto s = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(like.device().index());
  if ((int64_t)s.stream() == h.stream) return;
  for (const at::Tensor& t : {h.q_items, h.q_joins, h.k_items, h.k_joins})
    if (t.defined()) t.record_stream(s.unwrap());
}

struct AttnOperands {
  at::Tensor q, k, v, pos_q, pos_k, slope;      // pos_k undefined: the queries' positions are the keys' too
};

cgtp_attn_args attn_args(const AttnOperands& o, const AttnHandle& h, double scale, double cap) {
  cgtp_attn_args a{};
  a.q = o.q.data_ptr();
  a.k = o.k.data_ptr();
  a.v = o.v.data_ptr();
  a.q_node = o.q.stride(0);
  a.q_head = o.q.stride(1);
  a.k_node = o.k.stride(0);
  a.k_head = o.k.stride(1);
  a.v_node = o.v.stride(0);
  a.v_head = o.v.stride(1);
  a.pos_q = (const float*)ptr_or_null(o.pos_q);
  a.pos_k = (const float*)ptr_or_null(o.pos_k.defined() ? o.pos_k : o.pos_q);
  a.slope = (const float*)ptr_or_null(o.slope);
  a.n_q = o.q.size(0);
  a.n_k = o.k.size(0);
  a.h_q = (int32_t)o.q.size(1);
  a.h_kv = (int32_t)o.k.size(1);
  a.dim = (int32_t)o.q.size(2);
  a.dtype = code_of(o.q);
  a.scale = (float)scale;
  a.cap = (float)cap;
  a.same_pos = !o.pos_k.defined();
  auto table = [](const at::Tensor& t, const cgtp_attn_item*& p, int32_t& n) {
    p = (const cgtp_attn_item*)ptr_or_null(t);
    n = t.defined() ? (int32_t)t.size(0) : 0;
  };
  table(h.q_items, a.q_items, a.n_q_items);
  table(h.q_joins, a.q_joins, a.n_q_joins);
  table(h.k_items, a.k_items, a.n_k_items);
  table(h.k_joins, a.k_joins, a.n_k_joins);
  a.n_q_slots = (int32_t)h.q_slots;
  a.n_k_slots = (int32_t)h.k_slots;
  a.wide_q = (int32_t)h.wide_q;
  a.wide_k = (int32_t)h.wide_k;
  return a;
}

at::Tensor attn_forward(const AttnOperands& o, const AttnHandle& h, double scale, double cap, at::Tensor* lse) {
  c10::hip::HIPGuardMasqueradingAsCUDA guard(o.q.device());
  cgtp_attn_args a = attn_args(o, h, scale, cap);
  at::Tensor out = at::empty(o.q.sizes(), o.q.options());
  if (lse) *lse = at::empty({a.n_q, (int64_t)a.h_q}, o.q.options().dtype(at::kFloat));
  a.out = out.data_ptr();
  a.lse = lse ? lse->data_ptr() : nullptr;
  at::Tensor ws;
  if (const int64_t n = cgtp_attn_workspace_bytes(&a, 0)) {
    ws = bytes_on(o.q, n);
    a.workspace = ws.data_ptr();
  }
  record_tables(h, o.q);
  check_status(cgtp_attn_forward(&a, current_stream(o.q)), "cgtp_attn_forward");
  return out;
}

struct Attn : torch::autograd::Function<Attn> {
  typedef c10::optional<at::Tensor> Optional;
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const Optional& pos_q,
                            const Optional& pos_k, const Optional& slope, const AttnHandle* h, double scale, double cap) {
    const AttnOperands o = {q, k, v, opt(pos_q), opt(pos_k), opt(slope)};
    at::Tensor lse;
    at::Tensor out = attn_forward(o, *h, scale, cap, &lse);
    ctx->save_for_backward({q, k, v, o.pos_q, o.pos_k, o.slope, out, lse, h->q_items, h->q_joins, h->k_items, h->k_joins});
    auto& d = ctx->saved_data;
    d["shape"] = std::vector<int64_t>{h->q_slots, h->k_slots, h->wide_q, h->wide_k, h->stream, h->fallback.id};
    d["scale"] = scale;
    d["cap"] = cap;
    d["keep"] = c10::IValue::make_capsule(c10::make_intrusive<FallbackHolder>(h->fallback));
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const variable_list s = ctx->get_saved_variables();
    const AttnOperands o = {s[0], s[1], s[2], s[3], s[4], s[5]};
    auto& d = ctx->saved_data;
    const std::vector<int64_t> shape = d["shape"].toIntVector();
    std::vector<bool> need;
    size_t edge = 0;                    // the node has an edge for each operand that is there
    for (size_t i = 0; i < 6; ++i) need.push_back(s[i].defined() && ctx->needs_input_grad(edge++));
    if (at::GradMode::is_enabled())
      return call_fallback(shape[5], grad[0], {s[0], s[1], s[2], s[3], s[4], s[5]}, need, 9, d["scale"].toDouble(),
                           d["cap"].toDouble());
    c10::hip::HIPGuardMasqueradingAsCUDA guard(o.q.device());
    const AttnHandle h{s[8], s[9], s[10], s[11], shape[0], shape[1], shape[2], shape[3], shape[4], {}};
    cgtp_attn_args a = attn_args(o, h, d["scale"].toDouble(), d["cap"].toDouble());
    at::Tensor g = grad[0].contiguous();
    if ((uintptr_t)g.data_ptr() & 15) g = g.clone();
    a.out = s[6].data_ptr();
    a.lse = s[7].data_ptr();
    a.grad_out = g.data_ptr();
    variable_list out(9);
    for (size_t i = 0; i < 6; ++i)
      if (need[i]) out[i] = at::empty(s[i].sizes(), s[i].options());
    a.grad_q = mutable_ptr(out[0]);
    a.grad_k = mutable_ptr(out[1]);
    a.grad_v = mutable_ptr(out[2]);
    a.grad_pos_q = (float*)mutable_ptr(out[3]);
    a.grad_pos_k = (float*)mutable_ptr(out[4]);
    a.grad_slope = (float*)mutable_ptr(out[5]);
    const at::Tensor ws = bytes_on(o.q, cgtp_attn_workspace_bytes(&a, 1));
    a.workspace = ws.data_ptr();
    record_tables(h, o.q);
    check_status(cgtp_attn_backward(&a, current_stream(o.q)), "cgtp_attn_backward");
    return out;
  }
};

void bind_node_operators(py::module& m) {
  m.def("embed", [](const at::Tensor& kind, const at::Tensor& table, double scale) { return Embed::apply(kind, table, scale); },
        "embedding of node kinds with its autograd node");
  py::class_<Fallback>(m, "Fallback").def(py::init([](py::object fn) {
    Fallback f;
    f.set(std::move(fn));
    return f;
  }));
  m.def("gff", [](const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd, int64_t act, bool keep,
                  const Fallback& fallback) {
    if (keep) return Gff::apply(x, wg, wu, wd, act, fallback.id);
    at::Tensor mid;
    return gff_forward(x, wg, wu, wd, act, false, &mid);
  }, "gated feed-forward block; with its autograd node where a backward may follow (keep)");
  py::class_<AttnHandle>(m, "AttnHandle")
      .def(py::init([](c10::optional<at::Tensor> q_items, c10::optional<at::Tensor> q_joins, c10::optional<at::Tensor> k_items,
                       c10::optional<at::Tensor> k_joins, int64_t q_slots, int64_t k_slots, int64_t wide_q, int64_t wide_k, int64_t stream) {
        return AttnHandle{opt(q_items), opt(q_joins), opt(k_items), opt(k_joins), q_slots, k_slots, wide_q, wide_k, stream, {}};
      }))
      .def("set_fallback", &AttnHandle::set_fallback, "callable (grad_out, inputs, need, scale, cap) -> gradients, for gradients of higher order");
  m.def("attn", [](const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& pos_q,
                   const c10::optional<at::Tensor>& pos_k, const c10::optional<at::Tensor>& slope, const AttnHandle& h, double scale,
                   double cap, bool keep) {
    if (keep) return Attn::apply(q, k, v, pos_q, pos_k, slope, &h, scale, cap);
    return attn_forward({q, k, v, opt(pos_q), opt(pos_k), opt(slope)}, h, scale, cap, nullptr);
  }, "attention among the nodes of a structure; with its autograd node where a backward may follow (keep)");
}

}  // namespace
