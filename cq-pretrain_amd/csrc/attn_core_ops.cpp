// PyTorch-ROCm operators of the attention over 16-bit keys and values: training over packed rows, the 16-bit cache.
//
// Schemas:
//   attend(q, k, v, limit, first?, positions?, slopes?, scale, cap) -> (out, lse), differentiable in q, k and v
//       q [T,Hq,D], k, v [S,Hk,D] of one type (bf16 or fp16); limit, first, positions int32 [T]; slopes fp32 [Hq]
//   attend_bwd(dy, dlse?, q, k, v, out, lse, limit, first?, positions?, slopes?, scale, cap, want_keys) -> (dq, dk, dv)
//   kv16_append(q?, k, v, positions?, turns?, axis?, adjacent, slots, data!) -> q'
//   kv16_attend(q, data, tables, starts, visible, positions?, slopes?, window, scale, cap, max_queries, want_lse)
//       -> (out, lse)

#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "attn_ops.hpp"

namespace {

typedef std::optional<Tensor> Maybe;

const Tensor* given(const Maybe& x) { return x.has_value() && x->defined() ? &*x : nullptr; }

// rows as the kernels read them: the offsets of a tile's tokens and heads fit 32 bits
Tensor core_rows(const Tensor& x) {
  return x.stride(0) < 1 << 24 && x.stride(1) * x.size(1) < 1 << 29 ? head_rows(x) : x.clone(at::MemoryFormat::Contiguous);
}

// an int32 value a row, dense, or none
Tensor row_values(const Maybe& x, int64_t T, const char* name) {
  const Tensor* t = given(x);
  if (!t) return {};
  int32_vector(*t, name);
  TORCH_CHECK_VALUE(t->numel() == T, name, " must hold a value a row");
  return t->contiguous();
}

Tensor head_slopes(const Maybe& x, int64_t heads) {
  const Tensor* t = given(x);
  if (!t) return {};
  TORCH_CHECK_VALUE(t->dim() == 1 && t->numel() == heads && t->scalar_type() == at::kFloat,
                    "slopes must hold an fp32 value a query head");
  TORCH_CHECK_VALUE(!t->requires_grad() || !at::GradMode::is_enabled(), "slopes are constants: no gradient passes to them");
  return t->contiguous();
}

const int32_t* ints(const Tensor& x) { return x.defined() ? x.data_ptr<int32_t>() : nullptr; }
const float* floats(const Tensor& x) { return x.defined() ? x.data_ptr<float>() : nullptr; }

void check_scores(double scale, double cap) {
  TORCH_CHECK_VALUE(std::isfinite((float)scale), "scale must be finite");
  TORCH_CHECK_VALUE(std::isfinite((float)cap) && cap >= 0 && (cap == 0 || (float)cap > 0), "cap must be positive and finite");
}

struct Packed {
  int dtype;
  int64_t T, S;
  int heads, kv, D;
  Tensor limit, first, positions, slopes;
};
Packed check_packed(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& limit, const Maybe& first,
                    const Maybe& positions, const Maybe& slopes, double scale, double cap) {
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && q.size(2) == k.size(2),
                    "q must be [T, heads, head_dim], k and v [S, kv_heads, head_dim]");
  Packed p{dtype_code(q, "q"), q.size(0), k.size(0), (int)q.size(1), (int)k.size(1), (int)q.size(2)};
  TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v must share one type");
  TORCH_CHECK_VALUE(p.D == 64 || p.D == 128 || p.D == 256, "head_dim must be 64, 128 or 256");
  TORCH_CHECK_VALUE(p.heads > 0 && p.kv > 0 && p.heads % p.kv == 0, p.heads, " query heads are no multiple of ", p.kv,
                    " key heads");
  check_scores(scale, cap);
  p.limit = row_values(limit, p.T, "limit");
  p.first = row_values(first, p.T, "first");
  p.positions = row_values(positions, p.T, "positions");
  p.slopes = head_slopes(slopes, p.heads);
  on_one_gpu({&q, &k, &v, &p.limit, p.first.defined() ? &p.first : &q, p.positions.defined() ? &p.positions : &q,
              p.slopes.defined() ? &p.slopes : &q});
  return p;
}

std::tuple<Tensor, Tensor> attend(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& limit,
                                  const Maybe& first, const Maybe& positions, const Maybe& slopes, double scale, double cap) {
  const Packed p = check_packed(q, k, v, limit, first, positions, slopes, scale, cap);
  const c10::DeviceGuard guard(q.device());
  const Tensor qc = core_rows(q), kc = core_rows(k), vc = core_rows(v);
  Tensor out = at::empty(q.sizes(), q.options()), lse = at::empty({p.T, p.heads}, q.options().dtype(at::kFloat));
  const size_t need = cqgdn_attend_fwd_workspace_size(p.T, p.S, p.heads, p.kv, p.D);
  Tensor ws;
  if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  check(cqgdn_attend_fwd(qc.data_ptr(), qc.stride(0), qc.stride(1), kc.data_ptr(), kc.stride(0), kc.stride(1), vc.data_ptr(),
                         vc.stride(0), vc.stride(1), p.dtype, p.T, p.S, p.heads, p.kv, p.D, ints(p.first), ints(p.limit),
                         ints(p.positions), (float)scale, (float)cap, floats(p.slopes), out.data_ptr(), lse.data_ptr<float>(),
                         need ? ws.data_ptr() : nullptr, need, stream_of(q)),
        "cqgdn_attend_fwd");
  return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> attend_bwd(const Tensor& dy, const Maybe& dlse, const Tensor& q, const Tensor& k,
                                              const Tensor& v, const Tensor& out, const Tensor& lse, const Tensor& limit,
                                              const Maybe& first, const Maybe& positions, const Maybe& slopes, double scale,
                                              double cap, bool want_keys) {
  const Packed p = check_packed(q, k, v, limit, first, positions, slopes, scale, cap);
  TORCH_CHECK_VALUE(dy.sizes() == q.sizes() && dy.scalar_type() == q.scalar_type() && out.sizes() == q.sizes() &&
                        out.scalar_type() == q.scalar_type(), "dy and out must be as q");
  const Tensor* dl = given(dlse);
  for (const Tensor* x : {&lse, dl ? dl : &lse})
    TORCH_CHECK_VALUE(x->dim() == 2 && x->size(0) == p.T && x->size(1) == p.heads && x->scalar_type() == at::kFloat,
                      "lse and dlse must be fp32 [T, heads]");
  on_one_gpu({&q, &dy, &out, &lse, dl ? dl : &lse});
  const c10::DeviceGuard guard(q.device());
  const Tensor qc = core_rows(q), kc = core_rows(k), vc = core_rows(v), dyc = core_rows(dy), yc = out.contiguous(),
               l = lse.contiguous(), d = dl ? dl->contiguous() : Tensor();
  Tensor dq = at::empty(q.sizes(), q.options()), dk, dv;
  if (want_keys) {
    dk = at::empty(k.sizes(), k.options());
    dv = at::empty(k.sizes(), k.options());
  }
  const size_t need = cqgdn_attend_bwd_workspace_size(p.T, p.S, p.heads, p.kv, p.D);
  Tensor ws;
  if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  check(cqgdn_attend_bwd(qc.data_ptr(), qc.stride(0), qc.stride(1), kc.data_ptr(), kc.stride(0), kc.stride(1), vc.data_ptr(),
                         vc.stride(0), vc.stride(1), dyc.data_ptr(), dyc.stride(0), dyc.stride(1), p.dtype, p.T, p.S, p.heads,
                         p.kv, p.D, ints(p.first), ints(p.limit), ints(p.positions), (float)scale, (float)cap,
                         floats(p.slopes), yc.data_ptr(), l.data_ptr<float>(), floats(d), dq.data_ptr(),
                         want_keys ? dk.data_ptr() : nullptr, want_keys ? dv.data_ptr() : nullptr,
                         need ? ws.data_ptr() : nullptr, need, stream_of(q)),
        "cqgdn_attend_bwd");
  return {dq, dk, dv};
}

// In C++, as rotary's: a Python function and its engine call cost more than the kernels of a small step.
struct Attend : torch::autograd::Function<Attend> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                const Tensor& v, const Tensor& limit, const Maybe& first,
                                                const Maybe& positions, const Maybe& slopes, double scale, double cap) {
    const at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("cqgdn::attend", "").typed<decltype(attend)>();
    const auto [out, lse] = op.call(q, k, v, limit, first, positions, slopes, scale, cap);
    const auto or_none = [](const Maybe& x) { return given(x) ? *x : Tensor(); };
    ctx->save_for_backward({q, k, v, out, lse, limit, or_none(first), or_none(positions), or_none(slopes)});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["cap"] = cap;
    return {out, lse};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 const torch::autograd::variable_list& grad) {
    if (!grad[0].defined() && !grad[1].defined()) return torch::autograd::variable_list(9);
    const auto x = ctx->get_saved_variables();
    const auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
    TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), "attend: second derivatives are not implemented");
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("cqgdn::attend_bwd", "").typed<decltype(attend_bwd)>();
    const bool keys = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const auto [dq, dk, dv] = op.call(grad[0].defined() ? grad[0] : at::zeros_like(x[3]), maybe(grad[1]), x[0], x[1], x[2], x[3],
                                      x[4], x[5], maybe(x[6]), maybe(x[7]), maybe(x[8]), ctx->saved_data["scale"].toDouble(),
                                      ctx->saved_data["cap"].toDouble(), keys);
    return {ctx->needs_input_grad(0) ? dq : Tensor(), ctx->needs_input_grad(1) ? dk : Tensor(),
            ctx->needs_input_grad(2) ? dv : Tensor(), {}, {}, {}, {}, {}, {}};
  }
};
std::tuple<Tensor, Tensor> attend_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& limit,
                                           const Maybe& first, const Maybe& positions, const Maybe& slopes, double scale,
                                           double cap) {
  for (const Tensor* x : {&q, &k, &v})
    TORCH_CHECK_NOT_IMPLEMENTED(!x->_fw_grad(0).defined(), "attend: derivatives in forward mode are not implemented");
  head_slopes(slopes, q.dim() == 3 ? q.size(1) : 0);  // refuses a gradient, which the calls below no longer see
  if (!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || v.requires_grad())) {
    const at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("cqgdn::attend", "").typed<decltype(attend)>();
    return op.call(q, k, v, limit, first, positions, slopes, scale, cap);
  }
  const auto out = Attend::apply(q, k, v, limit, first, positions, slopes, scale, cap);
  return {out[0], out[1]};
}

void check_data16(const Tensor& data) {
  TORCH_CHECK_VALUE(data.dim() == 5 && data.is_contiguous() && data.size(1) > 0 && data.size(1) <= 65535 && data.size(2) == 2,
                    "data must be contiguous [pages, kv_heads, 2, page, head_dim]");
  dtype_code(data, "data");
  const int64_t page = data.size(3), D = data.size(4);
  TORCH_CHECK_VALUE(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256");
  TORCH_CHECK_VALUE(page >= 16 && page <= 65536 && (page & (page - 1)) == 0, "page must be a power of two from 16 to 65536");
}

Tensor kv16_append(const Maybe& q, const Tensor& k, const Tensor& v, const Maybe& positions, const Maybe& turns,
                   const Maybe& axis, bool adjacent, const Tensor& slots, Tensor& data) {
  check_data16(data);
  TORCH_CHECK_VALUE(k.dim() == 3 && v.sizes() == k.sizes() && k.size(1) == data.size(1) && k.size(2) == data.size(4),
                    "k and v must be [T, kv_heads, head_dim], as the cache is");
  TORCH_CHECK_VALUE(k.scalar_type() == data.scalar_type() && v.scalar_type() == data.scalar_type(),
                    "k and v must be of the cache's type");
  int32_vector(slots, "slots");
  const int64_t T = k.size(0), D = k.size(2);
  TORCH_CHECK_VALUE(slots.numel() == T, "slots must hold a value a row");
  const Tensor* x = given(q);
  TORCH_CHECK_VALUE(!x || (x->dim() == 3 && x->size(0) == T && x->size(2) == D && x->scalar_type() == k.scalar_type()),
                    "q must be [T, heads, head_dim] of the type of k");
  const Tensor *p = given(positions), *u = given(turns), *w = given(axis);
  TORCH_CHECK_VALUE((p && u && w) || (!p && !u && !w), "positions come with a plan's turns and axis");
  if (p) {
    TORCH_CHECK_VALUE(p->dim() == 2 && p->size(0) > 0 && p->size(1) == T &&
                          (p->scalar_type() == at::kInt || p->scalar_type() == at::kLong),
                      "positions must be int32 or int64 [axes, T]");
    TORCH_CHECK_VALUE(u->dim() == 1 && u->scalar_type() == at::kLong && u->is_contiguous() && w->dim() == 1 &&
                          w->scalar_type() == at::kInt && w->is_contiguous() && w->numel() == u->numel(),
                      "the plan's turns (int64) and axis (int32) must be dense vectors of one length");
    TORCH_CHECK_VALUE(2 * u->numel() <= D, "the plan turns ", 2 * u->numel(), " values of a head, which has ", D);
  }
  on_one_gpu({&data, &k, &v, &slots, x ? x : &k, p ? p : &k, u ? u : &k, w ? w : &k});
  const c10::DeviceGuard guard(k.device());
  const auto rows = [](const Tensor& t) { return t.stride(2) == 1 ? t : t.contiguous(); };
  const Tensor kc = rows(k), vc = rows(v), qc = x ? rows(*x) : Tensor(), s = slots.contiguous();
  const Tensor pc = p ? (p->stride(1) == 1 ? *p : p->contiguous()) : Tensor();
  Tensor out = at::empty({T, x ? x->size(1) : 0, D}, k.options());
  check(cqgdn_kv16_append(x ? qc.data_ptr() : nullptr, x ? qc.stride(0) : 0, x ? qc.stride(1) : 0, (int)out.size(1),
                          kc.data_ptr(), kc.stride(0), kc.stride(1), vc.data_ptr(), vc.stride(0), vc.stride(1), T,
                          (int)k.size(1), (int)D, u ? (int)(2 * u->numel()) : 0, adjacent, dtype_code(k, "k"),
                          p ? pc.data_ptr() : nullptr, p && p->scalar_type() == at::kLong, p ? pc.stride(0) : 0,
                          p ? (int)p->size(0) : 0,
                          u ? reinterpret_cast<const uint64_t*>(u->data_ptr<int64_t>()) : nullptr,
                          w ? w->data_ptr<int32_t>() : nullptr, s.data_ptr<int32_t>(), out.data_ptr(), data.data_ptr(),
                          data.size(0), (int)data.size(3), stream_of(k)),
        "cqgdn_kv16_append");
  return out;
}

std::tuple<Tensor, Tensor> kv16_attend(const Tensor& q, const Tensor& data, const Tensor& tables, const Tensor& starts,
                                       const Tensor& visible, const Maybe& positions, const Maybe& slopes, int64_t window,
                                       double scale, double cap, int64_t max_queries, bool want_lse) {
  check_data16(data);
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(2) == data.size(4) && q.scalar_type() == data.scalar_type(),
                    "q must be [T, heads, head_dim] of the cache's type and head_dim");
  const int64_t T = q.size(0), heads = q.size(1), kv = data.size(1), N = tables.dim() == 2 ? tables.size(0) : -1;
  TORCH_CHECK_VALUE(heads > 0 && heads % kv == 0, heads, " query heads are no multiple of ", kv, " key heads");
  TORCH_CHECK_VALUE(N >= 0 && tables.scalar_type() == at::kInt, "tables must be int32 [requests, columns]");
  int32_vector(starts, "starts");
  int32_vector(visible, "visible");
  TORCH_CHECK_VALUE(starts.numel() == N + 1 && visible.numel() == T,
                    "starts must hold a value a request and one more, visible a value a row");
  const Tensor pos = row_values(positions, T, "positions");
  const at::NoGradGuard constants;  // no gradient passes through the cache
  const Tensor slope = head_slopes(slopes, heads);
  check_scores(scale, cap);
  TORCH_CHECK_VALUE(window >= 0 && window <= INT32_MAX, "window must be positive");
  TORCH_CHECK_VALUE(max_queries > 0, "max_queries must be positive");
  TORCH_CHECK_VALUE(tables.size(1) <= INT32_MAX && T <= INT32_MAX && N < INT32_MAX, "sizes are 32-bit");
  on_one_gpu({&q, &data, &tables, &starts, &visible, pos.defined() ? &pos : &q, slope.defined() ? &slope : &q});
  const c10::DeviceGuard guard(q.device());
  const Tensor qc = head_rows(q), st = starts.contiguous(), vis = visible.contiguous();
  const Tensor tab = (tables.stride(1) == 1 || tables.size(1) <= 1) && (N <= 1 || tables.stride(0) >= tables.size(1))
                         ? tables
                         : tables.contiguous();
  Tensor out = at::empty({T, heads, q.size(2)}, q.options());
  Tensor lse = at::empty({want_lse ? T : 0, heads}, q.options().dtype(at::kFloat));
  const int most = (int)std::min(max_queries, std::max<int64_t>(T, 1)), columns = (int)tab.size(1), page = (int)data.size(3);
  const size_t need = cqgdn_kv16_attend_workspace_size(T, (int)N, (int)heads, (int)kv, (int)q.size(2), most, columns, page);
  Tensor ws;
  if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  check(cqgdn_kv16_attend(qc.data_ptr(), qc.stride(0), qc.stride(1), dtype_code(q, "q"), T, (int)heads, (int)q.size(2),
                          data.data_ptr(), data.size(0), page, (int)kv, tab.data_ptr<int32_t>(),
                          N > 1 ? tab.stride(0) : columns, columns, st.data_ptr<int32_t>(), (int)N, vis.data_ptr<int32_t>(),
                          (int)window, ints(pos), (float)scale, (float)cap, floats(slope), most, out.data_ptr(),
                          want_lse ? lse.data_ptr<float>() : nullptr, need ? ws.data_ptr() : nullptr, need, stream_of(q)),
        "cqgdn_kv16_attend");
  return {out, lse};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(cqgdn, m) {
  m.def("attend(Tensor q, Tensor k, Tensor v, Tensor limit, Tensor? first, Tensor? positions, Tensor? slopes, float scale, "
        "float cap) -> (Tensor, Tensor)");
  m.def("attend_bwd(Tensor dy, Tensor? dlse, Tensor q, Tensor k, Tensor v, Tensor out, Tensor lse, Tensor limit, "
        "Tensor? first, Tensor? positions, Tensor? slopes, float scale, float cap, bool want_keys) -> (Tensor, Tensor, Tensor)");
  m.def("kv16_append(Tensor? q, Tensor k, Tensor v, Tensor? positions, Tensor? turns, Tensor? axis, bool adjacent, "
        "Tensor slots, Tensor(a!) data) -> Tensor");
  m.def("kv16_attend(Tensor q, Tensor data, Tensor tables, Tensor starts, Tensor visible, Tensor? positions, "
        "Tensor? slopes, int window, float scale, float cap, int max_queries, bool want_lse) -> (Tensor, Tensor)");
}

// no gradient passes through the cache
TORCH_LIBRARY_IMPL(cqgdn, Autograd, m) {
  m.impl("attend", &attend_autograd);
  for (const char* name : {"kv16_append", "kv16_attend"}) m.impl(name, torch::CppFunction::makeFallthrough());
}

TORCH_LIBRARY_IMPL(cqgdn, CUDA, m) {
  m.impl("attend", &attend);
  m.impl("attend_bwd", &attend_bwd);
  m.impl("kv16_append", &kv16_append);
  m.impl("kv16_attend", &kv16_attend);
}

// CPU tensors reach the same functions only to be rejected by their checks.
TORCH_LIBRARY_IMPL(cqgdn, CPU, m) {
  m.impl("attend", &attend);
  m.impl("attend_bwd", &attend_bwd);
  m.impl("kv16_append", &kv16_append);
  m.impl("kv16_attend", &kv16_attend);
}
