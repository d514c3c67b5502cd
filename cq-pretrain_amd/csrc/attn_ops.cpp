// PyTorch-ROCm operators of the attention layers: rotary positions, the pages of a step, the 4-bit
// cache and the attention that reads it.  As in torch_ops.cpp each op allocates its outputs, enqueues on
// the current HIP stream of the tensors' device and turns error codes into Python exceptions.  The
// contract checks run before any launch and, but for the last ("a ROCm GPU"), for tensors on any device.
//
// Schemas:
//   rotary(q, k, positions, turns, axis, adjacent, backward) -> (q', k'), differentiable in q and k (both modes)
//       q [T,Hq,D], k [T,Hk,D] of one type; positions [A,T] int32 or int64
//   step_pages(cached, new, tables!, free!, free_count, page, tokens)
//       -> (starts, lengths, admitted, free_count, slots, positions, visible)
//   step_pages_(cached!, new, tables!, free!, free_count!, page, tokens)
//       -> (starts, admitted, slots, positions, visible); lengths and the count are written in place
//   kv4_write(data!, k, v, slots, page) -> (), kv4_read(data, slots, page, head_dim, fp16) -> (k, v)
//   kv4_attend(q, data, tables, starts, visible, page, window, scale, max_queries, want_lse) -> (out, lse)

#include <ATen/ATen.h>
#include <ATen/ops/_make_dual.h>
#include <ATen/ops/as_strided_native.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "cqgdn.h"

namespace {

using at::Tensor;

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check(int rc, const char* what) {
  if (rc == CQGDN_OK) return;
  TORCH_CHECK_VALUE(rc != CQGDN_EINVAL, what, ": ", cqgdn_last_error());
  TORCH_CHECK_NOT_IMPLEMENTED(rc != CQGDN_EUNSUPPORTED, what, ": ", cqgdn_last_error());
  TORCH_CHECK(false, what, ": ", cqgdn_last_error());
}

void on_one_gpu(std::initializer_list<const Tensor*> all) {
  const auto device = (*all.begin())->device();
  for (const Tensor* x : all) TORCH_CHECK_VALUE(x->device() == device, "tensors lie on different devices");
  TORCH_CHECK_VALUE(device.is_cuda(), "the hip GDN backend requires tensors on a ROCm GPU");
}

int dtype_code(const Tensor& x, const char* name) {
  const auto t = x.scalar_type();
  TORCH_CHECK_VALUE(t == at::kBFloat16 || t == at::kHalf, name, " must be bf16 or fp16");
  return t == at::kHalf ? CQGDN_F16 : CQGDN_BF16;
}

void int32_vector(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.dim() == 1 && x.scalar_type() == at::kInt, name, " must be an int32 vector");
}

// x as the kernels read rows of heads: unit stride within a head, 16-byte aligned rows
Tensor head_rows(const Tensor& x) {
  const bool fit = x.stride(2) == 1 && x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  return fit ? x : x.clone(at::MemoryFormat::Contiguous);
}

// n elements of the vector x from `at` on: a view made without the dispatcher's overhead, which seven narrow()
// would cost more of than the kernel takes
Tensor part(const Tensor& x, int64_t at, int64_t n) { return at::native::as_strided_tensorimpl(x, {n}, {1}, at); }

std::tuple<Tensor, Tensor> rotary(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& turns,
                                  const Tensor& axis, bool adjacent, bool backward) {
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && q.size(0) == k.size(0) && q.size(2) == k.size(2),
                    "q and k must be [T, heads, D] with one T and D");
  const auto t = q.scalar_type();
  TORCH_CHECK_VALUE((t == at::kBFloat16 || t == at::kHalf || t == at::kFloat) && k.scalar_type() == t,
                    "q and k must share one type: bf16, fp16 or fp32");
  TORCH_CHECK_VALUE(positions.dim() == 2 && positions.size(0) > 0 && positions.size(1) == q.size(0) &&
                        (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong),
                    "positions must be int32 or int64 [axes, T]");
  TORCH_CHECK_VALUE(turns.dim() == 1 && turns.scalar_type() == at::kLong && turns.is_contiguous() &&
                        axis.dim() == 1 && axis.scalar_type() == at::kInt && axis.is_contiguous() &&
                        axis.numel() == turns.numel(),
                    "the plan's turns (int64) and axis (int32) must be dense vectors of one length");
  TORCH_CHECK_VALUE(q.size(2) % 2 == 0 && 2 * turns.numel() <= q.size(2), "the plan turns ", 2 * turns.numel(),
                    " values of a head, which has ", q.size(2));
  on_one_gpu({&q, &k, &positions, &turns, &axis});
  const c10::DeviceGuard guard(q.device());
  const Tensor qc = q.stride(2) == 1 ? q : q.contiguous(), kc = k.stride(2) == 1 ? k : k.contiguous();
  const Tensor p = positions.stride(1) == 1 ? positions : positions.contiguous();
  Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
  const int dtype = t == at::kFloat ? CQGDN_F32 : t == at::kHalf ? CQGDN_F16 : CQGDN_BF16;
  check(cqgdn_rotary(qc.data_ptr(), qc.stride(0), qc.stride(1), (int)q.size(1), kc.data_ptr(), kc.stride(0),
                     kc.stride(1), (int)k.size(1), q.size(0), (int)q.size(2), (int)(2 * turns.numel()), adjacent,
                     backward, dtype, p.data_ptr(), p.scalar_type() == at::kLong, p.stride(0), (int)p.size(0),
                     reinterpret_cast<const uint64_t*>(turns.data_ptr<int64_t>()), axis.data_ptr<int32_t>(),
                     qo.data_ptr(), ko.data_ptr(), stream_of(q)),
        "cqgdn_rotary");
  return {qo, ko};
}

// The gradient of a turn is the turn back.  In C++ because a Python function and its engine call cost 40 us more
// than the kernels of a small step.  An output whose input needs no gradient needs none, and only gradients that are
// there are turned: the other operand goes in without heads, and where its input wants a gradient all the same (its
// output has no part in the loss), that is zeros.
struct Rotate : torch::autograd::Function<Rotate> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                const Tensor& positions, const Tensor& turns, const Tensor& axis,
                                                bool adjacent, bool backward) {
    const at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, turns, axis});
    ctx->saved_data["adjacent"] = adjacent;
    ctx->saved_data["backward"] = backward;
    ctx->saved_data["q"] = q.sizes().vec();
    ctx->saved_data["k"] = k.sizes().vec();
    static const auto op = rotary_op();
    const auto [y, z] = op.call(q, k, positions, turns, axis, adjacent, backward);
    if (!q.requires_grad()) ctx->mark_non_differentiable({y});
    if (!k.requires_grad()) ctx->mark_non_differentiable({z});
    return {y, z};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 const torch::autograd::variable_list& grad) {
    if (!grad[0].defined() && !grad[1].defined()) return {{}, {}, {}, {}, {}, {}, {}};
    static const auto op = rotary_op();
    const auto saved = ctx->get_saved_variables();
    const Tensor& one = grad[0].defined() ? grad[0] : grad[1];
    auto [dq, dk] = op.call(grad[0].defined() ? grad[0] : one.detach().narrow(1, 0, 0),
                            grad[1].defined() ? grad[1] : one.detach().narrow(1, 0, 0), saved[0], saved[1], saved[2],
                            ctx->saved_data["adjacent"].toBool(), !ctx->saved_data["backward"].toBool());
    const auto missing = [&](int i, const char* name) {
      return ctx->needs_input_grad(i) ? at::zeros(ctx->saved_data[name].toIntVector(), one.options()) : Tensor();
    };
    if (!grad[0].defined()) dq = missing(0, "q");
    if (!grad[1].defined()) dk = missing(1, "k");
    return {dq, dk, {}, {}, {}, {}, {}};
  }
  static c10::TypedOperatorHandle<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                             const Tensor&, bool, bool)>
  rotary_op() {
    return c10::Dispatcher::singleton()
        .findSchemaOrThrow("cqgdn::rotary", "")
        .typed<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, bool,
                                          bool)>();
  }
};
std::tuple<Tensor, Tensor> rotary_autograd(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& turns,
                                           const Tensor& axis, bool adjacent, bool backward) {
  // a turn is linear: its forward derivative is the turn of the tangents, of no heads where an input has none
  if (q._fw_grad(0).defined() || k._fw_grad(0).defined()) {
    static const auto op = Rotate::rotary_op();
    const auto [y, z] = op.call(q._fw_primal(0), k._fw_primal(0), positions, turns, axis, adjacent, backward);
    const Tensor tq = q._fw_grad(0), tk = k._fw_grad(0);
    const auto [ty, tz] = op.call(tq.defined() ? tq : y.detach().narrow(1, 0, 0),
                                  tk.defined() ? tk : z.detach().narrow(1, 0, 0), positions, turns, axis, adjacent, backward);
    return {tq.defined() ? at::_make_dual(y, ty, 0) : y, tk.defined() ? at::_make_dual(z, tz, 0) : z};
  }
  if (!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad())) {
    const at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = Rotate::rotary_op();
    return op.call(q, k, positions, turns, axis, adjacent, backward);
  }
  const auto out = Rotate::apply(q, k, positions, turns, axis, adjacent, backward);
  return {out[0], out[1]};
}

// what a step's pages come to; in place, lengths and left are the caller's own
struct Step {
  Tensor starts, lengths, admitted, left, slots, positions, visible;
};
Step pages_of_step(const Tensor& cached, const Tensor& fresh, const Tensor& tables, const Tensor& pool,
                   const Tensor& count, int64_t page, int64_t tokens, bool in_place) {
  int32_vector(cached, "cached");
  int32_vector(fresh, "new");
  int32_vector(pool, "free");
  int32_vector(count, "free_count");
  const int64_t N = cached.numel();
  TORCH_CHECK_VALUE(fresh.numel() == N && count.numel() == 1, "new must hold a value a request, free_count one value");
  TORCH_CHECK_VALUE(tables.dim() == 2 && tables.size(0) == N && tables.scalar_type() == at::kInt &&
                        (tables.stride(1) == 1 || tables.size(1) <= 1) && (tables.stride(0) >= tables.size(1) || N <= 1),
                    "tables must be int32 [requests, columns] with unit column stride");
  TORCH_CHECK_VALUE(cached.is_contiguous() && fresh.is_contiguous() && pool.is_contiguous(),
                    "cached, new and free must be contiguous");
  TORCH_CHECK_VALUE(page >= 16 && page <= 65536 && (page & (page - 1)) == 0,
                    "page must be a power of two from 16 to 65536");
  TORCH_CHECK_VALUE(tokens >= 0 && tokens <= INT32_MAX, "tokens must be a row count of 32 bits");
  TORCH_CHECK_VALUE(N <= INT32_MAX && tables.size(1) <= INT32_MAX && pool.numel() <= INT32_MAX, "sizes are 32-bit");
  on_one_gpu({&cached, &fresh, &tables, &pool, &count});
  const c10::DeviceGuard guard(cached.device());
  // one buffer: starts, admitted, lengths and the count (unless in place), then the three rows' vectors
  const int64_t rows = (tokens + 3) / 4 * 4, heads = (N + 1 + 3) / 4 * 4;
  const Tensor all = at::empty({3 * heads + 4 + 3 * rows}, cached.options());
  const Tensor starts = part(all, 0, N + 1), admitted = part(all, heads, N);
  const Tensor lengths = in_place ? cached : part(all, 2 * heads, N);
  const Tensor left = in_place ? count : part(all, 3 * heads, 1);
  const int64_t at = 3 * heads + 4;
  const Tensor slots = part(all, at, tokens), positions = part(all, at + rows, tokens),
               visible = part(all, at + 2 * rows, tokens);
  const int columns = (int)tables.size(1);
  check(cqgdn_step_pages(cached.data_ptr<int32_t>(), fresh.data_ptr<int32_t>(), (int)N, tables.data_ptr<int32_t>(),
                         N > 1 ? tables.stride(0) : columns, columns, pool.data_ptr<int32_t>(), (int)pool.numel(),
                         count.data_ptr<int32_t>(), (int)page, tokens, starts.data_ptr<int32_t>(),
                         lengths.data_ptr<int32_t>(), admitted.data_ptr<int32_t>(), left.data_ptr<int32_t>(),
                         slots.data_ptr<int32_t>(), positions.data_ptr<int32_t>(), visible.data_ptr<int32_t>(),
                         stream_of(cached)),
        "cqgdn_step_pages");
  return {starts, lengths, admitted, left, slots, positions, visible};
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> step_pages(const Tensor& cached, const Tensor& fresh,
                                                                              Tensor& tables, Tensor& pool,
                                                                              const Tensor& count, int64_t page,
                                                                              int64_t tokens) {
  const Step s = pages_of_step(cached, fresh, tables, pool, count, page, tokens, false);
  return {s.starts, s.lengths, s.admitted, s.left, s.slots, s.positions, s.visible};
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> step_pages_(Tensor& cached, const Tensor& fresh, Tensor& tables,
                                                               Tensor& pool, Tensor& count, int64_t page,
                                                               int64_t tokens) {
  const Step s = pages_of_step(cached, fresh, tables, pool, count, page, tokens, true);
  return {s.starts, s.admitted, s.slots, s.positions, s.visible};
}

void check_data(const Tensor& data, int64_t page, int64_t head_dim) {
  TORCH_CHECK_VALUE(head_dim == 64 || head_dim == 128 || head_dim == 256, "head_dim must be 64, 128 or 256");
  TORCH_CHECK_VALUE(page >= 16 && page <= 65536 && (page & (page - 1)) == 0,
                    "page must be a power of two from 16 to 65536");
  TORCH_CHECK_VALUE(data.dim() == 3 && data.scalar_type() == at::kByte && data.is_contiguous() &&
                        data.size(2) == page * (head_dim + head_dim / 16) && data.size(1) > 0 && data.size(1) <= INT32_MAX,
                    "data must be contiguous uint8 [pages, kv_heads, page * (head_dim + head_dim / 16)]");
}

void kv4_write(Tensor& data, const Tensor& k, const Tensor& v, const Tensor& slots, int64_t page) {
  TORCH_CHECK_VALUE(k.dim() == 3 && v.sizes() == k.sizes(), "k and v must be [T, kv_heads, head_dim]");
  check_data(data, page, k.size(2));
  TORCH_CHECK_VALUE(k.size(1) == data.size(1), "k and v have ", k.size(1), " heads, the cache ", data.size(1));
  const int dtype = dtype_code(k, "k");
  TORCH_CHECK_VALUE(v.scalar_type() == k.scalar_type(), "k and v must share one type");
  int32_vector(slots, "slots");
  TORCH_CHECK_VALUE(slots.numel() == k.size(0), "slots must hold a value a row");
  on_one_gpu({&data, &k, &v, &slots});
  const c10::DeviceGuard guard(k.device());
  const Tensor kc = head_rows(k), vc = head_rows(v), s = slots.contiguous();
  check(cqgdn_kv4_write(kc.data_ptr(), kc.stride(0), kc.stride(1), vc.data_ptr(), vc.stride(0), vc.stride(1), dtype,
                        s.data_ptr<int32_t>(), k.size(0), (int)k.size(1), (int)k.size(2), data.data_ptr(), data.size(0),
                        (int)page, stream_of(k)),
        "cqgdn_kv4_write");
}

std::tuple<Tensor, Tensor> kv4_read(const Tensor& data, const Tensor& slots, int64_t page, int64_t head_dim, bool fp16) {
  check_data(data, page, head_dim);
  int32_vector(slots, "slots");
  on_one_gpu({&data, &slots});
  const c10::DeviceGuard guard(data.device());
  const Tensor s = slots.contiguous();
  const auto opt = data.options().dtype(fp16 ? at::kHalf : at::kBFloat16);
  Tensor k = at::empty({s.numel(), data.size(1), head_dim}, opt), v = at::empty_like(k);
  check(cqgdn_kv4_read(data.data_ptr(), data.size(0), (int)page, (int)data.size(1), (int)head_dim,
                       s.data_ptr<int32_t>(), s.numel(), fp16 ? CQGDN_F16 : CQGDN_BF16, k.data_ptr(), v.data_ptr(),
                       stream_of(data)),
        "cqgdn_kv4_read");
  return {k, v};
}

std::tuple<Tensor, Tensor> kv4_attend(const Tensor& q, const Tensor& data, const Tensor& tables, const Tensor& starts,
                                      const Tensor& visible, int64_t page, int64_t window, double scale,
                                      int64_t max_queries, bool want_lse) {
  TORCH_CHECK_VALUE(q.dim() == 3, "q must be [T, heads, head_dim]");
  const int dtype = dtype_code(q, "q");
  check_data(data, page, q.size(2));
  const int64_t T = q.size(0), heads = q.size(1), kv = data.size(1), N = tables.dim() == 2 ? tables.size(0) : -1;
  TORCH_CHECK_VALUE(heads > 0 && heads % kv == 0, heads, " query heads are no multiple of ", kv, " key heads");
  TORCH_CHECK_VALUE(N >= 0 && tables.scalar_type() == at::kInt, "tables must be int32 [requests, columns]");
  int32_vector(starts, "starts");
  int32_vector(visible, "visible");
  TORCH_CHECK_VALUE(starts.numel() == N + 1 && visible.numel() == T,
                    "starts must hold a value a request and one more, visible a value a row");
  TORCH_CHECK_VALUE(window >= 0 && window <= INT32_MAX, "window must be positive");
  TORCH_CHECK_VALUE(max_queries > 0, "max_queries must be positive");
  TORCH_CHECK_VALUE(tables.size(1) <= INT32_MAX && T <= INT32_MAX && N < INT32_MAX, "sizes are 32-bit");
  on_one_gpu({&q, &data, &tables, &starts, &visible});
  const c10::DeviceGuard guard(q.device());
  const Tensor qc = head_rows(q), st = starts.contiguous(), vis = visible.contiguous();
  const Tensor tab = (tables.stride(1) == 1 || tables.size(1) <= 1) && (N <= 1 || tables.stride(0) >= tables.size(1))
                         ? tables
                         : tables.contiguous();
  Tensor out = at::empty({T, heads, q.size(2)}, q.options());
  Tensor lse = at::empty({want_lse ? T : 0, heads}, q.options().dtype(at::kFloat));
  const int most = (int)std::min(max_queries, std::max<int64_t>(T, 1)), columns = (int)tab.size(1);
  const size_t need = cqgdn_kv4_attend_workspace_size(T, (int)N, (int)heads, (int)kv, (int)q.size(2), most, columns,
                                                      (int)page);
  Tensor ws;
  if (need) ws = at::empty({(int64_t)need}, data.options());
  check(cqgdn_kv4_attend(qc.data_ptr(), qc.stride(0), qc.stride(1), dtype, T, (int)heads, (int)q.size(2),
                         data.data_ptr(), data.size(0), (int)page, (int)kv, tab.data_ptr<int32_t>(),
                         N > 1 ? tab.stride(0) : columns, columns, st.data_ptr<int32_t>(), (int)N,
                         vis.data_ptr<int32_t>(), (int)window, (float)scale, most, out.data_ptr(),
                         want_lse ? lse.data_ptr<float>() : nullptr, need ? ws.data_ptr() : nullptr, need, stream_of(q)),
        "cqgdn_kv4_attend");
  return {out, lse};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(cqgdn, m) {
  m.def("rotary(Tensor q, Tensor k, Tensor positions, Tensor turns, Tensor axis, bool adjacent, bool backward) "
        "-> (Tensor, Tensor)");
  m.def("step_pages(Tensor cached, Tensor new, Tensor(a!) tables, Tensor(b!) free, Tensor free_count, int page, "
        "int tokens) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("step_pages_(Tensor(a!) cached, Tensor new, Tensor(b!) tables, Tensor(c!) free, Tensor(d!) free_count, int page, "
        "int tokens) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("kv4_write(Tensor(a!) data, Tensor k, Tensor v, Tensor slots, int page) -> ()");
  m.def("kv4_read(Tensor data, Tensor slots, int page, int head_dim, bool fp16) -> (Tensor, Tensor)");
  m.def("kv4_attend(Tensor q, Tensor data, Tensor tables, Tensor starts, Tensor visible, int page, int window, "
        "float scale, int max_queries, bool want_lse) -> (Tensor, Tensor)");
}

// The cache and what reads it are for serving: no gradient passes, and their outputs say so (by default they would
// require one and give none).
TORCH_LIBRARY_IMPL(cqgdn, Autograd, m) {
  m.impl("rotary", &rotary_autograd);
  for (const char* name : {"step_pages", "step_pages_", "kv4_write", "kv4_read", "kv4_attend"})
    m.impl(name, torch::CppFunction::makeFallthrough());
}

TORCH_LIBRARY_IMPL(cqgdn, CUDA, m) {
  m.impl("rotary", &rotary);
  m.impl("step_pages", &step_pages);
  m.impl("step_pages_", &step_pages_);
  m.impl("kv4_write", &kv4_write);
  m.impl("kv4_read", &kv4_read);
  m.impl("kv4_attend", &kv4_attend);
}

// CPU tensors reach the same functions only to be rejected by their checks.
TORCH_LIBRARY_IMPL(cqgdn, CPU, m) {
  m.impl("rotary", &rotary);
  m.impl("step_pages", &step_pages);
  m.impl("step_pages_", &step_pages_);
  m.impl("kv4_write", &kv4_write);
  m.impl("kv4_read", &kv4_read);
  m.impl("kv4_attend", &kv4_attend);
}
