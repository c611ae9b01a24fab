// The training operators as torch tensors see them: allocations, launches through the C entry points of b200moe.h, and the nodes of
// the autograd graph.  Native, because small steps are bound by the host: the backward pass runs in a thread of torch's own, and a
// node in Python costs that thread two handovers of the interpreter lock.  Gated activation of 512 x 1024 with its gradient: 87 us
// per step with such a node, 52 with this one, 50 for a multiplication by torch.
//
// Arguments come checked (core/moe/moe_train).
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <memory>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/b200moe.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A refusal of an entry point; the exception that Python raises for one.
struct EntryError : torch::PyTorchError {
  explicit EntryError(const std::string& what)
      : PyTorchError("[INTERNAL_ERROR] [NCC_INKI016] Kernel validation exception: " + what) {}
  PyObject* python_type() override { return PyExc_AssertionError; }
};
void check(int rc, const char* name) {
  if (rc != B200MOE_OK)
    throw EntryError(std::string(name) + " failed (" + std::to_string(rc) + "): " + b200moe_last_error());
}

// The device of a tensor made current, and its current stream.
struct On {
  c10::cuda::CUDAGuard guard;
  b200moe_stream_t stream;
  explicit On(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};

Tensor make(at::IntArrayRef sizes, const Tensor& like, at::ScalarType type) { return at::empty(sizes, like.options().dtype(type)); }
Tensor make(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options()); }
void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int type_code(const Tensor& t) { return t.defined() && t.scalar_type() == at::kBFloat16 ? B200MOE_BF16 : B200MOE_F32; }
int as_int(int64_t v) { return static_cast<int>(v); }

// Elements between two rows of a matrix with contiguous columns (a single row has none).
int64_t pitch_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
// The rows themselves if their columns are contiguous, else a copy.
Tensor unit_rows(const Tensor& t) { return t.stride(1) == 1 || t.size(1) <= 1 ? t : t.contiguous(); }
// The rows themselves if they do not overlap and all start on 16-byte boundaries, else a copy.
Tensor tile_rows(const Tensor& t) {
  const bool apart = t.size(0) <= 1 || (t.stride(0) >= t.size(1) && t.stride(0) * t.element_size() % 16 == 0);
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && t.stride(1) == 1 && apart) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

using Maybe = std::optional<Tensor>;
Tensor or_none(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

bool recorded(std::initializer_list<Tensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// What would take a launch for nothing.  Forward-mode derivatives: a dual tensor need not ask for a gradient, so that the call would
// pass every node by and its result come without a tangent, which reads as a derivative of zero.  A recording of torch's calls: it
// holds the allocation of a result and not the launch that fills it.
bool recording() {
  using c10::impl::TorchDispatchModeTLS;
  return torch::jit::tracer::isTracing() ||
         (TorchDispatchModeTLS::any_modes_set() && TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value());
}
void refuse_transforms(std::initializer_list<Tensor> tensors) {
  if (recording()) throw EntryError("the training operators cannot be traced: a recording of torch's calls lacks their launches");
  for (const Tensor& t : tensors)
    if (t.defined() && t._fw_grad(0).defined())
      throw EntryError("the training operators have no forward-mode derivatives, neither of their results nor of their gradients");
}

// Gradients that are themselves recorded (create_graph) raise when they are differentiated: whatever in them depends on the
// inputs would be lost otherwise.
variable_list once(variable_list gradients) {
  if (!at::GradMode::is_enabled()) return gradients;
  for (Tensor& g : gradients)
    if (g.defined()) g = g.detach().requires_grad_();
  const int n = as_int(static_cast<int64_t>(gradients.size()));
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", n);
  return (*error)(std::move(gradients));
}

// ------------------------------------------------------------------ order and rows
using Sorted = std::tuple<Tensor, Tensor, Tensor>;  // rows (undefined without hidden), expert_offsets, row_of_pair

Sorted sort(const Tensor& hidden, const Tensor& index, int64_t E) {
  const On on(index);
  const int64_t T = index.size(0), K = index.size(1), H = hidden.defined() ? hidden.size(1) : 0;
  Tensor row_of_pair = make({T, K}, index, at::kInt), offsets, rows;
  if (hidden.defined()) rows = make({T * K, H}, hidden);
  if (T * K == 0) return {rows, at::zeros({E + 1}, index.options().dtype(at::kInt)), row_of_pair};
  offsets = make({E + 1}, index, at::kInt);
  const Tensor ids = index.contiguous();
  const size_t size = b200moe_sort_workspace_bytes(T * K, as_int(E));
  const Tensor ws = size ? make({static_cast<int64_t>(size)}, index, at::kByte) : Tensor();
  const int bytes = as_int(ids.element_size());
  if (H > 0) {
    const Tensor from = unit_rows(hidden);
    check(b200moe_sort_tokens(from.data_ptr(), type_code(from), pitch_of(from), ids.data_ptr(), bytes, as_int(T), as_int(K),
                              as_int(H), as_int(E), offsets.data_ptr<int>(), row_of_pair.data_ptr<int>(), rows.data_ptr(),
                              address(ws), size, on.stream),
          "b200moe_sort_tokens");
  } else {
    check(b200moe_sort_pairs(ids.data_ptr(), bytes, as_int(T), as_int(K), as_int(E), offsets.data_ptr<int>(),
                             row_of_pair.data_ptr<int>(), address(ws), size, on.stream),
          "b200moe_sort_pairs");
  }
  return {rows, offsets, row_of_pair};
}

Tensor unsort(const Tensor& rows, const Tensor& affinities, const Tensor& row_of_pair) {
  const On on(rows);
  const int64_t T = row_of_pair.size(0), K = row_of_pair.size(1), H = rows.size(1);
  if (T * K * H == 0) return at::zeros({T, H}, rows.options());
  Tensor out = make({T, H}, rows);
  const Tensor from = unit_rows(rows), weights = affinities.defined() ? affinities.contiguous() : Tensor();
  check(b200moe_unsort_rows(from.data_ptr(), type_code(from), pitch_of(from), as_int(T), as_int(K), as_int(H),
                            row_of_pair.data_ptr<int>(), address(weights), type_code(weights), out.data_ptr(), on.stream),
        "b200moe_unsort_rows");
  return out;
}

struct SortTokens : torch::autograd::Function<SortTokens> {
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& index, int64_t E) {
    auto [rows, offsets, row_of_pair] = sort(hidden, index, E);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({offsets, row_of_pair});
    ctx->save_for_backward({row_of_pair});
    return {rows, offsets, row_of_pair};
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    if (!d[0].defined()) return {Tensor(), Tensor(), Tensor()};
    refuse_transforms({d[0]});
    return once({unsort(d[0], Tensor(), ctx->get_saved_variables()[0]), Tensor(), Tensor()});
  }
};

struct UnsortRows : torch::autograd::Function<UnsortRows> {
  // Inputs of a node are defined or absent: absent affinities are no input, and none has its gradient's number then.
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Maybe& weights, const Tensor& row_of_pair,
                        const Tensor& offsets) {
    const Tensor affinities = or_none(weights);
    // the rows are needed for the affinities' gradient only
    const bool keep = affinities.defined() && affinities.requires_grad();
    ctx->save_for_backward({keep ? rows : Tensor(), affinities, row_of_pair, offsets});
    return unsort(rows, affinities, row_of_pair);
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    refuse_transforms({d[0]});
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &affinities = saved[1], &row_of_pair = saved[2], &offsets = saved[3];
    const On on(d[0]);
    const int64_t T = row_of_pair.size(0), K = row_of_pair.size(1), H = d[0].size(1);
    const bool want_affinities = affinities.defined() && ctx->needs_input_grad(1);
    Tensor d_rows = ctx->needs_input_grad(0) ? make({T * K, H}, d[0]) : Tensor();
    Tensor d_affinities = want_affinities ? make({T, K}, affinities) : Tensor();
    if (T * K * H == 0) {
      if (want_affinities) d_affinities.zero_();
    } else if (d_rows.defined() || want_affinities) {
      const Tensor d_out = unit_rows(d[0]), rows = want_affinities ? unit_rows(saved[0]) : Tensor();
      const Tensor weights = affinities.defined() ? affinities.contiguous() : Tensor();
      check(b200moe_unsort_rows_backward(d_out.data_ptr(), pitch_of(d_out), address(rows), rows.defined() ? pitch_of(rows) : H,
                                         type_code(d_out), as_int(T), as_int(K), as_int(H), as_int(offsets.size(0) - 1),
                                         row_of_pair.data_ptr<int>(), offsets.data_ptr<int>(), address(weights),
                                         type_code(weights), address(d_rows), address(d_affinities), on.stream),
            "b200moe_unsort_rows_backward");
    }
    return once({d_rows, d_affinities, Tensor(), Tensor()});
  }
};

// ------------------------------------------------------------------ products
// Matrices the kernels can read: contiguous columns, rows and matrices apart and on 16-byte boundaries.
bool readable(const Tensor& w) {
  return w.stride(2) == 1 && reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0 &&
         (w.size(1) == 1 || (w.stride(1) >= w.size(2) && w.stride(1) % 8 == 0)) &&
         (w.size(0) == 1 || (w.stride(0) >= w.size(2) && w.stride(0) % 8 == 0));
}
// weight [E, K, N] as such matrices.  Transposed ones lie in memory as [E, N, K], like the weights of linear layers; anything
// else is copied.
struct Stored {
  Tensor matrices;
  bool turned;
};
Stored stored(const Tensor& weight) {
  if (readable(weight)) return {weight, false};
  Tensor turned = weight.transpose(1, 2);
  if (readable(turned)) return {turned, true};
  return {weight.clone(at::MemoryFormat::Contiguous), false};
}

// Waits for a product and raises if it has given up.
void read_status(const Tensor& status) {
  const int code = status[0].item<int>();
  if (code != 0) throw EntryError("device-side wait expired in a product of the experts (status " + std::to_string(code) + ")");
}

// rows[r] @ weight[e], with `transpose` rows[r] @ weight[e].T
Tensor product(const Tensor& rows, const Tensor& weight, const Tensor& offsets, bool transpose, bool check_status) {
  const On on(rows);
  const Stored w = stored(weight);
  const int64_t R = rows.size(0), E = w.matrices.size(0), D0 = w.matrices.size(1), D1 = w.matrices.size(2);
  const int contract_last = transpose != w.turned;
  Tensor out = make({R, contract_last ? D0 : D1}, rows);
  if (R == 0) return out;
  const Tensor from = tile_rows(rows);
  const size_t size = b200moe_expert_product_workspace_bytes(contract_last, as_int(R), as_int(E), as_int(D0), as_int(D1));
  const Tensor ws = size ? make({static_cast<int64_t>(size)}, rows, at::kByte) : Tensor();
  const Tensor status = make({2}, rows, at::kInt);
  const int64_t w_pitch = w.matrices.stride(1);
  check(b200moe_expert_product(from.data_ptr(), pitch_of(from), w.matrices.data_ptr(), w_pitch,
                               E > 1 ? w.matrices.stride(0) : D0 * w_pitch, contract_last, offsets.data_ptr<int>(), as_int(R),
                               as_int(E), as_int(D0), as_int(D1), out.data_ptr(), address(ws), size, status.data_ptr<int>(),
                               on.stream),
        "b200moe_expert_product");
  if (check_status) read_status(status);
  return out;
}

// Gradient of product() in `weight`, laid out in memory as the weight is.
Tensor weight_grad(const Tensor& rows, const Tensor& d_out, const Tensor& weight, const Tensor& offsets, bool check_status) {
  const On on(weight);
  const bool turned = weight.stride(2) != 1 && weight.stride(1) == 1;
  const int64_t R = rows.size(0), E = weight.size(0), M = weight.size(turned ? 2 : 1), N = weight.size(turned ? 1 : 2);
  Tensor out;
  if (R == 0) {
    out = at::zeros({E, M, N}, weight.options());
  } else {
    out = make({E, M, N}, weight);
    const Tensor a = tile_rows(turned ? d_out : rows), b = tile_rows(turned ? rows : d_out);
    const size_t size = b200moe_expert_weight_grad_workspace_bytes(as_int(R), as_int(E), as_int(M), as_int(N));
    const Tensor ws = size ? make({static_cast<int64_t>(size)}, weight, at::kByte) : Tensor();
    const Tensor status = make({2}, weight, at::kInt);
    check(b200moe_expert_weight_grad(a.data_ptr(), pitch_of(a), b.data_ptr(), pitch_of(b), offsets.data_ptr<int>(), as_int(R),
                                     as_int(E), as_int(M), as_int(N), out.data_ptr(), address(ws), size, status.data_ptr<int>(),
                                     on.stream),
          "b200moe_expert_weight_grad");
    if (check_status) read_status(status);
  }
  return turned ? out.transpose(1, 2) : out;
}

struct ExpertLinear : torch::autograd::Function<ExpertLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weight, const Tensor& offsets, bool check_status) {
    ctx->save_for_backward({weight.requires_grad() ? rows : Tensor(), weight, offsets});
    ctx->saved_data["check"] = check_status;
    return product(rows, weight, offsets, false, check_status);
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    refuse_transforms({d[0]});
    const variable_list saved = ctx->get_saved_variables();
    const Tensor d_out = tile_rows(d[0]);
    const bool check = ctx->saved_data["check"].toBool();
    Tensor d_rows, d_weight;
    if (ctx->needs_input_grad(0)) d_rows = product(d_out, saved[1], saved[2], true, check);
    if (ctx->needs_input_grad(1)) d_weight = weight_grad(saved[0], d_out, saved[1], saved[2], check);
    return once({d_rows, d_weight, Tensor(), Tensor()});
  }
};

// ------------------------------------------------------------------ gated activation
// (m, kept): the codes of all rows, then their scales; undefined unless `keep`.
std::tuple<Tensor, Tensor> glu_forward(const Tensor& gate_up, int64_t act, bool keep) {
  const On on(gate_up);
  const int64_t R = gate_up.size(0), I = gate_up.size(1) / 2;
  Tensor m = make({R, I}, gate_up);
  Tensor kept = keep ? make({R * (2 * I + 2 * ((I + 31) / 32))}, gate_up, at::kByte) : Tensor();
  if (R > 0) {
    const Tensor from = tile_rows(gate_up);
    uint8_t* codes = static_cast<uint8_t*>(address(kept));
    check(b200moe_glu(from.data_ptr(), pitch_of(from), R, as_int(I), as_int(act), m.data_ptr(), codes,
                      keep ? codes + R * 2 * I : nullptr, on.stream),
          "b200moe_glu");
  }
  return {m, kept};
}

// (d_gate_up, m) at the kept gate and up; the first undefined without d_m [R, I], the second unless wanted.
std::tuple<Tensor, Tensor> glu_backward(const Tensor& d_m, const Tensor& kept, int64_t R, int64_t I, int64_t act, bool want_m) {
  const On on(kept);
  const auto bf16 = kept.options().dtype(at::kBFloat16);
  Tensor d_gate_up = d_m.defined() ? at::empty({R, 2 * I}, bf16) : Tensor(), m = want_m ? at::empty({R, I}, bf16) : Tensor();
  if (R > 0) {
    const Tensor from = d_m.defined() ? tile_rows(d_m) : Tensor();
    const uint8_t* codes = kept.data_ptr<uint8_t>();
    check(b200moe_glu_backward(address(from), from.defined() ? pitch_of(from) : I, codes, codes + R * 2 * I, R, as_int(I),
                               as_int(act), address(d_gate_up), address(m), on.stream),
          "b200moe_glu_backward");
  }
  return {d_gate_up, m};
}

struct Glu : torch::autograd::Function<Glu> {
  static Tensor forward(AutogradContext* ctx, const Tensor& gate_up, int64_t act) {
    auto [m, kept] = glu_forward(gate_up, act, true);
    ctx->save_for_backward({kept});
    ctx->saved_data["act"] = act;
    return m;
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    refuse_transforms({d[0]});
    const Tensor kept = ctx->get_saved_variables()[0];
    return once({std::get<0>(glu_backward(d[0], kept, d[0].size(0), d[0].size(1), ctx->saved_data["act"].toInt(), false)), Tensor()});
  }
};

// ------------------------------------------------------------------ product, activation, product
struct ExpertMLP : torch::autograd::Function<ExpertMLP> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& gate_up_weight, const Tensor& down_weight,
                        const Tensor& offsets, int64_t act, bool check_status) {
    auto [m, kept] = glu_forward(product(rows, gate_up_weight, offsets, false, check_status), act, true);
    ctx->save_for_backward({gate_up_weight.requires_grad() ? rows : Tensor(), gate_up_weight, down_weight, offsets, kept});
    ctx->saved_data["act"] = act;
    ctx->saved_data["check"] = check_status;
    return product(m, down_weight, offsets, false, check_status);
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    refuse_transforms({d[0]});
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &rows = saved[0], &gate_up_weight = saved[1], &down_weight = saved[2], &offsets = saved[3];
    const bool want_rows = ctx->needs_input_grad(0), want_gate_up = ctx->needs_input_grad(1), want_down = ctx->needs_input_grad(2);
    const Tensor d_out = tile_rows(d[0]);
    const bool check = ctx->saved_data["check"].toBool();
    Tensor d_m, d_rows, d_gate_up_weight, d_down;
    if (want_rows || want_gate_up) d_m = product(d_out, down_weight, offsets, true, check);
    auto [d_gate_up, m] = glu_backward(d_m, saved[4], d_out.size(0), down_weight.size(1), ctx->saved_data["act"].toInt(), want_down);
    if (want_down) d_down = weight_grad(m, d_out, down_weight, offsets, check);
    if (want_rows) d_rows = product(d_gate_up, gate_up_weight, offsets, true, check);
    if (want_gate_up) d_gate_up_weight = weight_grad(rows, d_gate_up, gate_up_weight, offsets, check);
    return once({d_rows, d_gate_up_weight, d_down, Tensor(), Tensor(), Tensor()});
  }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, module) {
  // every exception the way torch's own calls raise it (out of memory, refusals)
  const auto def = [&](const char* name, auto&& f) { module.def(name, torch::wrap_pybind_function(f)); };
  def("sort", [](const Maybe& hidden, const Tensor& index, int64_t E) -> std::tuple<Maybe, Tensor, Tensor> {
    refuse_transforms({or_none(hidden)});
    if (hidden.has_value() && recorded({*hidden})) {
      const variable_list out = SortTokens::apply(*hidden, index, E);
      return {out[0], out[1], out[2]};
    }
    auto [rows, offsets, row_of_pair] = sort(or_none(hidden), index, E);
    return {maybe(rows), offsets, row_of_pair};
  });
  def("unsort", [](const Tensor& rows, const Maybe& affinities, const Tensor& row_of_pair, const Tensor& offsets) {
    refuse_transforms({rows, or_none(affinities)});
    if (recorded({rows, or_none(affinities)})) return UnsortRows::apply(rows, affinities, row_of_pair, offsets);
    return unsort(rows, or_none(affinities), row_of_pair);
  });
  def("linear", [](const Tensor& rows, const Tensor& weight, const Tensor& offsets, bool check_status) {
    refuse_transforms({rows, weight});
    return recorded({rows, weight}) ? ExpertLinear::apply(rows, weight, offsets, check_status)
                                    : product(rows, weight, offsets, false, check_status);
  });
  def("glu", [](const Tensor& gate_up, int64_t act) {
    refuse_transforms({gate_up});
    return recorded({gate_up}) ? Glu::apply(gate_up, act) : std::get<0>(glu_forward(gate_up, act, false));
  });
  def("mlp", [](const Tensor& rows, const Tensor& gate_up_weight, const Tensor& down_weight, const Tensor& offsets,
                int64_t act, bool check_status) {
    refuse_transforms({rows, gate_up_weight, down_weight});
    if (recorded({rows, gate_up_weight, down_weight}))
      return ExpertMLP::apply(rows, gate_up_weight, down_weight, offsets, act, check_status);
    const Tensor m = std::get<0>(glu_forward(product(rows, gate_up_weight, offsets, false, check_status), act, false));
    return product(m, down_weight, offsets, false, check_status);
  });
  def("product", &product);
  def("weight_grad", [](const Tensor& rows, const Tensor& d_out, const Tensor& weight, const Tensor& offsets) {
    return weight_grad(rows, d_out, weight, offsets, false);
  });
  def("glu_forward", [](const Tensor& gate_up, int64_t act, bool keep) -> std::tuple<Tensor, Maybe> {
    auto [m, kept] = glu_forward(gate_up, act, keep);
    return {m, maybe(kept)};
  });
  def("glu_backward", [](const Maybe& d_m, const Tensor& kept, int64_t R, int64_t I, int64_t act,
                                bool want_m) -> std::tuple<Maybe, Maybe> {
    auto [d_gate_up, m] = glu_backward(or_none(d_m), kept, R, I, act, want_m);
    return {maybe(d_gate_up), maybe(m)};
  });
}
