// ml4tspbench_amd/csrc/learning_ext.cpp -- autograd nodes of the learning operators (host code only)
//
// The forward and gradient entry points of libtsp2opt_hip.so as torch::autograd nodes.  Written in C++ because the
// losses are a few microseconds of GPU work: a node in Python has autograd's device thread wait for the interpreter
// lock on every backward pass (clipped_policy_loss on 16 x 49 steps, forward and gradient: 127 us through Python
// nodes, 58 us through these).  The entry points are handed over by ml4tspbench_amd/learning.py, so
// that there is one copy of the library in the process, the one that _lib.py loaded.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <limits>
#include <memory>
#include <optional>
#include <string>
#include <vector>

#include "tsp2opt.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

struct Api {
    decltype(&tsp2opt_last_error) last_error;
    decltype(&tsp2opt_tour_logprobs_state_bytes) logp_bytes;
    decltype(&tsp2opt_tour_logprobs) logp;
    decltype(&tsp2opt_tour_logprobs_grad) logp_grad;
    decltype(&tsp2opt_policy_loss_state_bytes) policy_bytes;
    decltype(&tsp2opt_policy_loss) policy;
    decltype(&tsp2opt_policy_loss_grad) policy_grad;
    decltype(&tsp2opt_preference_loss_state_bytes) pref_bytes;
    decltype(&tsp2opt_preference_loss) pref;
    decltype(&tsp2opt_preference_loss_grad) pref_grad;
} api;

PyObject* failure_class = nullptr;          // Tsp2optError

// What _lib.check() raises.  Autograd's device thread calls this too: it holds no interpreter lock, and the exception
// reaches the caller of backward() as it is.
int64_t checked(int64_t rc, const char* what)
{
    if (rc >= 0) return rc;
    const char* msg = api.last_error();
    const std::string text = std::string(what) + " failed (" + std::to_string(rc) + "): " + (msg ? msg : "");
    py::gil_scoped_acquire gil;
    PyErr_SetObject(failure_class, py::handle(failure_class)(text, rc).ptr());
    throw py::error_already_set();
}

int code_of(const Tensor& x)
{
    return x.scalar_type() == at::kFloat ? TSP2OPT_DTYPE_F32 : x.scalar_type() == at::kBFloat16 ? TSP2OPT_DTYPE_BF16
                                                                                                 : TSP2OPT_DTYPE_F16;
}

void* stream_of(const Tensor& x)
{
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.get_device()).stream();
}

template <typename T = void>
T* ptr(const Tensor& x)
{
    return x.defined() ? static_cast<T*>(x.data_ptr()) : nullptr;
}

using Maybe = std::optional<Tensor>;

Tensor one(const Maybe& x) { return x ? *x : Tensor(); }

// Device memory between a call and its gradient call: one allocation a call, so that calls on other streams and
// captured graphs never share it.
Tensor state_like(const Tensor& x, int64_t bytes) { return at::empty({bytes}, x.options().dtype(at::kByte)); }

// The kernels have no second derivative: with create_graph the gradient's own node is one that raises when it is reached,
// instead of the gradient being a constant.  It has the edges of the operator's inputs and of the incoming gradients, so
// that a derivative of an expression which mixes the gradient with others meets it on its way to any of them.
Tensor once(Tensor grad, const variable_list& incoming)
{
    if (!c10::GradMode::is_enabled()) return grad;
    const auto self = torch::autograd::get_current_node();
    TORCH_CHECK(self, "the learning operators' gradient is taken with create_graph outside of autograd's engine");
    auto edges = self->next_edges();
    for (auto& edge : torch::autograd::collect_next_edges(incoming)) edges.push_back(std::move(edge));
    torch::autograd::set_history(grad, std::make_shared<torch::autograd::Error>(
                                           "the learning operators have no second derivative", std::move(edges)));
    return grad;
}

struct LogProbs : public Function<LogProbs> {
    static Tensor forward(AutogradContext* ctx, Tensor logits, const Tensor& tours, int64_t per, int64_t rows,
                          int64_t state_bytes)
    {
        const int64_t T = tours.size(0), n = tours.size(1) - 1;
        if (n > 1 && logits.stride(2) != 1) logits = logits.contiguous();
        Tensor state = state_like(logits, state_bytes);
        Tensor out = at::empty({T, n - 1}, logits.options().dtype(at::kFloat));
        checked(api.logp(ptr(logits), ptr<int64_t>(tours), ptr<float>(out), ptr(state), state.numel(), T, (int)n, (int)per,
                         (int)rows, logits.stride(0), logits.stride(1), code_of(logits), logits.get_device(),
                         stream_of(logits)),
                "tsp2opt_tour_logprobs");
        ctx->save_for_backward({logits, tours, state});
        ctx->saved_data["how"] = std::vector<int64_t>{per, rows};
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &tours = saved[1], &state = saved[2];
        const auto how = ctx->saved_data["how"].toIntVector();
        const int64_t T = tours.size(0), n = tours.size(1) - 1;
        Tensor grad = at::empty(logits.sizes(), logits.options());
        if (n == 1) return {once(grad.zero_(), grads), Tensor(), Tensor(), Tensor(), Tensor()};
        const Tensor g = grads[0].to(at::kFloat).contiguous();
        checked(api.logp_grad(ptr(logits), ptr<int64_t>(tours), ptr(state), state.numel(), ptr<float>(g), ptr(grad), T,
                              (int)n, (int)how[0], (int)how[1], logits.stride(0), logits.stride(1), code_of(logits),
                              logits.get_device(), stream_of(logits)),
                "tsp2opt_tour_logprobs_grad");
        return {once(grad, grads), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

struct PolicyLoss : public Function<PolicyLoss> {
    static variable_list forward(AutogradContext* ctx, Tensor lp, const Tensor& old, const Maybe& maybe_ref,
                                 const Tensor& adv, const Maybe& maybe_mask, int64_t of_tour, int64_t of_tours, double low,
                                 double high, double kl_coef)
    {
        const Tensor ref = one(maybe_ref), mask = one(maybe_mask);
        lp = lp.contiguous();
        const int64_t T = lp.size(0), S = lp.size(1);
        Tensor state = state_like(lp, checked(api.policy_bytes(T), "tsp2opt_policy_loss_state_bytes"));
        const auto f32 = lp.options().dtype(at::kFloat);
        Tensor loss = at::empty({}, f32), stats = at::empty({2}, f32);
        checked(api.policy(ptr(lp), ptr(old), ptr(ref), ptr<float>(adv), ptr<uint8_t>(mask), ptr<float>(loss),
                           ptr<float>(stats), ptr(state), state.numel(), T, S, adv.dim() == 2, (int)of_tour,
                           (int)of_tours, low, high, kl_coef, code_of(lp), lp.get_device(), stream_of(lp)),
                "tsp2opt_policy_loss");
        ctx->save_for_backward({lp, old, ref, adv, mask, state});
        ctx->saved_data["mode"] = std::vector<int64_t>{of_tour, of_tours};
        ctx->saved_data["how"] = std::vector<double>{low, high, kl_coef};
        ctx->mark_non_differentiable({stats});
        ctx->set_materialize_grads(false);
        return {loss, stats};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const Tensor& lp = saved[0];
        variable_list none(10);
        if (!grads[0].defined()) return none;
        const auto mode = ctx->saved_data["mode"].toIntVector();
        const auto how = ctx->saved_data["how"].toDoubleVector();
        Tensor grad = at::empty(lp.sizes(), lp.options());
        const Tensor g = grads[0].to(at::kFloat);
        checked(api.policy_grad(ptr(lp), ptr(saved[1]), ptr(saved[2]), ptr<float>(saved[3]), ptr<uint8_t>(saved[4]),
                                ptr(saved[5]), saved[5].numel(), ptr<float>(g), ptr(grad), lp.size(0), lp.size(1),
                                saved[3].dim() == 2, (int)mode[0], (int)mode[1], how[0], how[1], how[2], code_of(lp),
                                lp.get_device(), stream_of(lp)),
                "tsp2opt_policy_loss_grad");
        none[0] = once(grad, grads);
        return none;
    }
};

struct PreferenceLoss : public Function<PreferenceLoss> {
    static variable_list forward(AutogradContext* ctx, Tensor lp, const Maybe& maybe_ref, const Tensor& lengths,
                                 const Maybe& maybe_mask, int64_t per, int64_t best, int64_t per_step, double beta,
                                 double smoothing)
    {
        const Tensor ref = one(maybe_ref), mask = one(maybe_mask);
        lp = lp.contiguous();
        const int64_t T = lp.size(0), S = lp.size(1);
        Tensor state = state_like(lp, checked(api.pref_bytes(T), "tsp2opt_preference_loss_state_bytes"));
        Tensor loss = at::empty({}, lp.options().dtype(at::kFloat)), pairs = at::empty({}, lp.options().dtype(at::kLong));
        checked(api.pref(ptr(lp), ptr(ref), ptr<double>(lengths), ptr<uint8_t>(mask), ptr<float>(loss),
                         ptr<int64_t>(pairs), ptr(state), state.numel(), T, S, (int)per, (int)best, (int)per_step, beta,
                         smoothing, code_of(lp), lp.get_device(), stream_of(lp)),
                "tsp2opt_preference_loss");
        ctx->save_for_backward({mask, state});
        ctx->saved_data["like"] = std::vector<int64_t>{T, S, (int64_t)lp.scalar_type()};
        ctx->mark_non_differentiable({pairs});
        ctx->set_materialize_grads(false);
        return {loss, pairs};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        variable_list none(9);
        if (!grads[0].defined()) return none;
        const auto like = ctx->saved_data["like"].toIntVector();
        const Tensor& state = saved[1];
        Tensor grad = at::empty({like[0], like[1]}, state.options().dtype((at::ScalarType)like[2]));
        const Tensor g = grads[0].to(at::kFloat);
        checked(api.pref_grad(ptr<uint8_t>(saved[0]), ptr(state), state.numel(), ptr<float>(g), ptr(grad), like[0], like[1],
                              code_of(grad), state.get_device(), stream_of(state)),
                "tsp2opt_preference_loss_grad");
        none[0] = once(grad, grads);
        return none;
    }
};

// The library takes 32-bit sizes.  What divides an empty batch may be larger without meaning more.
constexpr int64_t most = std::numeric_limits<int32_t>::max();

// constants of a loss: never differentiated, and in the layout that the kernels read
Tensor constant(const Tensor& x) { return x.detach().contiguous(); }

Maybe constant(const Maybe& x) { return x ? Maybe(x->detach().contiguous()) : x; }

}  // namespace

PYBIND11_MODULE(_learning_ext, m)
{
    m.def("bind", [](const std::vector<uintptr_t>& at, py::object error) {
        failure_class = error.release().ptr();
        if (at.size() != 10) throw std::runtime_error("bind: ten entry points");
        size_t k = 0;
        auto next = [&](auto& f) { f = reinterpret_cast<std::decay_t<decltype(f)>>(at[k++]); };
        next(api.last_error);
        next(api.logp_bytes); next(api.logp); next(api.logp_grad);
        next(api.policy_bytes); next(api.policy); next(api.policy_grad);
        next(api.pref_bytes); next(api.pref); next(api.pref_grad);
    });
    m.def("tour_log_probs", [](const Tensor& logits, const Tensor& tours, int64_t per, int64_t rows) {
        // what does not fit is refused here, before a copy of such arrays is made
        const int64_t n = std::min(tours.size(1) - 1, most);
        per = std::min(per, most);
        const int64_t bytes = checked(api.logp_bytes(tours.size(0), (int)n, (int)per, (int)rows),
                                      "tsp2opt_tour_logprobs_state_bytes");
        return LogProbs::apply(logits, tours.to(at::kLong).contiguous(), per, rows, bytes);
    });
    m.def("policy_loss", [](const Tensor& lp, const Tensor& old, const Maybe& ref, const Tensor& adv,
                            const Maybe& mask, bool of_tour, bool of_tours, double low, double high,
                            double kl_coef) {
        auto out = PolicyLoss::apply(lp, constant(old), constant(ref), constant(adv.detach().to(at::kFloat)),
                                     constant(mask), (int64_t)of_tour, (int64_t)of_tours, low, high, kl_coef);
        return std::make_tuple(out[0], out[1].select(0, 0), out[1].select(0, 1));
    });
    m.def("preference_loss", [](const Tensor& lp, const Maybe& ref, const Tensor& lengths,
                                const Maybe& mask, int64_t per, bool best, bool per_step, double beta,
                                double smoothing) {
        auto out = PreferenceLoss::apply(lp, constant(ref), constant(lengths.detach().to(at::kDouble)),
                                         constant(mask), std::min(per, most), (int64_t)best, (int64_t)per_step, beta, smoothing);
        return std::make_tuple(out[0], out[1]);
    });
}
