// Native host path of the layers: the operators of include/cgnn_b200.h called on torch tensors, with
// their autograd nodes, in C++.
//
// What bounds it is host time: a small propagation's six kernels take 26 us on the device.  Issued from Python it
// takes 135 us (argument checks, ctypes conversions, torch.empty calls and two autograd functions, the backward one
// behind a GIL hand-over), from here 62: the allocations and the launches.  Nothing below computes anything
// the C ABI does not.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <mutex>
#include <tuple>
#include <vector>

#include "../../include/cgnn_b200.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

void check(int rc) {
    if (rc != CGNN_OK) TORCH_CHECK(false, "cgnn_b200: ", cgnn_last_error());
}

int dtype_code(const Tensor &t) {
    if (t.scalar_type() == at::kFloat) return CGNN_F32;
    TORCH_CHECK(t.scalar_type() == at::kDouble, "only float32 and float64 are supported");
    return CGNN_F64;
}

cgnn_stream_t current_stream(const Tensor &t) {
    return reinterpret_cast<cgnn_stream_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

void *data(const Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

// These operators carry no forward-mode derivative: a dual number is refused, its tangent never dropped.
void refuse_dual(const char *what, at::TensorList inputs) {
    for (const Tensor &t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(t), what,
                                    " does not support forward-mode automatic differentiation");
}

// Is the current stream of the current device being captured?
bool capturing() { return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; }

// Runs `fill`, which makes a buffer that launches on any stream will read from now on, and returns when the buffer is
// complete.  While the current stream is captured the buffer is made on another one: the captured graph may be
// replayed late, after other users of the buffer, or never.
template <typename Fill>
auto complete(int device, Fill &&fill) {
    c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(device);
    c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
    if (capturing()) stream = c10::cuda::getStreamFromPool(false, device);
    const c10::cuda::CUDAStreamGuard guard(stream);
    auto made = fill();
    C10_CUDA_CHECK(cudaStreamSynchronize(stream));
    return made;
}

// Owner of a native plan and of its scratch: one zero-initialised buffer per (width, dtype, stream), since
// a launch leaves the ticket words zero, launches on one stream are ordered, and those that hand each other
// sums in the scratch are kept together by the plan.
class Plan {
  public:
    Plan(intptr_t handle, int device) : plan_(reinterpret_cast<cgnn_plan *>(handle)), device_(device) {
        int64_t info[8];
        check(cgnn_plan_info(plan_, info));
        rows = info[0];
        nnz = info[1];
        check(cgnn_plan_source_rows(plan_, source_rows));
    }
    Plan(const Plan &) = delete;
    ~Plan() { cgnn_plan_destroy(plan_); }

    const cgnn_plan *get() const { return plan_; }
    intptr_t address() const { return reinterpret_cast<intptr_t>(plan_); }
    int device() const { return device_; }

    std::pair<void *, size_t> scratch(int64_t width, int code, cgnn_stream_t stream) {
        std::lock_guard<std::mutex> held(lock_);
        for (const auto &s : scratch_)
            if (s.width == width && s.code == code && s.stream == stream) return {s.buffer.data_ptr(), s.buffer.numel()};
        const int64_t bytes = std::max<int64_t>((int64_t)cgnn_plan_scratch_bytes(plan_, width, code), 16);
        const c10::cuda::CUDAGuard guard(device_);
        auto zeros = [&] { return at::zeros({bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device_)); };
        const Tensor buffer = capturing() ? complete(device_, zeros) : zeros();
        TORCH_CHECK(buffer.data_ptr() != nullptr, "the operators of compressgnn_b200 need tensors with memory, not fake ones");
        buffer.record_stream(c10::cuda::getCurrentCUDAStream(device_));
        scratch_.push_back({width, code, stream, buffer});
        return {scratch_.back().buffer.data_ptr(), scratch_.back().buffer.numel()};
    }
    std::pair<intptr_t, size_t> scratch_py(int64_t width, int code, intptr_t stream) {
        auto s = scratch(width, code, reinterpret_cast<cgnn_stream_t>(stream));
        return {reinterpret_cast<intptr_t>(s.first), s.second};
    }

    int64_t rows = 0, nnz = 0;
    int64_t source_rows[2] = {0, 0};

  private:
    struct Scratch {
        int64_t width;
        int code;
        cgnn_stream_t stream;
        Tensor buffer;
    };
    cgnn_plan *plan_;
    int device_;
    std::mutex lock_;
    std::vector<Scratch> scratch_;
};
using PlanPtr = std::shared_ptr<Plan>;

// ---------------------------------------------------------------------------------------------
// compressed propagation
// ---------------------------------------------------------------------------------------------
// The launch tables of one graph: per direction the plans in launch order (rules, levels, vertices) with
// the value arrays behind them, brought into plan order once per element type.
class Propagation : public std::enable_shared_from_this<Propagation> {
  public:
    using Launch = std::pair<PlanPtr, std::vector<Tensor>>;
    Propagation(int64_t vertices, int64_t rules, std::vector<Launch> forward, std::vector<Launch> backward)
        : vertices_(vertices), rules_(rules) {
        launches_[0] = std::move(forward);
        launches_[1] = std::move(backward);
        for (auto &dir : launches_) {
            TORCH_CHECK(dir.size() >= 2, "a pass has a rule launch and a vertex launch");
            for (auto &launch : dir)
                TORCH_CHECK(launch.first && launch.first->device() == device(), "the plans must lie on one device");
        }
    }
    int device() const { return launches_[0].front().first->device(); }

    // Launches first .. last of one direction (last < 0: to the end) on the current stream.
    Tensor run(const Tensor &x_in, bool backward, const Tensor &out_in, const Tensor &rule_in, int first, int last) {
        TORCH_CHECK(x_in.is_cuda(), "compressgnn_b200 runs on CUDA tensors only (no CPU propagation path)");
        TORCH_CHECK(x_in.get_device() == device(), "the feature matrix is on cuda:", (int)x_in.get_device(),
                    " and the graph on cuda:", device());
        const Tensor x = x_in.contiguous();
        TORCH_CHECK(x.dim() == 2, "the feature matrix must have two dimensions");
        const c10::cuda::OptionalCUDAGuard guard(x.device());
        const int64_t width = x.size(1);
        Tensor out = out_in;
        if (!out.defined()) out = at::empty({vertices_, width}, x.options());
        else
            TORCH_CHECK(out.device() == x.device() && out.dim() == 2 && out.size(0) == vertices_ && out.size(1) == width &&
                            out.scalar_type() == x.scalar_type() && out.is_contiguous(),
                        "out does not match the graph and the feature matrix");
        if (out.numel() == 0) return out;
        // The rule matrix starts a whole number of rows away from x, so that the fused vertex pass reads both
        // through one base pointer and a row index (see cgnn_spmm_pair).
        Tensor rule = rule_in;
        char *rule_ptr = nullptr;
        if (rule.defined()) {
            TORCH_CHECK(rule.device() == x.device() && rule.dim() == 2 && rule.size(0) == rules_ && rule.size(1) == width &&
                            rule.scalar_type() == x.scalar_type() && rule.is_contiguous(),
                        "rule buffer does not match the graph and the feature matrix");
            rule_ptr = static_cast<char *>(data(rule));
        } else if (rules_ > 0) {
            rule = at::empty({(rules_ + 1) * width}, x.options());
            const int64_t row_bytes = width * x.element_size();
            rule_ptr = static_cast<char *>(rule.data_ptr());
            int64_t shift = (reinterpret_cast<intptr_t>(x.data_ptr()) - reinterpret_cast<intptr_t>(rule_ptr)) % row_bytes;
            rule_ptr += shift < 0 ? shift + row_bytes : shift;
        }
        const Table &t = table(backward, width, x);
        TORCH_CHECK(x.size(0) >= t.x_rows && rules_ >= t.rule_rows,
                    "propagate: the graph refers to rows beyond the feature or rule matrix");
        const int n = (int)t.plans.size();
        check(cgnn_propagate(n, t.plans.data(), t.values.data(), t.scratch.data(), t.scratch_bytes.data(), t.code, width,
                             x.data_ptr(), rule_ptr, out.data_ptr(), backward ? 1 : 0, first, last < 0 ? n - 1 : last,
                             t.stream));
        return out;
    }

    Tensor apply(const Tensor &x, bool backward);

  private:
    struct Table {
        bool backward;
        int64_t width;
        int code;
        cgnn_stream_t stream;
        int64_t x_rows, rule_rows;
        std::vector<const cgnn_plan *> plans;
        std::vector<const void *> values;
        std::vector<void *> scratch;
        std::vector<size_t> scratch_bytes;
    };

    // The value arrays of one direction in plan order.  Every stream reads the same ones, so they are complete before
    // the first launch that does.
    const std::vector<Tensor> &ordered(bool backward, const Tensor &x, int code) {
        auto &have = ordered_[backward][code];
        if (!have.empty()) return have;
        have = complete(x.get_device(), [&] {
            std::vector<Tensor> arrays;
            for (auto &launch : launches_[backward]) {
                Tensor dst = at::empty({launch.first->nnz}, x.options());
                if (launch.first->nnz) {
                    Tensor v0 = launch.second[0].to(x.scalar_type()).contiguous(), v1;
                    int64_t given = v0.numel();
                    if (launch.second.size() > 1) {
                        v1 = launch.second[1].to(x.scalar_type()).contiguous();
                        given += v1.numel();
                    }
                    TORCH_CHECK(given == launch.first->nnz, "values do not match the plan's entries");
                    check(cgnn_plan_permute_values(launch.first->get(), code, data(v0), data(v1), dst.data_ptr(),
                                                   current_stream(x)));
                }
                arrays.push_back(dst);
            }
            return arrays;
        });
        return have;
    }

    const Table &table(bool backward, int64_t width, const Tensor &x) {
        const int code = dtype_code(x);
        const cgnn_stream_t stream = current_stream(x);
        std::lock_guard<std::mutex> guard(lock_);
        for (const auto &t : tables_)
            if (t->backward == backward && t->width == width && t->code == code && t->stream == stream) return *t;
        auto t = std::make_unique<Table>();
        t->backward = backward;
        t->width = width;
        t->code = code;
        t->stream = stream;
        const auto &values = ordered(backward, x, code);
        const auto &launches = launches_[backward];
        for (size_t i = 0; i < launches.size(); ++i) {
            auto s = launches[i].first->scratch(width, code, stream);
            t->plans.push_back(launches[i].first->get());
            t->values.push_back(data(values[i]));
            values[i].record_stream(c10::cuda::getCurrentCUDAStream(x.get_device()));
            t->scratch.push_back(s.first);
            t->scratch_bytes.push_back(s.second);
        }
        const int64_t *last = launches.back().first->source_rows;
        t->x_rows = std::max(launches.front().first->source_rows[0], last[backward ? 0 : 1]);
        t->rule_rows = last[backward ? 1 : 0];
        tables_.push_back(std::move(t));
        return *tables_.back();
    }

    int64_t vertices_, rules_;
    std::vector<Launch> launches_[2];
    std::vector<Tensor> ordered_[2][2];
    std::mutex lock_;
    std::vector<std::unique_ptr<Table>> tables_;
};

// What arrives for an output whose consumer returned no gradient: zeros, as autograd functions get them.
Tensor materialized(Node &node, const Tensor &grad) { return grad.defined() ? grad : node.input_metadata(0).zeros_like(); }

struct PropagateBackward : public Node {
    std::shared_ptr<Propagation> graph;
    bool backward = false;  // direction of the pass this node differentiates
    variable_list apply(variable_list &&grads) override {
        if (!task_should_compute_output(0)) return {Tensor()};
        return {graph->apply(materialized(*this, grads[0]), !backward)};
    }
    std::string name() const override { return "CompressgnnPropagateBackward"; }
};

template <typename N>
std::shared_ptr<N> new_node() {
    return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

// One direction with autograd (its derivative is the other direction).
Tensor Propagation::apply(const Tensor &x, bool backward) {
    refuse_dual("the propagation", {x});
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = run(x, backward, Tensor(), Tensor(), 0, -1);
    }
    if (torch::autograd::compute_requires_grad(x)) {
        auto node = new_node<PropagateBackward>();
        node->graph = shared_from_this();
        node->backward = backward;
        node->set_next_edges(torch::autograd::collect_next_edges(x));
        torch::autograd::set_history(out, node);
    }
    return out;
}

// ---------------------------------------------------------------------------------------------
// bucket mean, Linear, reconstruction
// ---------------------------------------------------------------------------------------------
Tensor mean(const Tensor &x, const Tensor &counts, Plan &plan) {
    Tensor out = at::empty({counts.numel(), x.size(1)}, x.options());
    const int code = dtype_code(x);
    const cgnn_stream_t stream = current_stream(x);
    auto s = plan.scratch(x.size(1), code, stream);
    check(cgnn_cluster_mean(plan.get(), code, x.size(1), data(x), counts.const_data_ptr<int32_t>(), data(out), s.first,
                            s.second, stream));
    return out;
}

Tensor mean_backward(const Tensor &grad, const Tensor &index, const Tensor &counts) {
    Tensor out = at::empty({index.numel(), grad.size(1)}, grad.options());
    if (out.numel() == 0) return out;
    Tensor scaled = at::empty_like(grad);
    check(cgnn_cluster_mean_backward(dtype_code(grad), index.numel(), grad.size(1), grad.size(0), data(grad),
                                     index.const_data_ptr<int64_t>(), counts.const_data_ptr<int32_t>(), data(out),
                                     data(scaled), current_stream(grad)));
    return out;
}

Tensor reconstruct(const Tensor &reps, const Tensor &index, const Tensor &bias, bool relu, double p, uint64_t seed) {
    Tensor out = at::empty({index.numel(), reps.size(1)}, reps.options());
    if (out.numel() == 0) return out;
    const int code = dtype_code(reps);
    if (p > 0.0)
        check(cgnn_cluster_reconstruct_dropout(code, index.numel(), reps.size(1), reps.size(0), data(reps),
                                               index.const_data_ptr<int64_t>(), data(bias), p, seed, data(out),
                                               current_stream(reps)));
    else
        check(cgnn_cluster_reconstruct(code, index.numel(), reps.size(1), reps.size(0), data(reps),
                                       index.const_data_ptr<int64_t>(), data(bias), relu ? 1 : 0, data(out),
                                       current_stream(reps)));
    return out;
}

// relu: 0, 1 (mask row per node) or 2 (one mask row per group), as in cgnn_cluster_reconstruct_backward.
std::pair<Tensor, Tensor> reconstruct_backward(const Tensor &grad, const Tensor &output, int64_t groups, int relu,
                                               bool want_bias, Plan &plan) {
    const int64_t width = grad.size(1);
    Tensor out = at::empty({groups, width}, grad.options()), bias;
    if (want_bias) bias = at::empty({width}, grad.options());
    TORCH_CHECK(plan.rows == groups && plan.nnz == grad.size(0), "reconstruct backward: plan does not match index/groups");
    const int code = dtype_code(grad);
    const cgnn_stream_t stream = current_stream(grad);
    auto s = plan.scratch(width, code, stream);
    check(cgnn_cluster_reconstruct_backward(plan.get(), code, width, data(grad), relu ? data(output) : nullptr, relu,
                                            data(out), data(bias), s.first, s.second, stream));
    return {out, bias};
}

// a^T b for tall a [K, M] and b [K, N]: the weight gradient over the representatives.  The package's kernel splits K
// over the GPU; it takes fp32 at full precision with up to a GPU of output tiles (64 x 128), beyond which the
// library's tiles fill the GPU without a split, and leaves a caller who allowed TF32 products to the library.  (128 x 256 over
// 64 k rows: 158 us there, 90 here; beyond 148 tiles neither side is measured and the library stays.)
// The precision is asked for by the query that answers for all of torch's switches: the older one raises once the
// newer switch has been used.
bool full_precision_products() {
    const auto precision = at::globalContext().float32Precision(at::Float32Backend::CUDA, at::Float32Op::MATMUL);
    return precision == at::Float32Precision::NONE || precision == at::Float32Precision::IEEE;
}

Tensor matmul_tn(const Tensor &a, const Tensor &b) {
    const int64_t K = a.size(0), M = a.size(1), N = b.size(1);
    const int64_t tiles = ((M + 63) / 64) * ((N + 127) / 128);
    if (a.scalar_type() != at::kFloat || tiles > 148 || tiles == 0 || !full_precision_products())
        return at::mm(a.t(), b);
    Tensor out = at::empty({M, N}, a.options());
    const size_t bytes = cgnn_matmul_tn_scratch_bytes(K, M, N);
    const Tensor scratch = at::empty({(int64_t)bytes}, a.options().dtype(at::kByte));
    check(cgnn_matmul_tn(K, M, N, static_cast<const float *>(data(a)), static_cast<const float *>(data(b)),
                         static_cast<float *>(data(out)), data(scratch), bytes, current_stream(a)));
    return out;
}

// A fresh 63-bit key from torch's host generator (follows torch.manual_seed; no device synchronisation):
// the draw of torch.randint(0, 2**63 - 1, (1,)).
uint64_t dropout_key() {
    return (uint64_t)at::randint(0, std::numeric_limits<int64_t>::max(), {1}, at::TensorOptions().dtype(at::kLong))
        .const_data_ptr<int64_t>()[0];
}

void check_matrix(const Tensor &x) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2, "Expected contiguous CUDA matrix");
    TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kDouble, "Only float32 and float64 are supported");
}

void check_index(const Tensor &index, const Tensor &like) {
    TORCH_CHECK(index.device() == like.device() && index.dim() == 1 && index.is_contiguous() &&
                    index.scalar_type() == at::kLong,
                "Expected contiguous int64 index on input device");
}

void check_counts(const Tensor &counts, const Tensor &like) {
    TORCH_CHECK(counts.device() == like.device() && counts.dim() == 1 && counts.is_contiguous() &&
                    counts.scalar_type() == at::kInt && counts.numel() >= 1,
                "Expected nonempty int32 counts on input device");
}

void check_bias(const Tensor &bias, int64_t width, const Tensor &like) {
    if (bias.defined())
        TORCH_CHECK(bias.device() == like.device() && bias.scalar_type() == like.scalar_type() && bias.dim() == 1 &&
                        bias.numel() == width,
                    "Invalid reconstruction bias");
}

// (Saved tensors are unpacked with .contiguous(): what a saved-tensor hook hands back may have other strides.)
// The gradients of these nodes are final: differentiating them again raises.  That takes an incoming gradient that
// is differentiated itself; with a constant one the result is a constant.
variable_list first_order(variable_list &&result, const variable_list &incoming) {
    if (!torch::autograd::compute_requires_grad(incoming)) return std::move(result);
    variable_list wrapped;
    for (auto &t : result) {
        if (t.defined()) {
            auto error = std::make_shared<torch::autograd::Error>(
                "trying to differentiate twice a function that was marked with @once_differentiable");
            t = t.detach().requires_grad_();
            error->set_next_edges(torch::autograd::collect_next_edges(t));
            Tensor out = t.detach();
            torch::autograd::set_history(out, error);
            wrapped.push_back(out);
        } else {
            wrapped.push_back(t);
        }
    }
    return wrapped;
}

struct MeanBackward : public Node {
    SavedVariable index_, counts_;
    variable_list apply(variable_list &&grads) override {
        if (!task_should_compute_output(0)) return {Tensor()};
        Tensor dx;
        {
            at::NoGradGuard no_grad;
            const Tensor grad = materialized(*this, grads[0]).contiguous();
            const c10::cuda::OptionalCUDAGuard guard(grad.device());
            dx = mean_backward(grad, index_.unpack().contiguous(), counts_.unpack().contiguous());
        }
        return first_order({dx}, grads);
    }
    void release_variables() override {
        index_.reset_data();
        counts_.reset_data();
    }
    std::string name() const override { return "CompressgnnMeanBackward"; }
};

Tensor mean_autograd(const Tensor &x_in, const Tensor &index, const Tensor &counts, const PlanPtr &plan) {
    refuse_dual("the bucket mean", {x_in});
    check_matrix(x_in);
    check_index(index, x_in);
    check_counts(counts, x_in);
    TORCH_CHECK(index.numel() == x_in.size(0), "Input/index length mismatch");
    TORCH_CHECK(x_in.numel() == 0 || (plan && plan->rows == counts.numel() && plan->nnz == index.numel()),
                "cluster_mean: plan does not match index/count");
    const c10::cuda::OptionalCUDAGuard guard(x_in.device());
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor x = x_in.contiguous();
        out = x.numel() ? mean(x, counts, *plan) : at::zeros({counts.numel(), x.size(1)}, x.options());
    }
    if (torch::autograd::compute_requires_grad(x_in)) {
        auto node = new_node<MeanBackward>();
        node->index_ = SavedVariable(index, false);
        node->counts_ = SavedVariable(counts, false);
        node->set_next_edges(torch::autograd::collect_next_edges(x_in));
        torch::autograd::set_history(out, node);
    }
    return out;
}

// plan == null: the index did not come from an assignment; its plan is built when the backward needs it.
PlanPtr plan_for(const PlanPtr &plan, const Tensor &index, int64_t groups) {
    if (plan) return plan;
    pybind11::gil_scoped_acquire gil;
    return pybind11::module_::import("compressgnn_b200.runtime")
        .attr("index_plan")(index, groups)
        .attr("native")
        .cast<PlanPtr>();
}

std::pair<Tensor, Tensor> backward_or_zero(const Tensor &grad, const Tensor &output, int64_t groups, int relu,
                                           bool want_bias, const PlanPtr &plan) {
    if (grad.numel()) return reconstruct_backward(grad, output, groups, relu, want_bias, *plan);
    return {at::zeros({groups, grad.size(1)}, grad.options()),
            want_bias ? at::zeros({grad.size(1)}, grad.options()) : Tensor()};
}

struct ReconstructBackward : public Node {
    SavedVariable index_, output_;
    PlanPtr plan;
    int64_t groups = 0;
    bool relu = false, has_bias = false;
    double p = 0.0;
    variable_list apply(variable_list &&grads) override {
        std::pair<Tensor, Tensor> r;
        {
            at::NoGradGuard no_grad;
            const Tensor grad = materialized(*this, grads[0]).contiguous();
            const c10::cuda::OptionalCUDAGuard guard(grad.device());
            const Tensor output = relu ? output_.unpack(shared_from_this()).contiguous() : Tensor();
            const Tensor index = index_.unpack().contiguous();
            const PlanPtr segments = grad.numel() ? plan_for(plan, index, groups) : plan;
            // Without dropout the rows of a group are identical and one mask row per group suffices; with it every
            // row has its own zeros (dropped or clamped alike): exact mask, sums rescaled.
            r = backward_or_zero(grad, output, groups, relu ? (p > 0.0 ? 1 : 2) : 0, has_bias, segments);
            if (p > 0.0) {
                r.first.mul_(1.0 / (1.0 - p));
                if (has_bias) r.second.mul_(1.0 / (1.0 - p));
            }
        }
        return first_order({r.first, r.second}, grads);
    }
    void release_variables() override {
        index_.reset_data();
        output_.reset_data();
    }
    std::string name() const override { return "CompressgnnReconstructBackward"; }
};

Tensor reconstruct_autograd(const Tensor &src, const Tensor &index_in, const c10::optional<Tensor> &bias_in, bool relu,
                            double p, const PlanPtr &plan) {
    check_matrix(src);
    const Tensor index = index_in.contiguous();
    check_index(index, src);
    const Tensor bias = bias_in.has_value() ? *bias_in : Tensor();
    refuse_dual("the reconstruction", {src, bias});
    check_bias(bias, src.size(1), src);
    TORCH_CHECK(p >= 0.0 && p < 1.0, "dropout probability must lie in [0, 1)");
    TORCH_CHECK(p == 0.0 || relu, "the fused dropout follows a ReLU (the backward reads its mask off the zeros)");
    const c10::cuda::OptionalCUDAGuard guard(src.device());
    const uint64_t seed = p > 0.0 ? dropout_key() : 0;
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = reconstruct(src.contiguous(), index, bias.defined() ? bias.contiguous() : bias, relu, p, seed);
    }
    if (torch::autograd::compute_requires_grad(src, bias)) {
        auto node = new_node<ReconstructBackward>();
        node->plan = plan;
        node->groups = src.size(0);
        node->relu = relu;
        node->has_bias = bias.defined();
        node->p = p;
        node->index_ = SavedVariable(index, false);
        node->set_next_edges(torch::autograd::collect_next_edges(src, bias));
        torch::autograd::set_history(out, node);
        if (relu) node->output_ = SavedVariable(out, true);
    }
    return out;
}

// act(dropout)(Linear(bucket means of x)) spread back over the nodes: the three modules of a layer
// (ref: model/compressgnn/gcn.py:27-34) as one autograd node.
struct TransformBackward : public Node {
    SavedVariable index_, counts_, reps_, weight_, output_;
    PlanPtr plan;
    bool relu = false;
    double p = 0.0;
    variable_list apply(variable_list &&grads) override {
        Tensor dx, dw, db;
        {
            at::NoGradGuard no_grad;
            const Tensor grad = materialized(*this, grads[0]).contiguous();
            const c10::cuda::OptionalCUDAGuard guard(grad.device());
            // all of them, needed or not: one that was modified in place since the forward pass is an error
            const Tensor index = index_.unpack().contiguous(), counts = counts_.unpack().contiguous();
            const Tensor reps = reps_.unpack().contiguous(), weight = weight_.unpack();
            const Tensor output = relu ? output_.unpack(shared_from_this()).contiguous() : Tensor();
            auto r = backward_or_zero(grad, output, reps.size(0), relu ? (p > 0.0 ? 1 : 2) : 0, true, plan);
            if (p > 0.0) {
                r.first.mul_(1.0 / (1.0 - p));
                r.second.mul_(1.0 / (1.0 - p));
            }
            if (task_should_compute_output(1)) dw = matmul_tn(r.first, reps);
            if (task_should_compute_output(0))
                dx = mean_backward(at::mm(r.first, weight), index, counts);
            if (task_should_compute_output(2)) db = r.second;
        }
        return first_order({dx, dw, db}, grads);
    }
    void release_variables() override {
        for (SavedVariable *v : {&index_, &counts_, &reps_, &weight_, &output_}) v->reset_data();
    }
    std::string name() const override { return "CompressgnnTransformBackward"; }
};

Tensor transform_autograd(const Tensor &x_in, const Tensor &index, const Tensor &counts, const PlanPtr &plan,
                          const Tensor &weight, const c10::optional<Tensor> &bias_in, bool relu, double p) {
    check_matrix(x_in);
    check_index(index, x_in);
    check_counts(counts, x_in);
    TORCH_CHECK(index.numel() == x_in.size(0), "Input/index length mismatch");
    // (without columns the mean needs no plan, but the backward sums gradients as wide as the layer's output)
    TORCH_CHECK(x_in.size(0) == 0 || (plan && plan->rows == counts.numel() && plan->nnz == index.numel()),
                "transform: plan does not match index/count");
    const Tensor bias = bias_in.has_value() ? *bias_in : Tensor();
    refuse_dual("the transformation", {x_in, weight, bias});
    check_bias(bias, weight.size(0), x_in);
    TORCH_CHECK(p >= 0.0 && p < 1.0, "dropout probability must lie in [0, 1)");
    TORCH_CHECK(p == 0.0 || relu, "the fused dropout follows a ReLU (the backward reads its mask off the zeros)");
    const c10::cuda::OptionalCUDAGuard guard(x_in.device());
    Tensor reps, out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        reps = x_in.numel() ? mean(x_in.contiguous(), counts, *plan) : at::zeros({counts.numel(), x_in.size(1)}, x_in.options());
        const Tensor lin = at::mm(reps, weight.t());
        const uint64_t seed = p > 0.0 ? dropout_key() : 0;
        out = reconstruct(lin, index, bias.defined() ? bias.contiguous() : bias, relu, p, seed);
    }
    if (torch::autograd::compute_requires_grad(x_in, weight, bias)) {
        auto node = new_node<TransformBackward>();
        node->plan = plan;
        node->relu = relu;
        node->p = p;
        node->index_ = SavedVariable(index, false);
        node->counts_ = SavedVariable(counts, false);
        node->reps_ = SavedVariable(reps, false);
        node->weight_ = SavedVariable(weight, false);
        node->set_next_edges(torch::autograd::collect_next_edges(x_in, weight, bias));
        torch::autograd::set_history(out, node);
        if (relu) node->output_ = SavedVariable(out, true);
    }
    return out;
}

// ---------------------------------------------------------------------------------------------
// row operators of a training step: normalisation, dropout, loss
// ---------------------------------------------------------------------------------------------
int row_dtype(const Tensor &t, const char *what) {
    switch (t.scalar_type()) {
        case at::kFloat: return CGNN_F32;
        case at::kDouble: return CGNN_F64;
        case at::kBFloat16: return CGNN_BF16;
        case at::kHalf: return CGNN_F16;
        default: TORCH_CHECK(false, what, ": only float32, float64, bfloat16 and float16 are supported");
    }
}

Tensor dense(const Tensor &t) { return t.defined() ? t.contiguous() : t; }

at::ScalarType sum_type(const Tensor &t) { return t.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }

// A matrix [rows, last dimension] over `t` whose rows may lie apart; anything else is made dense.
struct Rows {
    Tensor held;
    int64_t rows, width, stride;
    explicit Rows(const Tensor &t) : width(t.size(-1)) {
        if (t.dim() == 2 && (t.stride(1) == 1 || width == 1) && t.stride(0) >= 0) {
            held = t;
            stride = t.stride(0);
        } else {
            held = t.contiguous();
            stride = width;
        }
        rows = width ? held.numel() / width : 0;
    }
};

// The engine lets the streams of a backward pass wait for those its leaves' gradients were first accumulated on.  While
// a graph is captured that would be a wait on work outside the capture, which breaks it off (and ends the process where
// the error meets a thread of the engine), so the call is refused before anything is recorded.
void refuse_foreign_leaves(const char *what, at::TensorList inputs) {
    const auto concerned = [](const Tensor &t) { return t.defined() && t.requires_grad() && t.is_leaf(); };
    if (!at::GradMode::is_enabled() || std::none_of(inputs.begin(), inputs.end(), concerned) || !capturing()) return;
    for (const Tensor &t : inputs) {
        if (!concerned(t)) continue;
        const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
        if (!accumulator) continue;
        const auto stream = accumulator->stream();
        TORCH_CHECK(!stream || *stream == c10::cuda::getCurrentCUDAStream(t.get_device()).unwrap(), what,
                    ": an eager graph over one of these leaves still lives, on another stream than the one being captured; "
                    "drop its outputs before the capture, or build it on the capture's stream");
    }
}

// The key of a dropout: a number, or one int64 on the device.  Neither given: a fresh one, inside a capture drawn by
// the captured graph itself, so that every replay has another.
struct Key {
    uint64_t seed = 0;
    Tensor on_device;
    const int64_t *pointer() const { return on_device.defined() ? on_device.const_data_ptr<int64_t>() : nullptr; }
};

Key key_of(const char *what, double p, const c10::optional<int64_t> &seed, const c10::optional<Tensor> &seed_tensor,
           const Tensor &like) {
    TORCH_CHECK(p >= 0.0 && p < 1.0, "dropout probability must lie in [0, 1)");
    Key key;
    if (seed_tensor.has_value()) {
        key.on_device = *seed_tensor;
        TORCH_CHECK(key.on_device.device() == like.device() && key.on_device.scalar_type() == at::kLong &&
                        key.on_device.numel() == 1,
                    what, ": a seed in a tensor is one int64 on the input's device");
    } else if (seed.has_value()) {
        key.seed = (uint64_t)*seed;
    } else if (p > 0.0) {
        if (capturing())
            key.on_device = at::randint(0, std::numeric_limits<int64_t>::max(), {1}, like.options().dtype(at::kLong).requires_grad(false));
        else
            key.seed = dropout_key();
    }
    return key;
}

void *second_row(const Tensor &t) {
    return t.defined() && t.numel() ? static_cast<char *>(t.data_ptr()) + t.size(1) * t.element_size() : nullptr;
}

struct NormSettings {
    int dtype = 0, param_dtype = 0;
    double eps = 0.0, p = 0.0;
    bool relu = false;
    uint64_t seed = 0;
};

struct LayerNormBackward : public Node {
    SavedVariable x_, weight_, bias_, statistics_, key_;
    NormSettings set;
    at::TensorOptions param_options;
    variable_list apply(variable_list &&grads) override {
        Tensor dx, dw, db;
        {
            at::NoGradGuard no_grad;
            const Tensor grad = materialized(*this, grads[0]).contiguous();
            const c10::cuda::OptionalCUDAGuard guard(grad.device());
            const Tensor x_in = x_.unpack(), weight = dense(weight_.unpack()), bias = dense(bias_.unpack());
            const Tensor statistics = statistics_.unpack().contiguous();  // [2, rows]: means, then 1 / deviations
            const Tensor key = dense(key_.unpack());
            const Rows x(x_in);
            const auto plain = grad.options().requires_grad(false);
            if (task_should_compute_output(0)) dx = at::empty(x_in.sizes(), plain);
            if (task_should_compute_output(1)) dw = at::empty({x.width}, param_options);
            if (task_should_compute_output(2)) db = at::empty({x.width}, param_options);
            Tensor scratch;
            size_t bytes = 0;
            if (dw.defined() || db.defined()) {
                bytes = cgnn_layer_norm_scratch_bytes(set.dtype, x.rows, x.width);
                scratch = at::empty({(int64_t)bytes}, plain.dtype(at::kByte));
            }
            check(cgnn_layer_norm_backward(set.dtype, set.param_dtype, x.rows, x.width, x.stride, data(x.held), data(weight),
                                           data(bias), data(statistics), second_row(statistics), data(grad), set.relu, set.p, set.seed,
                                           static_cast<const int64_t *>(data(key)), data(dx), data(dw), data(db), data(scratch),
                                           bytes, current_stream(grad)));
        }
        return first_order({dx, dw, db}, grads);
    }
    void release_variables() override {
        for (SavedVariable *v : {&x_, &weight_, &bias_, &statistics_, &key_}) v->reset_data();
    }
    std::string name() const override { return "CompressgnnLayerNormBackward"; }
};

Tensor layer_norm_autograd(const Tensor &x_in, const c10::optional<Tensor> &weight_in, const c10::optional<Tensor> &bias_in,
                           double eps, bool relu, double p, const c10::optional<int64_t> &seed,
                           const c10::optional<Tensor> &seed_tensor) {
    const Tensor weight = weight_in.value_or(Tensor()), bias = bias_in.value_or(Tensor());
    TORCH_CHECK(x_in.is_cuda() && x_in.dim() >= 1, "layer_norm: Expected a CUDA tensor of one dimension or more");
    refuse_dual("the layer normalisation", {x_in, weight, bias});
    NormSettings set;
    set.dtype = set.param_dtype = row_dtype(x_in, "layer_norm");
    const Tensor &either = weight.defined() ? weight : bias;
    if (either.defined()) {
        set.param_dtype = row_dtype(either, "layer_norm");
        TORCH_CHECK(set.param_dtype == set.dtype || (x_in.element_size() == 2 && set.param_dtype == CGNN_F32),
                    "layer_norm: weight and bias are of the input's type, or float32 beside a 16-bit one");
    }
    for (const Tensor &t : {weight, bias})
        TORCH_CHECK(!t.defined() || (t.device() == x_in.device() && t.dim() == 1 && t.size(0) == x_in.size(-1) &&
                                     t.scalar_type() == either.scalar_type()),
                    "layer_norm: weight and bias are vectors over the last dimension, of one type and on the input's device");
    TORCH_CHECK(eps >= 0.0, "layer_norm: eps must not be negative");
    const c10::cuda::OptionalCUDAGuard guard(x_in.device());
    const Key key = key_of("layer_norm", p, seed, seed_tensor, x_in);
    refuse_foreign_leaves("layer_norm", {x_in, weight, bias});
    set.eps = eps;
    set.p = p;
    set.relu = relu;
    set.seed = key.seed;
    const bool differentiated = torch::autograd::compute_requires_grad(x_in, weight, bias);
    Tensor out, statistics;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Rows x(x_in);
        const Tensor w = dense(weight), b = dense(bias);
        out = at::empty(x_in.sizes(), x_in.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
        if (differentiated) statistics = at::empty({2, x.rows}, x_in.options().dtype(sum_type(x_in)).requires_grad(false));
        check(cgnn_layer_norm(set.dtype, set.param_dtype, x.rows, x.width, x.stride, data(x.held), data(w), data(b), eps, relu, p,
                              key.seed, key.pointer(), data(out), data(statistics), second_row(statistics), current_stream(x_in)));
    }
    if (differentiated) {
        auto node = new_node<LayerNormBackward>();
        node->set = set;
        node->param_options = (either.defined() ? either : x_in).options().requires_grad(false);
        node->x_ = SavedVariable(x_in, false);
        node->weight_ = SavedVariable(weight, false);
        node->bias_ = SavedVariable(bias, false);
        node->statistics_ = SavedVariable(statistics, false);
        node->key_ = SavedVariable(key.on_device, false);
        node->set_next_edges(torch::autograd::collect_next_edges(x_in, weight, bias));
        torch::autograd::set_history(out, node);
    }
    return out;
}

Tensor dropout_pass(const Tensor &x, const Tensor &residual, double p, uint64_t seed, const int64_t *device_seed) {
    Tensor out = at::empty(x.sizes(), x.options().requires_grad(false));
    check(cgnn_dropout(row_dtype(x, "dropout"), x.numel(), data(x), data(residual), p, seed, device_seed, data(out),
                       current_stream(x)));
    return out;
}

struct DropoutBackward : public Node {
    SavedVariable key_;
    double p = 0.0;
    uint64_t seed = 0;
    variable_list apply(variable_list &&grads) override {
        Tensor dx, dresidual;
        {
            at::NoGradGuard no_grad;
            const Tensor key = dense(key_.unpack());
            const Tensor grad = materialized(*this, grads[0]);
            const c10::cuda::OptionalCUDAGuard guard(grad.device());
            if (task_should_compute_output(0))
                dx = dropout_pass(grad.contiguous(), Tensor(), p, seed, static_cast<const int64_t *>(data(key)));
            if (task_should_compute_output(1)) dresidual = grad;
        }
        return first_order({dx, dresidual}, grads);
    }
    void release_variables() override { key_.reset_data(); }
    std::string name() const override { return "CompressgnnDropoutBackward"; }
};

Tensor dropout_autograd(const Tensor &x_in, double p, const c10::optional<Tensor> &residual_in, const c10::optional<int64_t> &seed,
                        const c10::optional<Tensor> &seed_tensor) {
    const Tensor residual = residual_in.value_or(Tensor());
    TORCH_CHECK(x_in.is_cuda(), "dropout: Expected a CUDA tensor");
    row_dtype(x_in, "dropout");
    refuse_dual("the dropout", {x_in, residual});
    TORCH_CHECK(!residual.defined() || (residual.device() == x_in.device() && residual.scalar_type() == x_in.scalar_type() &&
                                        residual.sizes() == x_in.sizes()),
                "dropout: the residual has the input's shape, type and device");
    const c10::cuda::OptionalCUDAGuard guard(x_in.device());
    const Key key = key_of("dropout", p, seed, seed_tensor, x_in);
    refuse_foreign_leaves("dropout", {x_in, residual});
    Tensor out;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        out = dropout_pass(x_in.contiguous(), dense(residual), p, key.seed, key.pointer());
    }
    if (torch::autograd::compute_requires_grad(x_in, residual)) {
        auto node = new_node<DropoutBackward>();
        node->p = p;
        node->seed = key.seed;
        node->key_ = SavedVariable(key.on_device, false);
        node->set_next_edges(torch::autograd::collect_next_edges(x_in, residual));
        torch::autograd::set_history(out, node);
    }
    return out;
}

constexpr int64_t LABELLED_BYTES = 16;

// For a sum or a mean the forward pass has written the gradient for an incoming one (`unit_`).  The first backward pass
// hands that array on, after a launch that computes it anew unless the incoming gradient is one; further passes over a
// retained graph have an array of their own.
struct CrossEntropyBackward : public Node {
    SavedVariable logits_, target_, held_;  // held_: the number of labelled rows, and each row's statistics
    Tensor unit_;
    int dtype = 0, reduction = 0;
    int64_t ignore_index = 0;
    variable_list apply(variable_list &&grads) override {
        std::lock_guard<std::mutex> guard_of_node(mutex_);
        Tensor dlogits;
        {
            at::NoGradGuard no_grad;
            const Tensor grad = materialized(*this, grads[0]).contiguous();
            const c10::cuda::OptionalCUDAGuard guard(grad.device());
            const Tensor logits = logits_.unpack(), target = target_.unpack().contiguous();
            const Tensor held_bytes = held_.unpack().contiguous();
            char *const held = static_cast<char *>(data(held_bytes));
            const Rows z(logits);
            const bool unit = unit_.defined() && !capturing();
            if (unit) dlogits = std::move(unit_);
            else dlogits = at::empty(logits.sizes(), logits.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
            unit_.reset();
            check(cgnn_cross_entropy_backward(dtype, z.rows, z.width, z.stride, data(z.held), static_cast<const int64_t *>(data(target)),
                                              ignore_index, reduction, held + LABELLED_BYTES, reinterpret_cast<const int64_t *>(held),
                                              data(grad), unit, data(dlogits), current_stream(grad)));
        }
        return first_order({dlogits}, grads);
    }
    void release_variables() override {
        std::lock_guard<std::mutex> guard_of_node(mutex_);
        for (SavedVariable *v : {&logits_, &target_, &held_}) v->reset_data();
        unit_.reset();
    }
    std::string name() const override { return "CompressgnnCrossEntropyBackward"; }
};

Tensor cross_entropy_autograd(const Tensor &logits, const Tensor &target_in, int64_t ignore_index, int reduction) {
    TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.size(1) >= 1,
                "cross_entropy: Expected a CUDA matrix [rows, classes] of class scores");
    const int dtype = row_dtype(logits, "cross_entropy");
    TORCH_CHECK(target_in.device() == logits.device() && target_in.scalar_type() == at::kLong && target_in.dim() == 1 &&
                    target_in.size(0) == logits.size(0),
                "cross_entropy: Expected one int64 class per row on the scores' device");
    TORCH_CHECK(reduction >= CGNN_NONE && reduction <= CGNN_MEAN, "cross_entropy: unknown reduction");
    refuse_dual("the cross entropy", {logits});
    const c10::cuda::OptionalCUDAGuard guard(logits.device());
    refuse_foreign_leaves("cross_entropy", {logits});
    const bool differentiated = torch::autograd::compute_requires_grad(logits);
    const Tensor target = target_in.contiguous();
    Tensor loss, held, unit;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Rows z(logits);
        const auto plain = logits.options().requires_grad(false);
        const auto sums = plain.dtype(sum_type(logits));
        const bool reduced = reduction != CGNN_NONE;
        if (reduced) loss = at::empty({}, sums);
        else loss = at::empty({z.rows}, sums);
        // (a captured backward pass may be replayed more than once per forward pass: it computes the gradient itself)
        if (differentiated && reduced && !capturing())
            unit = at::empty(logits.sizes(), plain.memory_format(at::MemoryFormat::Contiguous));
        // one allocation: the number of labelled rows, the rows' statistics, and what the launches hand each other
        const int64_t stats_bytes = differentiated ? 2 * z.rows * (int64_t)sums.dtype().itemsize() : 0;
        const int64_t scratch_begin = (LABELLED_BYTES + stats_bytes + 15) / 16 * 16;
        const int64_t scratch_bytes = reduced ? (int64_t)cgnn_cross_entropy_scratch_bytes() : 0;
        char *place = nullptr;
        if (reduced || differentiated) {
            held = at::empty({scratch_begin + scratch_bytes}, plain.dtype(at::kByte));
            place = static_cast<char *>(data(held));
        }
        check(cgnn_cross_entropy(dtype, z.rows, z.width, z.stride, data(z.held), static_cast<const int64_t *>(data(target)),
                                 ignore_index, reduction, data(loss), stats_bytes ? place + LABELLED_BYTES : nullptr, data(unit),
                                 reinterpret_cast<int64_t *>(place), place ? place + scratch_begin : nullptr, scratch_bytes,
                                 current_stream(logits)));
    }
    if (differentiated) {
        auto node = new_node<CrossEntropyBackward>();
        node->dtype = dtype;
        node->reduction = reduction;
        node->ignore_index = ignore_index;
        node->logits_ = SavedVariable(logits, false);
        node->target_ = SavedVariable(target, false);
        node->held_ = SavedVariable(held, false);
        node->unit_ = unit;
        node->set_next_edges(torch::autograd::collect_next_edges(logits));
        torch::autograd::set_history(loss, node);
    }
    return loss;
}

// ---------------------------------------------------------------------------------------------
// a dense layer as one product
// ---------------------------------------------------------------------------------------------
struct LinearBackward : public Node {
    SavedVariable x_, weight_, mask_;  // the input where the weight has a gradient, the weight where the input has one
    int dtype = 0;
    double p = 0.0;
    std::vector<int64_t> sizes;  // of the input
    int64_t rows = 0, in = 0, out = 0;
    at::TensorOptions options;
    variable_list apply(variable_list &&grads) override {
        Tensor dx, dw, db, dresidual;
        {
            at::NoGradGuard no_grad;
            const Tensor incoming = materialized(*this, grads[0]);
            const c10::cuda::OptionalCUDAGuard guard(incoming.device());
            // all that was kept, needed this time or not: one that was modified in place since the forward pass is an error
            const Tensor x_in = x_.unpack(), weight = dense(weight_.unpack()), mask = dense(mask_.unpack());
            if (task_should_compute_output(0)) dx = at::empty(sizes, options);
            if (task_should_compute_output(1)) dw = at::empty({out, in}, options);
            if (task_should_compute_output(2)) db = at::empty({out}, options);
            if (dx.defined() || dw.defined() || db.defined()) {
                const Tensor grad = incoming.contiguous();
                Tensor x;
                int64_t stride = in;
                if (x_in.defined()) {
                    const Rows of_x(x_in);
                    x = of_x.held;
                    stride = of_x.stride;
                }
                const size_t bytes = cgnn_linear_backward_scratch_bytes(dtype, rows, in, out);
                const Tensor scratch = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
                check(cgnn_linear_backward(dtype, rows, in, out, stride, data(x), data(weight), data(mask), data(grad), p, data(dx),
                                           data(dw), data(db), data(scratch), bytes, current_stream(grad)));
            }
            if (task_should_compute_output(3)) dresidual = incoming;
        }
        return first_order({dx, dw, db, dresidual}, grads);
    }
    void release_variables() override {
        for (SavedVariable *v : {&x_, &weight_, &mask_}) v->reset_data();
    }
    std::string name() const override { return "CompressgnnLinearBackward"; }
};

Tensor linear_autograd(const Tensor &x_in, const Tensor &weight, const c10::optional<Tensor> &bias_in, bool relu, double p,
                       const c10::optional<Tensor> &residual_in, const c10::optional<int64_t> &seed,
                       const c10::optional<Tensor> &seed_tensor) {
    const Tensor bias = bias_in.value_or(Tensor()), residual = residual_in.value_or(Tensor());
    TORCH_CHECK(x_in.is_cuda() && x_in.dim() >= 1, "linear: Expected a CUDA tensor of one dimension or more");
    const int dtype = row_dtype(x_in, "linear");
    refuse_dual("the dense layer", {x_in, weight, bias, residual});
    TORCH_CHECK(weight.dim() == 2 && weight.size(1) == x_in.size(-1) && weight.device() == x_in.device() &&
                    weight.scalar_type() == x_in.scalar_type(),
                "linear: the weight is [out, in] for the input's last dimension, of its type and on its device");
    const int64_t in = weight.size(1), out = weight.size(0);
    TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == out && bias.device() == x_in.device() &&
                                    bias.scalar_type() == x_in.scalar_type()),
                "linear: the bias is a vector over the weight's rows, of the input's type and on its device");
    auto sizes = x_in.sizes().vec();
    sizes.back() = out;
    TORCH_CHECK(!residual.defined() || (residual.sizes() == at::IntArrayRef(sizes) && residual.device() == x_in.device() &&
                                        residual.scalar_type() == x_in.scalar_type()),
                "linear: the residual has the output's shape, type and device");
    const c10::cuda::OptionalCUDAGuard guard(x_in.device());
    const Key key = key_of("linear", p, seed, seed_tensor, x_in);
    refuse_foreign_leaves("linear", {x_in, weight, bias, residual});
    const bool differentiated = torch::autograd::compute_requires_grad(x_in, weight, bias, residual);
    const bool masked = differentiated && (relu || p > 0.0);
    const auto plain = x_in.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous);
    const int64_t rows = c10::multiply_integers(sizes.begin(), sizes.end() - 1);
    Tensor y, mask;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Rows x(x_in);
        y = at::empty(sizes, plain);
        if (masked) mask = at::empty({(int64_t)cgnn_linear_mask_bytes(rows, out)}, plain.dtype(at::kByte));
        const size_t bytes = cgnn_linear_scratch_bytes(dtype, rows, in, out);
        const Tensor scratch = at::empty({(int64_t)bytes}, plain.dtype(at::kByte));
        const Tensor w = weight.contiguous(), b = dense(bias), r = dense(residual);
        check(cgnn_linear(dtype, rows, in, out, x.stride, data(x.held), data(w), data(b), data(r), relu, p, key.seed, key.pointer(),
                          data(y), data(mask), data(scratch), bytes, current_stream(x_in)));
    }
    if (differentiated) {
        auto node = new_node<LinearBackward>();
        node->dtype = dtype;
        node->p = p;
        node->sizes = x_in.sizes().vec();
        node->rows = rows;
        node->in = in;
        node->out = out;
        node->options = plain;
        if (weight.requires_grad()) node->x_ = SavedVariable(x_in, false);
        if (x_in.requires_grad()) node->weight_ = SavedVariable(weight, false);
        if (masked) node->mask_ = SavedVariable(mask, false);
        node->set_next_edges(torch::autograd::collect_next_edges(x_in, weight, bias, residual));
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ---------------------------------------------------------------------------------------------
// one optimiser step over many tensors
// ---------------------------------------------------------------------------------------------
// The places that a step writes: no two of its tensors may share memory, nor one of them with what it reads.
struct Places {
    using Span = std::pair<uintptr_t, uintptr_t>;
    std::vector<Span> written, read;
    static Span span_of(const Tensor &t) {
        const uintptr_t first = reinterpret_cast<uintptr_t>(t.const_data_ptr());
        return {first, first + t.nbytes()};
    }
    void writes(const Tensor &t) {
        TORCH_CHECK(!t.is_inference() || c10::InferenceMode::is_enabled(), "adamw_step: an inference tensor is written in inference mode only");
        if (t.numel()) written.push_back(span_of(t));
    }
    void reads(const Tensor &t) {
        if (t.numel()) read.push_back(span_of(t));
    }
    bool apart() {
        std::sort(written.begin(), written.end());
        for (size_t i = 1; i < written.size(); ++i)
            if (written[i].first < written[i - 1].second) return false;
        for (const Span &r : read) {  // (the first written one that ends behind its beginning)
            const auto next = std::partition_point(written.begin(), written.end(), [&](const Span &w) { return w.second <= r.first; });
            if (next != written.end() && next->first < r.second) return false;
        }
        return true;
    }
};

c10::optional<Tensor> adamw_step(const std::vector<Tensor> &params, const std::vector<Tensor> &grads, const std::vector<Tensor> &firsts,
                                 const std::vector<Tensor> &seconds, const std::vector<Tensor> &steps,
                                 const std::vector<c10::optional<Tensor>> &first_scales,
                                 const std::vector<c10::optional<Tensor>> &second_scales, const std::vector<double> &rates,
                                 const std::vector<c10::optional<Tensor>> &rate_tensors, const std::vector<double> &decays, double beta1,
                                 double beta2, double eps, const c10::optional<double> &max_norm, int64_t seed) {
    const size_t n = params.size();
    // (of scales none at all, of rates one for all)
    TORCH_CHECK(grads.size() == n && firsts.size() == n && seconds.size() == n && steps.size() == n &&
                    (first_scales.size() == n || first_scales.empty()) && (second_scales.size() == n || second_scales.empty()) &&
                    (rates.size() == n || rates.size() == 1) && rate_tensors.size() == rates.size() &&
                    (decays.size() == n || decays.size() == 1),
                "adamw_step: as many gradients, moments, steps, scales and rates as parameters are needed");
    const auto scale_of = [](const std::vector<c10::optional<Tensor>> &scales, size_t i) {
        return scales.empty() || !scales[i].has_value() ? Tensor() : *scales[i];
    };
    // (the library's bounds, before anything is looked at: a list without tensors is checked too)
    TORCH_CHECK(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adamw_step: the betas must lie in [0, 1)");
    TORCH_CHECK(eps >= 0.0, "adamw_step: eps must not be negative");
    TORCH_CHECK(!max_norm.has_value() || *max_norm >= 0.0, "adamw_step: max_norm must not be negative");
    if (n == 0) return c10::nullopt;
    const auto device = params[0].device();
    TORCH_CHECK(device.is_cuda(), "compressgnn_b200 runs on CUDA tensors only (no CPU optimiser path)");
    std::vector<cgnn_adamw_tensor> list(n);
    Places places;
    places.written.reserve(6 * n);
    places.read.reserve(2 * n);
    for (size_t i = 0; i < n; ++i) {
        const Tensor &p = params[i], &g = grads[i], &m = firsts[i], &v = seconds[i], &t = steps[i];
        const int dtype = row_dtype(p, "adamw_step");
        TORCH_CHECK(p.device() == device && g.device() == device && m.device() == device && v.device() == device && t.device() == device,
                    "adamw_step: all tensors lie on one device");
        TORCH_CHECK(p.is_contiguous(), "adamw_step: parameters are contiguous");
        TORCH_CHECK(g.sizes() == p.sizes() && g.scalar_type() == p.scalar_type() && g.is_contiguous(),
                    "adamw_step: a gradient is contiguous and has its parameter's shape and type");
        const bool eight = m.scalar_type() == at::kFloat8_e4m3fn;
        TORCH_CHECK(m.sizes() == p.sizes() && v.sizes() == p.sizes() && m.is_contiguous() && v.is_contiguous(),
                    "adamw_step: moments are contiguous and have their parameter's shape");
        TORCH_CHECK(m.scalar_type() == v.scalar_type() && (eight ? dtype != CGNN_F64 : m.scalar_type() == sum_type(p)),
                    "adamw_step: moments are float32 (float64 beside float64 parameters) or, with scales, float8_e4m3fn");
        TORCH_CHECK(t.scalar_type() == at::kLong && t.numel() == 1, "adamw_step: the steps taken are one int64 for each parameter");
        const Tensor first_scale = scale_of(first_scales, i), second_scale = scale_of(second_scales, i);
        TORCH_CHECK(eight == first_scale.defined() && eight == second_scale.defined(),
                    "adamw_step: moments of 8 bits come with scales, others without");
        cgnn_adamw_tensor &e = list[i];
        const size_t rate_at = rates.size() == 1 ? 0 : i;
        e.lr = rates[rate_at];
        e.weight_decay = decays[decays.size() == 1 ? 0 : i];
        e.device_lr = nullptr;
        TORCH_CHECK(e.lr >= 0.0 && e.weight_decay >= 0.0, "adamw_step: lr and weight_decay must not be negative");
        if (rate_tensors[rate_at].has_value()) {
            const Tensor &rate = *rate_tensors[rate_at];
            TORCH_CHECK(rate.device() == device && rate.scalar_type() == at::kFloat && rate.numel() == 1,
                        "adamw_step: a learning rate in a tensor is one float32 on the parameters' device");
            e.device_lr = rate.const_data_ptr<float>();
            places.reads(rate);
        }
        if (eight)
            for (const Tensor &s : {first_scale, second_scale})
                TORCH_CHECK(s.device() == device && s.scalar_type() == at::kFloat && s.is_contiguous() && s.numel() == (p.numel() + 255) / 256,
                            "adamw_step: a moment has one float32 scale for each block of 256 elements");
        for (const Tensor *w : {&p, &m, &v, &t}) places.writes(*w);
        places.reads(g);
        e.param = data(p);
        e.grad = data(g);
        e.exp_avg = data(m);
        e.exp_avg_sq = data(v);
        e.exp_avg_scale = e.exp_avg_sq_scale = nullptr;
        if (eight) {
            places.writes(first_scale);
            places.writes(second_scale);
            // (of an empty tensor: no scales, which are not looked at, but moments of 8 bits all the same)
            e.exp_avg_scale = static_cast<float *>(p.numel() ? data(first_scale) : data(t));
            e.exp_avg_sq_scale = static_cast<float *>(p.numel() ? data(second_scale) : data(t));
        }
        e.step = t.data_ptr<int64_t>();
        e.n = p.numel();
        e.dtype = dtype;
    }
    TORCH_CHECK(places.apart(), "adamw_step: parameters, moments, scales and steps must not share memory, nor with gradients and rates");
    const c10::cuda::OptionalCUDAGuard guard(device);
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor norm, scratch;
    size_t bytes = 0;
    if (max_norm.has_value()) {
        const auto options = at::TensorOptions().device(device);
        norm = at::empty({}, options.dtype(at::kFloat));
        bytes = cgnn_adamw_scratch_bytes(list.data(), (int64_t)n);
        scratch = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
    }
    check(cgnn_adamw(list.data(), (int64_t)n, beta1, beta2, eps, max_norm.value_or(-1.0), (uint64_t)seed,
                     static_cast<float *>(data(norm)), data(scratch), bytes, current_stream(params[0])));
    // what was written in place is newer than what autograd may have saved of it
    for (size_t i = 0; i < n; ++i) {
        for (const Tensor *w : {&params[i], &firsts[i], &seconds[i], &steps[i]}) w->unsafeGetTensorImpl()->bump_version();
        if (list[i].exp_avg_scale != nullptr)
            for (const Tensor &s : {*first_scales[i], *second_scales[i]}) s.unsafeGetTensorImpl()->bump_version();
    }
    return norm.defined() ? c10::optional<Tensor>(norm) : c10::nullopt;
}

// ---------------------------------------------------------------------------------------------
// assignment
// ---------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, int64_t, PlanPtr> assign(const Tensor &x, const Tensor &planes, int bits, const Tensor &workspace) {
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    at::AutoDispatchBelowADInplaceOrView below;
    const cgnn_stream_t stream = current_stream(x);
    const int64_t n = x.size(0);
    const auto ints = x.options().dtype(at::kInt).requires_grad(false);
    Tensor codes = at::empty({n}, ints), ids = at::empty({n}, ints.dtype(at::kLong));
    check(cgnn_cluster_codes(dtype_code(x), data(x), data(planes), n, x.size(1), bits, codes.data_ptr<int32_t>(), stream));
    int64_t active = 0;
    check(cgnn_cluster_assign(codes.data_ptr<int32_t>(), n, bits, workspace.data_ptr(), workspace.numel(),
                              ids.data_ptr<int64_t>(), &active, stream));
    Tensor counts = at::empty({active + 1}, ints);
    cgnn_plan *plan = nullptr;
    check(cgnn_cluster_assign_export(workspace.data_ptr(), n, active, counts.data_ptr<int32_t>(), &plan, 0, stream));
    return {ids, counts, active, std::make_shared<Plan>(reinterpret_cast<intptr_t>(plan), x.get_device())};
}

}  // namespace

namespace py = pybind11;

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    using nogil = py::call_guard<py::gil_scoped_release>;
    py::class_<Plan, PlanPtr>(m, "Plan")
        .def(py::init<intptr_t, int>())
        .def_property_readonly("handle", &Plan::address)
        .def("scratch", &Plan::scratch_py, nogil());
    py::class_<Propagation, std::shared_ptr<Propagation>>(m, "Propagation")
        .def(py::init<int64_t, int64_t, std::vector<Propagation::Launch>, std::vector<Propagation::Launch>>())
        .def("apply", &Propagation::apply, nogil())
        .def("run",
             [](Propagation &p, const Tensor &x, bool backward, const c10::optional<Tensor> &out,
                const c10::optional<Tensor> &rule_out, int first, int last) {
                 at::NoGradGuard no_grad;
                 return p.run(x, backward, out.value_or(Tensor()), rule_out.value_or(Tensor()), first, last);
             },
             py::arg("x"), py::arg("backward"), py::arg("out") = py::none(), py::arg("rule_out") = py::none(),
             py::arg("first") = 0, py::arg("last") = -1, nogil());
    m.def("mean", &mean_autograd, nogil());
    m.def("reconstruct", &reconstruct_autograd, nogil());
    m.def("transform", &transform_autograd, nogil());
    m.def("layer_norm", &layer_norm_autograd, nogil());
    m.def("dropout", &dropout_autograd, nogil());
    m.def("cross_entropy", &cross_entropy_autograd, nogil());
    m.def("linear", &linear_autograd, nogil());
    m.def("adamw_step", &adamw_step, nogil());
    m.def("assign", &assign, nogil());
    m.def("matmul_tn", [](const Tensor &a, const Tensor &b) {
        TORCH_CHECK(a.is_cuda() && a.device() == b.device() && a.scalar_type() == b.scalar_type() && a.dim() == 2 &&
                        b.dim() == 2 && a.size(0) == b.size(0) && a.is_contiguous() && b.is_contiguous(),
                    "Expected contiguous CUDA matrices with equal row counts");
        const c10::cuda::OptionalCUDAGuard guard(a.device());
        at::NoGradGuard no_grad;
        return matmul_tn(a, b);
    }, nogil());
}
