// Host side of raft_amd.group_norm and raft_amd.AdamW between PyTorch and the C ABI (include/raftcorr.h): argument checks, memory from
// the caching allocator, the autograd node, the walk over a model's parameters.  In C++ because at these sizes the host decides: a
// training pass of the norm over a 1/8-resolution map takes some 50 us of GPU time and took 136 us of host time as a Python autograd
// function; reading the addresses of 124 parameters and gradients takes 75 us in Python.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <c10/core/DeviceGuard.h>
#include "../../include/raftcorr.h"

namespace {

using at::Tensor;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void require(int rc, const char* what)
{
    if (rc != RAFTCORR_OK) throw std::runtime_error(std::string("raftcorr ") + what + " failed (code " + std::to_string(rc) + "): " + raftcorr_last_error());
}

#define REFUSE(...) do { std::ostringstream s_; s_ << __VA_ARGS__; throw std::runtime_error(s_.str()); } while (0)

int dtype_of(const Tensor& t)
{
    switch (t.scalar_type()) {
        case at::kFloat: return RAFTCORR_DTYPE_FP32;
        case at::kHalf: return RAFTCORR_DTYPE_FP16;
        case at::kBFloat16: return RAFTCORR_DTYPE_BF16;
        default: return -1;
    }
}

// ---- group norm ---------------------------------------------------------------------------------------------------------

// A (N, C, *spatial) tensor as N x P rows of C neighbouring values, a tensor of any other layout copied to dense channels-last first.
struct Rows { Tensor t; int64_t batch, row, P; };

Rows rows_of(const Tensor& t)
{
    const int64_t C = t.size(1);
    int64_t row = -1, size = 1, P = 1;                  // stride of the rows so far, positions they cover
    bool ok = C == 1 || t.stride(1) == 1;
    for (int64_t d = t.dim() - 1; d >= 2; --d) {
        const int64_t n = t.size(d), s = t.stride(d);
        P *= n;
        if (n == 1) continue;
        if (row < 0) { row = s; ok = ok && s >= C; }
        ok = ok && s == row * size;
        size *= n;
    }
    if (!ok) return Rows{t.movedim(1, -1).contiguous().movedim(-1, 1), P * C, C, P};
    return Rows{t, t.size(0) > 1 ? t.stride(0) : 0, row < 0 ? C : row, P};
}

// uninitialised, dense channels-last, of x's sizes and type
Tensor like_rows(const Tensor& x)
{
    c10::SmallVector<int64_t, 6> strides(x.dim());
    const int64_t C = x.size(1);
    int64_t s = C;
    strides[1] = 1;
    for (int64_t d = x.dim() - 1; d >= 2; --d) { strides[d] = s; s *= std::max<int64_t>(x.size(d), 1); }
    strides[0] = s;
    return at::empty_strided(x.sizes(), strides, x.options().requires_grad(false));
}

const float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

struct NormForward { Rows x; Tensor y, stats; };

NormForward norm_forward(const Tensor& x_, const Tensor& weight, const Tensor& bias, int64_t groups, double eps, int64_t act)
{
    const c10::OptionalDeviceGuard guard(x_.device());
    NormForward f{rows_of(x_), Tensor(), Tensor()};
    const Tensor& x = f.x.t;
    const int64_t N = x.size(0), C = x.size(1);
    f.y = like_rows(x);
    f.stats = at::empty({N, groups, 2}, x.options().dtype(at::kDouble).requires_grad(false));
    if (x.numel() == 0) return f;
    if (N > INT_MAX || C > INT_MAX) REFUSE("group_norm: " << N << " samples of " << C << " channels are too many");
    const int64_t bytes = raftcorr_group_norm_workspace_bytes((int)N, (int)C, (int)groups);
    const Tensor work = at::empty({bytes}, x.options().dtype(at::kByte).requires_grad(false));
    require(raftcorr_group_norm_fwd(x.data_ptr(), f.x.batch, f.x.row, dtype_of(x), (int)N, f.x.P, (int)C, (int)groups, floats(weight), floats(bias),
                                    eps, (int)act, f.y.data_ptr(), f.stats.data_ptr<double>(), work.data_ptr(), bytes, stream_of(x)), "group_norm_fwd");
    return f;
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, int64_t groups,
                          double eps, int64_t act)
    {
        const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
        NormForward f = norm_forward(x, w, b, groups, eps, act);
        ctx->save_for_backward({f.x.t, w, b, f.stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        ctx->saved_data["leaves"] = (int64_t)(1 + 2 * (weight && weight->requires_grad()) + 4 * (bias && bias->requires_grad()));
        ctx->set_materialize_grads(false);
        return f.y;
    }

    static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grads)
    {
        Tensor dx, dw, db;
        if (grads[0].defined()) {
            const auto saved = ctx->get_saved_variables();
            const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
            const int64_t groups = ctx->saved_data["groups"].toInt(), act = ctx->saved_data["act"].toInt(), leaves = ctx->saved_data["leaves"].toInt();
            const bool again = at::GradMode::is_enabled();
            {
                const at::NoGradGuard no_grad;
                const c10::OptionalDeviceGuard guard(x.device());
                const int64_t N = x.size(0), C = x.size(1);
                const auto options = x.options().dtype(at::kFloat).requires_grad(false);
                if (ctx->needs_input_grad(0)) dx = like_rows(x);
                if (leaves & 2) dw = x.numel() ? at::empty({C}, options) : at::zeros({C}, options);
                if (leaves & 4) db = x.numel() ? at::empty({C}, options) : at::zeros({C}, options);
                if (x.numel()) {
                    const Rows r = rows_of(x), d = rows_of(grads[0].scalar_type() == x.scalar_type() ? grads[0] : grads[0].to(x.scalar_type()));
                    const int64_t bytes = raftcorr_group_norm_workspace_bytes((int)N, (int)C, (int)groups);
                    const Tensor work = at::empty({bytes}, x.options().dtype(at::kByte).requires_grad(false));
                    require(raftcorr_group_norm_bwd(r.t.data_ptr(), r.batch, r.row, d.t.data_ptr(), d.batch, d.row, dtype_of(x), (int)N, r.P, (int)C,
                                                    (int)groups, floats(weight), floats(bias), (int)act, stats.data_ptr<double>(),
                                                    dx.defined() ? dx.data_ptr() : nullptr, dw.defined() ? dw.data_ptr<float>() : nullptr,
                                                    db.defined() ? db.data_ptr<float>() : nullptr, work.data_ptr(), bytes, stream_of(x)),
                            "group_norm_bwd");
                }
            }
            if (again)                                   // a second derivative through these would be wrong without a word
                for (Tensor* t : {&dx, &dw, &db})
                    if (t->defined()) {
                        const auto error = std::make_shared<torch::autograd::DelayedError>("group_norm: trying to differentiate twice a function that was marked with once_differentiable", 1);
                        *t = (*error)({t->requires_grad_(true)})[0];
                    }
        }
        return {dx, dw, db, Tensor(), Tensor(), Tensor()};
    }
};

// A backward pass inside a capture ends the process where a leaf's accumulation node belongs to another stream, which it does while an
// eager graph of the leaf is alive: refused before anything is recorded.
void check_capture(const char* name, const Tensor& t)
{
    if (!t.defined() || !t.requires_grad() || !t.is_leaf()) return;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto stream = node ? node->stream() : std::nullopt;
    if (stream && *stream != c10::Stream(c10::hip::getCurrentHIPStream(t.device().index())))
        REFUSE("group_norm: an eager graph of " << name << " is alive (on another stream than the capture's); delete its results before the capture");
}

Tensor group_norm(const Tensor& x, int64_t groups, const Maybe& weight_, const Maybe& bias_, double eps, int64_t act)
{
    if (!x.is_cuda()) REFUSE("x must be a CUDA tensor");
    if (x.dim() < 2) REFUSE("x must be (N, C, *spatial), got shape " << x.sizes());
    if (x.layout() != at::kStrided || dtype_of(x) < 0) REFUSE("x must be a dense float32, float16 or bfloat16 tensor, got " << x.scalar_type() << " " << x.layout());
    const int64_t C = x.size(1);
    if (groups < 1 || C < 1 || C % groups) REFUSE("num_groups = " << groups << " does not divide " << C << " channels");
    if (!(eps >= 0)) REFUSE("eps = " << eps);
    Maybe weight = weight_, bias = bias_;
    for (auto& [name, t] : {std::pair<const char*, Maybe*>{"weight", &weight}, {"bias", &bias}}) {
        if (!*t) continue;
        if ((*t)->device() != x.device()) REFUSE(name << " is on " << (*t)->device() << ", expected " << x.device());
        if ((*t)->dim() != 1 || (*t)->size(0) != C || !(*t)->is_floating_point())
            REFUSE(name << " must be a floating-point tensor of shape (" << C << ",), got " << (*t)->scalar_type() << " " << (*t)->sizes());
        *t = (*t)->to(at::kFloat).contiguous();
    }
    if (at::GradMode::is_enabled() && (x.requires_grad() || (weight && weight->requires_grad()) || (bias && bias->requires_grad())))
    {
        const c10::OptionalDeviceGuard guard(x.device());
        if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) {
            check_capture("x", x);
            check_capture("weight", weight_.value_or(Tensor()));
            check_capture("bias", bias_.value_or(Tensor()));
        }
        return GroupNorm::apply(x, weight, bias, groups, eps, act);
    }
    return norm_forward(x, weight.value_or(Tensor()), bias.value_or(Tensor()), groups, eps, act).y;
}

std::tuple<Tensor, int64_t, int64_t> rows(const Tensor& t)
{
    Rows r = rows_of(t);
    return {r.t, r.batch, r.row};
}

// ---- AdamW --------------------------------------------------------------------------------------------------------------

// Whether the tensor's values fill one stretch of memory without gaps or overlaps, in whatever order.
bool dense(const Tensor& t) { return t.is_non_overlapping_and_dense(); }

// Whether two tensors of the same sizes keep their values in the same order (strides of axes of one value say nothing).
bool same_order(at::IntArrayRef sizes, at::IntArrayRef a, at::IntArrayRef b)
{
    if (a.size() != sizes.size() || b.size() != sizes.size()) return false;
    for (size_t d = 0; d < sizes.size(); ++d)
        if (sizes[d] != 1 && a[d] != b[d]) return false;
    return true;
}

// The parameters of one group that share device and type: where they start in the bucket's buffers, and what one step works on.
struct Bucket {
    std::vector<int64_t> numel, offset;
    std::vector<std::vector<int64_t>> strides;
    int64_t total = 0;
    c10::Device device;
    at::ScalarType dtype;
    // of the step that is being taken
    std::vector<void*> p;
    std::vector<const void*> g;
    std::vector<int64_t> n, at_;
    std::vector<int32_t> slot;
    std::vector<Tensor> copies;

    explicit Bucket(const std::vector<Tensor>& params) : device(params.at(0).device()), dtype(params.at(0).scalar_type())
    {
        for (const Tensor& t : params) {
            if (t.device() != device || t.scalar_type() != dtype) REFUSE("a bucket's parameters share device and type");
            if (!dense(t)) REFUSE("parameter of shape " << t.sizes() << " and strides " << t.strides() << " does not lie in one stretch of memory");
            numel.push_back(t.numel());
            offset.push_back(total);
            strides.push_back(t.strides().vec());
            total += (t.numel() + RAFTCORR_ADAMW_TILE - 1) / RAFTCORR_ADAMW_TILE * RAFTCORR_ADAMW_TILE;
        }
    }

    // whether any two of all parameters share memory: they would be updated at the same time
    static bool overlap(const std::vector<Tensor>& params)
    {
        std::vector<std::pair<uintptr_t, uintptr_t>> spans;
        for (const Tensor& t : params)
            if (t.numel()) spans.emplace_back((uintptr_t)t.data_ptr(), (uintptr_t)t.data_ptr() + t.numel() * t.element_size());
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i)
            if (spans[i].first < spans[i - 1].second) return true;
        return false;
    }

    // the addresses of the parameters that have a gradient; how many
    int64_t collect(py::list params)
    {
        if (params.size() != numel.size()) REFUSE("the number of parameters has changed since the state was made");
        const at::NoGradGuard no_grad;
        p.clear(); g.clear(); n.clear(); at_.clear(); slot.clear(); copies.clear();
        for (size_t i = 0; i < numel.size(); ++i) {
            const Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(params.ptr(), (Py_ssize_t)i));
            Tensor grad = t.grad();
            if (!grad.defined()) continue;
            if (grad.scalar_type() != dtype || grad.device() != device || grad.layout() != at::kStrided)
                REFUSE("gradient is " << grad.scalar_type() << ", " << grad.layout() << " on " << grad.device() << ", expected a dense " << dtype << " on " << device);
            if (t.scalar_type() != dtype || t.device() != device || t.numel() != numel[i] || grad.numel() != numel[i])
                REFUSE("a parameter's type, device or size has changed since the state was made");
            if (!same_order(t.sizes(), t.strides(), strides[i])) REFUSE("a parameter's memory order has changed since the state was made");
            if (!same_order(t.sizes(), t.strides(), grad.strides())) {
                grad = at::empty_like(t).copy_(grad);                   // the order of the parameter's memory
                copies.push_back(grad);
            }
            p.push_back(t.data_ptr());
            g.push_back(grad.data_ptr());
            n.push_back(numel[i]);
            at_.push_back(offset[i]);
            slot.push_back((int32_t)i);
        }
        return (int64_t)p.size();
    }

    int64_t partials() const { return raftcorr_adamw_norm_partials(n.data(), (int)n.size()); }

    void norm(const Tensor& partial, int64_t first) const
    {
        const c10::OptionalDeviceGuard guard(device);
        require(raftcorr_adamw_norm(g.data(), n.data(), (int)n.size(), code(), partial.data_ptr<double>() + first, stream_of(partial)), "adamw_norm");
    }

    // partial: the sums of squares and one value more, the coefficient
    void step(int64_t bits, const Tensor& m, const Tensor& v, const Tensor& me, const Tensor& ve, const Tensor& steps, const Maybe& lr_device, double lr,
              double b1, double b2, double eps, double decay, int64_t seed, const Maybe& partial, double max_norm, const Maybe& norm)
    {
        const c10::OptionalDeviceGuard guard(device);
        const Tensor scale = at::empty({2 * (int64_t)numel.size()}, steps.options());
        const int64_t partials = partial ? partial->numel() - 1 : 0;
        require(raftcorr_adamw_step(p.data(), g.data(), n.data(), at_.data(), slot.data(), (int)p.size(), code(), (int)bits, m.data_ptr(), v.data_ptr(),
                                    bits == 8 ? me.data_ptr<uint8_t>() : nullptr, bits == 8 ? ve.data_ptr<uint8_t>() : nullptr, steps.data_ptr<float>(),
                                    scale.data_ptr<float>(), lr, lr_device ? lr_device->data_ptr<float>() : nullptr, b1, b2, eps, decay, (uint32_t)seed,
                                    partial ? partial->data_ptr<double>() : nullptr, (int)partials, max_norm,
                                    partial ? partial->data_ptr<double>() + partials : nullptr, norm ? norm->data_ptr<float>() : nullptr,
                                    stream_of(steps)), "adamw_step");
        copies.clear();
    }

    int code() const { return dtype == at::kFloat ? RAFTCORR_DTYPE_FP32 : RAFTCORR_DTYPE_BF16; }
};

}  // namespace

PYBIND11_MODULE(_glue, m)
{
    m.def("group_norm", &group_norm, py::arg("x"), py::arg("groups"), py::arg("weight"), py::arg("bias"), py::arg("eps"), py::arg("act"));
    m.def("rows", &rows, "the tensor, batch and row strides under which a (N, C, *spatial) tensor is rows of C neighbouring values");
    m.def("dense", &dense);
    m.def("same_order", [](const Tensor& a, const Tensor& b) { return same_order(a.sizes(), a.strides(), b.strides()); });
    py::class_<Bucket>(m, "Bucket")
        .def(py::init<const std::vector<Tensor>&>())
        .def_static("overlap", &Bucket::overlap)
        .def_readonly("total", &Bucket::total)
        .def_readonly("offsets", &Bucket::offset)
        .def_readonly("numels", &Bucket::numel)
        .def("collect", &Bucket::collect)
        .def("partials", &Bucket::partials)
        .def("norm", &Bucket::norm)
        .def("step", &Bucket::step);
}
