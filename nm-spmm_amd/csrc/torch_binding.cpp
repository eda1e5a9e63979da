// What torch_op.py calls for every forward and backward pass: checks of torch tensors, outputs and workspaces from torch's
// caching allocator, and the C-ABI call on the tensors' device and current stream, without Python in between.  Small calls
// are bound by the host: with the same steps in Python a one-row product took 8.7 us, a norm of one row 13.4 and its
// forward and backward pass 112 (autograd's thread waits for the interpreter there); here 5.3, 5.5 and 54, of which 3.7 are a
// launch each.
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <climits>
#include <stdexcept>

#include "../../include/nmspmm.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

int type_of(at::ScalarType t)
{
    return t == at::kFloat ? NMSPMM_F32 : t == at::kBFloat16 ? NMSPMM_BF16 : t == at::kHalf ? NMSPMM_F16 : -1;
}

// A status of the C-ABI, on its way to Python's NmSpmmError.
struct Failure : std::runtime_error {
    const char* function;
    int status;
    Failure(const char* function, int status)
        : std::runtime_error(std::string(function) + " failed: " + nmspmm_status_string(status)), function(function), status(status)
    {
    }
};

void check(const char* function, int status)
{
    if (status != NMSPMM_OK)
        throw Failure(function, status);
}

// Refuses an argument: ValueError in Python.
template <class... What>
void require(bool held, const What&... what)
{
    if (!held)
        throw std::invalid_argument(c10::str(what...));
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

const void* at_of(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// Whether a call must go through the dispatcher: someone else is to see it (a tracer, a dispatch mode, a function transform), or a tensor has
// no memory of its own (a wrapper, a batched one).  Keys beside those of an ordinary tensor and of autograd say so.
bool intercepted(std::initializer_list<const Tensor*> given)
{
    constexpr c10::DispatchKeySet ours = c10::DispatchKeySet({c10::DispatchKey::Dense, c10::DispatchKey::BackendSelect, c10::DispatchKey::Negative,
                                                              c10::DispatchKey::ADInplaceOrView}) |
                                         c10::autograd_dispatch_keyset | c10::autocast_dispatch_keyset;
    const auto tls = c10::impl::tls_local_dispatch_key_set();
    c10::DispatchKeySet keys = tls.included_;
    for (const Tensor* t : given)
        if (t->defined())
            keys = keys | t->key_set();
    return ((keys - tls.excluded_ - ours).raw_repr() & ~c10::full_backend_mask) != 0;
}

// What lies in memory is what t stands for, and no tangent of forward-mode differentiation is lost.
Tensor plain(const Tensor& t)
{
    if (!t.defined())
        return t;
    require(!t._fw_grad(0).defined(), "there is no forward-mode derivative");
    return t.is_neg() ? t.resolve_neg() : t;
}

// ---- operands in 4 bits --------------------------------------------------------------------------------

Tensor quant_linear(const Tensor& x, const Tensor& codes, const Tensor& scales, const OptTensor& row_offsets, const OptTensor& bias,
                    int64_t K, int64_t N, int64_t n, int64_t m, int64_t group)
{
    require(K >= 1 && N >= 1 && K <= INT_MAX && N <= INT_MAX && n >= 1 && m >= n && m <= INT_MAX && group >= 1 && group <= 128,
            "no operand of ", K, " x ", N, " with pattern ", n, ":", m, " and groups of ", group);
    const int type = type_of(x.scalar_type());
    require(x.is_cuda() && type >= 0 && x.dim() >= 1 && x.size(-1) == K,
                      "x must be a float32, bfloat16 or float16 CUDA tensor whose last dimension is ", K);
    const Tensor rows = row_offsets.value_or(Tensor());
    Tensor plus = bias.value_or(Tensor());
    auto buffer = [&](const Tensor& t, size_t need) {
        return t.device() == x.device() && t.is_contiguous() && t.nbytes() >= need && need > 0;
    };
    require(buffer(codes, nmspmm_q4_codes_bytes(K, N, n, m)) && buffer(scales, nmspmm_q4_meta_bytes(K, N, n, m, group)) &&
                (n == m || (rows.defined() && buffer(rows, nmspmm_q4_row_offsets_bytes(K, N, n, m)))),
                      "codes, scales and row offsets must be those of an operand of ", K, " x ", N, ", on the device of x");
    if (plus.defined()) {
        require(plus.device() == x.device() && plus.dim() == 1 && plus.size(0) == N, "bias must have ", N, " elements on the device of x");
        plus = plain(plus).to(at::kFloat).contiguous();
    }
    const c10::DeviceGuard guard(x.device());
    auto shape = x.sizes().vec();
    shape.back() = N;
    Tensor y = at::empty(shape, x.options());
    const int64_t M = y.numel() / N;
    if (M == 0)
        return y;
    Tensor from = plain(x);
    int64_t ldx = K;
    if (!from.is_contiguous()) {
        from = from.reshape({M, K});
        if (M > 1)
            ldx = from.stride(0);
        if ((K > 1 && from.stride(1) != 1) || ldx < K || ldx > (1 << 24)) {
            from = from.contiguous();
            ldx = K;
        }
    }
    require(M <= 1 << 24, "at most 2^24 rows, got ", M);
    nmspmm_q4_operand op = {codes.data_ptr(), scales.data_ptr(), const_cast<void*>(at_of(rows)), static_cast<const float*>(at_of(plus)),
                            (int)K, (int)N, (int)n, (int)m, (int)group};
    Tensor workspace;
    size_t need = 0;
    if (M > 8) {        // below, no operand needs one
        need = nmspmm_q4_workspace_bytes((int)M, (int)K, (int)N, (int)n, (int)m, type);
        if (need > 0)
            workspace = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
    }
    check("nmspmm_q4_linear", nmspmm_q4_linear(&op, from.const_data_ptr(), ldx, y.data_ptr(), N, (int)M, type,
                                               const_cast<void*>(at_of(workspace)), need, stream_of(x)));
    return y;
}

// Nothing where the registered operator is to be called in its place.
OptTensor quant_linear_direct(const Tensor& x, const Tensor& codes, const Tensor& scales, const OptTensor& row_offsets, const OptTensor& bias,
                              int64_t K, int64_t N, int64_t n, int64_t m, int64_t group)
{
    const Tensor rows = row_offsets.value_or(Tensor()), plus = bias.value_or(Tensor());
    if (intercepted({&x, &codes, &scales, &rows, &plus}))
        return std::nullopt;
    return quant_linear(x, codes, scales, row_offsets, bias, K, N, n, m, group);
}

// ---- the norms around a block -----------------------------------------------------------------------------

struct Conf {
    double factor = 1.0;
    int64_t post = 0, pre = 0;
    double eps = 0.0, weight_offset = 0.0;
    int64_t gate_rows = 1;
    at::ScalarType dtype = at::kFloat;
    bool want_out = true;

    std::vector<double> packed() const
    {
        return {factor, (double)post, (double)pre, eps, weight_offset, (double)gate_rows, (double)(int)dtype, (double)want_out};
    }
    static Conf of(const std::vector<double>& p)
    {
        return {p[0], (int64_t)p[1], (int64_t)p[2], p[3], p[4], (int64_t)p[5], (at::ScalarType)(int)p[6], p[7] != 0.0};
    }
};

// residual, branch, gate, scale, post weight and bias, pre weight and bias; undefined where there is none.
constexpr int kGiven = 8;
using Given = std::array<Tensor, kGiven>;
const char* const kNames[kGiven] = {"residual", "branch", "gate", "residual_scale", "post_weight", "post_bias", "pre_weight", "pre_bias"};

// t where its leading dimensions can be walked as rows, else a copy; and the elements between its rows.
std::pair<Tensor, int64_t> as_rows(const Tensor& given, int64_t D)
{
    const Tensor t = plain(given);
    if (!t.defined() || t.is_contiguous())
        return {t, D};
    Tensor rows = t.reshape({-1, D});
    if ((D > 1 && rows.stride(1) != 1) || (rows.size(0) > 1 && rows.stride(0) < D))
        rows = rows.contiguous();
    return {rows, std::max(rows.stride(0), D)};
}

void check_given(const Given& g, const Conf& c)
{
    const Tensor& residual = g[0];
    require(residual.is_cuda() && type_of(residual.scalar_type()) >= 0 && residual.dim() >= 1,
                      "residual must be a float32, bfloat16 or float16 CUDA tensor");
    const int64_t D = residual.size(-1);
    require(D >= 1 && D <= 16384, "rows must have 1 to 16384 features, got ", D);
    require(c.post >= 0 && c.post <= 2 && c.pre >= 0 && c.pre <= 2, "post and pre are \"rms\", \"layer\" or None");
    require(type_of(c.dtype) >= 0 && (residual.scalar_type() == c.dtype || residual.scalar_type() == at::kFloat),
                      "residual must be float32 or of the type of what the next block takes");
    require(c.eps >= 0.0, "eps must not be negative");
    if (g[1].defined()) {
        require(g[1].sizes() == residual.sizes() && g[1].device() == residual.device() && g[1].scalar_type() == c.dtype,
                          "branch must have residual's shape and device and the type of what the next block takes");
    } else {
        require(!g[2].defined() && !g[3].defined() && c.factor == 1.0 && c.post == 0 && c.want_out,
                          "without a branch there is a norm before the next block and nothing else");
    }
    require((c.post != 0 || (!g[4].defined() && !g[5].defined())) && (c.pre != 0 || (!g[6].defined() && !g[7].defined())),
                      "a weight or a bias belongs to a norm");
    for (int i = 2; i < kGiven; ++i)
        if (g[i].defined())
            require(g[i].device() == residual.device() && type_of(g[i].scalar_type()) >= 0 &&
                        (i > 2 ? g[i].dim() == 1 && g[i].size(0) == D : residual.numel() == 0 || g[i].numel() * c.gate_rows == residual.numel()),
                    kNames[i], " must be a float32, bfloat16 or float16 tensor [", D, "] on residual's device");
}

// The struct of a call; `keep` holds the copies whose memory it names.
nmspmm_block_norm block_of(const Given& g, const Conf& c, const Tensor& total, const Tensor& out, const Tensor& stats, std::vector<Tensor>& keep)
{
    const int64_t D = g[0].size(-1);
    nmspmm_block_norm b = {};
    b.rows = g[0].numel() / D;
    b.gate_rows = c.gate_rows;
    b.ld_sum = b.ld_out = D;
    b.features = (int)D;
    auto [residual, ld_residual] = as_rows(g[0], D);
    auto [branch, ld_branch] = as_rows(g[1], D);
    b.residual = residual.const_data_ptr();
    b.ld_residual = ld_residual;
    b.branch = at_of(branch);
    b.ld_branch = ld_branch;
    keep.push_back(residual);
    keep.push_back(branch);
    b.sum = const_cast<void*>(at_of(total));
    b.out = const_cast<void*>(at_of(out));
    b.stats = static_cast<float*>(const_cast<void*>(at_of(stats)));
    const void** const data[6] = {&b.gate, &b.scale, &b.post_weight, &b.post_bias, &b.pre_weight, &b.pre_bias};
    int* const type[6] = {&b.gate_type, &b.scale_type, &b.post_weight_type, &b.post_bias_type, &b.pre_weight_type, &b.pre_bias_type};
    for (int i = 0; i < 6; ++i) {
        const Tensor& t = g[i + 2];
        if (!t.defined())
            continue;
        const Tensor whole = plain(t).contiguous();
        *data[i] = whole.const_data_ptr();
        *type[i] = type_of(whole.scalar_type());
        if (!whole.is_same(t))
            keep.push_back(whole);
    }
    b.type = type_of(c.dtype);
    b.residual_type = type_of(g[0].scalar_type());
    b.post = (int)c.post;
    b.pre = (int)c.pre;
    b.factor = (float)c.factor;
    b.eps = (float)c.eps;
    b.weight_offset = (float)c.weight_offset;
    return b;
}

// {sum, out, stats}; undefined where there is none or none is wanted.
std::array<Tensor, 3> forward_of(const Given& g, const Conf& c, bool want_stats)
{
    check_given(g, c);
    const Tensor& residual = g[0];
    const c10::DeviceGuard guard(residual.device());
    std::array<Tensor, 3> made;
    if (g[1].defined())
        made[0] = at::empty(residual.sizes(), residual.options());
    if (c.want_out)
        made[1] = at::empty(residual.sizes(), residual.options().dtype(c.dtype));
    if (want_stats)
        made[2] = at::empty({residual.numel() / residual.size(-1), 4}, residual.options().dtype(at::kFloat));
    if (residual.numel() == 0)
        return made;
    std::vector<Tensor> keep;
    const nmspmm_block_norm b = block_of(g, c, made[0], made[1], made[2], keep);
    check("nmspmm_block_norm_forward", nmspmm_block_norm_forward(&b, stream_of(residual)));
    return made;
}

// The gradients of what was given, undefined where they are not needed.
Given backward_of(const Given& g, const Conf& c, const Tensor& stats, const Tensor& grad_sum, const Tensor& grad_out,
                  const std::array<bool, kGiven>& needs)
{
    const Tensor& residual = g[0];
    const c10::DeviceGuard guard(residual.device());
    Given made;
    for (int i = 0; i < kGiven; ++i)
        if (needs[i] && g[i].defined())
            made[i] = residual.numel() == 0 ? at::zeros(g[i].sizes(), g[i].options()) : at::empty(g[i].sizes(), g[i].options());
    if (residual.numel() == 0)
        return made;
    const int64_t D = residual.size(-1);
    auto like = [&](const Tensor& t, at::ScalarType type) {
        return !t.defined() || (t.sizes() == residual.sizes() && t.scalar_type() == type && t.device() == residual.device());
    };
    require(like(grad_sum, residual.scalar_type()) && like(grad_out, c.dtype), "gradients must be like the results they belong to");
    require(stats.device() == residual.device() && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                stats.numel() == residual.numel() / D * 4, "stats must be those of the forward pass");
    check_given(g, c);
    std::vector<Tensor> keep;
    // of the forward pass's results only whether there was an `out` counts: any address stands for it
    const nmspmm_block_norm b = block_of(g, c, g[1].defined() ? residual : Tensor(), c.want_out ? stats : Tensor(), stats, keep);
    const auto [from_sum, ld_sum] = as_rows(grad_sum, D);
    const auto [from_out, ld_out] = as_rows(grad_out, D);
    auto to = [&](int i) { return const_cast<void*>(at_of(made[i])); };
    const nmspmm_block_norm_grads d = {ld_sum, ld_out, D, D, at_of(from_sum), at_of(from_out), to(0), to(1),
                                       to(2), to(3), to(4), to(5), to(6), to(7)};
    const size_t need = nmspmm_block_norm_workspace_bytes(b.rows, b.gate_rows, (int)D);
    Tensor workspace = at::empty({(int64_t)need}, residual.options().dtype(at::kByte));
    check("nmspmm_block_norm_backward", nmspmm_block_norm_backward(&b, &d, workspace.data_ptr(), need, stream_of(residual)));
    return made;
}

Given given_of(const std::vector<OptTensor>& given)
{
    require(given.size() == kGiven, "residual, branch and the six parameters");
    Given g;
    for (int i = 0; i < kGiven; ++i)
        g[i] = given[i].value_or(Tensor());
    return g;
}

std::vector<OptTensor> optional_of(const Tensor* t, int n)
{
    std::vector<OptTensor> r(n);
    for (int i = 0; i < n; ++i)
        if (t[i].defined())
            r[i] = t[i];
    return r;
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
    // an input that is not there is no variable of the node: it has no edge, and takes no number in needs_input_grad
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const OptTensor& residual, const OptTensor& branch,
                                                  const OptTensor& gate, const OptTensor& scale, const OptTensor& post_weight,
                                                  const OptTensor& post_bias, const OptTensor& pre_weight, const OptTensor& pre_bias,
                                                  const Conf& c)
    {
        const Given g = given_of({residual, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias});
        auto made = forward_of(g, c, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({g[0], g[1], g[2], g[3], g[4], g[5], g[6], g[7], made[2]});
        ctx->saved_data["conf"] = c.packed();
        // without a branch the sum is the residual, as an output of its own: its gradient comes to the same kernel
        const Tensor total = made[0].defined() ? made[0] : g[0].view_as(g[0]);
        if (!c.want_out)
            return {total};
        return {total, made[1]};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        torch::autograd::variable_list result(kGiven + 1);
        const Tensor grad_out = grads.size() > 1 ? grads[1] : Tensor();
        if (!grads[0].defined() && !grad_out.defined())
            return result;
        const auto saved = ctx->get_saved_variables();
        Given g;
        std::array<bool, kGiven> needs;
        size_t edge = 0;
        for (int i = 0; i < kGiven; ++i) {
            g[i] = saved[i];
            needs[i] = g[i].defined() && ctx->needs_input_grad(edge++);
        }
        {
            const at::AutoGradMode off(false);
            const Given made = backward_of(g, Conf::of(ctx->saved_data["conf"].toDoubleVector()), saved[kGiven], grads[0], grad_out, needs);
            for (int i = 0; i < kGiven; ++i)
                result[i] = made[i];
        }
        if (at::GradMode::is_enabled()) {       // a graph of the gradients is being made: they cannot be differentiated again
            for (int i = 0; i < kGiven; ++i)
                if (result[i].defined()) {
                    torch::autograd::variable_list one = {result[i].requires_grad_(true)};
                    auto error = std::make_shared<torch::autograd::DelayedError>("block_norm is differentiable once", 1);
                    result[i] = (*error)(std::move(one))[0];
                }
        }
        return result;
    }
};

// The gate as rows of `D`, and the consecutive rows that share one of them, for a gate that broadcasts against `shape`.
std::pair<Tensor, int64_t> gate_of(const Tensor& gate, at::IntArrayRef shape)
{
    const int64_t D = shape.back(), dims = (int64_t)shape.size();
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < dims; ++i)
        rows *= shape[i];
    if (gate.dim() == 1 && gate.size(0) == D)
        return {gate, rows};
    if (gate.dim() == dims && gate.size(-1) == D) {
        int64_t lead = 0, each = 1;
        while (lead < dims - 1 && gate.size(lead) == shape[lead])
            ++lead;
        bool ones = true;
        for (int64_t i = lead; i + 1 < dims; ++i) {
            each *= shape[i];
            ones = ones && gate.size(i) == 1;
        }
        if (ones)
            return {gate, each};
    }
    return {gate.expand(shape), 1};
}

// Nothing where the registered operators are to be called in its place.
std::optional<std::tuple<Tensor, OptTensor>> block_norm(const Tensor& residual, const OptTensor& branch, const OptTensor& gate,
                                                        const OptTensor& scale,
                                                        double factor, int64_t post, const OptTensor& post_weight, const OptTensor& post_bias,
                                                        int64_t pre, const OptTensor& pre_weight, const OptTensor& pre_bias, double eps,
                                                        double weight_offset, const std::optional<at::ScalarType>& dtype)
{
    Given g = {residual, branch.value_or(Tensor()), gate.value_or(Tensor()), scale.value_or(Tensor()), post_weight.value_or(Tensor()),
               post_bias.value_or(Tensor()), pre_weight.value_or(Tensor()), pre_bias.value_or(Tensor())};
    if (intercepted({&g[0], &g[1], &g[2], &g[3], &g[4], &g[5], &g[6], &g[7]}))
        return std::nullopt;
    require(residual.dim() >= 1 && residual.size(-1) >= 1, "rows must have 1 to 16384 features");
    Conf c;
    c.factor = factor;
    c.post = post;
    c.pre = pre;
    c.eps = eps;
    c.weight_offset = weight_offset;
    c.dtype = dtype.value_or(g[1].defined() ? g[1].scalar_type() : residual.scalar_type());
    c.want_out = pre != 0;
    const int64_t D = residual.size(-1);
    c.gate_rows = residual.numel() / D;
    if (g[2].defined()) {
        auto [rows, each] = gate_of(g[2], residual.sizes());
        g[2] = rows;
        c.gate_rows = each;
    }
    c.gate_rows = std::max<int64_t>(c.gate_rows, 1);
    if (g[3].defined() && !(g[3].dim() == 1 && g[3].size(0) == D))
        g[3] = g[3].reshape({-1}).expand({D});
    bool tracked = false;
    for (const Tensor& t : g)
        tracked = tracked || (t.defined() && t.requires_grad());
    if (tracked && at::GradMode::is_enabled()) {
        const auto o = optional_of(g.data(), kGiven);
        auto made = BlockNorm::apply(o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7], c);
        return std::make_tuple(made[0], c.want_out ? OptTensor(made[1]) : std::nullopt);
    }
    auto made = forward_of(g, c, false);
    return std::make_tuple(g[1].defined() ? made[0] : residual, c.want_out ? OptTensor(made[1]) : std::nullopt);
}

// gate_rows 0 stands for all rows, so that a recorded call takes any number of them.
Conf recorded(const Given& g, Conf c)
{
    if (c.gate_rows == 0 && g[0].defined() && g[0].dim() >= 1 && g[0].size(-1) >= 1)
        c.gate_rows = std::max<int64_t>(g[0].numel() / g[0].size(-1), 1);
    return c;
}

// The same in pieces, for the operators that tracing front ends see.
std::vector<OptTensor> block_norm_forward(const std::vector<OptTensor>& given, double factor, int64_t post, int64_t pre, double eps,
                                          double weight_offset, int64_t gate_rows, at::ScalarType dtype, bool want_out)
{
    const Given g = given_of(given);
    const auto made = forward_of(g, recorded(g, {factor, post, pre, eps, weight_offset, gate_rows, dtype, want_out}), true);
    return optional_of(made.data(), 3);
}

std::vector<OptTensor> block_norm_backward(const std::vector<OptTensor>& given, const Tensor& stats, const OptTensor& grad_sum,
                                           const OptTensor& grad_out, double factor, int64_t post, int64_t pre, double eps,
                                           double weight_offset, int64_t gate_rows, at::ScalarType dtype, bool want_out,
                                           const std::vector<bool>& needs)
{
    std::array<bool, kGiven> which;
    for (int i = 0; i < kGiven; ++i)
        which[i] = i < (int)needs.size() && needs[i];
    const Given g = given_of(given);
    const Given made = backward_of(g, recorded(g, {factor, post, pre, eps, weight_offset, gate_rows, dtype, want_out}), stats,
                                   grad_sum.value_or(Tensor()), grad_out.value_or(Tensor()), which);
    return optional_of(made.data(), kGiven);
}

} // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    // the package's exception of a failed call, handed over once (and never freed: it lives as long as the interpreter)
    static PyObject* error = nullptr;
    m.def("set_error", [](const py::object& type) { error = type.inc_ref().ptr(); });
    py::register_local_exception_translator([](std::exception_ptr p) {
        try {
            if (p)
                std::rethrow_exception(p);
        } catch (const Failure& f) {
            if (!error)
                throw;
            PyErr_SetObject(error, py::reinterpret_borrow<py::object>(error)(f.function, f.status).ptr());
        }
    });
    const py::call_guard<py::gil_scoped_release> others;
    m.def("quant_linear", &quant_linear, others);
    m.def("quant_linear_direct", &quant_linear_direct, others);
    m.def("block_norm", &block_norm, others);
    m.def("block_norm_forward", &block_norm_forward, others);
    m.def("block_norm_backward", &block_norm_backward, others);
}
