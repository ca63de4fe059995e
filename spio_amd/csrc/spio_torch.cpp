// Native call path of the package's operators (host C++, no device code): what a call of
// spio::conv2d_gw8 or spio::layernorm_2d does between the Python call and the kernel launch.
//
// The Python definitions (spio_amd/functional) register the operators with torch and carry every
// rule of them: argument checks, fake tensors, autocast, autograd, tracing.  They cost 20 us per
// inference call and 220 us per training step, several times what the kernels take at ordinary
// sizes.  The functions here run the plain case (dense GPU tensors, eager mode, no tracing or
// dispatch mode in the way) without touching Python: look up the launch plan of the shape, allocate
// the result, launch, record one autograd node.  Anything else returns NotImplemented and the
// Python definition runs, so its checks and errors are the operator's.
//
// A launch plan is made once per shape by the Python side (tuner, compiler, kernel caches) and
// holds what a launch needs.  spio_amd/native.py drops the plans whenever the kernels behind them
// may change and switches this path off while an overlay, a logger or a timer wants to see every
// launch.
#include <torch/extension.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/autocast_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <limits>
#include <memory>
#include <mutex>
#include <shared_mutex>
#include <unordered_map>

#include "spio_hip.h"
#include "spio_token_args.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr auto CL = at::MemoryFormat::ChannelsLast;

// ---- launch plans ---------------------------------------------------------------------------

enum Kind : int64_t {
    FPROP = 0, DGRAD = 1, WGRAD = 2, BGRAD = 3, NORM = 4, NORM_BWD = 5,
    GROUP_NORM = 6, GROUP_NORM_BWD = 7, ACTIVATION = 8, ACTIVATION_BWD = 9, PACK = 10, UNPACK = 11,
    CONV1D = 12, CONV1D_BWD = 13, CONV1D_SUMS = 14, CONV1D_STEP = 15, SCAN_ENDS = 16, SCAN = 17, SCAN_ENDS_BWD = 18, SCAN_BWD = 19,
    SCAN_SUMS = 20, SCAN_STEP = 21, SCAN_JOIN = 22, SCAN_JOIN_BWD = 23, ROTARY = 24, ROTARY_BWD = 25, ROTARY_SUMS = 26
};

// What selects a plan: the kind, the device and the numbers of the problem.
struct Key {
    int64_t v[12];
    bool operator==(const Key& o) const { return std::memcmp(v, o.v, sizeof v) == 0; }
};
struct KeyHash {
    size_t operator()(const Key& k) const {
        uint64_t h = 0x9e3779b97f4a7c15ull;
        for (int64_t x : k.v) {
            h ^= static_cast<uint64_t>(x);
            h *= 0xff51afd7ed558ccdull;
            h ^= h >> 32;
        }
        return h;
    }
};

struct Stage {
    void* function = nullptr;
    unsigned grid[3] = {0, 0, 0}, block[3] = {0, 0, 0}, lds = 0;
};
struct Plan {
    Stage main, second;         // `second` of two-stage kernels
    Stage second_half;          // the second stage that stores grad_weight as float16
    int64_t workspace = 0;      // bytes of partial results between the stages; element-wise: values of a workgroup
    bool present = false;       // false: the shape does not use this kind (no fused backward, no float32 output)
    bool overwrites = false;    // the kernel stores its sums whole instead of adding to them
    std::shared_ptr<PyObject> kernel;  // the Python kernel whose code object `main` and `second` point into
};
using PlanPtr = std::shared_ptr<const Plan>;

std::shared_mutex g_plans_mutex;
using Plans = std::unordered_map<Key, PlanPtr, KeyHash>;
Plans& g_plans = *new Plans;            // never destroyed: the plans hold Python objects
std::atomic<int64_t> g_bypass{1};      // > 0: every call takes the Python path
std::atomic<uint64_t> g_generation{0};  // of the plans: a plan made before a forget() is not kept
PyObject* g_make_plan = nullptr;        // Python: (key values) -> plan description

PlanPtr find_plan(const Key& key) {
    {
        std::shared_lock<std::shared_mutex> lock(g_plans_mutex);
        auto it = g_plans.find(key);
        if (it != g_plans.end()) return it->second;
    }
    const uint64_t generation = g_generation.load();
    auto plan = std::make_shared<Plan>();
    {
        // tunes and compiles on a shape's first use; its errors travel to the caller
        py::gil_scoped_acquire gil;
        py::tuple values(12);
        for (int i = 0; i < 12; ++i) values[i] = py::int_(key.v[i]);
        py::object made = py::reinterpret_borrow<py::object>(g_make_plan)(values);
        if (!made.is_none()) {
            auto t = made.cast<py::tuple>();  // (stages, workspace bytes, overwrites, kernel)
            auto stages = t[0].cast<py::list>();
            for (size_t i = 0; i < stages.size(); ++i) {
                auto s = stages[i].cast<std::vector<uint64_t>>();
                Stage& stage = i == 0 ? plan->main : i == 1 ? plan->second : plan->second_half;
                stage.function = reinterpret_cast<void*>(s[0]);
                for (int d = 0; d < 3; ++d) {
                    stage.grid[d] = static_cast<unsigned>(s[1 + d]);
                    stage.block[d] = static_cast<unsigned>(s[4 + d]);
                }
                stage.lds = static_cast<unsigned>(s[7]);
            }
            plan->workspace = t[1].cast<int64_t>();
            plan->overwrites = t[2].cast<bool>();
            plan->present = true;
            // the last owner may be a thread without the GIL
            plan->kernel = {py::object(t[3]).release().ptr(), [](PyObject* kernel) {
                                py::gil_scoped_acquire gil;
                                Py_DECREF(kernel);
                            }};
        }
    }
    std::unique_lock<std::shared_mutex> lock(g_plans_mutex);
    if (g_bypass.load() == 0 && g_generation.load() == generation) g_plans.emplace(key, plan);
    return plan;
}

void launch(const Stage& stage, hipStream_t stream, std::initializer_list<const void*> args) {
    const void* values[16];
    void* params[16];
    int n = 0;
    for (const void* a : args) {
        values[n] = a;
        params[n] = &values[n];
        ++n;
    }
    const int rc = spio_hip_launch(stage.function, stage.grid[0], stage.grid[1], stage.grid[2], stage.block[0],
                                   stage.block[1], stage.block[2], stage.lds, stream, params, n);
    TORCH_CHECK_VALUE(rc == 0, "kernel launch failed: ", spio_hip_last_error());
}

const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor empty_cl(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& like) {
    return at::detail::empty_cuda(sizes, dtype, like.device(), CL);
}
Tensor empty_1d(int64_t n, at::ScalarType dtype, const Tensor& like) {
    return at::detail::empty_cuda({n}, dtype, like.device(), std::nullopt);
}
// Clears one or two tensors (undefined: none) in one launch.
void zero(const Tensor& a, const Tensor& b, hipStream_t stream) {
    auto bytes = [](const Tensor& t) { return t.defined() ? static_cast<size_t>(t.nbytes()) : 0; };
    const int rc = spio_hip_zero_fill_pair_async(const_cast<void*>(ptr(a)), bytes(a), const_cast<void*>(ptr(b)), bytes(b), stream);
    TORCH_CHECK_VALUE(rc == 0, "zero fill failed: ", spio_hip_last_error());
}

// ---- which calls take this path -------------------------------------------------------------

// A dense GPU tensor with no wrapper, transform or lazy view on it.
bool is_plain(const Tensor& t) {
    static const c10::DispatchKeySet dense =
        c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
        c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) | c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA);
    return t.defined() && t.is_cuda() && dense.has_all(t.key_set()) && !t._fw_grad(0).defined();
}

// Eager mode: no tracing, functionalisation, transform or Python mode above the operator.
bool eager_mode() {
    static const c10::DispatchKeySet usual = c10::DispatchKeySet(c10::DispatchKey::BackendSelect) |
                                             c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView);
    return usual.has_all(c10::impl::tls_local_dispatch_key_set().included_) &&
           !at::impl::torch_function_mode_enabled();
}

// Whether a backward pass goes to the Python operators: somebody has come to see every launch, or to trace or
// transform the call, since the forward pass, or its gradients are to be differentiated (create_graph=True).
bool stands_aside(const Tensor& grad) {
    return g_bypass.load(std::memory_order_relaxed) != 0 || !eager_mode() || !is_plain(grad) || at::GradMode::is_enabled();
}

// What a profiler that records shapes is told of a call; evaluated only if one is active.
std::vector<c10::IValue> tensors(std::initializer_list<Tensor> args) {
    std::vector<c10::IValue> values;
    for (const Tensor& t : args) values.emplace_back(t);
    return values;
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

std::optional<Tensor> optional(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

struct Conv {  // the numbers of one convolution
    int64_t n, c, h, w, r, s, py, px;
    bool bias;
    int64_t p() const { return h + 2 * py - r + 1; }
    int64_t q() const { return w + 2 * px - s + 1; }
    Key key(Kind kind, int64_t device, int64_t mode = 0) const {
        return {{kind, device, n, c, h, w, r, s, py, px, bias, mode}};
    }
};

// SPIO_FUSED_BACKWARD as the Python operator reads it: 0 never, 1 whenever possible, 2 by time.
int64_t fused_mode() {
    const char* v = std::getenv("SPIO_FUSED_BACKWARD");
    if (!v) return 2;
    std::string s(v);
    const auto from = s.find_first_not_of(" \t\n");
    s = from == std::string::npos ? "" : s.substr(from, s.find_last_not_of(" \t\n") - from + 1);
    for (char& ch : s) ch = static_cast<char>(std::tolower(static_cast<unsigned char>(ch)));
    if (s == "0" || s == "false" || s == "off" || s == "no") return 0;
    if (s == "1" || s == "true" || s == "on" || s == "yes") return 1;
    return 2;
}

// ---- convolution ----------------------------------------------------------------------------

// Bits of a key's mode.  WIDE: the kernel stores its activations as float32.  HALF_WEIGHT: the caller's weights,
// and so their gradient, are float16.  READ_F32, WEIGHT_F32: it reads a float32 source (x forward, grad_output
// backward), float32 weights.  KEEP: it stores what it rounded of these as float16.
constexpr int64_t WIDE = 4, HALF_WEIGHT = 8, READ_F32 = 16, WEIGHT_F32 = 32, KEEP = 64;

// What the kernels read: float16, channels_last; the tensor itself where it is that already.
Tensor to_half_cl(const Tensor& t) {
    if (t.scalar_type() == at::kHalf) return t.is_contiguous(CL) ? t : t.contiguous(CL);
    return t.to(at::kHalf, /*non_blocking=*/false, /*copy=*/false, CL).contiguous(CL);
}
// A float32 tensor that a kernel can read as it is, in the order and with the alignment of its 16-byte loads.
bool readable_f32(const Tensor& t) {
    return t.scalar_type() == at::kFloat && t.is_contiguous(CL) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

struct ConvOutput {
    Tensor y, x, w;  // x, w: the float16 tensors that the products were taken of (wanted: `keep`)
};

// The result is in the type of `x` where the kernel has such a version, else float16, for the caller to convert.
ConvOutput conv_forward(const Conv& cv, const Tensor& x, const Tensor& w, const Tensor& bias, bool keep) {
    const auto device = x.get_device();
    hipStream_t stream = c10::hip::getCurrentHIPStream(device);
    const int64_t wide = x.scalar_type() == at::kFloat ? WIDE : 0;
    const int64_t reads = (readable_f32(x) ? READ_F32 : 0) | (readable_f32(w) ? WEIGHT_F32 : 0);
    if (reads) {
        const auto plan = find_plan(cv.key(FPROP, device, wide | reads | (keep ? KEEP : 0)));
        if (plan->present) {
            ConvOutput o;
            o.y = empty_cl({cv.n, cv.c, cv.p(), cv.q()}, wide ? at::kFloat : at::kHalf, x);
            const Tensor xr = reads & READ_F32 ? x : to_half_cl(x), wr = reads & WEIGHT_F32 ? w : to_half_cl(w);
            if (keep) {
                o.x = reads & READ_F32 ? empty_cl(x.sizes(), at::kHalf, x) : xr;
                o.w = reads & WEIGHT_F32 ? empty_cl(w.sizes(), at::kHalf, w) : wr;
                launch(plan->main, stream, {ptr(o.y), ptr(xr), ptr(wr), ptr(bias), ptr(o.x), ptr(o.w)});
            } else {
                launch(plan->main, stream, {ptr(o.y), ptr(xr), ptr(wr), ptr(bias)});
            }
            return o;
        }
    }
    ConvOutput o{Tensor(), to_half_cl(x), to_half_cl(w)};
    PlanPtr plan;
    if (wide) plan = find_plan(cv.key(FPROP, device, WIDE));
    const bool store_wide = plan && plan->present;
    if (!store_wide) plan = find_plan(cv.key(FPROP, device));
    o.y = empty_cl({cv.n, cv.c, cv.p(), cv.q()}, store_wide ? at::kFloat : at::kHalf, x);
    launch(plan->main, stream, {ptr(o.y), ptr(o.x), ptr(o.w), ptr(bias)});
    return o;
}

struct ConvGrads {
    Tensor x, w, b;
};

// The backward operator, x and w on channels_last tensors: one fused kernel where the shape uses it and
// both gradients are wanted, else the weight and the data gradient one after the other.
// `x_dtype`, `w_dtype`: what the caller's tensors are; a gradient is stored in that type where the kernel
// can (a two-stage one's grad_weight), else in the operator's and the caller converts it.
ConvGrads conv_backward(const Conv& cv, const Tensor& x, const Tensor& w, const Tensor& grad, bool need_x,
                        bool need_w, bool need_b, at::ScalarType x_dtype, at::ScalarType w_dtype) {
    ConvGrads g;
    const auto device = grad.get_device();
    hipStream_t stream = c10::hip::getCurrentHIPStream(device);
    const int64_t weight_mode = w_dtype == at::kHalf ? HALF_WEIGHT : 0;
    const bool read_f32 = readable_f32(grad);
    // grad as float16, made when a kernel that wants it comes first
    Tensor half_grad;
    auto dy = [&]() -> const Tensor& {
        if (!half_grad.defined()) half_grad = to_half_cl(grad);
        return half_grad;
    };
    // The version of a kernel for the caller's types: one whose grad_input is float32, one that reads a float32
    // grad_output (and leaves a float16 copy), where these are wanted and there is one.
    int64_t types = 0;
    auto version = [&](const PlanPtr& plan, Kind kind, int64_t mode, int64_t keep) {
        const int64_t wide = x_dtype == at::kFloat ? WIDE : 0;
        for (const int64_t t : {wide | (read_f32 ? READ_F32 | keep : 0), wide}) {
            if (t == 0) continue;
            const auto v = find_plan(cv.key(kind, device, mode | t));
            if (!v->present) continue;
            types = t;
            return v;
        }
        return plan;
    };
    auto make_grad_input = [&] { g.x = empty_cl({cv.n, cv.c, cv.h, cv.w}, types & WIDE ? at::kFloat : at::kHalf, grad); };
    // atomic kernels add into zeroed sums, two-stage ones store them whole
    auto sums = [&](const Plan& plan, bool with_bias, bool bias_is_stored) {
        g.w = empty_cl({cv.c, 8, cv.r, cv.s}, weight_mode && plan.second_half.function ? at::kHalf : at::kFloat, grad);
        if (with_bias) g.b = empty_1d(cv.c, at::kFloat, grad);
        // one launch for both: a launch is all that the fill of such small sums costs
        zero(plan.overwrites ? Tensor() : g.w, bias_is_stored ? Tensor() : g.b, stream);
    };
    auto second = [&](const Plan& plan) -> const Stage& {
        return g.w.scalar_type() == at::kHalf ? plan.second_half : plan.second;
    };
    auto data_gradient = [&](int64_t keep) {
        const auto plan = version(find_plan(cv.key(DGRAD, device)), DGRAD, 0, keep);
        make_grad_input();
        if (types & KEEP) half_grad = empty_cl(grad.sizes(), at::kHalf, grad);
        if (types & KEEP)
            launch(plan->main, stream, {ptr(g.x), ptr(grad), ptr(w), nullptr, ptr(half_grad), nullptr});
        else
            launch(plan->main, stream, {ptr(g.x), types & READ_F32 ? ptr(grad) : ptr(dy()), ptr(w), nullptr});
    };
    PlanPtr fused;
    if (need_x && need_w) {
        const int64_t mode = fused_mode();
        if (mode != 0) fused = find_plan(cv.key(BGRAD, device, mode | weight_mode));
        if (fused && !fused->present) fused.reset();
        if (fused) fused = version(fused, BGRAD, mode | weight_mode, 0);
    }
    if (fused) {
        make_grad_input();
        sums(*fused, cv.bias && need_b, fused->overwrites);
        Tensor workspace;
        if (fused->second.function) workspace = empty_1d(fused->workspace, at::kByte, grad);
        const void* dw = workspace.defined() ? ptr(workspace) : ptr(g.w);
        const void* dy_ptr = types & READ_F32 ? ptr(grad) : ptr(dy());
        if (cv.bias)
            launch(fused->main, stream, {ptr(g.x), dw, ptr(x), dy_ptr, ptr(w), ptr(g.b)});
        else
            launch(fused->main, stream, {ptr(g.x), dw, ptr(x), dy_ptr, ptr(w)});
        if (workspace.defined()) launch(second(*fused), stream, {ptr(g.w), ptr(workspace), ptr(g.b)});
    } else if (need_w) {
        // a data gradient that reads float32 goes first: it leaves the copy that the weight gradient reads
        if (need_x && read_f32) data_gradient(KEEP);
        const auto plan = find_plan(cv.key(WGRAD, device, weight_mode));
        // the second stage that stores float16 stores the bias sums as well; the other adds them with atomics
        const bool half = weight_mode && plan->second_half.function;
        sums(*plan, cv.bias && need_b, half);
        Tensor workspace;
        if (plan->second.function) workspace = empty_1d(plan->workspace, at::kByte, grad);
        const void* dw = workspace.defined() ? ptr(workspace) : ptr(g.w);
        if (cv.bias)
            launch(plan->main, stream, {dw, ptr(x), ptr(dy()), half ? nullptr : ptr(g.b)});
        else
            launch(plan->main, stream, {dw, ptr(x), ptr(dy())});
        if (half && cv.bias)
            launch(plan->second_half, stream, {ptr(g.w), ptr(workspace), ptr(g.b)});
        else if (workspace.defined())
            launch(second(*plan), stream, {ptr(g.w), ptr(workspace)});
    }
    if (need_b && !g.b.defined()) g.b = dy().sum({0, 2, 3}, /*keepdim=*/false, at::kFloat);
    if (need_x && !g.x.defined()) data_gradient(0);
    return g;
}

// Whether a saved tensor still is what the forward pass saved, up to its layout: hooks on saved tensors may
// unpack it with other strides (a copy packed into host memory, say) or elsewhere altogether.
bool is_again(const Tensor& t, const Tensor& grad, at::IntArrayRef sizes, at::ScalarType dtype = at::kHalf) {
    return is_plain(t) && t.sizes() == sizes && t.device() == grad.device() && t.scalar_type() == dtype;
}
// A float32 vector of channels.
Tensor to_float_1d(const Tensor& t) {
    if (!t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous())) return t;
    return t.to(at::kFloat).contiguous();
}

PyObject* g_backward_op = nullptr;  // the Python operator: gradients that are differentiated again

// A saved copy (`cast`) of input number `input` of the node that is running, made to depend on that input
// again: the forward pass cast it with gradients off.  What is computed from it then leads back to the input,
// by way of a node that refuses to be run, so that a gradient of it is never taken for a constant.
Tensor with_history(const Tensor& copy, bool cast, size_t input) {
    const auto node = torch::autograd::get_current_node();
    if (!cast || !node || input >= node->num_outputs() || !node->next_edge(input).is_valid()) return copy;
    Tensor t = copy.variable_data();
    torch::autograd::set_history(t, std::make_shared<torch::autograd::Error>(
        "spio::conv2d_gw8: second derivatives have no autograd formula", torch::autograd::edge_list{node->next_edge(input)}));
    return t;
}

struct ConvFunction : torch::autograd::Function<ConvFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w,
                          const std::optional<Tensor>& bias_arg, const Conv& cv) {
        const Tensor bias = bias_arg.value_or(Tensor());
        const Tensor bf = to_float_1d(bias);
        const auto [y, xh, wh] = conv_forward(cv, x, w, bf, /*keep=*/true);
        // the caller's own tensors unless their type was cast: with their history and their version, which
        // a second differentiation and a write to one of them before the backward pass are noticed by
        ctx->save_for_backward({x.scalar_type() == at::kHalf ? x : xh, w.scalar_type() == at::kHalf ? w : wh,
                                bias.defined() && bias.scalar_type() == at::kFloat ? bias : bf});
        ctx->saved_data["v"] = std::vector<int64_t>{
            cv.n, cv.c, cv.h, cv.w, cv.r, cv.s, cv.py, cv.px, cv.bias, static_cast<int64_t>(x.scalar_type()),
            static_cast<int64_t>(w.scalar_type()),
            bias.defined() ? static_cast<int64_t>(bias.scalar_type()) : static_cast<int64_t>(at::kFloat)};
        return y.to(x.scalar_type());
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto v = ctx->saved_data["v"].toIntVector();
        const Conv cv{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8] != 0};
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1];
        const bool native = !stands_aside(grads[0]) && is_again(x, grads[0], {cv.n, cv.c, cv.h, cv.w}) &&
                            is_again(w, grads[0], {cv.c, 8, cv.r, cv.s});
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1),
                   need_b = cv.bias && ctx->needs_input_grad(2);
        ConvGrads g;
        if (!native) {  // the Python operator, which refuses second derivatives and tensors it does not take
            const Tensor xa = with_history(x, v[9] != static_cast<int64_t>(at::kHalf), 0),
                         wa = with_history(w, v[10] != static_cast<int64_t>(at::kHalf), 1),
                         ba = with_history(saved[2], v[11] != static_cast<int64_t>(at::kFloat), 2);
            py::gil_scoped_acquire gil;
            py::tuple r = py::reinterpret_borrow<py::object>(g_backward_op)(
                xa, wa, ba.defined() ? py::cast(ba) : py::none(), grads[0].to(at::kHalf), cv.py, cv.px, need_x, need_w, need_b);
            auto get = [&](int i) { return r[i].is_none() ? Tensor() : r[i].cast<Tensor>(); };
            g = {get(0), get(1), get(2)};
        } else {
            RECORD_FUNCTION("spio::conv2d_gw8_backward", tensors({x, w, saved[2], grads[0]}));
            g = conv_backward(cv, to_half_cl(x), to_half_cl(w), grads[0], need_x, need_w, need_b,
                              static_cast<at::ScalarType>(v[9]), static_cast<at::ScalarType>(v[10]));
        }
        auto typed = [&](const Tensor& t, int i) {
            return t.defined() ? t.to(static_cast<at::ScalarType>(v[i])) : t;
        };
        return {typed(g.x, 9), typed(g.w, 10), typed(g.b, 11), Tensor()};
    }
};

// ---- layer norm -----------------------------------------------------------------------------

struct Norm {
    int64_t n, c, h, w;
    double eps;
    Key key(Kind kind, int64_t device, bool weight, bool bias) const {
        int64_t bits;
        std::memcpy(&bits, &eps, sizeof bits);
        return {{kind, device, n, c, h, w, bits, weight, bias, 0, 0, 0}};
    }
};

Tensor norm_forward(const Norm& nm, const Tensor& x, const Tensor& weight, const Tensor& bias) {
    const auto plan = find_plan(nm.key(NORM, x.get_device(), weight.defined(), bias.defined()));
    Tensor y = empty_cl({nm.n, nm.c, nm.h, nm.w}, at::kHalf, x);
    launch(plan->main, c10::hip::getCurrentHIPStream(x.get_device()), {ptr(y), ptr(x), ptr(weight), ptr(bias)});
    return y;
}

constexpr int64_t NORM_BACKWARD_MAX_CHANNELS = 1024;  // of the backward kernel
PyObject* g_norm_gradients = nullptr;  // Python: the gradients, by kernel or torch operations

struct NormFunction : torch::autograd::Function<NormFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight_arg,
                          const std::optional<Tensor>& bias_arg, const Norm& nm) {
        const Tensor weight = weight_arg.value_or(Tensor()), bias = bias_arg.value_or(Tensor());
        const Tensor xc = to_half_cl(x);
        Tensor y = norm_forward(nm, xc, to_float_1d(weight), to_float_1d(bias));
        ctx->save_for_backward({x, weight});  // as in ConvFunction
        ctx->saved_data["v"] = std::vector<int64_t>{
            nm.n, nm.c, nm.h, nm.w, bias.defined(),
            weight.defined() ? static_cast<int64_t>(weight.scalar_type()) : static_cast<int64_t>(at::kFloat)};
        ctx->saved_data["eps"] = nm.eps;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto v = ctx->saved_data["v"].toIntVector();
        const Norm nm{v[0], v[1], v[2], v[3], ctx->saved_data["eps"].toDouble()};
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1];
        const bool native = !stands_aside(grads[0]) && !std::getenv("SPIO_LAYERNORM_BACKWARD") &&
                            is_again(x, grads[0], {nm.n, nm.c, nm.h, nm.w}) &&
                            (!weight.defined() || is_again(weight, grads[0], {nm.c}, static_cast<at::ScalarType>(v[5])));
        // absent tensors have no edge: the bias's follows the weight's or the input's
        const bool has_weight = weight.defined();
        const bool need_x = ctx->needs_input_grad(0), need_w = has_weight && ctx->needs_input_grad(1),
                   need_b = v[4] != 0 && ctx->needs_input_grad(has_weight ? 2 : 1);
        if (!native) {
            py::gil_scoped_acquire gil;
            py::tuple r = py::reinterpret_borrow<py::object>(g_norm_gradients)(
                x, has_weight ? py::cast(weight) : py::none(), grads[0], nm.eps, need_x, need_w, need_b);
            auto get = [&](int i) { return r[i].is_none() ? Tensor() : r[i].cast<Tensor>(); };
            return {get(0), get(1), get(2), Tensor()};
        }
        RECORD_FUNCTION("spio::layernorm_2d_backward", tensors({x, grads[0], weight}));
        const Tensor dy = to_half_cl(grads[0]), xc = to_half_cl(x);
        const Tensor w = to_float_1d(weight);
        const auto device = dy.get_device();
        hipStream_t stream = c10::hip::getCurrentHIPStream(device);
        const auto plan = find_plan(nm.key(NORM_BWD, device, w.defined(), false));
        const Tensor dx = empty_cl({nm.n, nm.c, nm.h, nm.w}, at::kHalf, dy);
        const Tensor sums = at::detail::empty_cuda({2, nm.c}, at::kFloat, dy.device(), std::nullopt);
        const Tensor workspace = empty_1d(plan->workspace, at::kByte, dy);
        launch(plan->main, stream, {ptr(workspace), ptr(dx), ptr(xc), ptr(dy), ptr(w)});
        launch(plan->second, stream, {ptr(sums), ptr(workspace)});
        return {need_x ? dx : Tensor(), need_w ? sums.select(0, 0).to(weight.scalar_type()) : Tensor(),
                need_b ? sums.select(0, 1) : Tensor(), Tensor()};
    }
};

// ---- group norm, activations, the 8-bit form --------------------------------------------------------

const void* number(int64_t v) { return reinterpret_cast<const void*>(v); }  // as a kernel argument

// The numbers that the Python side has for types and activations; -1: none of them.
int64_t dtype_number(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kHalf: return 0;
        case at::kBFloat16: return 1;
        case at::kFloat: return 2;
        default: return -1;
    }
}
constexpr const char* ACTIVATIONS[4] = {"none", "relu", "silu", "gelu"};
constexpr int64_t RELU = 1;
int64_t activation_number(PyObject* o) {
    if (!PyUnicode_CheckExact(o)) return -1;
    for (int i = 0; i < 4; ++i)
        if (PyUnicode_CompareWithASCIIString(o, ACTIVATIONS[i]) == 0) return i;
    return -1;
}

// The tensor, or a copy where it does not start on 16 bytes (the kernels load that much at once).
Tensor aligned(const Tensor& t) {
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(at::MemoryFormat::Preserve);
}
Tensor empty_bytes(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& like) {
    return at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt);
}
constexpr int64_t BLOCK = 32;  // values of a block of the 8-bit form
int64_t blocks(int64_t n) { return (n + BLOCK - 1) / BLOCK; }

constexpr int64_t GROUP_NORM_MAX_CHANNELS = 4096;

struct GroupNorm {
    int64_t n, c, h, w, groups, dtype, act;
    bool kept;
    double eps;
    Key key(Kind kind, int64_t device, bool weight, bool bias) const {
        int64_t bits;
        std::memcpy(&bits, &eps, sizeof bits);
        return {{kind, device, n, c, h, w, groups, bits, dtype, act, weight * 2 + bias, kept}};
    }
    int64_t pixels() const { return h * w; }
    std::vector<int64_t> codes() const { return {n, h, w, c}; }
    std::vector<int64_t> exponents() const { return {n, h, w, blocks(c) + (act == RELU ? c / 8 : 0)}; }  // (and relu's bits)
};

struct GroupNormOutput {
    Tensor y, stats, codes, exponents;
};

GroupNormOutput group_norm_forward(const GroupNorm& gn, const Tensor& x, const Tensor& weight, const Tensor& bias,
                                   bool record) {
    const auto plan = find_plan(gn.key(GROUP_NORM, x.get_device(), weight.defined(), bias.defined()));
    hipStream_t stream = c10::hip::getCurrentHIPStream(x.get_device());
    GroupNormOutput o;
    o.y = empty_cl(x.sizes(), x.scalar_type(), x);
    if (record) o.stats = at::detail::empty_cuda({gn.n, gn.groups, 2}, at::kFloat, x.device(), std::nullopt);
    if (gn.kept) {
        o.codes = empty_bytes(gn.codes(), at::kChar, x);
        o.exponents = empty_bytes(gn.exponents(), at::kByte, x);
    }
    const void *px = number(gn.pixels()), *images = number(gn.n);
    if (!plan->second.function) {
        launch(plan->main, stream, {ptr(o.y), ptr(o.codes), ptr(o.exponents), ptr(o.stats), ptr(x), ptr(weight), ptr(bias),
                                    px, images});
    } else {
        const Tensor partials = empty_1d(plan->workspace, at::kByte, x);
        launch(plan->main, stream, {nullptr, nullptr, nullptr, ptr(partials), ptr(x), nullptr, nullptr, px, images});
        launch(plan->second, stream, {ptr(o.stats), ptr(partials), ptr(o.y), ptr(o.codes), ptr(o.exponents), ptr(x),
                                      ptr(weight), ptr(bias), px, images});
    }
    return o;
}

PyObject* g_group_norm_gradients = nullptr;  // Python: the gradients through the backward operator
PyObject* g_activation_gradient = nullptr;

// A gradient with the layout that the kernels read.
Tensor to_cl(const Tensor& t) { return aligned(t.is_contiguous(CL) ? t : t.contiguous(CL)); }

struct GroupNormFunction : torch::autograd::Function<GroupNormFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight_arg,
                          const std::optional<Tensor>& bias_arg, const GroupNorm& gn) {
        const Tensor weight = weight_arg.value_or(Tensor()), bias = bias_arg.value_or(Tensor());
        const auto o = group_norm_forward(gn, to_cl(x), to_float_1d(weight), to_float_1d(bias), /*record=*/true);
        ctx->save_for_backward({gn.kept ? o.codes : x, o.exponents, o.stats, weight, bias});
        auto type = [](const Tensor& t) { return static_cast<int64_t>(t.defined() ? t.scalar_type() : at::kFloat); };
        ctx->saved_data["v"] = std::vector<int64_t>{gn.n, gn.c, gn.h, gn.w, gn.groups, gn.dtype, gn.act, gn.kept,
                                                    type(x), type(weight), type(bias)};
        ctx->saved_data["eps"] = gn.eps;
        return o.y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto v = ctx->saved_data["v"].toIntVector();
        const GroupNorm gn{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7] != 0, ctx->saved_data["eps"].toDouble()};
        auto type = [&](int i) { return static_cast<at::ScalarType>(v[i]); };
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &exponents = saved[1], &stats = saved[2], &weight = saved[3], &bias = saved[4];
        const Tensor& dy = grads[0];
        const bool has_weight = weight.defined(), has_bias = bias.defined();
        const bool native = !stands_aside(dy) && dy.scalar_type() == type(8) && dy.sizes() == at::IntArrayRef({gn.n, gn.c, gn.h, gn.w}) &&
                            (gn.kept ? is_again(x, dy, gn.codes(), at::kChar) && is_again(exponents, dy, gn.exponents(), at::kByte)
                                     : is_again(x, dy, {gn.n, gn.c, gn.h, gn.w}, type(8))) &&
                            is_again(stats, dy, {gn.n, gn.groups, 2}, at::kFloat) &&
                            (!has_weight || is_again(weight, dy, {gn.c}, type(9))) &&
                            (!has_bias || is_again(bias, dy, {gn.c}, type(10)));
        // absent tensors have no edge (as in NormFunction)
        const bool need_x = ctx->needs_input_grad(0), need_w = has_weight && ctx->needs_input_grad(1),
                   need_b = has_bias && ctx->needs_input_grad(has_weight ? 2 : 1);
        if (!native) {
            py::gil_scoped_acquire gil;
            auto optional_py = [](const Tensor& t) { return t.defined() ? py::cast(t) : py::object(py::none()); };
            py::tuple r = py::reinterpret_borrow<py::object>(g_group_norm_gradients)(
                dy, x, optional_py(exponents), stats, gn.groups, optional_py(weight), optional_py(bias), gn.eps,
                ACTIVATIONS[gn.act], need_x, need_w, need_b);
            auto get = [&](int i) { return r[i].is_none() ? Tensor() : r[i].cast<Tensor>(); };
            return {get(0), get(1), get(2), Tensor()};
        }
        RECORD_FUNCTION("spio::group_norm_2d_backward", tensors({dy, x, exponents, stats, weight, bias}));
        const Tensor dyc = to_cl(dy);
        const Tensor xc = gn.kept ? aligned(x.contiguous()) : to_cl(x);
        const Tensor ec = exponents.defined() ? exponents.contiguous() : Tensor(), sc = stats.contiguous();
        const Tensor wf = to_float_1d(weight), bf = to_float_1d(bias);
        const auto device = dyc.get_device();
        hipStream_t stream = c10::hip::getCurrentHIPStream(device);
        const auto plan = find_plan(gn.key(GROUP_NORM_BWD, device, has_weight, has_bias));
        const Tensor dx = empty_cl(dyc.sizes(), dyc.scalar_type(), dyc);
        Tensor sums, workspace;
        if (has_weight || has_bias) sums = at::detail::empty_cuda({2, gn.c}, at::kFloat, dyc.device(), std::nullopt);
        if (plan->second.function) workspace = empty_1d(plan->workspace, at::kByte, dyc);
        const void *px = number(gn.pixels()), *images = number(gn.n);
        launch(plan->main, stream, {ptr(workspace), ptr(dx), ptr(xc), ptr(ec), ptr(dyc), ptr(sc), ptr(wf), ptr(bf), px, images});
        if (plan->overwrites)  // (images in stretches: the second launch makes grad_input)
            launch(plan->second, stream, {ptr(sums), ptr(workspace), ptr(dx), ptr(xc), ptr(ec), ptr(dyc), ptr(sc), ptr(wf),
                                          ptr(bf), px, images});
        else if (plan->second.function)
            launch(plan->second, stream, {ptr(sums), ptr(workspace), images});
        at::AutoDispatchBelowADInplaceOrView below;  // (nobody looks for a history or a base of these)
        auto row = [&](int i, at::ScalarType dtype) {
            const Tensor t = sums.select(0, i);
            return t.scalar_type() == dtype ? t : t.to(dtype);
        };
        return {need_x ? dx : Tensor(), need_w ? row(0, type(9)) : Tensor(), need_b ? row(1, type(10)) : Tensor(), Tensor()};
    }
};

// The launch of an element-wise kernel over n values.
void launch_values(const Plan& plan, int64_t n, hipStream_t stream, std::initializer_list<const void*> args) {
    Stage stage = plan.main;
    const int64_t grid = (n + plan.workspace - 1) / plan.workspace;
    TORCH_CHECK_VALUE(grid * stage.block[0] < (int64_t(1) << 32), "more workgroups than a launch can have");
    stage.grid[0] = static_cast<unsigned>(grid);
    launch(stage, stream, args);
}
Key values_key(Kind kind, const Tensor& like, int64_t dtype, int64_t act, bool kept) {
    return {{kind, like.get_device(), dtype, act, kept, 0, 0, 0, 0, 0, 0, 0}};
}
Tensor empty_as(const Tensor& t, at::ScalarType dtype) {  // sizes and strides of a tensor without gaps
    return at::detail::empty_strided_cuda(t.sizes(), t.strides(), dtype, t.device());
}
Tensor dense(const Tensor& t) { return aligned(t.is_non_overlapping_and_dense() ? t : t.contiguous()); }

struct Kept {
    Tensor codes, exponents;
};
// Bytes of codes and of exponents of n values: one a value and one a block, or, for relu, a bit a value and none.
int64_t code_bytes(int64_t n, int64_t act = 0) { return act == RELU ? (n + 7) / 8 : n; }
int64_t exponent_bytes(int64_t n, int64_t act = 0) { return act == RELU ? 0 : blocks(n); }
Kept empty_kept(const Tensor& x, int64_t act = 0) {
    return {empty_1d(code_bytes(x.numel(), act), at::kChar, x), empty_1d(exponent_bytes(x.numel(), act), at::kByte, x)};
}

// y of x, a tensor without gaps, and x in the 8-bit form where `kept` is given.
Tensor activation_forward(const Tensor& x, int64_t act, Kept* kept) {
    const auto plan = find_plan(values_key(ACTIVATION, x, dtype_number(x), act, kept != nullptr));
    const Tensor y = empty_as(x, x.scalar_type());
    if (kept) *kept = empty_kept(x, act);
    launch_values(*plan, x.numel(), c10::hip::getCurrentHIPStream(x.get_device()),
                  {ptr(y), kept ? ptr(kept->codes) : nullptr, kept ? ptr(kept->exponents) : nullptr, ptr(x), number(x.numel())});
    return y;
}

struct ActivationFunction : torch::autograd::Function<ActivationFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, int64_t act) {
        Kept kept;
        const Tensor y = activation_forward(dense(x), act, &kept);
        ctx->save_for_backward({kept.codes, kept.exponents});
        ctx->saved_data["strides"] = y.strides().vec();
        ctx->saved_data["v"] = std::vector<int64_t>{act, static_cast<int64_t>(x.scalar_type())};
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto v = ctx->saved_data["v"].toIntVector();
        const auto strides = ctx->saved_data["strides"].toIntVector();
        const auto saved = ctx->get_saved_variables();
        const Tensor &codes = saved[0], &exponents = saved[1], &grad = grads[0];
        const int64_t n = grad.numel();
        const bool native = !stands_aside(grad) && grad.scalar_type() == static_cast<at::ScalarType>(v[1]) &&
                            is_again(codes, grad, {code_bytes(n, v[0])}, at::kChar) &&
                            is_again(exponents, grad, {exponent_bytes(n, v[0])}, at::kByte);
        if (!native) {
            py::gil_scoped_acquire gil;
            return {py::reinterpret_borrow<py::object>(g_activation_gradient)(grad, codes, exponents, ACTIVATIONS[v[0]], strides)
                        .cast<Tensor>(), Tensor()};
        }
        RECORD_FUNCTION("spio::activation_8bit_backward", tensors({grad, codes, exponents}));
        Tensor dy = grad;
        if (dy.strides() != at::IntArrayRef(strides)) {
            dy = at::detail::empty_strided_cuda(grad.sizes(), strides, grad.scalar_type(), grad.device());
            dy.copy_(grad);
        }
        dy = aligned(dy);
        const Tensor cc = aligned(codes.contiguous()), ec = exponents.contiguous();
        const auto plan = find_plan(values_key(ACTIVATION_BWD, dy, dtype_number(dy), v[0], true));
        const Tensor dx = empty_as(dy, dy.scalar_type());
        launch_values(*plan, n, c10::hip::getCurrentHIPStream(dy.get_device()), {ptr(dx), ptr(cc), ptr(ec), ptr(dy), number(n)});
        return {dx, Tensor()};
    }
};

// ---- convolution with its input kept in 8 bits ----

Kept pack(const Tensor& x) {  // a tensor without gaps, on 16 bytes
    const auto plan = find_plan(values_key(PACK, x, dtype_number(x), 0, true));
    Kept kept = empty_kept(x);
    launch_values(*plan, x.numel(), c10::hip::getCurrentHIPStream(x.get_device()),
                  {ptr(kept.codes), ptr(kept.exponents), ptr(x), number(x.numel())});
    return kept;
}
void unpack(const Tensor& out, const Tensor& codes, const Tensor& exponents) {
    const Tensor cc = aligned(codes.contiguous()), ec = exponents.contiguous();
    const auto plan = find_plan(values_key(UNPACK, out, dtype_number(out), 0, true));
    launch_values(*plan, out.numel(), c10::hip::getCurrentHIPStream(out.get_device()),
                  {ptr(out), ptr(cc), ptr(ec), number(out.numel())});
}

PyObject* g_conv_kept_gradients = nullptr;  // Python: the gradients through the operators

struct ConvKeptFunction : torch::autograd::Function<ConvKeptFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w,
                          const std::optional<Tensor>& bias_arg, const Conv& cv) {
        const Tensor bias = bias_arg.value_or(Tensor());
        const auto o = conv_forward(cv, x, w, to_float_1d(bias), /*keep=*/true);
        const Kept kept = pack(aligned(o.x));
        ctx->save_for_backward({kept.codes, kept.exponents, w, bias});
        ctx->saved_data["v"] = std::vector<int64_t>{
            cv.n, cv.c, cv.h, cv.w, cv.r, cv.s, cv.py, cv.px, cv.bias, static_cast<int64_t>(x.scalar_type()),
            static_cast<int64_t>(w.scalar_type()),
            bias.defined() ? static_cast<int64_t>(bias.scalar_type()) : static_cast<int64_t>(at::kFloat)};
        return o.y.to(x.scalar_type());
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto v = ctx->saved_data["v"].toIntVector();
        const Conv cv{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8] != 0};
        auto type = [&](int i) { return static_cast<at::ScalarType>(v[i]); };
        const auto saved = ctx->get_saved_variables();
        const Tensor &codes = saved[0], &exponents = saved[1], &w = saved[2], &bias = saved[3], &grad = grads[0];
        const int64_t n = cv.n * cv.c * cv.h * cv.w;
        const bool native = !stands_aside(grad) && is_again(codes, grad, {n}, at::kChar) &&
                            is_again(exponents, grad, {blocks(n)}, at::kByte) &&
                            is_again(w, grad, {cv.c, 8, cv.r, cv.s}, type(10));
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1),
                   need_b = cv.bias && ctx->needs_input_grad(2);
        if (!native) {
            py::gil_scoped_acquire gil;
            py::tuple r = py::reinterpret_borrow<py::object>(g_conv_kept_gradients)(
                grad, codes, exponents, w, bias.defined() ? py::cast(bias) : py::object(py::none()),
                std::vector<int64_t>{cv.n, cv.c, cv.h, cv.w}, cv.py, cv.px, need_x, need_w, need_b);
            auto get = [&](int i) { return r[i].is_none() ? Tensor() : r[i].cast<Tensor>().to(type(9 + i)); };
            return {get(0), get(1), get(2), Tensor()};
        }
        RECORD_FUNCTION("spio::conv2d_gw8_backward", tensors({codes, w, bias, grad}));
        Tensor x;
        if (need_w) {
            x = empty_cl({cv.n, cv.c, cv.h, cv.w}, at::kHalf, grad);
            unpack(x, codes, exponents);
        }
        const ConvGrads g = conv_backward(cv, x, to_half_cl(w), grad, need_x, need_w, need_b, type(9), type(10));
        auto typed = [&](const Tensor& t, int i) { return t.defined() ? t.to(type(i)) : t; };
        return {typed(g.x, 9), typed(g.w, 10), typed(g.b, 11), Tensor()};
    }
};

// ---- operators over sequences of tokens -----------------------------------------------------------------

int64_t divup(int64_t n, int64_t d) { return (n + d - 1) / d; }

// The launch of a kernel that takes one structure of arguments.
void launch_structure(const Plan& plan, int64_t grid, hipStream_t stream, const void* args) {
    TORCH_CHECK_VALUE(grid * plan.main.block[0] < (int64_t(1) << 32), "more workgroups than a launch can have");
    void* params[1] = {const_cast<void*>(args)};
    const Stage& s = plan.main;
    const int rc = spio_hip_launch(s.function, static_cast<unsigned>(grid), 1, 1, s.block[0], 1, 1, s.lds, stream, params, 1);
    TORCH_CHECK_VALUE(rc == 0, "kernel launch failed: ", spio_hip_last_error());
}
Key token_key(Kind kind, int64_t device, int64_t a, int64_t b, int64_t c = 0, int64_t d = 0) {
    return {{kind, device, a, b, c, d, 0, 0, 0, 0, 0, 0}};
}
Tensor empty_of(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& like) {
    return at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt);
}
constexpr int64_t SUM_COLUMNS = 32;  // of a workgroup that adds up partial sums

// [.., values] as rows of values that are equally far apart, or a copy without gaps (functional/token_rows.py: rows_of)
struct Rows {
    Tensor t;
    int64_t row = 0;
};
Rows rows_of(const Tensor& t, int64_t step = 1) {
    if (!t.defined()) return {};
    const int64_t last = t.size(-1);
    int64_t row = last, outer = -1;  // outer: the distance that the next dimension outwards must have
    bool even = true, seen = false;
    for (int64_t i = t.dim() - 2; i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (!seen) row = t.stride(i);
        even = even && (!seen || t.stride(i) == outer);
        outer = t.size(i) * t.stride(i);
        seen = true;
    }
    const int64_t size = row * t.element_size();
    const bool fits = step == 1 ? size < 1 << 27 : size % 16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    if (even && fits && (last == 1 || t.stride(-1) == 1)) return {t, row};
    return {t.clone(at::MemoryFormat::Contiguous), last};
}
Tensor whole(const Tensor& t) { return t.defined() ? aligned(t.contiguous()) : t; }  // without gaps, on 16 bytes

// Whether the bytes from a tensor's first to its last value meet another's
bool overlap(const Tensor& a, const Tensor& b) {
    auto end = [](const Tensor& t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        return reinterpret_cast<uintptr_t>(t.data_ptr()) + (last + 1) * t.element_size();
    };
    return a.numel() && b.numel() && reinterpret_cast<uintptr_t>(a.data_ptr()) < end(b) &&
           reinterpret_cast<uintptr_t>(b.data_ptr()) < end(a);
}
bool on_16_bytes(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// Whether a state may be written to `out`: the same tensor, or one like it that shares nothing with it; nor with the inputs
bool writable_state(const Tensor& state, const Tensor& out, std::initializer_list<Tensor> inputs) {
    if (!is_plain(out) || out.sizes() != state.sizes() || out.scalar_type() != state.scalar_type() ||
        out.device() != state.device() || !state.is_contiguous() || !out.is_contiguous() || !on_16_bytes(state) ||
        !on_16_bytes(out) || (state.data_ptr() != out.data_ptr() && overlap(state, out)) || wants_grad(out) ||
        (out.is_inference() && !c10::InferenceMode::is_enabled()))
        return false;
    return std::none_of(inputs.begin(), inputs.end(), [&](const Tensor& t) { return t.defined() && overlap(t, out); });
}
// A state was written to (tensors of inference mode have no versions)
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void* mut(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return static_cast<float*>(mut(t)); }

PyObject *g_conv1d_gradients = nullptr, *g_scan_gradients = nullptr, *g_rotary_gradients = nullptr;
py::object to_py(const Tensor& t) { return t.defined() ? py::cast(t) : py::object(py::none()); }
Tensor from_py(const py::tuple& r, int i) { return r[i].is_none() ? Tensor() : r[i].cast<Tensor>(); }
int64_t type_of(const Tensor& t) { return static_cast<int64_t>(t.defined() ? t.scalar_type() : at::kFloat); }
Tensor typed(const Tensor& t, int64_t type) {
    return t.scalar_type() == static_cast<at::ScalarType>(type) ? t : t.to(static_cast<at::ScalarType>(type));
}

// ---- causal convolution ----

struct Conv1d {
    int64_t n, l, c, width, act;
    bool keep_state = false;
    Tensor before, after;  // states, which have no history
};
int64_t conv1d_slice(int64_t tokens, int64_t channels, int64_t sequences, bool backward) {
    const int64_t lanes = channels / 8 * sequences, even = divup(tokens * lanes, 1 << 17);
    if (backward) return std::max({int64_t(16), std::min(int64_t(256), even), divup(tokens * sequences, 4096)});
    return std::max(int64_t(4), std::min(int64_t(32), even));
}
PlanPtr conv1d_plan(Kind kind, const Conv1d& cv, const Tensor& x, const Tensor& weight) {
    return find_plan(token_key(kind, x.get_device(), cv.width, dtype_number(x), dtype_number(weight), cv.act));
}
Tensor conv1d_forward(Conv1d& cv, const Tensor& x, const Tensor& weight, const Tensor& bias) {
    const auto plan = conv1d_plan(CONV1D, cv, x, weight);
    const Rows rows = rows_of(x, 8);
    const Tensor w = whole(weight), b = whole(bias), before = whole(cv.before);
    const Tensor y = empty_of({cv.n, cv.l, cv.c}, x.scalar_type(), x);
    if (cv.keep_state) cv.after = empty_of({cv.n, cv.width - 1, cv.c}, x.scalar_type(), x);
    SpioConv1dArgs a = {};
    a.x = ptr(rows.t), a.weight = ptr(w), a.bias = ptr(b), a.before = ptr(before), a.out = mut(y), a.after = mut(cv.after);
    a.tokens = cv.l, a.channels = cv.c, a.sequences = cv.n, a.x_row = rows.row;
    a.slice = conv1d_slice(cv.l, cv.c, cv.n, false);
    launch_structure(*plan, divup(cv.n * divup(cv.l, a.slice) * (cv.c / 8), 256), c10::hip::getCurrentHIPStream(x.get_device()), &a);
    return y;
}

struct Conv1dFunction : torch::autograd::Function<Conv1dFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_arg,
                          Conv1d* cv) {
        const Tensor bias = bias_arg.value_or(Tensor());
        const Tensor y = conv1d_forward(*cv, x, weight, bias);
        ctx->save_for_backward({x, weight, bias, cv->before});
        ctx->saved_data["v"] = std::vector<int64_t>{cv->n, cv->l, cv->c, cv->width, cv->act, type_of(x), type_of(weight), type_of(bias)};
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto v = ctx->saved_data["v"].toIntVector();
        const Conv1d cv{v[0], v[1], v[2], v[3], v[4]};
        auto type = [&](int i) { return static_cast<at::ScalarType>(v[i]); };
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &before = saved[3], &dy = grads[0];
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1),
                   need_b = bias.defined() && ctx->needs_input_grad(2);
        const bool native = !stands_aside(dy) && is_again(dy, dy, {cv.n, cv.l, cv.c}, type(5)) &&
                            is_again(x, dy, {cv.n, cv.l, cv.c}, type(5)) && is_again(weight, dy, {cv.c, cv.width}, type(6)) &&
                            (!bias.defined() || is_again(bias, dy, {cv.c}, type(7))) &&
                            (!before.defined() || is_again(before, dy, {cv.n, cv.width - 1, cv.c}, type(5)));
        if (!native) {
            py::gil_scoped_acquire gil;
            py::tuple r = py::reinterpret_borrow<py::object>(g_conv1d_gradients)(
                dy, x, weight, to_py(bias), cv.act ? "silu" : "none", to_py(before), need_x, need_w, need_b);
            return {from_py(r, 0), from_py(r, 1), from_py(r, 2), Tensor()};
        }
        RECORD_FUNCTION("spio::causal_conv1d_backward", tensors({dy, x, weight, bias}));
        const Rows rows = rows_of(x, 8);
        const Tensor g = whole(dy), w = whole(weight), b = whole(bias), first = whole(before);
        const auto main = conv1d_plan(CONV1D_BWD, cv, x, weight), second = conv1d_plan(CONV1D_SUMS, cv, x, weight);
        const Tensor dx = empty_of(x.sizes(), x.scalar_type(), x);
        SpioConv1dArgs a = {};
        a.slice = conv1d_slice(cv.l, cv.c, cv.n, true);
        const int64_t slices = divup(cv.l, a.slice);
        const Tensor partials = empty_1d(cv.n * slices * (cv.width + 1) * cv.c, at::kFloat, x);
        const Tensor dweight = empty_of({cv.c, cv.width}, at::kFloat, x), dbias = empty_1d(cv.c, at::kFloat, x);
        a.x = ptr(rows.t), a.weight = ptr(w), a.bias = ptr(b), a.dy = ptr(g), a.before = ptr(first), a.dx = mut(dx);
        a.partials = floats(partials), a.dweight = floats(dweight), a.dbias = floats(dbias);
        a.tokens = cv.l, a.channels = cv.c, a.sequences = cv.n, a.x_row = rows.row;
        hipStream_t stream = c10::hip::getCurrentHIPStream(x.get_device());
        launch_structure(*main, divup(cv.n * slices * (cv.c / 8), 256), stream, &a);
        if (need_w || need_b) launch_structure(*second, divup((cv.width + 1) * cv.c, SUM_COLUMNS), stream, &a);
        at::AutoDispatchBelowADInplaceOrView below;
        return {need_x ? dx : Tensor(), need_w ? typed(dweight, v[6]) : Tensor(), need_b ? typed(dbias, v[7]) : Tensor(), Tensor()};
    }
};

// ---- selective scan ----

constexpr int64_t SCAN_MAX_STATES = 32, SCAN_LANES = 64;
int64_t scan_tile(int64_t states) { return states <= 8 ? 8 : 4; }
int64_t scan_chunk(int64_t tokens, int64_t channels, int64_t sequences, bool backward) {
    const int64_t waves = divup(channels, SCAN_LANES) * sequences;
    if (waves >= (backward ? 1024 : 700)) return tokens;
    int64_t chunks = 4096 / waves;
    if (tokens < 48 * chunks) chunks = std::max(int64_t(1), std::min(2048 / waves, tokens / 16));
    return divup(divup(tokens, chunks), 8) * 8;
}

struct Scan {
    int64_t n, l, c, s;
    bool softplus;
    bool keep_state = false;
    Tensor before, after;  // states, which have no history
};
// What a scan's launches share: u, delta, A, B, C, D, gate, bias in this order, as the kernels read them
struct ScanInputs {
    SpioScanArgs a = {};
    std::vector<Tensor> held;
    ScanInputs(const Scan& sc, const variable_list& t, bool backward = false) {
        auto rows = [&](int i, const void*& p, long long& row) {
            const Rows r = rows_of(t[i]);
            held.push_back(r.t);
            p = ptr(r.t), row = r.row;
        };
        auto parameter = [&](int i, const float*& p, bool to_16_bytes = false) {
            held.push_back(to_float_1d(t[i]));
            if (to_16_bytes) held.back() = aligned(held.back());
            p = floats(held.back());
        };
        rows(0, a.u, a.u_row), rows(1, a.delta, a.delta_row), rows(3, a.B, a.b_row), rows(4, a.C, a.c_row), rows(6, a.gate, a.gate_row);
        parameter(2, a.A, true), parameter(5, a.D), parameter(7, a.bias);
        a.tokens = sc.l, a.channels = sc.c, a.sequences = sc.n;
        a.chunk = scan_chunk(sc.l, sc.c, sc.n, backward);
    }
};
// (the first pass forward reads no gate; the sums and joins neither that nor time steps)
PlanPtr scan_plan(Kind kind, const Scan& sc, const Tensor& u, bool gate, bool keep = false) {
    const int64_t flags = kind == SCAN_SUMS || kind == SCAN_JOIN || kind == SCAN_JOIN_BWD ? 0 : (gate && kind != SCAN_ENDS) + 2 * sc.softplus + 4 * keep;
    return find_plan(token_key(kind, u.get_device(), sc.s, dtype_number(u), flags));
}
Tensor scan_forward(Scan& sc, const variable_list& t, Tensor* kept) {
    const Tensor& u = t[0];
    ScanInputs in(sc, t);
    const int64_t chunks = divup(sc.l, in.a.chunk), grid = sc.n * chunks * divup(sc.c, SCAN_LANES);
    hipStream_t stream = c10::hip::getCurrentHIPStream(u.get_device());
    const Tensor y = empty_of({sc.n, sc.l, sc.c}, u.scalar_type(), u);
    const Tensor before = sc.before.defined() ? sc.before.contiguous() : sc.before;
    if (sc.keep_state) sc.after = empty_of({sc.n, sc.c, sc.s}, at::kFloat, u);
    if (kept) *kept = empty_of({sc.n, divup(sc.l, scan_tile(sc.s)), sc.s, sc.c}, at::kFloat, u);
    Tensor ends;
    if (chunks > 1) ends = empty_1d(sc.n * chunks * (sc.s + 1) * sc.c, at::kFloat, u);
    in.a.before = floats(before), in.a.out = mut(y), in.a.after = floats(sc.after), in.a.ends = floats(ends);
    in.a.kept = kept ? floats(*kept) : nullptr;
    if (chunks > 1) {
        launch_structure(*scan_plan(SCAN_ENDS, sc, u, false), grid, stream, &in.a);
        launch_structure(*scan_plan(SCAN_JOIN, sc, u, false), sc.n * sc.s * divup(sc.c, SCAN_LANES), stream, &in.a);
    }
    launch_structure(*scan_plan(SCAN, sc, u, t[6].defined(), kept != nullptr), grid, stream, &in.a);
    return y;
}

struct ScanFunction : torch::autograd::Function<ScanFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B,
                          const Tensor& C, const std::optional<Tensor>& D, const std::optional<Tensor>& gate,
                          const std::optional<Tensor>& bias, Scan* sc) {
        const variable_list t = {u, delta, A, B, C, D.value_or(Tensor()), gate.value_or(Tensor()), bias.value_or(Tensor())};
        Tensor kept;
        const Tensor y = scan_forward(*sc, t, &kept);
        variable_list saved = t;
        saved.push_back(kept);
        ctx->save_for_backward(saved);
        std::vector<int64_t> v = {sc->n, sc->l, sc->c, sc->s, sc->softplus};
        for (const Tensor& one : t) v.push_back(type_of(one));
        ctx->saved_data["v"] = v;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto v = ctx->saved_data["v"].toIntVector();
        const Scan sc{v[0], v[1], v[2], v[3], v[4] != 0};
        const auto saved = ctx->get_saved_variables();
        const variable_list t(saved.begin(), saved.begin() + 8);
        const Tensor &kept = saved[8], &dy = grads[0], &u = t[0];
        const std::vector<int64_t> tensor = {sc.n, sc.l, sc.c}, row = {sc.n, sc.l, sc.s}, rate = {sc.c, sc.s}, channel = {sc.c};
        const std::vector<int64_t>* shapes[8] = {&tensor, &tensor, &rate, &row, &row, &channel, &tensor, &channel};
        bool native = !stands_aside(dy) && is_again(dy, dy, tensor, static_cast<at::ScalarType>(v[5])) &&
                      is_again(kept, dy, {sc.n, divup(sc.l, scan_tile(sc.s)), sc.s, sc.c}, at::kFloat);
        std::vector<bool> needs(8);
        int edge = 0;  // absent tensors have none
        for (int i = 0; i < 8; ++i) {
            if (!t[i].defined()) continue;
            needs[i] = ctx->needs_input_grad(edge++);
            native = native && is_again(t[i], dy, *shapes[i], static_cast<at::ScalarType>(v[5 + i]));
        }
        if (!native) {
            py::gil_scoped_acquire gil;
            py::tuple r = py::reinterpret_borrow<py::object>(g_scan_gradients)(
                dy, u, t[1], t[2], t[3], t[4], to_py(t[5]), to_py(t[6]), to_py(t[7]), sc.softplus, kept, needs);
            variable_list out;
            for (int i = 0; i < 8; ++i) out.push_back(from_py(r, i));
            out.emplace_back();
            return out;
        }
        RECORD_FUNCTION("spio::selective_scan_backward", tensors({dy, u, t[1], t[2], t[3], t[4], t[5], t[6], t[7]}));
        ScanInputs in(sc, t, true);
        const int64_t chunks = divup(sc.l, in.a.chunk), blocks = divup(sc.c, SCAN_LANES), grid = sc.n * chunks * blocks;
        hipStream_t stream = c10::hip::getCurrentHIPStream(u.get_device());
        const Tensor g = dy.contiguous(), k = kept.contiguous();
        const Tensor du = empty_of(tensor, u.scalar_type(), u), ddelta = empty_of(tensor, u.scalar_type(), u);
        const Tensor dgate = t[6].defined() ? empty_of(tensor, u.scalar_type(), u) : Tensor();
        const Tensor dB = empty_of(row, u.scalar_type(), u), dC = empty_of(row, u.scalar_type(), u);
        const Tensor dA = empty_of(rate, at::kFloat, u), dD = empty_1d(sc.c, at::kFloat, u), dbias = empty_1d(sc.c, at::kFloat, u);
        const int64_t of_tokens = sc.n * sc.l * blocks * 2 * sc.s, of_channels = sc.n * chunks * (sc.s + 2) * sc.c,
                      of_ends = chunks > 1 ? sc.n * chunks * (sc.s + 1) * sc.c : 0;
        const Tensor workspace = empty_1d(of_tokens + of_channels + of_ends, at::kFloat, u);
        in.a.dout = ptr(g), in.a.kept = floats(k), in.a.du = mut(du), in.a.ddelta = mut(ddelta);
        in.a.dgate = mut(dgate), in.a.dB = mut(dB), in.a.dC = mut(dC), in.a.dA = floats(dA), in.a.dD = floats(dD), in.a.dbias = floats(dbias);
        in.a.token_sums = floats(workspace), in.a.channel_sums = in.a.token_sums + of_tokens;
        in.a.ends = in.a.channel_sums + of_channels;
        if (chunks > 1) {
            launch_structure(*scan_plan(SCAN_ENDS_BWD, sc, u, t[6].defined()), grid, stream, &in.a);
            launch_structure(*scan_plan(SCAN_JOIN_BWD, sc, u, false), sc.n * sc.s * blocks, stream, &in.a);
        }
        launch_structure(*scan_plan(SCAN_BWD, sc, u, t[6].defined()), grid, stream, &in.a);
        launch_structure(*scan_plan(SCAN_SUMS, sc, u, false), divup(sc.n * sc.l * 2 * sc.s, 256) + divup((sc.s + 2) * sc.c, SUM_COLUMNS),
                         stream, &in.a);
        at::AutoDispatchBelowADInplaceOrView below;
        return {needs[0] ? du : Tensor(), needs[1] ? ddelta : Tensor(), needs[2] ? typed(dA, v[7]) : Tensor(),
                needs[3] ? dB : Tensor(), needs[4] ? dC : Tensor(), needs[5] ? typed(dD, v[10]) : Tensor(),
                needs[6] ? dgate : Tensor(), needs[7] ? typed(dbias, v[12]) : Tensor(), Tensor()};
    }
};

// ---- rotary positions and norms of heads ----

constexpr int64_t ROTARY_MAX_HEAD = 256, ROTARY_THREADS = 256, ROTARY_SUMMED = 512;
int64_t rotary_lanes(int64_t head, bool norm) {
    int64_t lanes = norm ? 1 : divup(head, 16);
    while (lanes * 16 < head) lanes *= 2;
    return lanes;
}
int64_t rotary_parts(int64_t tokens, int64_t heads, int64_t head, bool norm) {
    const int64_t most = divup(heads, 2);
    if (divup(tokens * rotary_lanes(head, norm), 64) * most < 256) return most;
    int64_t parts = 1;
    while (parts * 8 <= heads) parts *= 2;
    return parts;
}
int64_t rotary_grid(int64_t tokens, int64_t parts, int64_t head, bool norm, bool summed) {
    const int64_t grid = divup(tokens * parts, ROTARY_THREADS / rotary_lanes(head, norm));
    return summed ? std::min(grid, ROTARY_SUMMED) : grid;
}

struct Rotary {
    int64_t n, l, q_heads, k_heads, d;
    bool interleaved;
    double eps, scale;
    Tensor positions, frequencies;  // have no gradients
    int64_t tokens() const { return n * l; }
    std::vector<int64_t> shape(int64_t heads) const { return {n, l, heads, d}; }
    SpioRotaryArgs args(bool norm) const {
        SpioRotaryArgs a = {};
        a.positions = ptr(positions), a.frequencies = static_cast<const double*>(ptr(frequencies));
        a.tokens = tokens(), a.q_heads = q_heads, a.k_heads = k_heads, a.parts = rotary_parts(tokens(), std::max(q_heads, k_heads), d, norm), a.pairs = frequencies.numel();
        a.position_tokens = positions.numel(), a.wide_positions = positions.scalar_type() == at::kLong;
        a.eps = eps, a.scale = scale;
        return a;
    }
};
PlanPtr rotary_plan(Kind kind, const Rotary& r, const Tensor& q, bool norm) {
    return find_plan(token_key(kind, q.get_device(), r.d, dtype_number(q), norm, r.interleaved));
}
// Rows (tokens) and heads that are equally far apart and start on 16 bytes, or a copy without gaps
struct Heads {
    Tensor t;
    int64_t row, head;
};
Heads heads_of(const Tensor& t) {
    const int64_t n = t.size(0), l = t.size(1), h = t.size(2), d = t.size(3), size = t.element_size();
    const int64_t row = l != 1 ? t.stride(1) : n != 1 ? t.stride(0) : h * d, head = h != 1 ? t.stride(2) : d;
    const bool even = n == 1 || l == 1 || t.stride(0) == l * t.stride(1);
    if (even && t.stride(3) == 1 && on_16_bytes(t) && row * size % 16 == 0 && head * size % 16 == 0) return {t, row, head};
    return {t.clone(at::MemoryFormat::Contiguous), h * d, d};
}
variable_list rotary_forward(const Rotary& r, const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight) {
    const Heads qh = heads_of(q), kh = heads_of(k);
    const Tensor wq = whole(to_float_1d(q_weight)), wk = whole(to_float_1d(k_weight));
    const Tensor qo = empty_of(r.shape(r.q_heads), q.scalar_type(), q), ko = empty_of(r.shape(r.k_heads), k.scalar_type(), k);
    SpioRotaryArgs a = r.args(wq.defined());
    a.q = ptr(qh.t), a.q_row = qh.row, a.q_head = qh.head, a.k = ptr(kh.t), a.k_row = kh.row, a.k_head = kh.head;
    a.q_weight = floats(wq), a.k_weight = floats(wk), a.q_out = mut(qo), a.k_out = mut(ko);
    launch_structure(*rotary_plan(ROTARY, r, q, wq.defined()), rotary_grid(r.tokens(), a.parts, r.d, wq.defined(), false),
                     c10::hip::getCurrentHIPStream(q.get_device()), &a);
    return {qo, ko};
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const std::optional<Tensor>& q_weight,
                                 const std::optional<Tensor>& k_weight, const Rotary& r) {
        const Tensor wq = q_weight.value_or(Tensor()), wk = k_weight.value_or(Tensor());
        const bool norm = wq.defined();
        variable_list out = rotary_forward(r, q, k, wq, wk);
        ctx->set_materialize_grads(false);
        // without a norm the gradients need no inputs
        ctx->save_for_backward({norm ? q : Tensor(), norm ? k : Tensor(), wq, wk, r.positions, r.frequencies});
        ctx->saved_data["v"] = std::vector<int64_t>{r.n, r.l, r.q_heads, r.k_heads, r.d, r.interleaved, type_of(q), type_of(wq),
                                                    type_of(wk), type_of(r.positions), q.get_device()};
        ctx->saved_data["eps"] = r.eps;
        ctx->saved_data["scale"] = r.scale;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined() && !grads[1].defined()) return variable_list(5);
        const auto v = ctx->saved_data["v"].toIntVector();
        const auto saved = ctx->get_saved_variables();
        const Rotary r{v[0], v[1], v[2], v[3], v[4], v[5] != 0, ctx->saved_data["eps"].toDouble(), ctx->saved_data["scale"].toDouble(),
                       saved[4], saved[5]};
        auto type = [&](int i) { return static_cast<at::ScalarType>(v[i]); };
        const Tensor &q = saved[0], &k = saved[1], &wq = saved[2], &wk = saved[3];
        const bool norm = wq.defined();
        const auto options = at::TensorOptions().dtype(type(6)).device(at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(v[10])));
        const Tensor gq = grads[0].defined() ? grads[0] : at::zeros(r.shape(r.q_heads), options);
        const Tensor gk = grads[1].defined() ? grads[1] : at::zeros(r.shape(r.k_heads), options);
        const bool native =
            !stands_aside(gq) && !stands_aside(gk) && is_again(gq, gq, r.shape(r.q_heads), type(6)) &&
            is_again(gk, gq, r.shape(r.k_heads), type(6)) &&
            (!norm || (is_again(q, gq, r.shape(r.q_heads), type(6)) && is_again(k, gq, r.shape(r.k_heads), type(6)) &&
                       is_again(wq, gq, {r.d}, type(7)) && is_again(wk, gq, {r.d}, type(8)))) &&
            is_again(r.positions, gq, r.positions.sizes(), type(9)) && r.positions.is_contiguous() &&
            (r.positions.numel() == r.l || r.positions.numel() == r.tokens()) &&
            is_again(r.frequencies, gq, r.frequencies.sizes(), at::kDouble) && r.frequencies.is_contiguous();
        const bool needs[4] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), norm && ctx->needs_input_grad(2),
                               norm && ctx->needs_input_grad(3)};
        if (!native) {
            py::gil_scoped_acquire gil;
            py::tuple out = py::reinterpret_borrow<py::object>(g_rotary_gradients)(
                gq, gk, to_py(q), to_py(k), to_py(wq), to_py(wk), r.positions, r.frequencies, r.eps, r.interleaved, r.scale,
                std::vector<bool>(needs, needs + 4));
            return {from_py(out, 0), from_py(out, 1), from_py(out, 2), from_py(out, 3), Tensor()};
        }
        RECORD_FUNCTION("spio::head_norm_rotary_backward", tensors({gq, gk, q, k, wq, wk}));
        const Tensor gqc = whole(gq), gkc = whole(gk), wqf = whole(to_float_1d(wq)), wkf = whole(to_float_1d(wk));
        const Tensor dq = empty_of(gq.sizes(), type(6), gq), dk = empty_of(gk.sizes(), type(6), gk);
        SpioRotaryArgs a = r.args(norm);
        const int64_t grid = rotary_grid(r.tokens(), a.parts, r.d, norm, norm);
        Heads qh, kh;
        Tensor partials, dwq, dwk;
        if (norm) {
            qh = heads_of(q), kh = heads_of(k);
            a.q = ptr(qh.t), a.q_row = qh.row, a.q_head = qh.head, a.k = ptr(kh.t), a.k_row = kh.row, a.k_head = kh.head;
            partials = empty_1d(grid * 2 * r.d, at::kFloat, gq);
            dwq = empty_1d(r.d, at::kFloat, gq), dwk = empty_1d(r.d, at::kFloat, gq);
        }
        a.dq = ptr(gqc), a.dk = ptr(gkc), a.q_weight = floats(wqf), a.k_weight = floats(wkf), a.q_out = mut(dq), a.k_out = mut(dk);
        a.partials = floats(partials), a.dq_weight = floats(dwq), a.dk_weight = floats(dwk);
        hipStream_t stream = c10::hip::getCurrentHIPStream(gq.get_device());
        launch_structure(*rotary_plan(ROTARY_BWD, r, gq, norm), grid, stream, &a);
        if (needs[2] || needs[3]) {
            a.parts = grid;
            launch_structure(*rotary_plan(ROTARY_SUMS, r, gq, norm), divup(2 * r.d, SUM_COLUMNS), stream, &a);
        }
        at::AutoDispatchBelowADInplaceOrView below;
        return {needs[0] ? dq : Tensor(), needs[1] ? dk : Tensor(), needs[2] ? typed(dwq, v[7]) : Tensor(),
                needs[3] ? typed(dwk, v[8]) : Tensor(), Tensor()};
    }
};

// ---- Python boundary ------------------------------------------------------------------------

// Arguments of a Python call by position or keyword; false if they do not fit the names.
template <size_t N>
bool parse(PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames, PyObject* const (&names)[N], PyObject* (&out)[N]) {
    if (nargs > static_cast<Py_ssize_t>(N)) return false;
    for (Py_ssize_t i = 0; i < nargs; ++i) out[i] = args[i];
    const Py_ssize_t nkw = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
    for (Py_ssize_t k = 0; k < nkw; ++k) {
        PyObject* name = PyTuple_GET_ITEM(kwnames, k);
        size_t i = 0;
        while (i < N && name != names[i]) ++i;
        if (i == N) {
            i = 0;
            while (i < N && PyUnicode_Compare(name, names[i]) != 0) ++i;
        }
        if (i == N || out[i]) return false;
        out[i] = args[nargs + k];
    }
    return true;
}

bool tensor_arg(PyObject* o, Tensor* t) {
    if (!o || !THPVariable_CheckExact(o)) return false;
    *t = THPVariable_Unpack(o);
    return true;
}
bool int_arg(PyObject* o, int64_t* v) {
    if (!o) return true;
    if (!PyLong_CheckExact(o)) return false;
    int overflow = 0;
    *v = PyLong_AsLongLongAndOverflow(o, &overflow);
    return overflow == 0;
}

PyObject* not_implemented() { Py_RETURN_NOTIMPLEMENTED; }

// Paddings above this are the Python operator's to refuse: twice one near 2^63 would wrap around to a small image.
constexpr int64_t MAX_PADDING = 1 << 24;

// conv2d_gw8(inputs, weight, bias=None, stride=1, padding_y=0, padding_x=0, dilation=1, groups=1), with `Function` for calls
// whose gradients are recorded
template <class Function>
PyObject* convolution(PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames, const char* name) {
    static PyObject* const names[8] = {
        PyUnicode_InternFromString("inputs"),    PyUnicode_InternFromString("weight"),
        PyUnicode_InternFromString("bias"),      PyUnicode_InternFromString("stride"),
        PyUnicode_InternFromString("padding_y"), PyUnicode_InternFromString("padding_x"),
        PyUnicode_InternFromString("dilation"),  PyUnicode_InternFromString("groups")};
    if (g_bypass.load(std::memory_order_relaxed) != 0 || !eager_mode()) return not_implemented();
    PyObject* a[8] = {};
    if (!parse(args, nargs, kwnames, names, a)) return not_implemented();
    Tensor x, w, bias;
    int64_t stride = 1, py = 0, px = 0, dilation = 1, groups = 1;
    if (!tensor_arg(a[0], &x) || !tensor_arg(a[1], &w) || (a[2] && a[2] != Py_None && !tensor_arg(a[2], &bias)) ||
        !int_arg(a[3], &stride) || !int_arg(a[4], &py) || !int_arg(a[5], &px) || !int_arg(a[6], &dilation) ||
        !int_arg(a[7], &groups))
        return not_implemented();
    if (!is_plain(x) || !is_plain(w) || x.dim() != 4 || w.dim() != 4 || w.device() != x.device())
        return not_implemented();
    if (bias.defined() && (!is_plain(bias) || bias.dim() != 1 || bias.device() != x.device() || bias.size(0) != w.size(0)))
        return not_implemented();
    const Conv cv{x.size(0), x.size(1), x.size(2), x.size(3), w.size(2), w.size(3), py, px, bias.defined()};
    if (stride != 1 || dilation != 1 || groups != cv.c / 8 || cv.c % 8 || w.size(0) != cv.c || w.size(1) != 8 || py < 0 ||
        px < 0 || py > MAX_PADDING || px > MAX_PADDING || cv.r < 1 || cv.r > 7 || cv.s < 1 || cv.s > 7 || cv.n < 1 ||
        cv.c < 8 || cv.h < 1 || cv.w < 1 || cv.p() < 1 || cv.q() < 1)
        return not_implemented();
    const bool autocast = at::autocast::is_autocast_enabled(at::kCUDA);
    auto floating = [](const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf; };
    if (autocast) {  // any of the two types is cast to what the kernels take; others are the Python operator's
        if (!floating(x) || !floating(w) || (bias.defined() && !floating(bias))) return not_implemented();
    } else if (x.scalar_type() != at::kHalf || w.scalar_type() != at::kHalf ||
               (bias.defined() && bias.scalar_type() != at::kFloat)) {
        return not_implemented();
    }
    Tensor y;
    {
        py::gil_scoped_release no_gil;
        c10::DeviceGuard device(x.device());
        RECORD_FUNCTION(name, tensors({x, w, bias}));
        // the casts and copies inside are the operator's own, whatever autocast thinks of them
        c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
        if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(bias))) {
            y = Function::apply(x, w, optional(bias), cv);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            y = conv_forward(cv, x, w, to_float_1d(bias), /*keep=*/false).y.to(x.scalar_type());
        }
    }
    return THPVariable_Wrap(y);
}
PyObject* conv2d_gw8(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    return convolution<ConvFunction>(args, nargs, kwnames, "spio::conv2d_gw8");
    END_HANDLE_TH_ERRORS
}
// The same with its input kept in 8 bits
PyObject* conv2d_gw8_8bit(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    return convolution<ConvKeptFunction>(args, nargs, kwnames, "spio::conv2d_gw8_8bit_forward");
    END_HANDLE_TH_ERRORS
}

// layernorm_2d(inputs, weight=None, bias=None, eps=1e-6)
PyObject* layernorm_2d(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    static PyObject* const names[4] = {PyUnicode_InternFromString("inputs"), PyUnicode_InternFromString("weight"),
                                       PyUnicode_InternFromString("bias"), PyUnicode_InternFromString("eps")};
    if (g_bypass.load(std::memory_order_relaxed) != 0 || !eager_mode()) return not_implemented();
    PyObject* a[4] = {};
    if (!parse(args, nargs, kwnames, names, a)) return not_implemented();
    Tensor x, weight, bias;
    if (!tensor_arg(a[0], &x) || (a[1] && a[1] != Py_None && !tensor_arg(a[1], &weight)) ||
        (a[2] && a[2] != Py_None && !tensor_arg(a[2], &bias)) || (a[3] && !PyFloat_CheckExact(a[3])))
        return not_implemented();
    if (!is_plain(x) || x.dim() != 4 || x.scalar_type() != at::kHalf) return not_implemented();
    const Norm nm{x.size(0), x.size(1), x.size(2), x.size(3), a[3] ? PyFloat_AS_DOUBLE(a[3]) : 1e-6};
    for (const Tensor& t : {weight, bias})
        if (t.defined() && (!is_plain(t) || t.dim() != 1 || t.size(0) != nm.c || t.device() != x.device() ||
                            (t.scalar_type() != at::kFloat && t.scalar_type() != at::kHalf)))
            return not_implemented();
    if (nm.n < 1 || nm.h < 1 || nm.w < 1 || nm.c < 8 || nm.c % 8 || !(nm.eps > 0)) return not_implemented();
    const bool record = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias));
    // the backward pass by torch operations is the Python operator's
    if (record && nm.c > NORM_BACKWARD_MAX_CHANNELS) return not_implemented();
    Tensor y;
    {
        py::gil_scoped_release no_gil;
        c10::DeviceGuard device(x.device());
        RECORD_FUNCTION("spio::layernorm_2d", tensors({x, weight, bias}));
        if (record) {
            y = NormFunction::apply(x, optional(weight), optional(bias), nm);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            y = norm_forward(nm, to_half_cl(x), to_float_1d(weight), to_float_1d(bias));
        }
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// group_norm_2d(inputs, num_groups, weight=None, bias=None, eps=1e-5, activation="none", checkpoint_8bit=False)
PyObject* group_norm_2d(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    static PyObject* const names[7] = {
        PyUnicode_InternFromString("inputs"), PyUnicode_InternFromString("num_groups"), PyUnicode_InternFromString("weight"),
        PyUnicode_InternFromString("bias"), PyUnicode_InternFromString("eps"), PyUnicode_InternFromString("activation"),
        PyUnicode_InternFromString("checkpoint_8bit")};
    if (g_bypass.load(std::memory_order_relaxed) != 0 || !eager_mode()) return not_implemented();
    PyObject* a[7] = {};
    if (!parse(args, nargs, kwnames, names, a)) return not_implemented();
    Tensor x, weight, bias;
    int64_t groups = 0;
    if (!tensor_arg(a[0], &x) || !a[1] || !int_arg(a[1], &groups) || (a[2] && a[2] != Py_None && !tensor_arg(a[2], &weight)) ||
        (a[3] && a[3] != Py_None && !tensor_arg(a[3], &bias)) || (a[4] && !PyFloat_CheckExact(a[4])) || (a[6] && !PyBool_Check(a[6])))
        return not_implemented();
    if (!is_plain(x) || x.dim() != 4 || dtype_number(x) < 0) return not_implemented();
    GroupNorm gn{x.size(0), x.size(1), x.size(2), x.size(3), groups, dtype_number(x), a[5] ? activation_number(a[5]) : 0,
                 a[6] == Py_True, a[4] ? PyFloat_AS_DOUBLE(a[4]) : 1e-5};
    for (const Tensor& t : {weight, bias})
        if (t.defined() && (!is_plain(t) || t.dim() != 1 || t.size(0) != gn.c || t.device() != x.device() || dtype_number(t) < 0))
            return not_implemented();
    if (gn.n < 1 || gn.h < 1 || gn.w < 1 || gn.c < 8 || gn.c % 8 || gn.c > GROUP_NORM_MAX_CHANNELS || groups < 1 ||
        gn.c % groups || gn.act < 0 || !(gn.eps > 0) || gn.eps > std::numeric_limits<double>::max())
        return not_implemented();
    const bool record = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias));
    gn.kept = gn.kept && record;
    Tensor y;
    {
        py::gil_scoped_release no_gil;
        c10::DeviceGuard device(x.device());
        RECORD_FUNCTION("spio::group_norm_2d_forward", tensors({x, weight, bias}));
        if (record) {
            y = GroupNormFunction::apply(x, optional(weight), optional(bias), gn);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            y = group_norm_forward(gn, to_cl(x), to_float_1d(weight), to_float_1d(bias), /*record=*/false).y;
        }
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// activation_8bit(inputs, activation="gelu")
PyObject* activation_8bit(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    static PyObject* const names[2] = {PyUnicode_InternFromString("inputs"), PyUnicode_InternFromString("activation")};
    if (g_bypass.load(std::memory_order_relaxed) != 0 || !eager_mode()) return not_implemented();
    PyObject* a[2] = {};
    Tensor x;
    if (!parse(args, nargs, kwnames, names, a) || !tensor_arg(a[0], &x)) return not_implemented();
    const int64_t act = a[1] ? activation_number(a[1]) : 3;
    if (!is_plain(x) || dtype_number(x) < 0 || act < 1 || x.numel() == 0) return not_implemented();
    Tensor y;
    {
        py::gil_scoped_release no_gil;
        c10::DeviceGuard device(x.device());
        RECORD_FUNCTION("spio::activation_8bit_forward", tensors({x}));
        if (at::GradMode::is_enabled() && x.requires_grad()) {
            y = ActivationFunction::apply(x, act);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            y = activation_forward(dense(x), act, nullptr);
        }
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// pack_8bit(inputs): (codes, exponents) of a tensor without gaps
PyObject* pack_8bit(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    if (g_bypass.load(std::memory_order_relaxed) != 0 || !eager_mode() || nargs != 1 || kwnames) return not_implemented();
    Tensor x;
    if (!tensor_arg(args[0], &x) || !is_plain(x) || dtype_number(x) < 0 || x.numel() == 0 || !x.is_non_overlapping_and_dense())
        return not_implemented();
    Kept kept;
    {
        py::gil_scoped_release no_gil;
        c10::DeviceGuard device(x.device());
        at::AutoDispatchBelowADInplaceOrView below;
        RECORD_FUNCTION("spio::pack_8bit", tensors({x}));
        kept = pack(aligned(x));
    }
    return py::make_tuple(kept.codes, kept.exponents).release().ptr();
    END_HANDLE_TH_ERRORS
}

// A tuple of integers, at most 16.
bool ints_arg(PyObject* o, std::vector<int64_t>* v) {
    if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) > 16) return false;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(o); ++i) {
        int64_t item = 0;
        if (!int_arg(PyTuple_GET_ITEM(o, i), &item) || item < 0) return false;
        v->push_back(item);
    }
    return true;
}

// unpack_8bit(codes, exponents, shape, strides, dtype)
PyObject* unpack_8bit(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    if (g_bypass.load(std::memory_order_relaxed) != 0 || !eager_mode() || nargs != 5 || kwnames) return not_implemented();
    Tensor codes, exponents;
    std::vector<int64_t> shape, strides;
    if (!tensor_arg(args[0], &codes) || !tensor_arg(args[1], &exponents) || !ints_arg(args[2], &shape) ||
        !ints_arg(args[3], &strides) || !THPDtype_Check(args[4]) || shape.size() != strides.size())
        return not_implemented();
    const at::ScalarType dtype = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    const int64_t n = codes.numel();
    if (!is_plain(codes) || !is_plain(exponents) || codes.dim() != 1 || exponents.dim() != 1 || n == 0 ||
        codes.scalar_type() != at::kChar || exponents.scalar_type() != at::kByte || exponents.device() != codes.device() ||
        exponents.numel() != blocks(n) || (dtype != at::kHalf && dtype != at::kBFloat16 && dtype != at::kFloat))
        return not_implemented();
    int64_t count = 1;
    for (int64_t size : shape) {
        if (size < 1 || count > n / size) return not_implemented();
        count *= size;
    }
    if (count != n) return not_implemented();
    Tensor out;
    bool dense_strides = true;
    {
        py::gil_scoped_release no_gil;
        c10::DeviceGuard device(codes.device());
        at::AutoDispatchBelowADInplaceOrView below;
        std::vector<size_t> order;
        for (size_t i = 0; i < shape.size(); ++i)
            if (shape[i] != 1) order.push_back(i);
        std::sort(order.begin(), order.end(), [&](size_t i, size_t j) { return strides[i] < strides[j]; });
        int64_t expected = 1;
        for (size_t i : order) {
            dense_strides = dense_strides && strides[i] == expected;
            expected *= shape[i];
        }
        if (dense_strides) {
            RECORD_FUNCTION("spio::unpack_8bit", tensors({codes, exponents}));
            out = at::detail::empty_strided_cuda(shape, strides, dtype, codes.device());
            unpack(out, codes, exponents);
        }
    }
    if (!dense_strides) return not_implemented();
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// What the functions below are called with: positional arguments, by the functions of spio_amd/functional, in their order.
bool optional_tensor(PyObject* o, Tensor* t) { return o == Py_None || tensor_arg(o, t); }
bool number_arg(PyObject* o, double* v) {
    if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
    *v = PyFloat_AsDouble(o);
    if (*v == -1.0 && PyErr_Occurred()) {  // an integer that no float64 is near
        PyErr_Clear();
        return false;
    }
    return true;
}
bool bool_arg(PyObject* o, bool* v) {
    *v = o == Py_True;
    return PyBool_Check(o);
}
bool ready(Py_ssize_t nargs, Py_ssize_t expected, PyObject* kwnames) {
    return g_bypass.load(std::memory_order_relaxed) == 0 && eager_mode() && nargs == expected && !kwnames;
}
// A plain tensor of that shape, on the device of `like`; with `typed` of its type, too, else of one of the three
bool fits(const Tensor& t, const Tensor& like, at::IntArrayRef sizes, bool typed) {
    return is_plain(t) && t.sizes() == sizes && t.device() == like.device() &&
           (typed ? t.scalar_type() == like.scalar_type() : dtype_number(t) >= 0);
}
bool absent_or_fits(const Tensor& t, const Tensor& like, at::IntArrayRef sizes, bool typed) {
    return !t.defined() || fits(t, like, sizes, typed);
}
bool state_fits(const Tensor& t, const Tensor& like, at::IntArrayRef sizes, at::ScalarType dtype) {
    return !t.defined() || (is_plain(t) && t.sizes() == sizes && t.device() == like.device() && t.scalar_type() == dtype);
}
PyObject* with_state(const Tensor& y, const Tensor& state) {
    return state.defined() ? py::make_tuple(y, state).release().ptr() : THPVariable_Wrap(y);
}
constexpr int64_t CONV1D_MIN_WIDTH = 2, CONV1D_MAX_WIDTH = 8;

// Whether weight and bias are what the convolution's kernels read; `act`: its number
bool conv1d_fits(PyObject* activation, const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t* act) {
    *act = activation_number(activation);
    const int64_t c = x.size(-1);
    return (*act == 0 || *act == 2) && dtype_number(x) >= 0 && c > 0 && c % 8 == 0 && is_plain(weight) && weight.dim() == 2 &&
           weight.size(1) >= CONV1D_MIN_WIDTH && weight.size(1) <= CONV1D_MAX_WIDTH &&
           fits(weight, x, {c, weight.size(1)}, false) && absent_or_fits(bias, x, {c}, false) &&
           (!bias.defined() || bias.scalar_type() == weight.scalar_type());
}

// causal_conv1d(inputs, weight, bias, activation, initial_state, return_state)
PyObject* causal_conv1d(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    if (!ready(nargs, 6, kwnames)) return not_implemented();
    Tensor x, weight, bias;
    Conv1d cv{};
    if (!tensor_arg(args[0], &x) || !tensor_arg(args[1], &weight) || !optional_tensor(args[2], &bias) ||
        !optional_tensor(args[4], &cv.before) || !bool_arg(args[5], &cv.keep_state))
        return not_implemented();
    if (!is_plain(x) || x.dim() != 3 || x.numel() == 0 || !conv1d_fits(args[3], x, weight, bias, &cv.act)) return not_implemented();
    cv.n = x.size(0), cv.l = x.size(1), cv.c = x.size(2), cv.width = weight.size(1);
    if (!state_fits(cv.before, x, {cv.n, cv.width - 1, cv.c}, x.scalar_type())) return not_implemented();
    const bool grad = at::GradMode::is_enabled();
    if (grad && wants_grad(cv.before)) return not_implemented();
    Tensor y;
    {
        py::gil_scoped_release no_gil;
        c10::DeviceGuard device(x.device());
        RECORD_FUNCTION("spio::causal_conv1d_forward", tensors({x, weight, bias, cv.before}));
        c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
        if (grad && (wants_grad(x) || wants_grad(weight) || wants_grad(bias))) {
            y = Conv1dFunction::apply(x, weight, optional(bias), &cv);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            y = conv1d_forward(cv, x, weight, bias);
        }
    }
    return with_state(y, cv.after);
    END_HANDLE_TH_ERRORS
}

// causal_conv1d_step(inputs, state, weight, bias, activation, out_state)
PyObject* causal_conv1d_step(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    if (!ready(nargs, 6, kwnames)) return not_implemented();
    Tensor x, weight, bias, after;
    Conv1d cv{};
    if (!tensor_arg(args[0], &x) || !tensor_arg(args[1], &cv.before) || !tensor_arg(args[2], &weight) ||
        !optional_tensor(args[3], &bias) || !tensor_arg(args[5], &after))
        return not_implemented();
    if (!is_plain(x) || x.dim() != 2 || x.numel() == 0 || !conv1d_fits(args[4], x, weight, bias, &cv.act)) return not_implemented();
    cv.n = x.size(0), cv.l = 1, cv.c = x.size(1), cv.width = weight.size(1);
    if (!state_fits(cv.before, x, {cv.n, cv.width - 1, cv.c}, x.scalar_type()) || !writable_state(cv.before, after, {x}))
        return not_implemented();
    Tensor y;
    {
        py::gil_scoped_release no_gil;
        c10::DeviceGuard device(x.device());
        RECORD_FUNCTION("spio::causal_conv1d_step", tensors({x, cv.before, weight, bias}));
        at::AutoDispatchBelowADInplaceOrView below;
        const Rows rows = rows_of(x, 8);
        const Tensor w = whole(weight), b = whole(bias);
        const auto plan = conv1d_plan(CONV1D_STEP, cv, x, weight);
        y = empty_of({cv.n, cv.c}, x.scalar_type(), x);
        SpioConv1dArgs a = {};
        a.x = ptr(rows.t), a.weight = ptr(w), a.bias = ptr(b), a.before = ptr(cv.before), a.out = mut(y), a.after = mut(after);
        a.tokens = a.slice = 1, a.channels = cv.c, a.sequences = cv.n, a.x_row = rows.row;
        launch_structure(*plan, divup(cv.n * (cv.c / 8), 64), c10::hip::getCurrentHIPStream(x.get_device()), &a);
        written(after);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// Shapes and types of a scan's tensors: u, delta, A, B, C, D, gate, bias
bool scan_fits(const variable_list& t) {
    const Tensor &u = t[0], &A = t[2];
    if (dtype_number(u) < 0 || u.numel() == 0 || !is_plain(A) || A.dim() != 2 || A.size(1) < 1 || A.size(1) > SCAN_MAX_STATES)
        return false;
    std::vector<int64_t> row = u.sizes().vec();
    const int64_t c = row.back();
    if (c >= 1 << 24) return false;
    row.back() = A.size(1);
    return fits(t[1], u, u.sizes(), true) && fits(A, u, {c, A.size(1)}, false) && fits(t[3], u, row, true) &&
           fits(t[4], u, row, true) && absent_or_fits(t[5], u, {c}, false) && absent_or_fits(t[6], u, u.sizes(), true) &&
           absent_or_fits(t[7], u, {c}, false);
}
bool scan_tensors(PyObject* const* args, const int (&at)[8], variable_list* t) {
    t->resize(8);
    for (int i = 0; i < 8; ++i)
        if (!(i < 5 ? tensor_arg(args[at[i]], &(*t)[i]) : optional_tensor(args[at[i]], &(*t)[i]))) return false;
    return is_plain((*t)[0]);
}

// selective_scan(inputs, delta, A, B, C, D, gate, delta_bias, delta_softplus, initial_state, return_state)
PyObject* selective_scan(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    if (!ready(nargs, 11, kwnames)) return not_implemented();
    variable_list t;
    Scan sc{};
    if (!scan_tensors(args, {0, 1, 2, 3, 4, 5, 6, 7}, &t) || !bool_arg(args[8], &sc.softplus) ||
        !optional_tensor(args[9], &sc.before) || !bool_arg(args[10], &sc.keep_state))
        return not_implemented();
    const Tensor& u = t[0];
    if (u.dim() != 3 || u.size(1) >= int64_t(1) << 30 || !scan_fits(t)) return not_implemented();
    sc.n = u.size(0), sc.l = u.size(1), sc.c = u.size(2), sc.s = t[2].size(1);
    if (!state_fits(sc.before, u, {sc.n, sc.c, sc.s}, at::kFloat)) return not_implemented();
    const bool grad = at::GradMode::is_enabled();
    if (grad && wants_grad(sc.before)) return not_implemented();
    Tensor y;
    {
        py::gil_scoped_release no_gil;
        c10::DeviceGuard device(u.device());
        RECORD_FUNCTION("spio::selective_scan_forward", tensors({u, t[1], t[2], t[3], t[4], t[5], t[6], t[7], sc.before}));
        c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
        if (grad && std::any_of(t.begin(), t.end(), wants_grad)) {
            y = ScanFunction::apply(u, t[1], t[2], t[3], t[4], optional(t[5]), optional(t[6]), optional(t[7]), &sc);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            y = scan_forward(sc, t, nullptr);
        }
    }
    return with_state(y, sc.after);
    END_HANDLE_TH_ERRORS
}

// selective_scan_step(inputs, state, delta, A, B, C, D, gate, delta_bias, delta_softplus, out_state)
PyObject* selective_scan_step(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    if (!ready(nargs, 11, kwnames)) return not_implemented();
    variable_list t;
    Tensor after;
    Scan sc{};
    if (!scan_tensors(args, {0, 2, 3, 4, 5, 6, 7, 8}, &t) || !tensor_arg(args[1], &sc.before) || !bool_arg(args[9], &sc.softplus) ||
        !tensor_arg(args[10], &after))
        return not_implemented();
    const Tensor& u = t[0];
    if (u.dim() != 2 || !scan_fits(t)) return not_implemented();
    sc.n = u.size(0), sc.l = 1, sc.c = u.size(1), sc.s = t[2].size(1);
    if (!state_fits(sc.before, u, {sc.n, sc.c, sc.s}, at::kFloat) || !writable_state(sc.before, after, {u, t[1], t[3], t[4], t[6]}))
        return not_implemented();
    Tensor y;
    {
        py::gil_scoped_release no_gil;
        c10::DeviceGuard device(u.device());
        RECORD_FUNCTION("spio::selective_scan_step", tensors({u, sc.before, t[1], t[2], t[3], t[4], t[5], t[6], t[7]}));
        at::AutoDispatchBelowADInplaceOrView below;
        ScanInputs in(sc, t);
        const auto plan = scan_plan(SCAN_STEP, sc, u, t[6].defined());
        y = empty_of({sc.n, sc.c}, u.scalar_type(), u);
        in.a.before = floats(sc.before), in.a.out = mut(y), in.a.after = floats(after);
        const int64_t lanes = sc.s <= 4 ? 1 : sc.s <= 8 ? 2 : sc.s <= 16 ? 4 : 8;
        launch_structure(*plan, divup(sc.n * sc.c * lanes, 256), c10::hip::getCurrentHIPStream(u.get_device()), &in.a);
        written(after);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// head_norm_rotary(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, scale); without weights no norm
PyObject* head_norm_rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
    HANDLE_TH_ERRORS
    if (!ready(nargs, 9, kwnames)) return not_implemented();
    Tensor q, k, wq, wk;
    Rotary r{};
    if (!tensor_arg(args[0], &q) || !tensor_arg(args[1], &k) || !optional_tensor(args[2], &wq) || !optional_tensor(args[3], &wk) ||
        !tensor_arg(args[4], &r.positions) || !tensor_arg(args[5], &r.frequencies) || !number_arg(args[6], &r.eps) ||
        !bool_arg(args[7], &r.interleaved) || !number_arg(args[8], &r.scale))
        return not_implemented();
    if (!is_plain(q) || q.dim() != 4 || dtype_number(q) < 0 || !is_plain(k) || k.dim() != 4) return not_implemented();
    r.n = q.size(0), r.l = q.size(1), r.q_heads = q.size(2), r.k_heads = k.size(2), r.d = q.size(3);
    const int64_t pairs = is_plain(r.frequencies) && r.frequencies.dim() == 1 ? r.frequencies.size(0) : 0;
    if (q.numel() == 0 || k.numel() == 0 || r.tokens() * std::max(r.q_heads, r.k_heads) >= int64_t(1) << 31 ||
        !fits(k, q, r.shape(r.k_heads), true) || r.d % 8 || r.d > ROTARY_MAX_HEAD ||
        wq.defined() != wk.defined() || !absent_or_fits(wq, q, {r.d}, false) || !absent_or_fits(wk, q, {r.d}, false) ||
        !(r.eps > 0) || r.eps > std::numeric_limits<double>::max() || !(std::fabs(r.scale) <= std::numeric_limits<float>::max()) || pairs < 1 || 2 * pairs > r.d ||
        (!r.interleaved && pairs % 8) || r.frequencies.scalar_type() != at::kDouble || wants_grad(r.frequencies) || r.frequencies.device() != q.device() ||
        !is_plain(r.positions) || (r.positions.scalar_type() != at::kLong && r.positions.scalar_type() != at::kInt) ||
        r.positions.device() != q.device() ||
        !(r.positions.sizes() == at::IntArrayRef({r.l}) || r.positions.sizes() == at::IntArrayRef({r.n, r.l})))
        return not_implemented();
    variable_list out;
    {
        py::gil_scoped_release no_gil;
        c10::DeviceGuard device(q.device());
        RECORD_FUNCTION("spio::head_norm_rotary_forward", tensors({q, k, wq, wk, r.positions, r.frequencies}));
        c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
        r.positions = r.positions.contiguous(), r.frequencies = r.frequencies.contiguous();
        if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(wq) || wants_grad(wk))) {
            out = RotaryFunction::apply(q, k, optional(wq), optional(wk), r);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            out = rotary_forward(r, q, k, wq, wk);
        }
    }
    return py::make_tuple(out[0], out[1]).release().ptr();
    END_HANDLE_TH_ERRORS
}

PyMethodDef g_methods[] = {
    {"causal_conv1d", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(causal_conv1d)),
     METH_FASTCALL | METH_KEYWORDS, "causal_conv1d on plain GPU tensors, else NotImplemented"},
    {"causal_conv1d_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(causal_conv1d_step)),
     METH_FASTCALL | METH_KEYWORDS, "causal_conv1d_step on plain GPU tensors, else NotImplemented"},
    {"selective_scan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(selective_scan)),
     METH_FASTCALL | METH_KEYWORDS, "selective_scan on plain GPU tensors, else NotImplemented"},
    {"selective_scan_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(selective_scan_step)),
     METH_FASTCALL | METH_KEYWORDS, "selective_scan_step on plain GPU tensors, else NotImplemented"},
    {"head_norm_rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(head_norm_rotary)),
     METH_FASTCALL | METH_KEYWORDS, "head_norm_rotary on plain GPU tensors, else NotImplemented"},
    {"group_norm_2d", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(group_norm_2d)),
     METH_FASTCALL | METH_KEYWORDS, "group_norm_2d on plain GPU tensors, else NotImplemented"},
    {"activation_8bit", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(activation_8bit)),
     METH_FASTCALL | METH_KEYWORDS, "activation_8bit on plain GPU tensors, else NotImplemented"},
    {"conv2d_gw8_8bit", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(conv2d_gw8_8bit)),
     METH_FASTCALL | METH_KEYWORDS, "conv2d_gw8 with its input kept in 8 bits on plain GPU tensors, else NotImplemented"},
    {"pack_8bit", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(pack_8bit)), METH_FASTCALL | METH_KEYWORDS,
     "codes and exponents of a plain GPU tensor without gaps, else NotImplemented"},
    {"unpack_8bit", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(unpack_8bit)), METH_FASTCALL | METH_KEYWORDS,
     "the tensor of codes, exponents, shape, strides and type, else NotImplemented"},
    {"layernorm_2d", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layernorm_2d)),
     METH_FASTCALL | METH_KEYWORDS, "spio::layernorm_2d on plain GPU tensors, else NotImplemented"},
    {"conv2d_gw8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(conv2d_gw8)),
     METH_FASTCALL | METH_KEYWORDS, "spio::conv2d_gw8 on plain GPU tensors, else NotImplemented"},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

// Found in the built file by spio_amd/build.py.
#define SPIO_TEXT_(x) #x
#define SPIO_TEXT(x) SPIO_TEXT_(x)

PYBIND11_MODULE(_native, m) {
    m.attr("built_from") = "spio-built-from:" SPIO_TEXT(SPIO_BUILT_FROM);
    m.attr("WIDE") = WIDE;
    m.attr("HALF_WEIGHT") = HALF_WEIGHT;
    m.attr("READ_F32") = READ_F32;
    m.attr("WEIGHT_F32") = WEIGHT_F32;
    m.attr("KEEP") = KEEP;
    m.def("configure", [](py::object make_plan, py::object backward_op, py::object norm_gradients) {
        g_make_plan = make_plan.release().ptr();
        g_backward_op = backward_op.release().ptr();
        g_norm_gradients = norm_gradients.release().ptr();
    });
    m.def("configure_kept", [](py::object group_norm_gradients, py::object activation_gradient, py::object conv_gradients) {
        g_group_norm_gradients = group_norm_gradients.release().ptr();
        g_activation_gradient = activation_gradient.release().ptr();
        g_conv_kept_gradients = conv_gradients.release().ptr();
    });
    m.def("configure_tokens", [](py::object conv1d_gradients, py::object scan_gradients, py::object rotary_gradients) {
        g_conv1d_gradients = conv1d_gradients.release().ptr();
        g_scan_gradients = scan_gradients.release().ptr();
        g_rotary_gradients = rotary_gradients.release().ptr();
    });
    // how work over sequences of tokens is cut, which kernels/*_kernel.py compute as well
    m.def("conv1d_slice", &conv1d_slice);
    m.def("scan_chunk", &scan_chunk);
    m.def("scan_tile", &scan_tile);
    m.def("rotary_parts", &rotary_parts);
    m.def("rotary_grid", &rotary_grid);
    m.def("bypass", [](int64_t change) { g_bypass.fetch_add(change); });
    m.def("forget", [] {
        g_generation.fetch_add(1);
        Plans dropped;  // destroyed behind the lock: a kernel that goes with its plan runs Python code
        std::unique_lock<std::shared_mutex> lock(g_plans_mutex);
        dropped.swap(g_plans);
    });
    m.def("plans", [] {
        std::shared_lock<std::shared_mutex> lock(g_plans_mutex);
        return g_plans.size();
    });
    PyModule_AddFunctions(m.ptr(), g_methods);
}
