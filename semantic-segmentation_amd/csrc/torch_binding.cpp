// Python binding of the class-score and gradient-norm operators: argument checks, output tensors, autograd and launches in C++.
//
// These calls are made once per training step or per request on small tensors as often as on large ones, and a launch takes the GPU
// less time than Python needs to describe it: looking at a list of 500 gradients took 180 us in Python against 125 us of kernels,
// and a forward and backward pass through a Python autograd function 140 us against 30 us.  The kernels stay behind the C ABI of
// include/dsaspp.h; the addresses of its functions come from the Python side, which has loaded the library.  No HIP header is needed:
// the current stream is handed in as its handle, and a backward pass runs on the stream of its forward pass, as autograd arranges.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>
#include <vector>

#include "dsaspp.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

#ifndef DSASPP_BINDING_HASH
#define DSASPP_BINDING_HASH "unknown"
#endif
const char g_hash[] = "DSASPP_BIND=" DSASPP_BINDING_HASH;

constexpr int64_t MAX_PIECES = 1 << 16;
constexpr int64_t MAX_CLASSES_UPSAMPLED = 32;

struct Api {
    int (*scores_fwd)(const dsaspp_scores_desc*, dsaspp_stream_t);
    int (*scores_bwd)(const dsaspp_scores_desc*, dsaspp_stream_t);
    int64_t (*scores_workspace)(const dsaspp_scores_desc*);
    int64_t (*scores8_workspace)(const dsaspp_scores8_desc*);
    int (*scores8_fwd)(const dsaspp_scores8_desc*, dsaspp_stream_t);
    int (*scores8_bwd)(const dsaspp_scores8_desc*, dsaspp_stream_t);
    int64_t (*grad_norm_workspace)(const dsaspp_clip_desc*);
    int (*grad_ranges_overlap)(const dsaspp_clip_desc*);
    int (*grad_norm_partials)(const dsaspp_clip_desc*, dsaspp_stream_t);
    int (*grad_norm_finish)(const dsaspp_clip_desc*, dsaspp_stream_t);
    int (*clip_scale)(const dsaspp_clip_desc*, dsaspp_stream_t);
    int (*clip_grads)(const dsaspp_clip_desc*, dsaspp_stream_t);
    int (*adam_step_clipped)(const dsaspp_adam_clip_desc*, const dsaspp_clip_desc*, dsaspp_stream_t);
    const char* (*last_error)(void);
} api;

std::string text(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
std::string text(const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return buf;
}
#define VALUE_CHECK(cond, ...) \
    if (!(cond)) throw py::value_error(text(__VA_ARGS__))
#define TYPE_CHECK(cond, ...) \
    if (!(cond)) throw py::type_error(text(__VA_ARGS__))

void call(int rc) {
    if (rc != 0) throw std::runtime_error(api.last_error());
}

std::string shape_text(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + (s.size() == 1 ? ",)" : ")");
}

int dtype_code(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kFloat ? 1 : t == at::kHalf ? 2 : -1; }
std::string dtype_name(const Tensor& t) {
    std::string s = c10::toString(t.scalar_type());        // "Double" and the like
    return s == "Double" ? "float64" : s == "Long" ? "int64" : s == "Int" ? "int32" : s;
}
template <typename T>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
dsaspp_stream_t handle(int64_t stream) { return reinterpret_cast<dsaspp_stream_t>(stream); }

// The results below are new tensors filled by kernels of which torch knows nothing: a trace would record the empty tensors alone, and a
// tangent would be dropped without a word.
void no_trace(const char* who) {
    if (torch::jit::tracer::getTracingState()) throw std::runtime_error(text("%s cannot be traced: a trace does not hold its kernels", who));
}
void no_tangent(const Tensor& t, const char* who) {
    if (t.defined() && t._fw_grad(0).defined()) throw std::runtime_error(text("%s has no forward-mode derivative, but was given a dual tensor", who));
}

// ---------------------------------------------------------------- class scores
struct Plan : torch::CustomClassHolder {
    int64_t n, c, ignore_index, stream = 0;
    int top_k, upsample;
    bool entropy, empty;
    std::vector<int64_t> rows;            // of labels, logp and entropy
    Tensor labels;
};

c10::intrusive_ptr<Plan> make_plan(at::IntArrayRef shape, at::Device device, const OptTensor& labels, int64_t top_k, int64_t ignore_index, bool entropy,
                                   int64_t upsample) {
    VALUE_CHECK(device.is_cuda(), "label_scores needs logits on a GPU");
    VALUE_CHECK(upsample == 1 || upsample == 8, "upsample must be 1 or 8, got %lld", (long long)upsample);
    const bool up = upsample == 8;
    VALUE_CHECK(shape.size() >= 2 && (!up || shape.size() == 4), "logits must be N x C x ...%s, got %s", up ? " (N x C x h x w with upsample=8)" : "",
                shape_text(shape).c_str());
    auto p = c10::make_intrusive<Plan>();
    p->n = shape[0];
    p->c = shape[1];
    VALUE_CHECK(p->c >= 1 && p->c < (1 << 30) && (!up || p->c <= MAX_CLASSES_UPSAMPLED), "%lld classes: at least one%s", (long long)p->c,
                up ? ", at most 32 with upsample=8" : "");
    // before the narrowing to the descriptor's 32 bits, which would make another picture of it
    VALUE_CHECK(!up || (p->n < (1ll << 31) && shape[2] < (1 << 20) && shape[3] < (1 << 20)), "logits of shape %s are too large for upsample=8: pictures below 2^20 x 2^20, "
                "fewer than 2^31", shape_text(shape).c_str());
    VALUE_CHECK(top_k >= 0 && top_k <= std::min<int64_t>(DSASPP_SCORES_MAX_TOP, p->c), "top_k must be in [0, %d] and at most the %lld classes, got %lld",
                DSASPP_SCORES_MAX_TOP, (long long)p->c, (long long)top_k);
    VALUE_CHECK(labels.has_value() || entropy || top_k, "nothing to compute: no labels, no entropy, top_k = 0");
    p->rows.assign(1, p->n);
    for (size_t i = 2; i < shape.size(); ++i) p->rows.push_back(up ? 8 * shape[i] : shape[i]);
    if (labels.has_value()) {
        VALUE_CHECK(labels->scalar_type() == at::kLong && labels->sizes() == at::IntArrayRef(p->rows) && labels->device() == device,
                    "labels must be an int64 tensor of shape %s on the device of the logits", shape_text(p->rows).c_str());
        p->labels = labels->contiguous().resolve_neg();
    }
    p->top_k = (int)top_k;
    p->ignore_index = ignore_index;
    p->entropy = entropy;
    p->upsample = (int)upsample;
    p->empty = std::find(shape.begin(), shape.end(), 0) != shape.end();
    return p;
}

// Row dimensions (without the classes) merged into at most three (size, stride) pairs, the first of them dimension 0 by itself.
bool row_strides(at::IntArrayRef sizes, at::IntArrayRef strides, int64_t (&n)[3], int64_t (&st)[3]) {
    n[0] = sizes[0];
    st[0] = strides[0];
    n[1] = n[2] = 1;
    st[1] = st[2] = 0;
    std::vector<std::pair<int64_t, int64_t>> rest;
    for (size_t i = 2; i < sizes.size(); ++i) {
        if (sizes[i] == 1) continue;
        if (!rest.empty() && rest.back().second == sizes[i] * strides[i]) rest.back() = {rest.back().first * sizes[i], strides[i]};
        else rest.emplace_back(sizes[i], strides[i]);
    }
    if (rest.size() > 2) return false;
    for (size_t k = 0; k < rest.size(); ++k) {
        n[3 - rest.size() + k] = rest[k].first;
        st[3 - rest.size() + k] = rest[k].second;
    }
    return true;
}

// The logits as the kernels of both passes read them: themselves, unless
//  - the rows are scattered over more than three strides;
//  - few rows have many classes that do not lie side by side.  A lane walks the classes of a row then, and a lane per row leaves the GPU idle: one
//    row of 21841 classes, every second element, 2671 us against 17 with the copy, 16 pixels of 50257 class planes 6494 against 18 (its backward
//    pass 10 ms).  16384 pixels of 1024 and 4096 planes 115 and 470 against 91 and 355; 256 planes of 1024 pixels 22 against 15.
constexpr int64_t COPY_CLASSES = 512, COPY_ROWS = 16384;
Tensor readable(const Tensor& logits, const Plan& p) {
    int64_t n[3], st[3];
    if (p.upsample != 1 || p.empty) return logits;
    if (p.c >= COPY_CLASSES && logits.stride(1) != 1 && logits.numel() <= COPY_ROWS * p.c) return logits.movedim(1, -1).contiguous().movedim(-1, 1);
    return row_strides(logits.sizes(), logits.strides(), n, st) ? logits : logits.contiguous();
}

void fill(dsaspp_scores_desc& d, const Plan& p, const Tensor& logits) {
    int64_t n[3], st[3];
    row_strides(logits.sizes(), logits.strides(), n, st);
    d.d0 = n[0]; d.d1 = n[1]; d.d2 = n[2];
    d.s0 = st[0]; d.s1 = st[1]; d.s2 = st[2];
    d.sc = logits.stride(1);
}
void fill(dsaspp_scores8_desc& d, const Plan& p, const Tensor& logits) {
    d.n_img = (int32_t)p.n;
    d.h = (int32_t)logits.size(2);
    d.w = (int32_t)logits.size(3);
    d.sn = logits.stride(0); d.sc = logits.stride(1); d.sy = logits.stride(2); d.sx = logits.stride(3);
}
template <typename D>
void fill_common(D& d, const Plan& p, const Tensor& logits) {
    fill(d, p, logits);
    d.dtype = dtype_code(logits.scalar_type());
    d.n_class = (int32_t)p.c;
    d.top_k = p.top_k;
    d.logits = logits.data_ptr();
    d.labels = ptr<int64_t>(p.labels);
    d.ignore_index = p.ignore_index;
}

struct Out { Tensor logp, entropy, top_logp, top_class, stats; };

Out scores_forward(const Plan& p, const Tensor& given, bool need_stats) {
    const c10::DeviceGuard guard(given.device());
    const Tensor logits = readable(given, p);
    const auto f32 = at::TensorOptions().dtype(at::kFloat).device(logits.device());
    Out o;
    if (p.labels.defined()) o.logp = at::empty(p.rows, f32);
    if (p.entropy) o.entropy = at::empty(p.rows, f32);
    if (p.top_k) {
        std::vector<int64_t> shape = p.rows;
        shape.insert(shape.begin() + 1, p.top_k);
        o.top_logp = at::empty(shape, f32);
        o.top_class = at::empty(shape, f32.dtype(at::kLong));
    }
    if (need_stats) {
        std::vector<int64_t> shape = p.rows;
        if (p.upsample == 1) shape.push_back(2);
        o.stats = at::empty(shape, f32);
    }
    if (p.empty) return o;
    auto outputs = [&](auto& d) {
        d.logp = ptr<float>(o.logp);
        d.entropy = ptr<float>(o.entropy);
        d.top_logp = ptr<float>(o.top_logp);
        d.top_class = ptr<int64_t>(o.top_class);
        d.stats = ptr<float>(o.stats);
    };
    if (p.upsample == 8) {
        dsaspp_scores8_desc d = {};
        fill_common(d, p, logits);
        outputs(d);
        call(api.scores8_fwd(&d, handle(p.stream)));
    } else {
        dsaspp_scores_desc d = {};
        fill_common(d, p, logits);
        outputs(d);
        const int64_t need = api.scores_workspace(&d);
        if (need < 0) call(1);
        Tensor ws;
        if (need) ws = at::empty({need}, f32);
        d.ws = ptr<float>(ws);
        d.ws_len = need;
        call(api.scores_fwd(&d, handle(p.stream)));
    }
    return o;
}

// An upstream gradient for the kernels: dense, or one value for all (what sum() and mean() send back).
Tensor upstream(const Tensor& g, const float*& at, int32_t& one) {
    if (!g.defined()) return g;
    no_tangent(g, "the backward pass of label_scores");
    Tensor t = (g.scalar_type() == at::kFloat ? g : g.to(at::kFloat)).resolve_neg();
    one = 1;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.stride(i) != 0 && t.size(i) != 1) one = 0;
    if (!one) t = t.contiguous();
    at = ptr<float>(t);
    return t;
}

// Gradient of the logits in their shape and type, dense in the order that the kernels write; `out` receives it instead (upsample=8).
Tensor scores_backward(const Plan& p, const Tensor& given, const Tensor& stats, const Tensor& entropy, const Tensor& top_class, const Tensor& g_logp,
                       const Tensor& g_entropy, const Tensor& g_top, Tensor out) {
    const c10::DeviceGuard guard(given.device());
    const Tensor logits = readable(given, p);
    auto classes_last = [&]() {
        std::vector<int64_t> shape(logits.sizes().begin(), logits.sizes().end());
        shape.erase(shape.begin() + 1);
        shape.push_back(p.c);
        return at::empty(shape, logits.options()).movedim(-1, 1);
    };
    auto inputs = [&](auto& d, Tensor (&up)[3]) {
        fill_common(d, p, logits);
        d.entropy = ptr<float>(entropy);
        d.top_class = ptr<int64_t>(top_class);
        d.stats = ptr<float>(stats);
        up[0] = upstream(g_logp, d.g_logp, d.g_logp_one);
        up[1] = upstream(g_entropy, d.g_entropy, d.g_entropy_one);
        up[2] = upstream(g_top, d.g_top, d.g_top_one);
    };
    Tensor up[3];                         // alive until the launch; freed in the order of the stream
    const bool none = !g_logp.defined() && !g_entropy.defined() && !g_top.defined();
    if (!out.defined()) out = logits.stride(1) == 1 || p.c == 1 ? classes_last() : at::empty(logits.sizes(), logits.options());
    if (p.empty) return out;
    if (none) return out.zero_();
    if (p.upsample == 8) {
        dsaspp_scores8_desc d = {};
        inputs(d, up);
        d.dlogits = out.data_ptr();
        d.g_dtype = dtype_code(out.scalar_type());
        d.gn = out.stride(0); d.gc = out.stride(1); d.gy = out.stride(2); d.gx = out.stride(3);
        const int64_t need = api.scores8_workspace(&d);
        if (need < 0) call(1);
        const Tensor ws = at::empty({need}, logits.options().dtype(at::kFloat));
        d.ws = ptr<float>(ws);
        d.ws_len = need;
        call(api.scores8_bwd(&d, handle(p.stream)));
    } else {
        dsaspp_scores_desc d = {};
        inputs(d, up);
        d.dlogits = out.data_ptr();
        call(api.scores_bwd(&d, handle(p.stream)));
    }
    return out;
}

// The result of a backward pass that autograd was asked to differentiate again (create_graph): an error if that happens.
Tensor differentiable_once(Tensor g) {
    if (!at::GradMode::is_enabled()) return g;
    Tensor v = g.detach();
    v.set_requires_grad(true);
    auto err = std::make_shared<torch::autograd::DelayedError>("label_scores: trying to differentiate twice, its backward pass has no derivative", 1);
    return (*err)(torch::autograd::variable_list{v})[0];
}

// A leaf's gradient accumulator keeps the stream of the oldest live graph that reaches it.  If that is not the stream being captured,
// handing it a gradient would pull a stream that is not captured into the graph, which ends the process: refused here, before it happens.
void check_capture(const Tensor& logits) {
    if (!logits.is_leaf() || !logits.requires_grad()) return;
    const auto acc = torch::autograd::impl::try_get_grad_accumulator(logits);
    const auto stream = acc ? acc->stream() : std::nullopt;
    if (!stream || *stream == c10::impl::VirtualGuardImpl(logits.device().type()).getStream(logits.device())) return;
    const c10::DeviceGuard guard(logits.device());
    const py::gil_scoped_acquire gil;
    if (py::module_::import("torch.cuda").attr("is_current_stream_capturing")().cast<bool>())
        throw std::runtime_error("label_scores: a backward pass is captured while a graph made on another stream still holds the same logits: "
                                 "drop that graph first, or detach the logits for the capture");
}

struct LabelScores : torch::autograd::Function<LabelScores> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits, c10::intrusive_ptr<Plan> plan) {
        const Out o = scores_forward(*plan, logits, true);
        ctx->set_materialize_grads(false);
        // the labels too: autograd then notices if any of them is overwritten before the backward pass
        ctx->save_for_backward({logits, o.stats, o.entropy, o.top_class, plan->labels});
        ctx->saved_data["plan"] = c10::IValue::make_capsule(plan);
        torch::autograd::variable_list outs;
        for (const Tensor& t : {o.logp, o.entropy, o.top_logp, o.top_class})
            if (t.defined()) outs.push_back(t);
        if (o.top_class.defined()) ctx->mark_non_differentiable({o.top_class});
        return outs;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        const auto saved = ctx->get_saved_variables();
        check_capture(saved[0]);
        const auto holder = ctx->saved_data["plan"].toCapsule();
        const Plan& p = *static_cast<Plan*>(holder.get());
        size_t k = 0;
        const Tensor g_logp = p.labels.defined() ? g[k++] : Tensor(), g_entropy = p.entropy ? g[k++] : Tensor(), g_top = p.top_k ? g[k++] : Tensor();
        Tensor out;
        {
            at::NoGradGuard no_grad;
            out = scores_backward(p, saved[0], saved[1], saved[2], saved[3], g_logp, g_entropy, g_top, Tensor());
        }
        return {differentiable_once(out), Tensor()};
    }
};

py::object opt(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }

py::tuple label_scores(const Tensor& given, const OptTensor& labels, int64_t top_k, int64_t ignore_index, bool entropy, int64_t upsample, int64_t stream) {
    no_trace("label_scores");
    no_tangent(given, "label_scores");
    TYPE_CHECK(dtype_code(given.scalar_type()) >= 0 && given.layout() == at::kStrided, "logits must be a float32, bfloat16 or float16 tensor, got %s",
               dtype_name(given).c_str());
    const Tensor logits = given.resolve_neg();        // itself, unless it is a view that torch negates when it is read
    auto p = make_plan(logits.sizes(), logits.device(), labels, top_k, ignore_index, entropy, upsample);
    p->stream = stream;
    Out o;
    if (at::GradMode::is_enabled() && logits.requires_grad()) {
        const auto outs = LabelScores::apply(logits, p);
        size_t k = 0;
        if (p->labels.defined()) o.logp = outs[k++];
        if (entropy) o.entropy = outs[k++];
        if (top_k) { o.top_logp = outs[k++]; o.top_class = outs[k++]; }
    } else {
        at::NoGradGuard no_grad;
        o = scores_forward(*p, logits.detach(), false);
    }
    return py::make_tuple(opt(o.logp), opt(o.entropy), opt(o.top_logp), opt(o.top_class));
}

void check_image(const Tensor& x) {
    no_trace("DenseASPP.score");
    no_tangent(x, "DenseASPP.score");
}

void check_scores(const std::vector<int64_t>& shape, const std::string& device, const OptTensor& labels, int64_t top_k, bool entropy, int64_t upsample) {
    make_plan(shape, at::Device(device), labels, top_k, 0, entropy, upsample);
}

// The two halves of DenseASPP.score, whose logits and gradient live in the engine's buffers.
py::tuple upsampled_forward(const Tensor& low, const OptTensor& labels, int64_t top_k, int64_t ignore_index, bool entropy, bool stats, int64_t stream) {
    at::NoGradGuard no_grad;
    auto p = make_plan(low.sizes(), low.device(), labels, top_k, ignore_index, entropy, 8);
    p->stream = stream;
    const Out o = scores_forward(*p, low, stats);
    return py::make_tuple(opt(o.logp), opt(o.entropy), opt(o.top_logp), opt(o.top_class), opt(o.stats));
}
void upsampled_backward(const Tensor& low, const OptTensor& labels, int64_t ignore_index, const Tensor& stats, const OptTensor& entropy,
                        const OptTensor& top_class, const OptTensor& g_logp, const OptTensor& g_entropy, const OptTensor& g_top, const Tensor& out, int64_t stream) {
    at::NoGradGuard no_grad;
    auto p = make_plan(low.sizes(), low.device(), labels, top_class.has_value() ? top_class->size(1) : 0, ignore_index, true, 8);
    p->stream = stream;
    auto t = [](const OptTensor& x) { return x.has_value() ? *x : Tensor(); };
    scores_backward(*p, low, stats, t(entropy), t(top_class), t(g_logp), t(g_entropy), t(g_top), out);
}

// ---------------------------------------------------------------- gradient norm
// The dense pieces of a tensor whose elements do not fill one piece of memory: its dimensions are merged from the innermost stride
// outwards as far as they are contiguous, the rest is walked (expanded ones over and over).
void add_pieces(const Tensor& t, int code, std::vector<dsaspp_grad_range>& out) {
    std::vector<std::pair<int64_t, int64_t>> dims;       // (stride, size)
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) != 1) dims.emplace_back(t.stride(i), t.size(i));
    std::sort(dims.begin(), dims.end(), [](auto& a, auto& b) { return std::make_pair(a.first == 0, a.first) < std::make_pair(b.first == 0, b.first); });
    int64_t run = 1, pieces = 1;
    size_t i = 0;
    for (; i < dims.size() && dims[i].first == run; ++i) run *= dims[i].second;
    for (size_t k = i; k < dims.size(); ++k) {
        pieces *= dims[k].second;
        VALUE_CHECK(pieces <= MAX_PIECES, "a gradient of shape %s and strides %s lies in more than %lld separate pieces: make it contiguous",
                    shape_text(t.sizes()).c_str(), shape_text(t.strides()).c_str(), (long long)MAX_PIECES);
    }
    char* base = static_cast<char*>(t.data_ptr());
    for (int64_t piece = 0; piece < pieces; ++piece) {
        int64_t off = 0, rest = piece;
        for (size_t k = i; k < dims.size(); ++k) {
            off += rest % dims[k].second * dims[k].first;
            rest /= dims[k].second;
        }
        out.push_back({base + off * t.element_size(), run, code, 0});
    }
}

struct Grads {
    std::vector<dsaspp_grad_range> ranges;
    std::vector<const Tensor*> tensors;
    dsaspp_clip_desc d = {};
    Tensor ws, norm;
    at::Device device = at::kCPU;

    void add(const Tensor& t, const char* who) {
        no_tangent(t, who);
        const int code = dtype_code(t.scalar_type());
        TYPE_CHECK(t.layout() == at::kStrided && code >= 0, "%s needs dense float32, bfloat16 or float16 gradients, got %s%s", who, dtype_name(t).c_str(),
                   t.layout() == at::kStrided ? "" : " in another layout");
        if (tensors.empty()) device = t.device();
        VALUE_CHECK(t.is_cuda() && t.device() == device, "%s: the gradients must be on one GPU, got %s and %s", who, device.str().c_str(),
                    t.device().str().c_str());
        tensors.push_back(&t);
        if (t.numel() == 0) return;
        if (t.is_contiguous() || t.is_non_overlapping_and_dense()) ranges.push_back({t.data_ptr(), t.numel(), code, 0});
        else add_pieces(t, code, ranges);
    }
    void set_norm_type(double type, const char* who) {
        VALUE_CHECK(type == 2.0 || (std::isinf(type) && type > 0), "%s: norm_type must be 2 or inf, got %g", who, type);
        d.norm_type = type == 2.0 ? 2 : 0;
    }
    void ready(bool in_place, const char* who) {
        d.ranges = ranges.data();
        d.n_ranges = (int32_t)ranges.size();
        if (d.scale == 0.f) d.scale = 1.f;
        if (in_place) {
            const int o = api.grad_ranges_overlap(&d);
            VALUE_CHECK(o != 1, "%s: two gradients (or two elements of one) share memory: each would be scaled twice", who);
            if (o) call(1);
        }
        const int64_t need = api.grad_norm_workspace(&d);
        if (need < 0) call(1);
        // from the caching allocator for this call: two calls, streams or captured graphs never share a workspace
        const auto on = at::TensorOptions().device(device);
        ws = at::empty({need}, on.dtype(at::kDouble));
        norm = at::empty({}, on.dtype(at::kFloat));
        d.ws = ptr<double>(ws);
        d.ws_len = need;
        d.norm = ptr<float>(norm);
    }
};

void written(const Tensor& t) {           // as torch's own in-place operations tell autograd
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The gradients of a Python list: the tensors themselves, or the .grad of parameters that have one.
Grads gather(const py::list& list, bool of_parameters, const char* who) {
    no_trace(who);
    Grads g;
    const size_t n = list.size();
    g.ranges.reserve(n);
    g.tensors.reserve(n);
    for (size_t i = 0; i < n; ++i) {
        PyObject* o = PyList_GET_ITEM(list.ptr(), (Py_ssize_t)i);
        TYPE_CHECK(THPVariable_Check(o), "%s needs tensors, got %s", who, Py_TYPE(o)->tp_name);
        const Tensor& t = THPVariable_Unpack(o);
        if (!of_parameters) g.add(t, who);
        else if (t.grad().defined()) g.add(t.grad(), who);
    }
    return g;
}

Tensor grad_norm(const py::list& grads, double norm_type, int64_t stream) {
    Grads g = gather(grads, false, "grad_norm");
    g.set_norm_type(norm_type, "grad_norm");
    if (g.tensors.empty()) return at::zeros({}, at::kFloat);
    const c10::DeviceGuard guard(g.device);
    g.ready(false, "grad_norm");
    call(api.grad_norm_partials(&g.d, handle(stream)));
    call(api.grad_norm_finish(&g.d, handle(stream)));
    return g.norm;
}

Tensor clip_grads(const py::list& grads, bool of_parameters, double max_norm, double norm_type, bool error_if_nonfinite, int64_t stream) {
    const char* who = of_parameters ? "clip_grad_norm_" : "clip_grads_";
    VALUE_CHECK(max_norm >= 0.0, "%s: max_norm must be >= 0, got %g", who, max_norm);
    Grads g = gather(grads, of_parameters, who);
    g.set_norm_type(norm_type, who);
    if (g.tensors.empty()) return at::zeros({}, at::kFloat);
    for (const Tensor* t : g.tensors)
        VALUE_CHECK(!t->requires_grad(), "%s writes plain gradient tensors in place; a tensor that requires grad is not one (pass p.grad, or use "
                    "clip_grad_norm_ on the parameters)", who);
    const c10::DeviceGuard guard(g.device);
    g.ready(true, who);
    g.d.max_norm = (float)max_norm;
    std::vector<Tensor> held;
    std::vector<c10::Storage> memory;
    if (error_if_nonfinite) {
        call(api.grad_norm_partials(&g.d, handle(stream)));
        call(api.grad_norm_finish(&g.d, handle(stream)));
        double v;
        {
            // Other Python threads run on while this one waits: the queue ahead may itself wait for what one of them has yet to launch.  The
            // list and the parameters are theirs to change then, so the tensors and their memory are held here.
            held.reserve(g.tensors.size());
            memory.reserve(g.tensors.size());
            for (const Tensor*& t : g.tensors) {
                held.push_back(*t);
                memory.push_back(t->storage());
                t = &held.back();
            }
            const py::gil_scoped_release no_gil;
            v = g.norm.item<double>();
        }
        if (!std::isfinite(v)) throw std::runtime_error(text("the norm of the gradients is not finite (%g): nothing was clipped", v));
        call(api.clip_scale(&g.d, handle(stream)));
    } else {
        call(api.clip_grads(&g.d, handle(stream)));
    }
    for (const Tensor* t : g.tensors) written(*t);
    return g.norm;
}

Tensor adam_update(const Tensor& p, const Tensor& grad, const Tensor& m, const Tensor& v, int64_t step, double lr, double beta1, double beta2, double eps,
                   double weight_decay, double grad_scale, double max_grad_norm, double norm_type, const OptTensor& shadow, int64_t stream) {
    no_trace("adam_update_");
    for (const Tensor* t : {&p, &grad, &m, &v}) no_tangent(*t, "adam_update_");
    for (const Tensor* t : {&p, &grad, &m, &v})
        VALUE_CHECK(t->is_cuda() && t->scalar_type() == at::kFloat && t->numel() == p.numel() && t->device() == p.device() && t->is_contiguous() && !t->is_neg(),
                    "adam_update_ needs contiguous float32 tensors of one size on one GPU");
    if (shadow.has_value())
        VALUE_CHECK(shadow->scalar_type() == at::kBFloat16 && shadow->numel() == p.numel() && shadow->device() == p.device() && shadow->is_contiguous() &&
                        !shadow->is_neg(),
                    "adam_update_: shadow must be a contiguous bfloat16 tensor of the size of param");
    VALUE_CHECK(p.numel() > 0, "adam_update_ needs at least one element");
    std::vector<std::pair<char*, char*>> spans;
    for (const Tensor* t : {&p, &grad, &m, &v, shadow.has_value() ? &*shadow : nullptr})
        if (t) spans.emplace_back((char*)t->data_ptr(), (char*)t->data_ptr() + t->nbytes());
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i) VALUE_CHECK(spans[i].first >= spans[i - 1].second, "adam_update_: two of the tensors share memory");
    VALUE_CHECK(step >= 1, "adam_update_: step counts from 1, got %lld", (long long)step);
    VALUE_CHECK(grad_scale > 0.0 && (float)grad_scale > 0.f && (float)grad_scale < INFINITY, "adam_update_: grad_scale must be positive and finite, got %g", grad_scale);
    VALUE_CHECK(max_grad_norm >= 0.0, "adam_update_: max_grad_norm must be >= 0, got %g", max_grad_norm);
    VALUE_CHECK(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adam_update_: betas must be in [0, 1), got (%g, %g)", beta1, beta2);
    Grads g;
    g.add(grad, "adam_update_");
    g.set_norm_type(norm_type, "adam_update_");
    g.d.scale = (float)grad_scale;
    const c10::DeviceGuard guard(g.device);
    g.ready(false, "adam_update_");
    g.d.max_norm = (float)max_grad_norm;
    call(api.grad_norm_partials(&g.d, handle(stream)));
    dsaspp_adam_clip_desc a = {};
    a.n = p.numel();
    a.p = ptr<float>(p); a.g = ptr<float>(grad); a.m = ptr<float>(m); a.v = ptr<float>(v);
    a.w16 = shadow.has_value() ? shadow->data_ptr() : nullptr;
    a.lr = lr; a.beta1 = beta1; a.beta2 = beta2; a.eps = eps; a.weight_decay = weight_decay;
    a.step = step;
    call(api.adam_step_clipped(&a, &g.d, handle(stream)));
    for (const Tensor* t : {&p, &m, &v, shadow.has_value() ? &*shadow : nullptr})
        if (t) written(*t);
    return g.norm;
}

// for tests: (address, elements, dtype code) of the ranges a list of gradients makes, and the merged row dimensions of logits
py::list ranges_of(const Tensor& t) {
    std::vector<dsaspp_grad_range> r;
    if (t.is_contiguous() || t.is_non_overlapping_and_dense()) r.push_back({t.data_ptr(), t.numel(), dtype_code(t.scalar_type()), 0});
    else add_pieces(t, dtype_code(t.scalar_type()), r);
    py::list out;
    for (auto& x : r) out.append(py::make_tuple((int64_t)x.p, x.n));
    return out;
}
py::object rows_of(const Tensor& logits) {
    int64_t n[3], st[3];
    if (!row_strides(logits.sizes(), logits.strides(), n, st)) return py::none();
    py::list out;
    for (int k = 0; k < 3; ++k) out.append(py::make_tuple(n[k], st[k]));
    return std::move(out);
}

void init(const py::dict& f) {
    auto take = [&](const char* name, auto& fn) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(f[name].cast<int64_t>()); };
    take("dsaspp_scores_fwd", api.scores_fwd);
    take("dsaspp_scores_bwd", api.scores_bwd);
    take("dsaspp_scores_workspace", api.scores_workspace);
    take("dsaspp_scores8_workspace", api.scores8_workspace);
    take("dsaspp_scores8_fwd", api.scores8_fwd);
    take("dsaspp_scores8_bwd", api.scores8_bwd);
    take("dsaspp_grad_norm_workspace", api.grad_norm_workspace);
    take("dsaspp_grad_ranges_overlap", api.grad_ranges_overlap);
    take("dsaspp_grad_norm_partials", api.grad_norm_partials);
    take("dsaspp_grad_norm_finish", api.grad_norm_finish);
    take("dsaspp_clip_scale", api.clip_scale);
    take("dsaspp_clip_grads", api.clip_grads);
    take("dsaspp_adam_step_clipped", api.adam_step_clipped);
    take("dsaspp_last_error", api.last_error);
}

}  // namespace

PYBIND11_MODULE(_dsaspp_torch, m) {
    m.def("init", &init);
    m.def("source_hash", [] { return std::string(g_hash + 12); });
    m.def("label_scores", &label_scores);
    m.def("check_image", &check_image);
    m.def("check_scores", &check_scores);
    m.def("upsampled_forward", &upsampled_forward);
    m.def("upsampled_backward", &upsampled_backward);
    m.def("grad_norm", &grad_norm);
    m.def("clip_grads", &clip_grads);
    m.def("adam_update", &adam_update);
    m.def("ranges_of", &ranges_of);
    m.def("rows_of", &rows_of);
}
