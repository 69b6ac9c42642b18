// mvf_torch.cpp -- the token-attention operators as torch autograd functions over the C ABI (include/mvf_hotpath.h).
//
// At the coarse levels of a pyramid the kernels of a training step take some ten microseconds each and the host decides: an
// autograd.Function written in Python costs its arguments, its descriptor, its allocations and a hand-over of the interpreter
// lock to the engine's thread in every backward.  Here both directions run without the interpreter.  The module holds no kernel: it is
// given the entry points of the library that the ctypes binding loaded (bind), and mono-vifi_amd/ops.py offers its functions.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/version.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <map>
#include <optional>
#include <unordered_set>

#include "../../include/mvf_hotpath.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct Api {
    decltype(&mvf_error_string) error_string;
    decltype(&mvf_cross_attention_fwd_workspace_bytes) attn_fwd_bytes;
    decltype(&mvf_cross_attention_fwd) attn_fwd;
    decltype(&mvf_cross_attention_bwd_workspace_bytes) attn_bwd_bytes;
    decltype(&mvf_cross_attention_bwd) attn_bwd;
    decltype(&mvf_qk_norm_rope_fwd) norm_fwd;
    decltype(&mvf_qk_norm_rope_bwd_workspace_floats) norm_bwd_floats;
    decltype(&mvf_qk_norm_rope_bwd) norm_bwd;
} api = {};

void bind(const std::map<std::string, uintptr_t> &at)
{
    auto get = [&](const char *name, auto &fn) { fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(at.at(name)); };
    get("mvf_error_string", api.error_string);
    get("mvf_cross_attention_fwd_workspace_bytes", api.attn_fwd_bytes);
    get("mvf_cross_attention_fwd", api.attn_fwd);
    get("mvf_cross_attention_bwd_workspace_bytes", api.attn_bwd_bytes);
    get("mvf_cross_attention_bwd", api.attn_bwd);
    get("mvf_qk_norm_rope_fwd", api.norm_fwd);
    get("mvf_qk_norm_rope_bwd_workspace_floats", api.norm_bwd_floats);
    get("mvf_qk_norm_rope_bwd", api.norm_bwd);
}

void check(int err, const char *what)
{
    TORCH_CHECK(err == 0, what, " failed: HIP error ", err, " (", api.error_string(err), ")");
}
// the kernels go to the current stream of the current device, as all of the library's
void *stream_now() { return (void *)c10::hip::getCurrentHIPStream().stream(); }

std::string shape_of(const Tensor &t)
{
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + (t.dim() == 1 ? ",)" : ")");
}

// all tensors on one HIP device, and that is the current one (mono-vifi_amd/_native.py: require_device)
void require_device(std::initializer_list<const Tensor *> ts)
{
    std::optional<c10::Device> dev;
    for (const Tensor *t : ts) {
        if (!t->defined()) continue;
        TORCH_CHECK(t->is_cuda(), "mono_vifi_amd hot-path ops run on a HIP device (MI355X) only; got a ", t->device(),
                    " tensor. There is no CPU fallback.");
        if (!dev) dev = t->device();
        TORCH_CHECK(*dev == t->device(), "hot-path op got tensors on different devices: ", *dev, " and ", t->device());
    }
    const int cur = c10::hip::current_device();
    TORCH_CHECK(!dev || dev->index() == cur, "hot-path op got ", *dev, " tensors while the current device is cuda:", cur,
                "; call torch.cuda.set_device(local_rank) (or use `with torch.cuda.device(t.device)`) so that the kernels are "
                "enqueued on the stream of the GPU that owns the data");
}

// [batch, token, head, channel] with adjacent channels, float32 or bfloat16; any strides otherwise
Tensor token_heads(const char *what, const char *name, const Tensor &t, std::optional<at::ScalarType> dtype)
{
    TORCH_CHECK(t.defined() && t.dim() == 4, what, ": ", name, " must be [batch, tokens, heads, channels], got ", t.defined() ? shape_of(t) : "None");
    TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, what, ": ", name, " must be float32 or bfloat16, got ",
                t.scalar_type());
    TORCH_CHECK(!dtype || t.scalar_type() == *dtype, what, ": ", name, " is ", t.scalar_type(), ", the queries are ", *dtype);
    TORCH_CHECK(t.size(2) >= 1 && t.size(3) >= 1 && t.size(3) <= MVF_ATTN_MAX_D, what, ": ", name, " needs at least one head of 1..",
                MVF_ATTN_MAX_D, " channels, got ", shape_of(t));
    for (int i = 0; i < 3; ++i)
        TORCH_CHECK(t.size(i) <= INT32_MAX, what, ": ", name, " is too large: ", shape_of(t));
    return t.size(3) == 1 || t.stride(3) == 1 ? t : t.contiguous();
}
int type_of(const Tensor &t) { return t.scalar_type() == at::kFloat ? MVF_DTYPE_F32 : MVF_DTYPE_BF16; }

// an incoming gradient as the kernels read it: contiguous, of the forward's type, 16-byte aligned
Tensor aligned(Tensor g, at::ScalarType type)
{
    g = g.to(type).contiguous();
    return (uintptr_t)g.data_ptr() & 15 ? g.clone() : g;
}
// These functions call the kernels themselves, past torch's dispatcher.  A trace would hold the allocation of the output and not what
// fills it, and a forward gradient of an input would be dropped: both are errors, in the call and in its backward.
void direct(const char *what, std::initializer_list<const Tensor *> ts)
{
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY), what,
                " cannot be traced: its kernels are called directly, the trace would not hold them");
    for (const Tensor *t : ts)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative, and got a tensor with a forward gradient");
}
void once(const char *what, const variable_list &grads)
{
    // (a second derivative through the saved inputs would be silently missing)
    TORCH_CHECK(!at::GradMode::is_enabled(), what, " is differentiable once: its backward does not run under create_graph=True");
    for (const Tensor &g : grads) direct(what, {&g});
}
// A leaf's gradient is accumulated on the stream that was current when the first graph that still lives first used the leaf.  If that is the
// default stream, a backward that is being captured on another would order captured work before a stream that cannot join a
// capture, and the process ends.  Refused while it is an error that can be caught: for every leaf that this backward will reach
// from its inputs whose gradients are needed (a leaf may lie behind a copy or a view of it).
void capturable(const char *what, std::initializer_list<std::pair<const Tensor *, bool>> inputs)
{
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    std::vector<std::shared_ptr<torch::autograd::Node>> todo;
    for (const auto &[t, needed] : inputs)
        if (needed && t->defined()) todo.push_back(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    const c10::Stream eager = c10::hip::getDefaultHIPStream().unwrap();
    const auto *task = torch::autograd::get_current_graph_task_exec_info();        // which nodes run; empty: all
    std::unordered_set<torch::autograd::Node *> seen;
    while (!todo.empty()) {
        const auto node = todo.back();
        todo.pop_back();
        if (!node || !seen.insert(node.get()).second) continue;
        if (task && !task->empty()) {
            const auto it = task->find(node.get());
            if (it == task->end() || !it->second.should_execute()) continue;
        }
        if (dynamic_cast<torch::autograd::AccumulateGrad *>(node.get())) {
            const auto stream = node->stream();
            TORCH_CHECK(!stream || stream->id() != eager.id(), what, ": this backward is being captured while an eager graph of the same "
                        "leaves lives on the default stream; drop its outputs, or run the eager calls on a side stream");
        }
        for (const auto &edge : node->next_edges()) todo.push_back(edge.function);
    }
}
Tensor dense(const Tensor &like) { return at::empty(like.sizes(), like.options(), at::MemoryFormat::Contiguous); }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor or_none(const std::optional<Tensor> &t) { return t && t->defined() ? *t : Tensor(); }
std::optional<Tensor> opt(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// ------------------------------------------------------------------------------------------------- cross attention
mvf_attn_desc attn_desc(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &mask, const Tensor &lens, double scale)
{
    mvf_attn_desc d = {};
    d.q = ptr(q); d.k = ptr(k); d.v = ptr(v);
    d.key_mask = (const uint8_t *)ptr(mask);
    d.kv_lens = (const int32_t *)ptr(lens);
    for (int i = 0; i < 3; ++i) { d.q_stride[i] = q.stride(i); d.k_stride[i] = k.stride(i); d.v_stride[i] = v.stride(i); }
    if (mask.defined()) { d.mask_stride[0] = mask.stride(0); d.mask_stride[1] = mask.stride(1); }
    d.B = (int)q.size(0); d.Lq = (int)q.size(1); d.Hq = (int)q.size(2); d.D = (int)q.size(3);
    d.Lk = (int)k.size(1); d.Hk = (int)k.size(2);
    d.dtype = type_of(q);
    d.scale = (float)scale;
    return d;
}
// lse, low: what a backward needs besides the output, or null (low: the rest of a bfloat16 output; lse of float32: and 1 / the sums behind it)
Tensor attn_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &mask, const Tensor &lens, double scale, Tensor *lse, Tensor *low)
{
    mvf_attn_desc d = attn_desc(q, k, v, mask, lens, scale);
    Tensor out = dense(q), ws;
    if (lse) *lse = at::empty({d.dtype == MVF_DTYPE_F32 ? 2 : 1, q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    if (lse && d.dtype == MVF_DTYPE_F32) d.inv_sum = (float *)ptr(*lse) + lse->numel() / 2;
    if (low && d.dtype == MVF_DTYPE_BF16) {
        *low = dense(q);
        d.out_low = ptr(*low);
    }
    if (const size_t n = api.attn_fwd_bytes(&d)) ws = at::empty({(int64_t)n}, q.options().dtype(at::kByte));
    check(api.attn_fwd(&d, ptr(out), lse ? (float *)ptr(*lse) : nullptr, ptr(ws), stream_now()), "cross_attention_fwd");
    return out;
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const std::optional<Tensor> &mask_,
                          const std::optional<Tensor> &lens_, double scale)
    {
        const Tensor mask = or_none(mask_), lens = or_none(lens_);
        Tensor lse, low;
        const Tensor out = attn_forward(q, k, v, mask, lens, scale, &lse, &low);
        ctx->save_for_backward({q, k, v, mask, lens, out, lse, low});
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        once("cross_attention", grads);
        const auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2];
        mvf_attn_desc d = attn_desc(q, k, v, s[3], s[4], ctx->saved_data["scale"].toDouble());
        const Tensor g = aligned(grads[0], q.scalar_type()), out = aligned(s[5], q.scalar_type()), lse = s[6].contiguous();
        const Tensor low = s[7].defined() ? aligned(s[7], q.scalar_type()) : Tensor();
        d.out_low = ptr(low);
        if (d.dtype == MVF_DTYPE_F32) d.inv_sum = (float *)ptr(lse) + lse.numel() / 2;
        const bool need_q = ctx->needs_input_grad(0), need_k = ctx->needs_input_grad(1), need_v = ctx->needs_input_grad(2);
        capturable("cross_attention", {{&q, need_q}, {&k, need_k}, {&v, need_v}});
        Tensor gq = dense(q), gk, gv;
        if (need_k || need_v) { gk = dense(k); gv = dense(v); }
        const Tensor ws = at::empty({(int64_t)api.attn_bwd_bytes(&d)}, q.options().dtype(at::kByte));
        check(api.attn_bwd(&d, ptr(out), (const float *)ptr(lse), ptr(g), ptr(gq), ptr(gk), ptr(gv), ptr(ws), stream_now()), "cross_attention_bwd");
        return {need_q ? gq : Tensor(), need_k ? gk : Tensor(), need_v ? gv : Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor cross_attention(Tensor q, Tensor k, Tensor v, std::optional<double> scale_, std::optional<Tensor> mask_, std::optional<Tensor> lens_)
{
    const char *what = "cross_attention";
    direct(what, {&q, &k, &v});
    q = token_heads(what, "q", q, {});
    k = token_heads(what, "k", k, q.scalar_type());
    v = token_heads(what, "v", v, q.scalar_type());
    TORCH_CHECK(k.sizes() == v.sizes(), what, ": k ", shape_of(k), " and v ", shape_of(v), " differ");
    const int64_t B = q.size(0), Lk = k.size(1);
    TORCH_CHECK(k.size(0) == B && k.size(3) == q.size(3) && q.size(2) % k.size(2) == 0, what, ": states ", shape_of(k), " do not fit queries ",
                shape_of(q), " (same batch and channels, query heads a multiple of the states' heads)");
    const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)q.size(3));
    TORCH_CHECK(scale > 0.0 && scale < 1e38, what, ": scale must be positive and finite, got ", scale);
    const Tensor mask = or_none(mask_);
    Tensor lens = or_none(lens_);
    if (mask.defined())
        TORCH_CHECK((mask.scalar_type() == at::kBool || mask.scalar_type() == at::kByte) && mask.dim() == 2 && mask.size(0) == B && mask.size(1) == Lk,
                    what, ": key_mask must be bool or uint8 (", B, ", ", Lk, "), got ", mask.scalar_type(), " ", shape_of(mask));
    if (lens.defined())
        TORCH_CHECK((lens.scalar_type() == at::kInt || lens.scalar_type() == at::kLong) && lens.dim() == 1 && lens.size(0) == B, what,
                    ": kv_lens must be int32 or int64 (", B, ",), got ", lens.scalar_type(), " ", shape_of(lens));
    require_device({&q, &k, &v, &mask, &lens});
    if (lens.defined()) {
        if (lens.scalar_type() != at::kInt) lens = lens.clamp(0, Lk).to(at::kInt);
        lens = lens.contiguous();
    }
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
        return CrossAttention::apply(q, k, v, opt(mask), opt(lens), scale);
    return attn_forward(q, k, v, mask, lens, scale, nullptr, nullptr);
}

// ------------------------------------------------------------------------------------------------- norm and rotation
// turns per unit of position of the ra / 2 frequencies, as 64-bit fractions of a turn
const std::vector<uint64_t> &turn_fractions(int64_t ra, double base)
{
    static thread_local std::map<std::pair<int64_t, double>, std::vector<uint64_t>> tables;
    if (tables.size() > 64) tables.clear();
    auto &t = tables[{ra, base}];
    if (t.empty()) {
        const long double turn = 2.0L * 3.14159265358979323846264338327950288L, whole = 18446744073709551616.0L;
        for (int64_t j = 0; j < ra / 2; ++j) {
            const long double f = std::fmod(std::pow((long double)base, -2.0L * j / ra) / turn, 1.0L) * whole;
            t.push_back(f < whole - 0.5L ? (uint64_t)(f + 0.5L) : 0);
        }
        if (t.empty()) t.push_back(0);
    }
    return t;
}

struct NormConfig {
    int64_t rot, axes;
    double base, eps;
    bool interleaved;
};
mvf_qk_norm_desc norm_desc(const Tensor &q, const Tensor &k, const Tensor &wq, const Tensor &wk, const Tensor &pq, const Tensor &pk, const NormConfig &c)
{
    mvf_qk_norm_desc d = {};
    d.q = ptr(q); d.k = ptr(k);
    d.q_weight = (const float *)ptr(wq); d.k_weight = (const float *)ptr(wk);
    d.q_pos = ptr(pq); d.k_pos = ptr(pk);
    d.freq = turn_fractions(c.rot / c.axes, c.base).data();
    for (int i = 0; i < 3; ++i) {
        d.q_stride[i] = q.stride(i);
        d.k_stride[i] = k.defined() ? k.stride(i) : 0;
    }
    d.q_pos_stride = pq.defined() && pq.dim() == 3 ? pq.stride(0) : 0;
    d.k_pos_stride = pk.defined() && pk.dim() == 3 ? pk.stride(0) : 0;
    d.B = (int)q.size(0); d.Lq = (int)q.size(1); d.Hq = (int)q.size(2); d.D = (int)q.size(3);
    d.Lk = k.defined() ? (int)k.size(1) : 0;
    d.Hk = k.defined() ? (int)k.size(2) : 1;
    d.dtype = type_of(q);
    d.axes = (int)c.axes; d.rot = (int)c.rot;
    d.interleaved = c.interleaved;
    d.pos64 = (pq.defined() ? pq : pk).defined() && (pq.defined() ? pq : pk).scalar_type() == at::kLong;
    d.eps = (float)c.eps;
    return d;
}
variable_list norm_forward(const Tensor &q, const Tensor &k, const Tensor &wq, const Tensor &wk, const Tensor &pq, const Tensor &pk, const NormConfig &c)
{
    const mvf_qk_norm_desc d = norm_desc(q, k, wq, wk, pq, pk, c);
    variable_list out = {dense(q)};
    if (k.defined()) out.push_back(dense(k));
    check(api.norm_fwd(&d, ptr(out[0]), k.defined() ? ptr(out[1]) : nullptr, stream_now()), "qk_norm_rope_fwd");
    return out;
}

struct QkNormRope : torch::autograd::Function<QkNormRope> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const std::optional<Tensor> &k_, const std::optional<Tensor> &wq_,
                                 const std::optional<Tensor> &wk_, const std::optional<Tensor> &pq_, const std::optional<Tensor> &pk_, int64_t rot,
                                 int64_t axes, double base, double eps, bool interleaved)
    {
        const Tensor k = or_none(k_), wq = or_none(wq_), wk = or_none(wk_), pq = or_none(pq_), pk = or_none(pk_);
        ctx->save_for_backward({q, k, wq, wk, pq, pk});
        auto &s = ctx->saved_data;
        s["rot"] = rot; s["axes"] = axes; s["base"] = base; s["eps"] = eps; s["interleaved"] = interleaved;
        return norm_forward(q, k, wq, wk, pq, pk, {rot, axes, base, eps, interleaved});
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        once("qk_norm_rope", grads);
        const auto s = ctx->get_saved_variables();
        auto &c = ctx->saved_data;
        const Tensor &q = s[0], &k = s[1], &wq = s[2], &wk = s[3];
        const mvf_qk_norm_desc d = norm_desc(q, k, wq, wk, s[4], s[5],
                                             {c["rot"].toInt(), c["axes"].toInt(), c["base"].toDouble(), c["eps"].toDouble(), c["interleaved"].toBool()});
        const Tensor gyq = aligned(grads[0], q.scalar_type()), gyk = k.defined() ? aligned(grads[1], q.scalar_type()) : Tensor();
        Tensor gq = dense(q), gk = k.defined() ? dense(k) : Tensor(), gwq, gwk, ws;
        // (edges are counted over the tensors that are there)
        const int ek = 1, ewq = ek + k.defined(), ewk = ewq + wq.defined();
        const bool need_k = k.defined() && ctx->needs_input_grad(ek), need_wq = wq.defined() && ctx->needs_input_grad(ewq),
                   need_wk = wk.defined() && ctx->needs_input_grad(ewk);
        capturable("qk_norm_rope", {{&q, ctx->needs_input_grad(0)}, {&k, need_k}, {&wq, need_wq}, {&wk, need_wk}});
        if (need_wq) gwq = dense(wq);
        if (need_wk) gwk = dense(wk);
        if (need_wq || need_wk) ws = at::empty({(int64_t)api.norm_bwd_floats(&d) + 1}, q.options().dtype(at::kFloat));
        check(api.norm_bwd(&d, ptr(gyq), ptr(gyk), ptr(gq), ptr(gk), (float *)ptr(gwq), (float *)ptr(gwk), (float *)ptr(ws), stream_now()),
              "qk_norm_rope_bwd");
        return {ctx->needs_input_grad(0) ? gq : Tensor(), need_k ? gk : Tensor(), gwq, gwk,
                Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor positions(const char *what, const char *name, Tensor p, int64_t B, int64_t L)
{
    TORCH_CHECK(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong, what, ": ", name, " must be int32 or int64, got ", p.scalar_type());
    if (p.dim() == 1) p = p.unsqueeze(1);
    TORCH_CHECK((p.dim() == 2 || (p.dim() == 3 && p.size(0) == B)) && p.size(-2) == L && p.size(-1) >= 1 && p.size(-1) <= 3, what, ": ", name,
                " must be [", L, ", axes] or [", B, ", ", L, ", axes] with 1..3 axes, got ", shape_of(p));
    return p.contiguous();
}
Tensor head_weight(const char *what, const char *name, const Tensor &w, at::ScalarType type, int64_t D)
{
    TORCH_CHECK((w.scalar_type() == at::kFloat || w.scalar_type() == type) && w.dim() == 1 && w.size(0) == D, what, ": ", name, " must be [", D,
                "] in float32 or ", type, ", got ", w.scalar_type(), " ", shape_of(w));
    return w.to(at::kFloat).contiguous();
}

py::object qk_norm_rope(Tensor q, std::optional<Tensor> k_, std::optional<Tensor> wq_, std::optional<Tensor> wk_, std::optional<Tensor> pq_,
                        std::optional<Tensor> pk_, std::optional<int64_t> rot_, double base, double eps, bool interleaved)
{
    const char *what = "qk_norm_rope";
    Tensor k = or_none(k_), wq = or_none(wq_), wk = or_none(wk_), pq = or_none(pq_), pk = or_none(pk_);
    direct(what, {&q, &k, &wq, &wk});
    q = token_heads(what, "q", q, {});
    const int64_t B = q.size(0), D = q.size(3);
    if (k.defined()) {
        k = token_heads(what, "k", k, q.scalar_type());
        TORCH_CHECK(k.size(0) == B && k.size(3) == D, what, ": k ", shape_of(k), " does not fit q ", shape_of(q), " (same batch and channels)");
    } else {
        TORCH_CHECK(!wk.defined() && !pk.defined(), what, ": k_weight / k_pos without k");
    }
    int64_t axes = 0;
    if (pq.defined()) {
        pq = positions(what, "q_pos", pq, B, q.size(1));
        axes = pq.size(-1);
    }
    if (pk.defined()) {
        pk = positions(what, "k_pos", pk, B, k.size(1));
        TORCH_CHECK(!axes || axes == pk.size(-1), what, ": q_pos and k_pos have different numbers of axes");
        axes = pk.size(-1);
        if (pq.defined() && pq.scalar_type() != pk.scalar_type()) {
            pq = pq.to(at::kLong);
            pk = pk.to(at::kLong);
        }
    }
    if (!axes) axes = 1;
    const int64_t rot = rot_ ? *rot_ : D / (2 * axes) * (2 * axes);
    TORCH_CHECK(rot >= 0 && rot <= D && rot % (2 * axes) == 0, what, ": rot_dim ", rot, " must be a multiple of ", 2 * axes,
                " (two per axis) of at most ", D, " channels");
    TORCH_CHECK(base > 0.0 && base < INFINITY && eps >= 0.0 && eps < INFINITY, what, ": base must be positive and eps not negative, got ", base, " and ", eps);
    if (wq.defined()) wq = head_weight(what, "q_weight", wq, q.scalar_type(), D);
    if (wk.defined()) wk = head_weight(what, "k_weight", wk, q.scalar_type(), D);
    require_device({&q, &k, &wq, &wk, &pq, &pk});
    const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()) || (wq.defined() && wq.requires_grad()) ||
                                                     (wk.defined() && wk.requires_grad()));
    const variable_list out = grad ? QkNormRope::apply(q, opt(k), opt(wq), opt(wk), opt(pq), opt(pk), rot, axes, base, eps, interleaved)
                                   : norm_forward(q, k, wq, wk, pq, pk, {rot, axes, base, eps, interleaved});
    if (!k.defined()) return py::cast(out[0]);
    return py::make_tuple(out[0], out[1]);
}

}  // namespace

PYBIND11_MODULE(_mvf_torch, m)
{
    m.def("bind", &bind);
    m.attr("abi") = MVF_ABI_VERSION;                             // of the descriptors, and the torch, that this was compiled against
    m.attr("torch") = TORCH_VERSION;
    m.def("cross_attention", &cross_attention);
    m.def("qk_norm_rope", &qk_norm_rope);
}
