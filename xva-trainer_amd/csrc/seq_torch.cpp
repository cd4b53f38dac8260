// seq_torch.cpp — the sequence operators as torch sees them: argument checks, allocation, autograd nodes and the calls of the C ABI (include/xva_hip.h), for
// seq_ops.py.
//
// Why not ctypes and torch.autograd.Function, as the rest of the package: these operators take 5 - 50 us on the card, and a backward pass in Python runs on torch's
// worker thread with every Python object it touches in another core's cache.  Host time of a group norm, forward and backward: 123 us that way, 68 us here, of
// which torch's engine takes 42 (negating one tensor); differential attention 84 us; a call without a gradient 6 - 8 us.
//
// The kernel library is not linked: seq_ops.py hands over the addresses of its entry points (`bind`), so that both sides use the one that _lib.py has loaded.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <algorithm>
#include <cmath>
#include <vector>
#include "../../include/xva_hip.h"

namespace {
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> MaybeTensor;

struct Failure : std::runtime_error { using std::runtime_error::runtime_error; };      // XvaError in Python
#define REFUSE(cond, ...) do { if (cond) throw Failure(c10::str(__VA_ARGS__)); } while (0)

struct Entries {
    decltype(&xva_last_error) last_error;
    decltype(&xva_rotary) rotary;
    decltype(&xva_group_norm_workspace_bytes) norm_ws;
    decltype(&xva_group_norm_act_fwd) norm_fwd, norm_bwd;
    decltype(&xva_recurrence_workspace_bytes) rec_ws;
    decltype(&xva_recurrence_state_floats) rec_states;
    decltype(&xva_recurrence_fwd) rec_fwd, rec_bwd;
    decltype(&xva_diff_attention_workspace_bytes) diff_ws;
    decltype(&xva_diff_attention_fwd) diff_fwd, diff_bwd;
} lib;

void call(int rc, const char* what) { REFUSE(rc != 0, what, " failed (rc=", rc, "): ", lib.last_error()); }
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor or_none(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }
// (autograd takes a missing tensor as an empty optional only)
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

int dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: return -1;
    }
}
bool has_tangent(const Tensor& t) { return t.defined() && torch::autograd::isFwGradDefined(t); }
// all of them on the GPU of the first one, and nothing of torch's under way that the launches would drop out of without a word
void on_one_device(const Tensor& first, std::initializer_list<Tensor> others) {
    bool dual = has_tangent(first);
    for (const Tensor& t : others) dual = dual || has_tangent(t);
    REFUSE(dual, "forward-mode derivatives: these operators have backward passes only");
    REFUSE(torch::jit::tracer::isTracing(), "torch.jit.trace would record none of these operators' launches");
    REFUSE(!first.is_cuda(), "libxvahip ops need device tensors; got a ", first.device(), " tensor (no CPU fallback exists)");
    for (const Tensor& t : others) REFUSE(t.defined() && t.device() != first.device(), "tensors on ", first.device(), " and ", t.device());
    // (a fake tensor or a wrapper around others has no address, which would be taken for an argument that was left out)
    auto empty_handed = [](const Tensor& t) { return t.defined() && t.numel() > 0 && !t.const_data_ptr(); };
    bool bare = empty_handed(first);
    for (const Tensor& t : others) bare = bare || empty_handed(t);
    REFUSE(bare, "a tensor without memory of its own (fake, functional, or a wrapper around others)");
}
Tensor lengths(const Tensor& lens, int64_t B, int64_t T, const char* what) {
    if (!lens.defined()) return lens;
    REFUSE(lens.dim() != 1 || lens.size(0) != B, what, ": ", lens.sizes(), ", expected (", B, ",)");
    REFUSE(lens.scalar_type() != at::kInt && lens.scalar_type() != at::kLong, what, ": int32 or int64, got ", lens.scalar_type());
    return (lens.scalar_type() == at::kLong ? lens.clamp(0, T) : lens).to(at::kInt).contiguous();        // (64 bits have numbers that 32 take for others)
}
Tensor fp32(const Tensor& t) { return t.defined() ? t.to(at::kFloat).contiguous() : t; }
// elements from one index of dimension e to the next (a dimension of 1 has none: torch leaves any number there)
int64_t step(const Tensor& t, int e) { return t.size(e) > 1 ? t.stride(e) : 0; }
// with a contiguous last dimension
Tensor rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
Tensor aligned(const Tensor& t) { return (uintptr_t)t.data_ptr() % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous); }
bool wants_grad(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}
Tensor workspace(int64_t bytes, const Tensor& like) { return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor(); }
Tensor floats(at::IntArrayRef size, const Tensor& like) { return at::empty(size, like.options().dtype(at::kFloat)); }
int small(int64_t v, const char* what) { REFUSE(v < 0 || v > INT32_MAX, what, " ", v); return (int)v; }

// A gradient taken with create_graph is right, and says so if it is differentiated again.  Whether the incoming gradients require one does not matter: the result
// depends on the saved inputs too (of a linear map it does not: without such a gradient it is a constant).
variable_list once(variable_list out, const variable_list& grads, bool linear = false) {
    for (const Tensor& g : grads) REFUSE(has_tangent(g), "forward-mode derivatives of a backward pass");
    if (!at::GradMode::is_enabled()) return out;
    bool any = !linear;
    for (const Tensor& g : grads) any = any || (g.defined() && g.requires_grad());
    if (!any) return out;
    auto fn = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", (int)out.size());
    for (Tensor& t : out) {
        if (!t.defined()) continue;
        t = (*fn)({t.detach().requires_grad_()})[0];
    }
    return out;
}

// ---------------------------------------------------------------------------------------------------------------------------------- rotary ----
// Do elements of (items, rows, heads, D) views lie on each other: of q and k, or, without k, of two different heads of q?  torch's own answer is "too hard" for views
// that are not dense, and slices of one projection are not.  Two elements meet where sum n_e s_e + r equals the distance of the two views, n_e a difference of indices
// along one of the strides s_e, |r| < D: a search over the n_e from the widest stride down, which has a candidate or two each where strides enclose each other.
enum Overlap { APART, MEETING, UNKNOWN };
struct Search {
    struct Dim { int64_t stride, lo, hi; };
    std::vector<Dim> dims;
    std::vector<std::pair<int64_t, int64_t>> rest;         // least and largest sum over dims e ..
    bool same;                                             // all n_e = 0 is an element's own place
    int left = 4096;                                       // candidates that are tried: beyond them nothing is promised
    void add(const Tensor& t, bool other) {
        for (int e = 0; e < 3; ++e) {
            if (t.size(e) < 2) continue;
            const int64_t n = t.size(e) - 1;
            Dim* d = nullptr;
            for (Dim& x : dims) d = x.stride == t.stride(e) && !same ? &x : d;
            if (!d) { dims.push_back({t.stride(e), 0, 0}); d = &dims.back(); }
            if (other || same) d->lo -= n;
            if (!other || same) d->hi += n;
        }
    }
    bool meets(size_t e, int64_t target, bool moved) {
        if (--left < 0) return true;
        if (e == dims.size()) return (moved || !same) && target >= rest[e].first && target <= rest[e].second;
        const Dim& d = dims[e];
        for (int64_t n = d.lo; n <= d.hi; ++n) {
            if (d.stride > 0) {
                const int64_t least = target - rest[e + 1].second, most = target - rest[e + 1].first;      // of n * stride
                const int64_t first = least > 0 ? (least + d.stride - 1) / d.stride : -(-least / d.stride);
                if (n < first) n = first;
                if (n > d.hi || n * d.stride > most) return false;
            }
            if (meets(e + 1, target - n * d.stride, moved || n != 0)) return true;
        }
        return false;
    }
    Overlap run(int64_t target, int64_t D) {
        std::sort(dims.begin(), dims.end(), [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
        rest.assign(dims.size() + 1, {1 - D, D - 1});
        for (size_t e = dims.size(); e-- > 0;) rest[e] = {rest[e + 1].first + dims[e].lo * dims[e].stride, rest[e + 1].second + dims[e].hi * dims[e].stride};
        const bool found = meets(0, target, false);
        return left < 0 ? UNKNOWN : (found ? MEETING : APART);
    }
};
Overlap overlap(const Tensor& q, const Tensor& k) {
    if (q.numel() == 0 || (k.defined() && k.numel() == 0)) return APART;
    Search s;
    s.same = !k.defined();
    s.add(q, false);
    if (s.same) return s.run(0, q.size(3));
    s.add(k, true);
    const int64_t bytes = (const char*)k.data_ptr() - (const char*)q.data_ptr(), es = q.element_size();
    return bytes % es ? UNKNOWN : s.run(bytes / es, q.size(3));       // (q + i = k + j: i - j is the distance from q to k)
}

struct RotaryArgs { Tensor turns, pos; int64_t rd; bool interleaved; double gain; };

std::pair<Tensor, Tensor> rotary_launch(const Tensor& q_, const Tensor& k_, const RotaryArgs& r, bool inverse, bool inplace) {
    const c10::DeviceGuard guard(q_.device());
    const Tensor q = rows(q_), k = k_.defined() ? rows(k_) : k_;
    const Tensor qo = inplace ? q : at::empty(q.sizes(), q.options()), ko = !k.defined() ? k : (inplace ? k : at::empty(k.sizes(), k.options()));
    xva_rotary_args a = {};
    a.q = q.data_ptr(); a.k = ptr(k); a.q_out = qo.data_ptr(); a.k_out = ptr(ko);
    for (int e = 0; e < 3; ++e) {
        a.q_stride[e] = step(q, e); a.q_out_stride[e] = step(qo, e);
        if (k.defined()) { a.k_stride[e] = step(k, e); a.k_out_stride[e] = step(ko, e); }
    }
    a.turns = (const uint64_t*)r.turns.data_ptr();
    if (r.pos.defined()) {
        a.positions = r.pos.data_ptr();
        a.positions64 = r.pos.scalar_type() == at::kLong;
        a.pos_stride[0] = r.pos.dim() == 2 && r.pos.size(0) > 1 ? r.pos.stride(0) : 0;
        a.pos_stride[1] = r.pos.size(-1) > 1 ? r.pos.stride(-1) : 0;
    }
    a.dtype = dtype_of(q); a.B = small(q.size(0), "B"); a.T = small(q.size(1), "T"); a.H = small(q.size(2), "H"); a.Hk = k.defined() ? small(k.size(2), "Hk") : 0;
    a.D = small(q.size(3), "D"); a.rd = (int)r.rd; a.interleaved = r.interleaved; a.inverse = inverse; a.gain = (float)r.gain;
    call(lib.rotary(&a, stream_of(q)), "xva_rotary");
    return {qo, ko};
}

struct Rotary : torch::autograd::Function<Rotary> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const MaybeTensor& k_, const Tensor& turns, const MaybeTensor& pos_, int64_t rd, bool interleaved,
                                 double gain) {
        const Tensor k = or_none(k_), pos = or_none(pos_);
        ctx->save_for_backward({turns, pos});
        ctx->saved_data["rd"] = rd; ctx->saved_data["interleaved"] = interleaved; ctx->saved_data["gain"] = gain;
        ctx->saved_data["k"] = k.defined();
        ctx->set_materialize_grads(false);
        const auto out = rotary_launch(q, k, {turns, pos, rd, interleaved, gain}, false, false);
        if (k.defined()) return {out.first, out.second};
        return {out.first};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const RotaryArgs r = {saved[0], saved[1], ctx->saved_data["rd"].toInt(), ctx->saved_data["interleaved"].toBool(), ctx->saved_data["gain"].toDouble()};
        const bool both = ctx->saved_data["k"].toBool();
        Tensor dq = grads[0], dk = both ? grads[1] : Tensor();
        variable_list out(7);
        if (dq.defined()) {
            const auto got = rotary_launch(dq, dk, r, true, false);
            out[0] = got.first; out[1] = got.second;
        } else if (dk.defined()) out[1] = rotary_launch(dk, Tensor(), r, true, false).first;
        return once(out, grads, true);
    }
};

variable_list rotary(const Tensor& turns, int64_t rd, bool interleaved, double gain, const Tensor& q, const MaybeTensor& k_, const MaybeTensor& pos_, bool inplace) {
    const Tensor k = or_none(k_), pos = or_none(pos_);
    on_one_device(q, {k, pos, turns});
    REFUSE(q.dim() != 4 || (k.defined() && (k.dim() != 4 || k.size(0) != q.size(0) || k.size(1) != q.size(1) || k.size(3) != q.size(3))), "q ", q.sizes(), ", k ",
           k.defined() ? c10::str(k.sizes()) : std::string("None"), ": (B, T, heads, D)");
    REFUSE(dtype_of(q) < 0 || (k.defined() && k.scalar_type() != q.scalar_type()), "q is ", q.scalar_type(), ", k ", k.defined() ? k.scalar_type() : q.scalar_type());
    REFUSE(rd > q.size(3), "rotary_dim ", rd, " of heads of ", q.size(3));
    if (pos.defined()) {
        REFUSE(pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong, "positions: int32 or int64, got ", pos.scalar_type());
        REFUSE((pos.dim() != 1 && pos.dim() != 2) || (pos.size(-1) != 1 && pos.size(-1) != q.size(1)) || (pos.dim() == 2 && pos.size(0) != 1 && pos.size(0) != q.size(0)),
               "positions ", pos.sizes(), " of (", q.size(0), ", ", q.size(1), ") rows");
    }
    if (wants_grad({q, k})) {
        REFUSE(inplace, "inplace: no gradient");
        return Rotary::apply(q, maybe(k), turns, maybe(pos), rd, interleaved, gain);
    }
    if (inplace) {
        REFUSE(q.stride(3) != 1 || (k.defined() && k.stride(3) != 1), "inplace: a contiguous last dimension");
        for (const Tensor& t : {q, k}) REFUSE(t.defined() && overlap(t, Tensor()) != APART, "inplace: heads of an expanded or overlapping tensor lie on each other, or may");
        REFUSE(k.defined() && overlap(q, k) != APART, "inplace: q and k share memory, or may");
        for (const Tensor& t : {q, k})
            if (t.defined()) t.unsafeGetTensorImpl()->bump_version();       // (a graph that saved it says so when it is run)
    }
    const auto out = rotary_launch(q, k, {turns, pos, rd, interleaved, gain}, false, inplace);
    if (k.defined()) return {out.first, out.second};
    return {out.first};
}

// ------------------------------------------------------------------------------------------------------------------ differential attention ----
// as the kernels read it: 16-byte rows, 64 of them and their maps within 32-bit offsets
Tensor wide(const Tensor& t) {
    bool ok = t.stride(-1) == 1 && (uintptr_t)t.data_ptr() % 16 == 0 && step(t, 1) < (1 << 24) && (t.dim() < 5 || step(t, 3) < (1 << 24));
    for (int e = 0; e + 1 < t.dim(); ++e) ok = ok && step(t, e) % 8 == 0;
    if (ok) return t;
    return aligned(t.contiguous());
}
xva_diff_attention_args diff_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const Tensor& ql, const Tensor& kl, bool causal, double scale) {
    xva_diff_attention_args a = {};
    a.q = ptr(q); a.k = ptr(k); a.v = ptr(v); a.lam = ptr(lam); a.lam_dtype = dtype_of(lam); a.q_lens = (const int32_t*)ptr(ql); a.k_lens = (const int32_t*)ptr(kl);
    for (int e = 0; e < 4; ++e) { a.q_stride[e] = step(q, e); a.k_stride[e] = step(k, e); }
    for (int e = 0; e < 3; ++e) a.v_stride[e] = step(v, e);
    a.dtype = dtype_of(q); a.B = small(q.size(0), "B"); a.Tq = small(q.size(1), "Tq"); a.Tk = small(k.size(1), "Tk"); a.H = small(q.size(2), "H"); a.Hk = small(k.size(2), "Hk");
    a.d = small(q.size(4), "d"); a.causal = causal; a.scale = (float)scale;
    return a;
}
// (out, maps, lse); the last two only with `train`
variable_list diff_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const Tensor& ql, const Tensor& kl, bool causal, double scale, bool train) {
    const c10::DeviceGuard guard(q.device());
    const int64_t B = q.size(0), Tq = q.size(1), H = q.size(2), d = q.size(4);
    const Tensor out = at::empty({B, Tq, H, 2 * d}, q.options());
    const Tensor maps = train ? at::empty({2, B, Tq, H, 2 * d}, q.options()) : Tensor(), lse = train ? floats({2, B, H, Tq}, q) : Tensor();
    xva_diff_attention_args a = diff_args(q, k, v, lam, ql, kl, causal, scale);
    a.out = ptr(out); a.maps = ptr(maps); a.lse = (float*)ptr(lse);
    for (int e = 0; e < 3; ++e) a.out_stride[e] = step(out, e);
    const int64_t n = lib.diff_ws(&a, 0);
    const Tensor ws = workspace(n, q);
    call(lib.diff_fwd(&a, ptr(ws), n, stream_of(q)), "xva_diff_attention_fwd");
    return {out, maps, lse};
}

struct DiffAttention : torch::autograd::Function<DiffAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const MaybeTensor& ql_, const MaybeTensor& kl_, bool causal,
                          double scale) {
        const Tensor ql = or_none(ql_), kl = or_none(kl_);
        const variable_list out = diff_forward(q, k, v, lam, ql, kl, causal, scale, true);
        ctx->save_for_backward({q, k, v, lam, out[1], out[2], ql, kl});
        ctx->saved_data["causal"] = causal; ctx->saved_data["scale"] = scale;
        return out[0];
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &lam = s[3];
        const c10::DeviceGuard guard(q.device());
        const Tensor dout = wide(grads[0].to(q.scalar_type()));
        const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), q.options()), dv = at::empty(v.sizes(), q.options()), dlam = at::empty(lam.sizes(), lam.options());
        if (q.numel() == 0) {
            dk.zero_(); dv.zero_(); dlam.zero_();
        } else {
            xva_diff_attention_args a = diff_args(q, k, v, lam, s[6], s[7], ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
            a.maps = ptr(s[4]); a.lse = (float*)ptr(s[5]); a.dout = ptr(dout); a.dq = ptr(dq); a.dk = ptr(dk); a.dv = ptr(dv); a.dlam = ptr(dlam);
            for (int e = 0; e < 3; ++e) a.dout_stride[e] = step(dout, e);
            const int64_t n = lib.diff_ws(&a, 1);
            const Tensor ws = workspace(n, q);
            call(lib.diff_bwd(&a, ptr(ws), n, stream_of(q)), "xva_diff_attention_bwd");
        }
        return once({dq, dk, dv, dlam, Tensor(), Tensor(), Tensor(), Tensor()}, grads);
    }
};

Tensor differential_attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& lam_, c10::optional<double> scale_, bool causal, const MaybeTensor& ql_,
                              const MaybeTensor& kl_) {
    Tensor ql = or_none(ql_), kl = or_none(kl_);
    on_one_device(q_, {k_, v_, lam_, ql, kl});
    REFUSE(q_.dim() != 5 || k_.dim() != 5 || v_.dim() != 4 || q_.size(3) != 2 || k_.size(3) != 2, "q ", q_.sizes(), " (B, Tq, H, 2, d), k ", k_.sizes(), " (B, Tk, Hk, 2, d), v ",
           v_.sizes(), " (B, Tk, Hk, 2 d)");
    const int64_t B = q_.size(0), H = q_.size(2), d = q_.size(4), Tk = k_.size(1), Hk = k_.size(2);
    REFUSE(k_.size(0) != B || k_.size(4) != d || v_.size(0) != B || v_.size(1) != Tk || v_.size(2) != Hk || v_.size(3) != 2 * d, "q ", q_.sizes(), ", k ", k_.sizes(), ", v ",
           v_.sizes(), " do not belong together");
    REFUSE(Hk < 1 || H < 1 || H % Hk, H, " query heads on ", Hk, " key heads");
    REFUSE(d % 8 || d < 8 || d > 64, "head width ", d, ": a multiple of 8 up to 64");
    REFUSE(dtype_of(q_) < 1 || k_.scalar_type() != q_.scalar_type() || v_.scalar_type() != q_.scalar_type(), "q, k, v are ", q_.scalar_type(), ", ", k_.scalar_type(), ", ",
           v_.scalar_type(), ": one of bf16, fp16");
    REFUSE(lam_.dim() != 1 || lam_.size(0) != H || !lam_.is_floating_point(), "lam ", lam_.sizes(), " ", lam_.scalar_type(), ": (", H, ",), a float type");
    const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)d);
    REFUSE(!(scale > 0.0 && std::isfinite(scale)), "scale ", scale);
    const c10::DeviceGuard guard(q_.device());
    ql = lengths(ql, B, q_.size(1), "q_lens"); kl = lengths(kl, B, Tk, "k_lens");
    const Tensor q = wide(q_), k = wide(k_), v = wide(v_), lam = dtype_of(lam_) < 0 ? fp32(lam_) : lam_.contiguous();
    if (wants_grad({q, k, v, lam})) return DiffAttention::apply(q, k, v, lam, maybe(ql), maybe(kl), causal, scale);
    return diff_forward(q, k, v, lam, ql, kl, causal, scale, false)[0];
}

// ------------------------------------------------------------------------------------------------------------------------ gated recurrence ----
xva_recurrence_args rec_args(const Tensor& x, const Tensor& gate, const Tensor& lens, bool reverse, bool unit) {
    xva_recurrence_args a = {};
    a.x = ptr(x); a.gate = ptr(gate); a.lens = (const int32_t*)ptr(lens);
    for (int e = 0; e < 2; ++e) { a.x_stride[e] = step(x, e); a.gate_stride[e] = step(gate, e); }
    a.dtype = dtype_of(x); a.B = small(x.size(0), "B"); a.T = small(x.size(1), "T"); a.C = small(x.size(2), "C"); a.reverse = reverse; a.unit_gain = unit;
    return a;
}
// (h, last, states); the last one only with `train`
variable_list rec_forward(const Tensor& x, const Tensor& gate, const Tensor& h0, const Tensor& lens, bool reverse, bool unit, bool train) {
    const c10::DeviceGuard guard(x.device());
    xva_recurrence_args a = rec_args(x, gate, lens, reverse, unit);
    const Tensor h = at::empty(x.sizes(), x.options()), last = floats({x.size(0), x.size(2)}, x);
    const Tensor states = train ? floats({lib.rec_states(a.B, a.T, a.C)}, x) : Tensor();
    a.h = ptr(h); a.h0 = (const float*)ptr(h0); a.last = (float*)ptr(last); a.states = (float*)ptr(states);
    for (int e = 0; e < 2; ++e) a.h_stride[e] = step(h, e);
    const int64_t n = lib.rec_ws(a.B, a.T, a.C);
    const Tensor ws = workspace(n, x);
    call(lib.rec_fwd(&a, ptr(ws), n, stream_of(x)), "xva_recurrence_fwd");
    return {h, last, states};
}

struct Recurrence : torch::autograd::Function<Recurrence> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const MaybeTensor& h0_, const MaybeTensor& lens_, bool reverse, bool unit) {
        const Tensor h0 = or_none(h0_), lens = or_none(lens_);
        const variable_list out = rec_forward(x, gate, h0, lens, reverse, unit, true);
        ctx->save_for_backward({x, gate, out[2], lens});
        ctx->saved_data["reverse"] = reverse; ctx->saved_data["unit"] = unit; ctx->saved_data["h0"] = h0.defined();
        ctx->set_materialize_grads(false);
        return {out[0], out[1]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Tensor &x = s[0], &gate = s[1];
        const c10::DeviceGuard guard(x.device());
        xva_recurrence_args a = rec_args(x, gate, s[3], ctx->saved_data["reverse"].toBool(), ctx->saved_data["unit"].toBool());
        const Tensor dh = grads[0].defined() ? rows(grads[0].to(x.scalar_type())) : at::zeros({1, 1, x.size(2)}, x.options()).expand(x.sizes());
        const Tensor dlast = fp32(grads[1]);
        const Tensor dx = at::empty(x.sizes(), x.options()), dgate = at::empty(x.sizes(), x.options());
        const Tensor dh0 = ctx->saved_data["h0"].toBool() ? floats({x.size(0), x.size(2)}, x) : Tensor();
        a.states = (float*)ptr(s[2]); a.dh = ptr(dh); a.dlast = (const float*)ptr(dlast); a.dx = ptr(dx); a.dgate = ptr(dgate); a.dh0 = (float*)ptr(dh0);
        for (int e = 0; e < 2; ++e) { a.dh_stride[e] = step(dh, e); a.dx_stride[e] = step(dx, e); a.dgate_stride[e] = step(dgate, e); }
        const int64_t n = lib.rec_ws(a.B, a.T, a.C);
        const Tensor ws = workspace(n, x);
        call(lib.rec_bwd(&a, ptr(ws), n, stream_of(x)), "xva_recurrence_bwd");
        return once({dx, dgate, dh0, Tensor(), Tensor(), Tensor()}, grads);
    }
};

std::tuple<Tensor, Tensor> gated_recurrence(const Tensor& x_, const Tensor& gate_, const MaybeTensor& h0_, const MaybeTensor& lens_, bool reverse, const std::string& gain) {
    Tensor h0 = or_none(h0_), lens = or_none(lens_);
    on_one_device(x_, {gate_, h0, lens});
    REFUSE(x_.dim() != 3 || gate_.sizes() != x_.sizes(), "x ", x_.sizes(), ", gate ", gate_.sizes(), ": (B, T, C)");
    REFUSE(dtype_of(x_) < 0 || gate_.scalar_type() != x_.scalar_type(), "x is ", x_.scalar_type(), ", gate ", gate_.scalar_type());
    REFUSE(gain != "convex" && gain != "unit", "gain ", gain, ": convex or unit");
    REFUSE(x_.size(2) < 1, "x ", x_.sizes(), ": no channels");
    REFUSE(h0.defined() && (h0.dim() != 2 || h0.size(0) != x_.size(0) || h0.size(1) != x_.size(2) || !h0.is_floating_point()), "h0 ", h0.sizes(), ": (", x_.size(0), ", ",
           x_.size(2), "), a float type");
    const c10::DeviceGuard guard(x_.device());
    lens = lengths(lens, x_.size(0), x_.size(1), "lens");
    const Tensor x = rows(x_), gate = rows(gate_);
    h0 = fp32(h0);
    const bool unit = gain == "unit";
    const variable_list out = wants_grad({x, gate, h0}) ? Recurrence::apply(x, gate, maybe(h0), maybe(lens), reverse, unit) : rec_forward(x, gate, h0, lens, reverse, unit, false);
    return {out[0], out[1]};
}

// -------------------------------------------------------------------------------------------------------------------------------- group norm ----
struct NormHow { int64_t groups; int act; double eps, slope; };

xva_group_norm_args norm_args(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& lens, const Tensor& stats, const NormHow& how) {
    xva_group_norm_args a = {};
    a.x = ptr(x); a.weight = (const float*)ptr(weight); a.bias = (const float*)ptr(bias); a.lens = (const int32_t*)ptr(lens);
    a.mean = (float*)ptr(stats); a.rstd = a.mean + x.size(0) * how.groups;
    for (int e = 0; e < 2; ++e) a.x_stride[e] = step(x, e);
    a.dtype = dtype_of(x); a.B = small(x.size(0), "B"); a.T = small(x.size(1), "T"); a.C = small(x.size(2), "C"); a.G = (int)how.groups; a.act = how.act;
    a.eps = (float)how.eps; a.slope = (float)how.slope;
    return a;
}
// as the kernels read it: one whose strides or address rule out vectors that its many channels, or groups, need is copied
Tensor norm_rows(const Tensor& t_, int64_t groups) {
    const Tensor t = rows(t_);
    const int64_t C = t.size(2), all = step(t, 0) | step(t, 1), wide = t.scalar_type() == at::kFloat ? 4 : 8, bytes = t.element_size();
    const auto at_address = [&](int64_t v) { return all % v == 0 && (uintptr_t)t.data_ptr() % (v * bytes) == 0; };
    const int64_t v = C % wide == 0 && at_address(wide) ? wide : (C % 2 == 0 && at_address(2) ? 2 : 1);
    return C / v <= 1024 && groups <= 2048 ? t : aligned(t.contiguous());
}
// (y, stats)
variable_list norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& lens, const NormHow& how) {
    const c10::DeviceGuard guard(x.device());
    const Tensor y = at::empty(x.sizes(), x.options()), stats = floats({2, x.size(0), how.groups}, x);
    xva_group_norm_args a = norm_args(x, weight, bias, lens, stats, how);
    a.out = ptr(y);
    for (int e = 0; e < 2; ++e) a.out_stride[e] = step(y, e);
    const int64_t n = lib.norm_ws(&a, 0);
    const Tensor ws = workspace(n, x);
    call(lib.norm_fwd(&a, ptr(ws), n, stream_of(x)), "xva_group_norm_act_fwd");
    return {y, stats};
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight_, const MaybeTensor& bias_, const MaybeTensor& lens_, int64_t groups, int64_t act,
                          double eps, double slope) {
        const Tensor weight = or_none(weight_), bias = or_none(bias_), lens = or_none(lens_);
        const variable_list out = norm_forward(x, weight, bias, lens, {groups, (int)act, eps, slope});
        ctx->save_for_backward({x, weight, bias, lens, out[1]});
        ctx->saved_data["groups"] = groups; ctx->saved_data["act"] = act; ctx->saved_data["eps"] = eps; ctx->saved_data["slope"] = slope;
        return out[0];
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Tensor &x = s[0], &weight = s[1], &bias = s[2];
        const c10::DeviceGuard guard(x.device());
        auto& d = ctx->saved_data;
        xva_group_norm_args a = norm_args(x, weight, bias, s[3], s[4], {d["groups"].toInt(), (int)d["act"].toInt(), d["eps"].toDouble(), d["slope"].toDouble()});
        const Tensor dy = norm_rows(grads[0].to(x.scalar_type()), a.G), dx = at::empty(x.sizes(), x.options());
        // (needs_input_grad counts the inputs that were there)
        const Tensor dw = weight.defined() && ctx->needs_input_grad(1) ? at::empty(weight.sizes(), weight.options()) : Tensor();
        const Tensor db = bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1) ? at::empty(bias.sizes(), bias.options()) : Tensor();
        a.dy = ptr(dy); a.out = ptr(dx); a.dweight = (float*)ptr(dw); a.dbias = (float*)ptr(db);
        for (int e = 0; e < 2; ++e) { a.dy_stride[e] = step(dy, e); a.out_stride[e] = step(dx, e); }
        const int64_t n = lib.norm_ws(&a, 1);
        const Tensor ws = workspace(n, x);
        call(lib.norm_bwd(&a, ptr(ws), n, stream_of(x)), "xva_group_norm_act_bwd");
        return once({dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, grads);
    }
};

Tensor group_norm_act(const Tensor& x_, int64_t groups, const MaybeTensor& weight_, const MaybeTensor& bias_, const MaybeTensor& lens_, double eps, const std::string& act,
                      double slope) {
    static const char* const acts[] = {"none", "relu", "lrelu", "tanh", "silu", "gelu"};
    Tensor weight = or_none(weight_), bias = or_none(bias_), lens = or_none(lens_);
    const bool flat = x_.dim() == 2;
    REFUSE((x_.dim() != 2 && x_.dim() != 3) || (flat && lens.defined()), "x ", x_.sizes(), ": (B, T, C), or (B, C) without lens");
    on_one_device(x_, {weight, bias, lens});
    REFUSE(dtype_of(x_) < 0, "x is ", x_.scalar_type());
    int which = 0;
    while (which < 6 && act != acts[which]) ++which;
    REFUSE(which == 6, "act ", act, ": one of none, relu, lrelu, tanh, silu, gelu");
    const int64_t C = x_.size(-1);
    REFUSE(groups < 1 || C < 1 || C % groups, C, " channels in ", groups, " groups");
    REFUSE(!(eps >= 0.0 && std::isfinite(eps)), "eps ", eps);
    for (const Tensor& t : {weight, bias}) REFUSE(t.defined() && (t.dim() != 1 || t.size(0) != C || !t.is_floating_point()), "weight / bias ", t.sizes(), ": (", C, ",), a float type");
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = norm_rows(flat ? x_.unsqueeze(1) : x_, groups);
    lens = lengths(lens, x.size(0), x.size(1), "lens");
    weight = fp32(weight); bias = fp32(bias);
    const NormHow how = {groups, which, eps, slope};
    const Tensor y = wants_grad({x, weight, bias}) ? GroupNormAct::apply(x, maybe(weight), maybe(bias), maybe(lens), groups, (int64_t)which, eps, slope) : norm_forward(x, weight, bias, lens, how)[0];
    return flat ? y.squeeze(1) : y;
}

template <class F> void set(F& f, const py::dict& d, const char* name) { f = reinterpret_cast<F>(d[name].cast<uintptr_t>()); }
}   // namespace

PYBIND11_MODULE(_seq_torch, m) {
    // entries: name -> address of libxvahip.so's entry points; error: the exception type to raise
    m.def("bind", [](const py::dict& e, py::object error) {
        static py::object* type = nullptr;
        type = new py::object(error);                 // (lives as long as the process)
        py::register_exception_translator([](std::exception_ptr p) {
            try { if (p) std::rethrow_exception(p); }
            catch (const Failure& f) { PyErr_SetString(type->ptr(), f.what()); }
        });
        set(lib.last_error, e, "xva_last_error"); set(lib.rotary, e, "xva_rotary");
        set(lib.norm_ws, e, "xva_group_norm_workspace_bytes"); set(lib.norm_fwd, e, "xva_group_norm_act_fwd"); set(lib.norm_bwd, e, "xva_group_norm_act_bwd");
        set(lib.rec_ws, e, "xva_recurrence_workspace_bytes"); set(lib.rec_states, e, "xva_recurrence_state_floats"); set(lib.rec_fwd, e, "xva_recurrence_fwd");
        set(lib.rec_bwd, e, "xva_recurrence_bwd"); set(lib.diff_ws, e, "xva_diff_attention_workspace_bytes"); set(lib.diff_fwd, e, "xva_diff_attention_fwd");
        set(lib.diff_bwd, e, "xva_diff_attention_bwd");
    });
    m.def("rotary", &rotary);
    m.def("overlap", [](const Tensor& q, const MaybeTensor& k) { return (int)overlap(q, or_none(k)); });      // 0: apart, 1: elements meet, 2: not known
    m.def("differential_attention", &differential_attention);
    m.def("gated_recurrence", &gated_recurrence);
    m.def("group_norm_act", &group_norm_act);
}
