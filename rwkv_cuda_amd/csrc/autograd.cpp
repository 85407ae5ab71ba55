// The operators as torch::autograd::Function, over the C ABI of librwkv_hip.so: what the Python classes of rwkv_cuda_amd/*.py
// run.  Everything the reference's wrapper classes do on the host (checks, allocations, saved tensors, the launches of one
// direction) happens here in one call from Python and one from the autograd engine, which needs no interpreter for it: for the
// small shapes the host is what a step waits for.  With the classes in Python and the library called through ctypes, wkv4 B4 T512
// C768, forward + backward, took 147 us, of which the GPU worked 27; it takes 72 (most of it torch.autograd.grad and the hand-over
// to the engine's thread).  rwkv7 B1 T16 C2048, forward: 33 -> 9 us.
#include <torch/extension.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include "rwkv_hip.h"

namespace py = pybind11;

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;

constexpr auto BF = torch::kBFloat16;
constexpr auto F32 = torch::kFloat32;
constexpr int64_t HEAD = 64, MAX_HEAD = 128, CHUNK7 = 16;

// the reference's wrappers use bare asserts (e.g. wkv6_state/run.py:84-100): an AssertionError keeps that contract.  Only
// called from the forwards, which run under the interpreter's lock.
void require(bool cond, const std::string& msg) {
    if (cond) return;
    PyErr_SetString(PyExc_AssertionError, msg.c_str());
    throw py::error_already_set();
}
std::string str(c10::ScalarType t) { return std::string("torch.") + (t == BF ? "bfloat16" : (t == F32 ? "float32" : c10::toString(t))); }
// one device, one dtype, contiguous
void check(std::initializer_list<std::pair<const Tensor*, const char*>> ts, c10::ScalarType dt, const Tensor& first) {
    for (const auto& t : ts) {
        const Tensor& x = *t.first;
        if (x.is_cuda() && x.scalar_type() == dt && x.is_contiguous() && x.device() == first.device()) continue;
        const std::string n = t.second;
        require(x.is_cuda() && first.is_cuda(), "tensors must live on a HIP device: there is no CPU path");
        require(x.scalar_type() == dt, n + ".dtype must be " + str(dt) + ", got " + str(x.scalar_type()));
        require(x.is_contiguous(), n + " must be contiguous");
        require(false, n + " is on " + x.device().str() + ", expected " + first.device().str());
    }
}
void check_head(int64_t C, int64_t H) {
    require(H > 0 && C % H == 0 && C / H <= MAX_HEAD, "C must be a multiple of H with a head size of at most 128");
}
// the package's own error type, in either direction: the engine's threads, which run the backwards, do not hold the interpreter's lock
[[noreturn]] void fail(const std::string& msg) {
    const py::gil_scoped_acquire lock;
    PyErr_SetString(py::module_::import("rwkv_cuda_amd._lib").attr("RwkvHipError").ptr(), msg.c_str());
    throw py::error_already_set();
}
// sizes as the C ABI takes them
int i32(int64_t x) {
    if (x <= 0 || x > std::numeric_limits<int>::max()) fail("size " + std::to_string(x) + " is outside 1 .. 2147483647");
    return static_cast<int>(x);
}
struct Dims { int B, T, C, H; };
Dims dims(int64_t B, int64_t T, int64_t C, int64_t H) { return {i32(B), i32(T), i32(C), i32(H)}; }

void* stream_of(const Tensor& t) { return static_cast<void*>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream()); }
void ok(int status) {
    if (status == RWKV_OK) return;
    std::string msg = "librwkv_hip: status " + std::to_string(status) + ": " + rwkv_strerror(status);
    if (status == RWKV_ERR_LAUNCH) msg += " (hipError " + std::to_string(rwkv_last_hip_error()) + ")";
    fail(msg);
}

// typed pointers; an undefined tensor is NULL
struct Ptr {
    void* p;
    template <class T> operator T*() const { return static_cast<T*>(p); }
};
Ptr P(const Tensor& t) { return {t.defined() ? t.data_ptr() : nullptr}; }
Tensor bytes(const Tensor& like, size_t n) { return at::empty({static_cast<int64_t>(n)}, like.options().dtype(torch::kUInt8)); }
bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!c10::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts) if (t->requires_grad()) return true;
    return false;
}
void put(AutogradContext* ctx, std::initializer_list<std::pair<const char*, int64_t>> xs) { for (const auto& x : xs) ctx->saved_data[x.first] = x.second; }
int64_t get(AutogradContext* ctx, const char* n) { return ctx->saved_data[n].toInt(); }
Dims get_dims(AutogradContext* ctx) { return dims(get(ctx, "B"), get(ctx, "T"), get(ctx, "C"), get(ctx, "H")); }
const Tensor NONE;

// --------------------------------------------------------------------------------------------- wkv (wkv/run.py:89-117)
struct Wkv4 : Function<Wkv4> {
    static Tensor forward(AutogradContext* ctx, int64_t B, int64_t T, int64_t C, const Tensor& w_, const Tensor& u_, const Tensor& k_, const Tensor& v_) {
        const Tensor w = w_.contiguous(), u = u_.contiguous(), k = k_.contiguous(), v = v_.contiguous();
        check({{&w, "w"}, {&u, "u"}, {&k, "k"}, {&v, "v"}}, F32, w);
        require(k.numel() == B * T * C && v.numel() == k.numel() && w.numel() == C && u.numel() == C, "shape mismatch");
        const Guard guard(w.device());
        Tensor y = at::empty({B, T, C}, k.options());
        // w = -exp(w) of the reference wrapper (:95) happens inside the kernels
        ok(rwkv_wkv4raw_forward(stream_of(w), i32(B), i32(T), i32(C), P(w), P(u), P(k), P(v), P(y)));
        ctx->save_for_backward({w, u, k, v});
        put(ctx, {{"B", B}, {"T", T}, {"C", C}});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const Tensor &w = s[0], &u = s[1], &k = s[2], &v = s[3], gy = g[0].contiguous();
        const int B = i32(get(ctx, "B")), T = i32(get(ctx, "T")), C = i32(get(ctx, "C"));
        const Guard guard(w.device());
        Tensor gw = at::empty({C}, w.options()), gu = at::empty({C}, w.options());      // summed over the batch by the library (:115-116)
        Tensor gk = at::empty({B, T, C}, w.options()), gv = at::empty({B, T, C}, w.options());
        const size_t n = rwkv_wkv4raw_backward_workspace_bytes(B, T, C);
        Tensor ws = bytes(w, n);
        ok(rwkv_wkv4raw_backward(stream_of(w), B, T, C, P(w), P(u), P(k), P(v), P(gy), P(gw), P(gu), P(gk), P(gv), P(ws), n));
        return {NONE, NONE, NONE, gw, gu, gk, gv};
    }
};
Tensor wkv4_op(int64_t B, int64_t T, int64_t C, const Tensor& w, const Tensor& u, const Tensor& k, const Tensor& v) { return Wkv4::apply(B, T, C, w, u, k, v); }

// --------------------------------------------------------------------------------------------- depthwise_conv1d (run.py:76-102)
constexpr int64_t T_MAX = 4096;
struct TimeX : Function<TimeX> {
    static Tensor forward(AutogradContext* ctx, const Tensor& w_, const Tensor& k_, int64_t B, int64_t C, int64_t T, double eps) {
        require(T % 4 == 0 && T <= T_MAX, "require T % 4 == 0 and T <= T_MAX");
        const Tensor w = w_.contiguous(), k = k_.contiguous();
        check({{&w, "w"}, {&k, "k"}}, F32, w);
        require(w.numel() == C * T && k.numel() == B * C * T, "shape mismatch");
        const Guard guard(w.device());
        Tensor x = at::empty({B, C, T}, k.options());
        ok(rwkv_timex_forward(stream_of(w), P(w), P(k), P(x), static_cast<float>(eps), i32(B), i32(C), i32(T)));
        ctx->save_for_backward({w, k});
        put(ctx, {{"B", B}, {"T", T}, {"C", C}});
        return x;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const Tensor &w = s[0], &k = s[1], gx = g[0].contiguous();
        const int B = i32(get(ctx, "B")), T = i32(get(ctx, "T")), C = i32(get(ctx, "C"));
        const Guard guard(w.device());
        Tensor gk = at::empty({B, C, T}, k.options()), gw = at::empty({C, T}, k.options());      // the sum over the batch of run.py:102 happens in the library
        const size_t n = rwkv_timex_backward_ws_bytes(B, C, T);
        const Tensor ws = n > 0 ? bytes(k, n) : Tensor();
        ok(rwkv_timex_backward_ws(stream_of(w), P(w), P(k), P(gx), P(gw), P(gk), B, C, T, P(ws), n));
        return {gw, gk, NONE, NONE, NONE, NONE};
    }
};
Tensor timex_op(const Tensor& w, const Tensor& k, int64_t B, int64_t C, int64_t T, double eps) { return TimeX::apply(w, k, B, C, T, eps); }

// --------------------------------------------------------------------------------------------- wkv5, fp32 (wkv5/run.py:469-504)
struct Wkv5F32 : Function<Wkv5F32> {
    static Tensor forward(AutogradContext* ctx, int64_t B, int64_t T, int64_t C, int64_t H, const Tensor& r, const Tensor& k, const Tensor& v,
                          const Tensor& w, const Tensor& u, int64_t flags, bool grad) {
        check({{&r, "r"}, {&k, "k"}, {&v, "v"}, {&w, "w"}, {&u, "u"}}, F32, r);
        check_head(C, H);
        require(r.numel() == B * T * C && k.numel() == r.numel() && v.numel() == r.numel() && w.numel() == C && u.numel() == C, "shape mismatch");
        const Guard guard(r.device());
        const Dims d = dims(B, T, C, H);
        Tensor y = at::empty({B, T, C}, r.options());
        // head size 64: the raw decay and the sums over the batch (:482-483,:497-501) are the library's; other head sizes, and
        // the sequential kernels on request, sit behind the reference's own signature
        const bool chunked = C == H * HEAD && !(flags & RWKV_FLAG_SWEEPS);
        if (chunked) {
            const size_t n = grad ? rwkv_wkv5f32s_saved_bytes(d.B, d.T, d.C, d.H) : 0;
            const Tensor saved = grad ? bytes(r, n) : Tensor();
            const size_t nw = rwkv_wkv5f32s_forward_workspace_bytes(d.B, d.T, d.C, d.H);
            const Tensor ws = nw > 0 ? bytes(r, nw) : Tensor();
            ok(rwkv_wkv5f32s_forward_ws(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(w), P(u), P(y), P(saved), n, P(ws), nw));
            if (grad) ctx->save_for_backward({r, k, v, w, u, saved});
        } else {
            const Tensor ew = w.exp().neg_(), eew = ew.exp();
            ok(rwkv_wkv5f32_forward(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(eew), P(u), P(y)));
            if (grad) ctx->save_for_backward({r, k, v, w, u, eew, ew});
        }
        put(ctx, {{"B", B}, {"T", T}, {"C", C}, {"H", H}, {"chunked", chunked}});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const Tensor &r = s[0], &k = s[1], &v = s[2], &w = s[3], &u = s[4], gy = g[0].contiguous();
        const Dims d = get_dims(ctx);
        const Guard guard(r.device());
        const auto o = r.options();
        Tensor gr = at::empty({d.B, d.T, d.C}, o), gk = at::empty({d.B, d.T, d.C}, o), gv = at::empty({d.B, d.T, d.C}, o), gw, gu;
        if (get(ctx, "chunked")) {
            const Tensor& saved = s[5];
            gw = at::empty(w.sizes(), o); gu = at::empty(u.sizes(), o);
            const size_t n = rwkv_wkv5f32s_backward_workspace_bytes(d.B, d.T, d.C, d.H);
            Tensor ws = bytes(r, n);
            ok(rwkv_wkv5f32s_backward(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(w), P(u), P(gy), P(gr), P(gk), P(gv), P(gw), P(gu),
                                      P(saved), saved.numel(), P(ws), n));
        } else {
            Tensor pw = at::empty({d.B, d.C}, o), pu = at::empty({d.B, d.C}, o);
            ok(rwkv_wkv5f32_backward(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(s[5]), P(s[6]), P(u), P(gy), P(gr), P(gk), P(gv), P(pw), P(pu)));
            gw = pw.sum(0).view(w.sizes()); gu = pu.sum(0).view(u.sizes());
        }
        return {NONE, NONE, NONE, NONE, gr, gk, gv, gw, gu, NONE, NONE};
    }
};
Tensor wkv5_f32_op(int64_t B, int64_t T, int64_t C, int64_t H, const Tensor& r, const Tensor& k, const Tensor& v, const Tensor& w, const Tensor& u, int64_t flags) {
    return Wkv5F32::apply(B, T, C, H, r, k, v, w, u, flags, wants_grad({&r, &k, &v, &w, &u}));
}

// --------------------------------------------------------------------------------------------- wkv5a, fp32 (wkv5a/run.py:100-154)
struct Wkv5A : Function<Wkv5A> {
    static Tensor forward(AutogradContext* ctx, const Tensor& r, const Tensor& k, const Tensor& v, const Tensor& w1, const Tensor& u1,
                          const Tensor& w2, const Tensor& u2, int64_t flags, bool grad) {
        check({{&r, "r"}, {&k, "k"}, {&v, "v"}, {&w1, "w1"}, {&u1, "u1"}, {&w2, "w2"}, {&u2, "u2"}}, F32, r);
        require(r.dim() == 3 && w1.dim() == 2, "r,k,v are [B,T,C]; w1,u1,w2,u2 are [H,N]");
        const int64_t B = r.size(0), T = r.size(1), C = r.size(2), H = w1.size(0);
        require(H > 0 && C % H == 0 && w1.size(1) == C / H && C / H <= MAX_HEAD, "w1 is [H, C/H] with a head size of at most 128");
        require(k.sizes() == r.sizes() && v.sizes() == r.sizes(), "shape mismatch");
        require(u1.sizes() == w1.sizes() && w2.sizes() == w1.sizes() && u2.sizes() == w1.sizes(), "shape mismatch");
        const Guard guard(r.device());
        const Dims d = dims(B, T, C, H);
        Tensor y = at::empty({B, T, C}, r.options());
        const bool chunked = C == H * HEAD && !(flags & RWKV_FLAG_SWEEPS);
        if (chunked) {
            const size_t n = grad ? rwkv_wkv5as_saved_bytes(d.B, d.T, d.C, d.H) : 0;
            const Tensor saved = grad ? bytes(r, n) : Tensor();
            const size_t nw = rwkv_wkv5as_forward_workspace_bytes(d.B, d.T, d.C, d.H);
            const Tensor ws = nw > 0 ? bytes(r, nw) : Tensor();
            ok(rwkv_wkv5as_forward_ws(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(w1), P(u1), P(w2), P(u2), P(y), P(saved), n, P(ws), nw));
            if (grad) ctx->save_for_backward({r, k, v, w1, u1, w2, u2, saved});
        } else {
            const Tensor ew1 = w1.exp().neg_(), eew1 = ew1.exp(), ew2 = w2.exp().neg_(), eew2 = ew2.exp();
            ok(rwkv_wkv5a_forward(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(eew1), P(u1), P(eew2), P(u2), P(y)));
            if (grad) ctx->save_for_backward({r, k, v, w1, u1, w2, u2, eew1, ew1, eew2, ew2});
        }
        put(ctx, {{"B", B}, {"T", T}, {"C", C}, {"H", H}, {"chunked", chunked}});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const Tensor &r = s[0], &k = s[1], &v = s[2], &w1 = s[3], &u1 = s[4], &w2 = s[5], &u2 = s[6], gy = g[0].contiguous();
        const Dims d = get_dims(ctx);
        const Guard guard(r.device());
        const auto o = r.options();
        Tensor gr = at::empty({d.B, d.T, d.C}, o), gk = at::empty({d.B, d.T, d.C}, o), gv = at::empty({d.B, d.T, d.C}, o);
        Tensor gp[4];                                     // w1, u1, w2, u2
        if (get(ctx, "chunked")) {
            const Tensor& saved = s[7];
            for (Tensor& x : gp) x = at::empty(w1.sizes(), o);                      // summed over the batch by the library (:150-153)
            const size_t n = rwkv_wkv5as_backward_workspace_bytes(d.B, d.T, d.C, d.H);
            Tensor ws = bytes(r, n);
            ok(rwkv_wkv5as_backward(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(w1), P(u1), P(w2), P(u2), P(gy), P(gr), P(gk), P(gv),
                                    P(gp[0]), P(gp[1]), P(gp[2]), P(gp[3]), P(saved), saved.numel(), P(ws), n));
        } else {
            for (Tensor& x : gp) x = at::empty({d.B, d.C}, o);
            ok(rwkv_wkv5a_backward(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(s[7]), P(s[8]), P(u1), P(s[9]), P(s[10]), P(u2), P(gy),
                                   P(gr), P(gk), P(gv), P(gp[0]), P(gp[1]), P(gp[2]), P(gp[3])));
            for (Tensor& x : gp) x = x.sum(0).view(w1.sizes());
        }
        return {gr, gk, gv, gp[0], gp[1], gp[2], gp[3], NONE, NONE};
    }
};
Tensor wkv5a_op(const Tensor& r, const Tensor& k, const Tensor& v, const Tensor& w1, const Tensor& u1, const Tensor& w2, const Tensor& u2, int64_t flags) {
    return Wkv5A::apply(r, k, v, w1, u1, w2, u2, flags, wants_grad({&r, &k, &v, &w1, &u1, &w2, &u2}));
}

// --------------------------------------------------------------------------------------------- wkv5, bf16 (wkv5_bf16/run.py:44-88)
struct Wkv5Bf16 : Function<Wkv5Bf16> {
    static Tensor forward(AutogradContext* ctx, int64_t B, int64_t T, int64_t C, int64_t H, const Tensor& r, const Tensor& k, const Tensor& v,
                          const Tensor& w, const Tensor& u, int64_t flags, bool grad) {
        check({{&r, "r"}, {&k, "k"}, {&v, "v"}, {&w, "w"}, {&u, "u"}}, BF, r);
        check_head(C, H);
        require(r.numel() == B * T * C && k.numel() == r.numel() && v.numel() == r.numel() && w.numel() == C && u.numel() == C, "shape mismatch");
        const Guard guard(r.device());
        const Dims d = dims(B, T, C, H);
        // ew = -exp(w.float()), eew = exp(ew) (:63-64) are made by the library into `decay` = [eew | ew]
        Tensor decay = at::empty({2 * C}, r.options().dtype(F32)), y = at::empty({B, T, C}, r.options());
        const bool whole = C == H * MAX_HEAD && flags == 0;
        const size_t n = C == H * HEAD || whole ? rwkv_wkv5s_saved_bytes(d.B, d.T, d.C, d.H) : 0;
        if (n > 0) {
            // head sizes 64 and 128: one forward and one reverse sweep; the forward keeps the state entering every 64th token
            // (at 128 only if a backward can follow)
            const bool keep = grad || !whole;
            const Tensor saved = keep ? bytes(r, n) : Tensor();
            const size_t nw = rwkv_wkv5s_blocks_workspace_bytes(d.B, d.T, d.C, d.H, 0);
            const Tensor ws = nw > 0 ? bytes(r, nw) : Tensor();
            ok(rwkv_wkv5s_forward_ws(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(w), P(u), P(y), P(decay), P(saved), keep ? n : 0, P(ws), nw, flags));
            if (keep) ctx->save_for_backward({r, k, v, decay, u, w, saved});
        } else {
            // heads of 128 channels with options run as four heads of 64 whose fp32 terms need scratch; every other size needs none
            const size_t nf = rwkv_wkv5_forward_workspace_bytes(d.B, d.T, d.C, d.H);
            Tensor ws = bytes(r, nf < 16 ? 16 : nf);
            ok(rwkv_wkv5raw_forward_ws(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(w), P(u), P(y), P(decay), P(ws), nf, flags));
            ctx->save_for_backward({r, k, v, decay, u});
        }
        put(ctx, {{"B", B}, {"T", T}, {"C", C}, {"H", H}, {"flags", flags}});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        const auto s = ctx->get_saved_variables();
        const Tensor &r = s[0], &k = s[1], &v = s[2], &decay = s[3], &u = s[4], gy = g[0].contiguous();
        const Dims d = get_dims(ctx);
        const unsigned flags = static_cast<unsigned>(get(ctx, "flags"));
        const Guard guard(r.device());
        const auto o = r.options();
        Tensor gr = at::empty({d.B, d.T, d.C}, o), gk = at::empty({d.B, d.T, d.C}, o), gv = at::empty({d.B, d.T, d.C}, o);
        Tensor gw = at::empty({d.H, d.C / d.H}, o), gu = at::empty({d.H, d.C / d.H}, o);       // summed over the batch by the library (:86-87)
        if (s.size() > 5) {
            const Tensor &w = s[5], &saved = s[6];
            // (at head size 128 without options the per-batch rows of gw and gu are all, and what blocks of time take)
            const size_t nb = rwkv_wkv5s_blocks_workspace_bytes(d.B, d.T, d.C, d.H, 1);
            const size_t n = nb > 0 ? nb : d.C == d.H * MAX_HEAD ? 4 * static_cast<size_t>(d.B) * d.C : rwkv_wkv5s_backward_workspace_bytes(d.B, d.T, d.C, d.H);
            Tensor ws = bytes(r, n);
            ok(rwkv_wkv5s_backward(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(w), P(decay), P(u), P(gy), P(gr), P(gk), P(gv), P(gw), P(gu),
                                   P(saved), saved.numel(), P(ws), n, flags));
        } else {
            const size_t n = rwkv_wkv5raw_backward_workspace_bytes(d.B, d.T, d.C, d.H);
            Tensor ws = bytes(r, n);
            ok(rwkv_wkv5raw_backward(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(decay), P(u), P(gy), P(gr), P(gk), P(gv), P(gw), P(gu),
                                     P(ws), n, flags));
        }
        return {NONE, NONE, NONE, NONE, gr, gk, gv, gw, gu, NONE, NONE};
    }
};
Tensor wkv5_bf16_op(int64_t B, int64_t T, int64_t C, int64_t H, const Tensor& r, const Tensor& k, const Tensor& v, const Tensor& w, const Tensor& u, int64_t flags) {
    return Wkv5Bf16::apply(B, T, C, H, r, k, v, w, u, flags, wants_grad({&r, &k, &v, &w, &u}));
}

// ------------------------------------------------------- wkv6 and wkv6_state, bf16 (wkv6/run.py:128-170, wkv6_state/run.py:80-124)
// (s: the initial state, undefined for wkv6; the saved variables are taken once: hooks on them run per taking, and a checkpoint
// refuses a second one)
variable_list wkv6_grads(AutogradContext* ctx, const Tensor& gy_, bool state) {
    const auto s = ctx->get_saved_variables();
    const Tensor &r = s[0], &k = s[1], &v = s[2], &w = s[3], &u = s[4], &saved = s[5], s0 = state ? s[6] : Tensor(), gy = gy_.contiguous();
    const Dims d = get_dims(ctx);
    const Guard guard(r.device());
    const auto o = r.options();
    Tensor gr = at::empty({d.B, d.T, d.C}, o), gk = at::empty({d.B, d.T, d.C}, o), gv = at::empty({d.B, d.T, d.C}, o), gw = at::empty({d.B, d.T, d.C}, o);
    const int64_t N = d.C / d.H;
    Tensor gu = at::empty({d.H, N}, o), gs = s0.defined() ? at::empty({d.B, d.H, N, N}, o) : Tensor();    // gu summed over the batch by the library (:169, :123)
    const size_t n = rwkv_wkv6f_backward_saved_workspace_bytes(d.B, d.T, d.C, d.H);
    Tensor ws = bytes(r, n);
    ok(rwkv_wkv6f_backward_saved(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(w), P(u), P(s0), P(gy), P(gr), P(gk), P(gv), P(gw), P(gu), P(gs),
                                 saved.numel() > 0 ? P(saved) : Ptr{nullptr}, saved.numel(), P(ws), n, static_cast<unsigned>(get(ctx, "flags"))));
    return {NONE, NONE, NONE, NONE, gr, gk, gv, gw, gu, gs, NONE};
}
Tensor wkv6_run(AutogradContext* ctx, int64_t B, int64_t T, int64_t C, int64_t H, const Tensor& r, const Tensor& k, const Tensor& v, const Tensor& w,
                const Tensor& u, const Tensor& s, int64_t flags) {
    check({{&r, "r"}, {&k, "k"}, {&v, "v"}, {&w, "w"}, {&u, "u"}}, BF, r);
    check_head(C, H);
    require(r.numel() == B * T * C && k.numel() == r.numel() && v.numel() == r.numel() && w.numel() == r.numel() && u.numel() == C, "shape mismatch");
    const Guard guard(r.device());
    const Dims d = dims(B, T, C, H);
    Tensor y = at::empty({B, T, C}, r.options());
    // the forward keeps the state entering every 64th token for the backward's single reverse sweep (no bytes for head sizes
    // and options that take the two-sweep kernels)
    const size_t n = rwkv_wkv6f_saved_bytes(d.B, d.T, d.C, d.H);
    Tensor saved = bytes(r, n);
    ok(rwkv_wkv6f_forward(stream_of(r), d.B, d.T, d.C, d.H, P(r), P(k), P(v), P(w), P(u), P(s), P(y), n > 0 ? P(saved) : Ptr{nullptr}, n,
                          static_cast<unsigned>(flags)));
    if (s.defined()) ctx->save_for_backward({r, k, v, w, u, saved, s});
    else ctx->save_for_backward({r, k, v, w, u, saved});
    put(ctx, {{"B", B}, {"T", T}, {"C", C}, {"H", H}, {"flags", flags}});
    return y;
}
struct Wkv6 : Function<Wkv6> {
    static Tensor forward(AutogradContext* ctx, int64_t B, int64_t T, int64_t C, int64_t H, const Tensor& r, const Tensor& k, const Tensor& v,
                          const Tensor& w, const Tensor& u, int64_t flags) {
        return wkv6_run(ctx, B, T, C, H, r, k, v, w, u, NONE, flags);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        variable_list x = wkv6_grads(ctx, g[0], false);
        x.erase(x.begin() + 9);
        return x;
    }
};
struct Wkv6State : Function<Wkv6State> {
    static Tensor forward(AutogradContext* ctx, int64_t B, int64_t T, int64_t C, int64_t H, const Tensor& r, const Tensor& k, const Tensor& v,
                          const Tensor& w, const Tensor& u, const Tensor& s, int64_t flags) {
        check({{&s, "s"}}, BF, r);
        check_head(C, H);
        require(s.numel() == B * C * (C / H), "shape mismatch");
        return wkv6_run(ctx, B, T, C, H, r, k, v, w, u, s, flags);
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) { return wkv6_grads(ctx, g[0], true); }
};
Tensor wkv6_op(int64_t B, int64_t T, int64_t C, int64_t H, const Tensor& r, const Tensor& k, const Tensor& v, const Tensor& w, const Tensor& u, int64_t flags) {
    return Wkv6::apply(B, T, C, H, r, k, v, w, u, flags);
}
Tensor wkv6_state_op(int64_t B, int64_t T, int64_t C, int64_t H, const Tensor& r, const Tensor& k, const Tensor& v, const Tensor& w, const Tensor& u,
                  const Tensor& s, int64_t flags) {
    return Wkv6State::apply(B, T, C, H, r, k, v, w, u, s, flags);
}

// --------------------------------------------- rwkv7 clamp-w (rwkv7_cuda_benchmark_state_passing.py:75-103, _state.py:75-102, .py:76-100)
// One body for the three siblings: s0 may be undefined (no state), passing = the final state is an output too.  r is
// [B,T,H*64] (flat: the functions) or [B,T,H,64] (the classes), the others either (the same memory); y has the shape of r, with
// `passing` always [B,T,H*64].  The checkpoint tensors `s` and `sa` are scratch
// whose layout belongs to the library.  The backward must run with the flags of the forward (the kernel families lay `s` out
// differently), so they ride on the context.
variable_list rwkv7_run(AutogradContext* ctx, const Tensor& s0, const Tensor& r, const Tensor& w, const Tensor& k, const Tensor& v, const Tensor& a,
                        const Tensor& b, int64_t flags, bool passing, bool flat, bool grad) {
    const auto dt = r.scalar_type();
    require(dt == BF || dt == F32, "r.dtype must be bfloat16 or float32, got " + str(dt));
    require(r.dim() == (flat ? 3 : 4), flat ? "r must be [B,T,H*64]" : "r must be [B,T,H,64]");
    require(flat ? r.size(2) % HEAD == 0 : r.size(3) == HEAD, "head size must be 64");
    const int64_t B = r.size(0), T = r.size(1), H = flat ? r.size(2) / HEAD : r.size(2);
    require(T % CHUNK7 == 0, "T must be a multiple of CHUNK_LEN");
    check({{&r, "r"}, {&w, "w"}, {&k, "k"}, {&v, "v"}, {&a, "a"}, {&b, "b"}}, dt, r);
    for (const Tensor* x : {&w, &k, &v, &a, &b}) require(x->numel() == r.numel(), "shape mismatch");
    if (s0.defined()) {
        check({{&s0, "s0"}}, F32, r);
        require(s0.sizes() == at::IntArrayRef({B, H, HEAD, HEAD}), "s0 must be [B,H,N,N] on the same device");
    }
    const Guard guard(r.device());
    const int b_ = i32(B), t_ = i32(T), h_ = i32(H);
    const auto f32 = r.options().dtype(F32);
    Tensor y = flat || passing ? at::empty({B, T, H * HEAD}, r.options()) : at::empty({B, T, H, HEAD}, r.options());
    Tensor sT = passing ? at::empty({B, H, HEAD, HEAD}, f32) : Tensor();
    void* st = stream_of(r);
    const bool sweeps = flags & RWKV_FLAG_SWEEPS;
    const size_t n = sweeps ? 0 : rwkv7_workspace_bytes(b_, t_, h_, 0);
    const Tensor ws = n > 0 ? bytes(r, n) : Tensor();
    if (!grad && !sweeps) {
        // no backward can follow: nothing is kept for one
        ok(rwkv7_forward_ws(st, b_, t_, h_, dt == F32, P(s0), P(r), P(w), P(k), P(v), P(a), P(b), P(y), P(sT), nullptr, nullptr, P(ws), n));
        if (passing) return {y, sT};
        return {y};
    }
    Tensor s = at::empty({B, H, T / CHUNK7, HEAD, HEAD}, f32), sa = at::empty({B, T, H, HEAD}, f32);
    if (!sweeps)
        ok(rwkv7_forward_ws(st, b_, t_, h_, dt == F32, P(s0), P(r), P(w), P(k), P(v), P(a), P(b), P(y), P(sT), P(s), P(sa), P(ws), n));
    else if (dt == BF)
        ok(rwkv7_statepassing_forward_ex(st, b_, t_, h_, P(s0), P(r), P(w), P(k), P(v), P(a), P(b), P(y), P(sT), P(s), P(sa), static_cast<unsigned>(flags)));
    else
        ok(rwkv7_statepassing_forward_f32_ex(st, b_, t_, h_, P(s0), P(r), P(w), P(k), P(v), P(a), P(b), P(y), P(sT), P(s), P(sa), static_cast<unsigned>(flags)));
    ctx->save_for_backward({r, w, k, v, a, b, s, sa});
    put(ctx, {{"B", B}, {"T", T}, {"H", H}, {"flags", flags}});
    if (passing) return {y, sT};
    return {y};
}
// ds0 (undefined without a state), dr, dw, dk, dv, da, db; dsT undefined: no gradient comes back for a final state
variable_list rwkv7_grads(AutogradContext* ctx, const Tensor& dy_, const Tensor& dsT_, bool state) {
    const auto x = ctx->get_saved_variables();
    const Tensor &r = x[0], &w = x[1], &k = x[2], &v = x[3], &a = x[4], &b = x[5], &s = x[6], &sa = x[7];
    const Tensor dy = dy_.contiguous(), dsT = dsT_.defined() ? dsT_.contiguous() : Tensor();
    const int B = i32(get(ctx, "B")), T = i32(get(ctx, "T")), H = i32(get(ctx, "H"));
    const Guard guard(r.device());
    Tensor ds0 = state ? at::empty({B, H, HEAD, HEAD}, r.options().dtype(F32)) : Tensor(), d[6];
    for (int i = 0; i < 6; ++i) d[i] = at::empty(x[i].sizes(), r.options());       // (each input may have come in either shape)
    void* st = stream_of(r);
    if (!(get(ctx, "flags") & RWKV_FLAG_SWEEPS)) {
        const size_t n = rwkv7_workspace_bytes(B, T, H, 1);
        const Tensor ws = n > 0 ? bytes(r, n) : Tensor();
        ok(rwkv7_backward_ws(st, B, T, H, r.scalar_type() == F32, P(r), P(w), P(k), P(v), P(a), P(b), P(dy), P(dsT), P(s), P(sa), P(ds0), P(d[0]), P(d[1]),
                             P(d[2]), P(d[3]), P(d[4]), P(d[5]), P(ws), n));
    } else if (r.scalar_type() == BF)
        ok(rwkv7_statepassing_backward_ex(st, B, T, H, P(r), P(w), P(k), P(v), P(a), P(b), P(dy), P(dsT), P(s), P(sa), P(ds0), P(d[0]), P(d[1]), P(d[2]),
                                          P(d[3]), P(d[4]), P(d[5]), static_cast<unsigned>(get(ctx, "flags"))));
    else
        ok(rwkv7_statepassing_backward_f32_ex(st, B, T, H, P(r), P(w), P(k), P(v), P(a), P(b), P(dy), P(dsT), P(s), P(sa), P(ds0), P(d[0]), P(d[1]), P(d[2]),
                                              P(d[3]), P(d[4]), P(d[5]), static_cast<unsigned>(get(ctx, "flags"))));
    return {ds0, d[0], d[1], d[2], d[3], d[4], d[5], NONE, NONE};
}
struct Rwkv7Passing : Function<Rwkv7Passing> {
    static variable_list forward(AutogradContext* ctx, const Tensor& s0, const Tensor& r, const Tensor& w, const Tensor& k, const Tensor& v, const Tensor& a,
                                 const Tensor& b, int64_t flags, bool flat, bool grad) { return rwkv7_run(ctx, s0, r, w, k, v, a, b, flags, true, flat, grad); }
    static variable_list backward(AutogradContext* ctx, variable_list g) { variable_list x = rwkv7_grads(ctx, g[0], g[1], true); x.push_back(NONE); return x; }
};
struct Rwkv7State : Function<Rwkv7State> {
    static variable_list forward(AutogradContext* ctx, const Tensor& s0, const Tensor& r, const Tensor& w, const Tensor& k, const Tensor& v, const Tensor& a,
                                 const Tensor& b, int64_t flags, bool flat, bool grad) { return rwkv7_run(ctx, s0, r, w, k, v, a, b, flags, false, flat, grad); }
    static variable_list backward(AutogradContext* ctx, variable_list g) { variable_list x = rwkv7_grads(ctx, g[0], NONE, true); x.push_back(NONE); return x; }
};
struct Rwkv7 : Function<Rwkv7> {
    static variable_list forward(AutogradContext* ctx, const Tensor& r, const Tensor& w, const Tensor& k, const Tensor& v, const Tensor& a, const Tensor& b,
                                 int64_t flags, bool flat, bool grad) { return rwkv7_run(ctx, NONE, r, w, k, v, a, b, flags, false, flat, grad); }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        variable_list x = rwkv7_grads(ctx, g[0], NONE, false);
        x.erase(x.begin());
        x.push_back(NONE);
        return x;
    }
};
std::tuple<Tensor, Tensor> rwkv7_passing_op(const Tensor& s0, const Tensor& r, const Tensor& w, const Tensor& k, const Tensor& v, const Tensor& a, const Tensor& b, int64_t flags, bool flat) {
    variable_list o = Rwkv7Passing::apply(s0, r, w, k, v, a, b, flags, flat, wants_grad({&s0, &r, &w, &k, &v, &a, &b}));
    return {o[0], o[1]};
}
Tensor rwkv7_state_op(const Tensor& s0, const Tensor& r, const Tensor& w, const Tensor& k, const Tensor& v, const Tensor& a, const Tensor& b, int64_t flags, bool flat) {
    return Rwkv7State::apply(s0, r, w, k, v, a, b, flags, flat, wants_grad({&s0, &r, &w, &k, &v, &a, &b}))[0];
}
Tensor rwkv7_op(const Tensor& r, const Tensor& w, const Tensor& k, const Tensor& v, const Tensor& a, const Tensor& b, int64_t flags, bool flat) {
    return Rwkv7::apply(r, w, k, v, a, b, flags, flat, wants_grad({&r, &w, &k, &v, &a, &b}))[0];
}

// --------------------------------------------------------------------------------------------- gated recurrence, attention, paged attention
using Maybe = c10::optional<Tensor>;
Tensor or_none(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
int dtype_of(const Tensor& t, const char* n, bool with_f32) {
    const auto d = t.scalar_type();
    require(d == BF || d == torch::kFloat16 || (with_f32 && d == F32), std::string(n) + ".dtype must be torch.bfloat16" + (with_f32 ? ", torch.float16 or torch.float32" : " or torch.float16") + ", got " + str(d));
    return d == BF ? RWKV_DTYPE_BF16 : (d == F32 ? RWKV_DTYPE_FP32 : RWKV_DTYPE_FP16);
}
// one device, one dtype, a dense innermost dimension
void check_rows(std::initializer_list<std::pair<const Tensor*, const char*>> ts, const Tensor& first) {
    for (const auto& t : ts) {
        const Tensor& x = *t.first;
        const std::string n = t.second;
        require(x.is_cuda() && first.is_cuda(), "tensors must live on a HIP device: there is no CPU path");
        require(x.device() == first.device(), n + " is on " + x.device().str() + ", expected " + first.device().str());
        require(x.scalar_type() == first.scalar_type(), n + ".dtype must be " + str(first.scalar_type()) + ", got " + str(x.scalar_type()));
        require(x.stride(-1) == 1 || x.size(-1) == 1, n + " must be dense in its last dimension");
    }
}
// an optional dense tensor of a given shape beside `first`
void check_side(const Tensor& x, const char* n, c10::ScalarType dt, at::IntArrayRef shape, const Tensor& first) {
    if (!x.defined()) return;
    check({{&x, n}}, dt, first);
    require(x.sizes() == shape, std::string(n) + " has the wrong shape");
}
// the strides of a dimension of size 1 are arbitrary: 0 for the kernels' checks
int64_t stride_of(const Tensor& x, int64_t d) { return x.size(d) == 1 ? 0 : x.stride(d); }
// a gradient that may be a view from anywhere, for kernels that read 16 bytes at once
Tensor on_16(const Tensor& x) { return reinterpret_cast<uintptr_t>(x.data_ptr()) & 15 ? x.clone() : x; }
// whether two tensors have memory in common (or may have: the spans that they lie in)
bool touch(const Tensor& a, const Tensor& b) {
    if (!a.storage().is_alias_of(b.storage())) return false;
    const auto span = [](const Tensor& x) {
        int64_t last = 0;
        for (int64_t d = 0; d < x.dim(); ++d) last += (x.size(d) - 1) * x.stride(d);
        const char* p = static_cast<const char*>(x.data_ptr());
        return std::make_pair(p, p + (last + 1) * static_cast<int64_t>(x.element_size()));
    };
    const auto s = span(a), t = span(b);
    return s.first < t.second && t.first < s.second;
}
// torch refuses to raise an inference tensor's version outside of inference mode: found out before the kernel writes it
void check_writable(const Tensor& x, const char* n) {
    require(!x.is_inference() || c10::InferenceMode::is_enabled(), std::string(n) + " is an inference tensor: it can be written in inference mode only");
}
// a tensor that a kernel writes: a graph that has saved it finds out
void written(const Tensor& x) { x.unsafeGetTensorImpl()->bump_version(); }
void once_only(const char* n) {
    if (c10::GradMode::is_enabled()) fail(std::string(n) + " has no second derivatives: its backward cannot run with create_graph");
}

rwkv_grec_args grec_args(const Tensor& w, const Tensor& x, int64_t gate, bool tied) {
    rwkv_grec_args a{};
    a.dtype = dtype_of(w, "w", true);
    a.gate = static_cast<int>(gate);
    a.tied = tied;
    a.B = i32(w.size(0)); a.T = i32(w.size(1)); a.C = i32(w.size(2));
    a.w = w.data_ptr(); a.w_sb = stride_of(w, 0); a.w_st = stride_of(w, 1);
    a.x = x.data_ptr(); a.x_sb = stride_of(x, 0); a.x_st = stride_of(x, 1);
    return a;
}
struct Grec : Function<Grec> {
    static variable_list forward(AutogradContext* ctx, const Tensor& w, const Tensor& x, const Maybe& h0_, const Maybe& doc_, int64_t gate, bool tied, bool grad) {
        const Tensor h0 = or_none(h0_), doc = or_none(doc_);
        require(w.dim() == 3 && x.sizes() == w.sizes(), "w and x are [B,T,C]");
        check_rows({{&w, "w"}, {&x, "x"}}, w);
        const int64_t B = w.size(0), T = w.size(1), C = w.size(2);
        check_side(h0, "h0", F32, {B, C}, w);
        check_side(doc, "doc", torch::kInt32, {B, T}, w);
        const Guard guard(w.device());
        rwkv_grec_args a = grec_args(w, x, gate, tied);
        Tensor y = at::empty({B, T, C}, w.options()), hT = at::empty({B, C}, w.options().dtype(F32)), saved;
        a.h0 = P(h0); a.doc = P(doc); a.y = P(y); a.hT = P(hT);
        if (grad) {
            a.saved_bytes = rwkv_grec_saved_bytes(a.B, a.T, a.C);
            saved = bytes(w, a.saved_bytes);
            a.saved = P(saved);
        }
        a.workspace_bytes = rwkv_grec_workspace_bytes(a.B, a.T, a.C);
        const Tensor ws = a.workspace_bytes > 0 ? bytes(w, a.workspace_bytes) : Tensor();
        a.workspace = P(ws);
        ok(rwkv_grec_forward(stream_of(w), &a));
        if (grad) ctx->save_for_backward({w, x, doc, saved});
        put(ctx, {{"gate", gate}, {"tied", tied}, {"state", h0.defined()}});
        ctx->set_materialize_grads(false);
        return {y, hT};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once_only("gated_recurrence");
        const auto s = ctx->get_saved_variables();
        const Tensor &w = s[0], &x = s[1], &doc = s[2], &saved = s[3];
        const Tensor dy = g[0].defined() ? g[0].contiguous() : Tensor(), dhT = g[1].defined() ? g[1].contiguous() : Tensor();
        const Guard guard(w.device());
        rwkv_grec_args a = grec_args(w, x, get(ctx, "gate"), get(ctx, "tied") != 0);
        Tensor dw = at::empty(w.sizes(), w.options()), dx = at::empty(w.sizes(), w.options());
        Tensor dh0 = get(ctx, "state") ? at::empty({a.B, a.C}, w.options().dtype(F32)) : Tensor();
        a.doc = P(doc); a.saved = P(saved); a.saved_bytes = saved.numel();
        a.dy = P(dy); a.dhT = P(dhT); a.dw = P(dw); a.dx = P(dx); a.dh0 = P(dh0);
        a.workspace_bytes = rwkv_grec_workspace_bytes(a.B, a.T, a.C);
        const Tensor ws = a.workspace_bytes > 0 ? bytes(w, a.workspace_bytes) : Tensor();
        a.workspace = P(ws);
        ok(rwkv_grec_backward(stream_of(w), &a));
        return {dw, dx, dh0, NONE, NONE, NONE, NONE};
    }
};
std::tuple<Tensor, Tensor> grec_op(const Tensor& w, const Tensor& x, const Maybe& h0, const Maybe& doc, int64_t gate, bool tied) {
    const Tensor h = or_none(h0);
    variable_list o = Grec::apply(w, x, h0, doc, gate, tied, wants_grad({&w, &x}) || (h.defined() && wants_grad({&h})));
    return {o[0], o[1]};
}
Tensor grec_step_op(const Tensor& w, const Tensor& x, const Tensor& h, const Tensor& out, int64_t gate, bool tied) {
    require(!wants_grad({&w, &x, &h, &out}), "STEP has no gradients: call it under torch.no_grad()");
    require(w.dim() == 2 && x.sizes() == w.sizes(), "w and x are [B,C]");
    const Tensor w3 = w.unsqueeze(1), x3 = x.unsqueeze(1);
    check_rows({{&w, "w"}, {&x, "x"}}, w);
    check_side(h, "h", F32, w.sizes(), w);
    check_side(out, "out", F32, w.sizes(), w);
    check_writable(out, "the new state");
    require(!touch(out, w) && !touch(out, x) && (out.data_ptr() == h.data_ptr() || !touch(out, h)), "out must be h, or share no memory with w, x and h");
    const Guard guard(w.device());
    rwkv_grec_args a = grec_args(w3, x3, gate, tied);
    Tensor y = at::empty(w.sizes(), w.options());
    a.h0 = P(h); a.hT = P(out); a.y = P(y);
    a.workspace_bytes = rwkv_grec_workspace_bytes(a.B, a.T, a.C);
    const Tensor ws = a.workspace_bytes > 0 ? bytes(w, a.workspace_bytes) : Tensor();
    a.workspace = P(ws);
    ok(rwkv_grec_forward(stream_of(w), &a));
    written(out);
    return y;
}

float scale_of(const c10::optional<double>& scale, int64_t N) { return static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(N))); }
rwkv_attn_args attn_args(const Tensor& q, const Tensor& k, const Tensor& v, double cap, double scale, bool causal) {
    rwkv_attn_args a{};
    a.dtype = dtype_of(q, "q", false);
    a.causal = causal;
    a.B = i32(q.size(0)); a.Tq = i32(q.size(1)); a.H = i32(q.size(2)); a.N = i32(q.size(3));
    a.Tk = i32(k.size(1)); a.Hk = i32(k.size(2));
    a.scale = static_cast<float>(scale); a.cap = static_cast<float>(cap);
    a.q = q.data_ptr(); a.q_sb = stride_of(q, 0); a.q_st = stride_of(q, 1); a.q_sh = stride_of(q, 2);
    a.k = k.data_ptr(); a.k_sb = stride_of(k, 0); a.k_st = stride_of(k, 1); a.k_sh = stride_of(k, 2);
    a.v = v.data_ptr(); a.v_sb = stride_of(v, 0); a.v_st = stride_of(v, 1); a.v_sh = stride_of(v, 2);
    return a;
}
struct Attn : Function<Attn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& doc_, const Maybe& prefix_, const Maybe& slopes_, double cap,
                          double scale, bool causal, bool grad) {
        const Tensor doc = or_none(doc_), prefix = or_none(prefix_), slopes = or_none(slopes_);
        const int64_t B = q.size(0), Tq = q.size(1), H = q.size(2), N = q.size(3), Tk = k.size(1);
        check_side(doc, "doc", torch::kInt32, {B, Tk}, q);
        check_side(prefix, "prefix", torch::kInt32, {B}, q);
        check_side(slopes, "slopes", F32, {H}, q);
        const Guard guard(q.device());
        rwkv_attn_args a = attn_args(q, k, v, cap, scale, causal);
        Tensor y = at::empty({B, Tq, H, N}, q.options()), rest, lse;
        a.doc = P(doc); a.prefix = P(prefix); a.slopes = P(slopes); a.y = P(y);
        if (grad) {
            rest = at::empty_like(y);
            lse = at::empty({B, H, Tq}, q.options().dtype(F32));
            a.y_rest = P(rest); a.lse = P(lse);
        }
        a.workspace_bytes = rwkv_attn_workspace_bytes(a.B, a.Tq, a.Tk, a.H, a.Hk, a.N, doc.defined(), 0);
        const Tensor ws = a.workspace_bytes > 0 ? bytes(q, a.workspace_bytes) : Tensor();
        a.workspace = P(ws);
        ok(rwkv_attn_forward(stream_of(q), &a));
        if (grad) ctx->save_for_backward({q, k, v, doc, prefix, slopes, y, rest, lse});
        ctx->saved_data["cap"] = cap;
        ctx->saved_data["scale"] = scale;
        put(ctx, {{"causal", causal}});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once_only("attention");
        const auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &y = s[6], &rest = s[7], &lse = s[8], dy = on_16(g[0].contiguous());
        const Guard guard(q.device());
        rwkv_attn_args a = attn_args(q, k, v, ctx->saved_data["cap"].toDouble(), ctx->saved_data["scale"].toDouble(), get(ctx, "causal") != 0);
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
        a.doc = P(s[3]); a.prefix = P(s[4]); a.slopes = P(s[5]); a.y = P(y); a.y_rest = P(rest); a.lse = P(lse);
        a.dy = P(dy); a.dq = P(dq); a.dk = P(dk); a.dv = P(dv);
        a.workspace_bytes = rwkv_attn_workspace_bytes(a.B, a.Tq, a.Tk, a.H, a.Hk, a.N, s[3].defined(), 1);
        const Tensor ws = bytes(q, a.workspace_bytes);
        a.workspace = P(ws);
        ok(rwkv_attn_backward(stream_of(q), &a));
        return {dq, dk, dv, NONE, NONE, NONE, NONE, NONE, NONE, NONE};
    }
};
Tensor attention_op(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& doc, const Maybe& prefix, const Maybe& slopes, double cap,
                    c10::optional<double> scale, bool causal) {
    require(q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes(), "q is [B,Tq,H,N], k and v are [B,Tk,Hk,N]");
    check_rows({{&q, "q"}, {&k, "k"}, {&v, "v"}}, q);
    const int64_t N = q.size(3);
    require(k.size(0) == q.size(0) && k.size(3) == N && k.size(1) >= q.size(1), "q is [B,Tq,H,N], k and v are [B,Tk,Hk,N] with Tk >= Tq");
    require(k.size(2) > 0 && q.size(2) % k.size(2) == 0, "H must be a multiple of Hk");
    require(N >= 8 && N <= MAX_HEAD && N % 8 == 0, "the head size must be a multiple of 8 up to 128");
    require(causal || !prefix.has_value(), "prefix goes with causal");
    require(cap == 0.0 || (cap >= 0x1p-20 && cap <= 4096.0), "cap must be 0, or from 2^-20 to 4096");
    const float sc = scale_of(scale, N);
    require(sc > 0.f && std::isfinite(sc), "scale must be positive");
    require(!slopes.has_value() || sc >= 0x1p-60f, "with slopes scale must be at least 2^-60");
    require(!slopes.has_value() || !wants_grad({&*slopes}), "slopes have no gradient");
    return Attn::apply(q, k, v, doc, prefix, slopes, cap, static_cast<double>(sc), causal, wants_grad({&q, &k, &v}));
}

Tensor paged_op(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& table, const Tensor& lens, const Maybe& k_, const Maybe& v_, const Maybe& slopes_,
                double cap, c10::optional<double> scale) {
    const Tensor k = or_none(k_), v = or_none(v_), slopes = or_none(slopes_);
    require(!wants_grad({&q, &kp, &vp}) && !(k.defined() && wants_grad({&k})) && !(v.defined() && wants_grad({&v})), "paged_attention has no gradients: call it under torch.no_grad()");
    require(q.dim() == 3 && kp.dim() == 4 && vp.sizes() == kp.sizes(), "q is [B,H,N], k_pages and v_pages are [P,page,Hk,N]");
    const int64_t B = q.size(0), H = q.size(1), N = q.size(2), page = kp.size(1), Hk = kp.size(2);
    check({{&q, "q"}}, q.scalar_type(), q);
    check_rows({{&q, "q"}, {&kp, "k_pages"}, {&vp, "v_pages"}}, q);
    require(kp.size(3) == N && Hk > 0 && H % Hk == 0, "H must be a multiple of Hk, and the head size that of the pages");
    require(N >= 8 && N <= MAX_HEAD && N % 8 == 0, "the head size must be a multiple of 8 up to 128");
    require(page > 0 && (page & (page - 1)) == 0, "page must be a power of two");
    require(table.dim() == 2, "table is [B,M]");
    check_side(table, "table", torch::kInt32, {B, table.size(1)}, q);
    check_side(lens, "lens", torch::kInt32, {B}, q);
    check_side(slopes, "slopes", F32, {H}, q);
    require(k.defined() == v.defined(), "k and v go together");
    check_side(k, "k", q.scalar_type(), {B, Hk, N}, q);
    check_side(v, "v", q.scalar_type(), {B, Hk, N}, q);
    if (k.defined()) check_writable(kp, "k_pages"), check_writable(vp, "v_pages");
    require(cap == 0.0 || (cap >= 0x1p-20 && cap <= 4096.0), "cap must be 0, or from 2^-20 to 4096");
    const Guard guard(q.device());
    rwkv_paged_args a{};
    a.dtype = dtype_of(q, "q", false);
    a.B = i32(B); a.H = i32(H); a.Hk = i32(Hk); a.N = i32(N); a.P = i32(kp.size(0)); a.page = i32(page); a.M = i32(table.size(1));
    a.scale = scale_of(scale, N); a.cap = static_cast<float>(cap);
    require(a.scale > 0.f && std::isfinite(a.scale), "scale must be positive");
    a.k_sp = stride_of(kp, 0); a.k_st = stride_of(kp, 1); a.k_sh = stride_of(kp, 2);
    a.v_sp = stride_of(vp, 0); a.v_st = stride_of(vp, 1); a.v_sh = stride_of(vp, 2);
    Tensor y = at::empty({B, H, N}, q.options());
    a.q = P(q); a.k_pages = P(kp); a.v_pages = P(vp); a.table = P(table); a.lens = P(lens); a.slopes = P(slopes); a.k = P(k); a.v = P(v); a.y = P(y);
    a.workspace_bytes = rwkv_paged_workspace_bytes(a.B, a.H, a.Hk, a.N, a.page, a.M);
    const Tensor ws = a.workspace_bytes > 0 ? bytes(q, a.workspace_bytes) : Tensor();
    a.workspace = P(ws);
    ok(rwkv_paged_attn(stream_of(q), &a));
    if (k.defined()) written(kp), written(vp);
    return y;
}

// --------------------------------------------------------------------------------------------- gated delta rule
rwkv_delta_args delta_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, double scale) {
    rwkv_delta_args a{};
    a.dtype = dtype_of(q, "q", false);
    a.B = i32(v.size(0)); a.T = i32(v.size(1)); a.H = i32(v.size(2)); a.N = i32(v.size(3)); a.Hk = i32(k.size(2));
    a.scale = static_cast<float>(scale);
    a.q = q.data_ptr(); a.q_sb = stride_of(q, 0); a.q_st = stride_of(q, 1); a.q_sh = stride_of(q, 2);
    a.k = k.data_ptr(); a.k_sb = stride_of(k, 0); a.k_st = stride_of(k, 1); a.k_sh = stride_of(k, 2);
    a.v = v.data_ptr(); a.v_sb = stride_of(v, 0); a.v_st = stride_of(v, 1); a.v_sh = stride_of(v, 2);
    a.g = g.data_ptr(); a.g_sb = stride_of(g, 0); a.g_st = stride_of(g, 1);
    a.beta = beta.data_ptr(); a.beta_sb = stride_of(beta, 0); a.beta_st = stride_of(beta, 1);
    return a;
}
// [B,T,heads,N] and [B,T,H]; returns the scale
float check_delta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, const c10::optional<double>& scale) {
    check_rows({{&q, "q"}, {&k, "k"}, {&v, "v"}, {&g, "g"}, {&beta, "beta"}}, q);
    const int64_t H = v.size(2), N = v.size(3);
    require(k.sizes() == q.sizes() && k.size(0) == v.size(0) && k.size(1) == v.size(1) && k.size(3) == N, "q and k are [B,T,Hk,N], v is [B,T,H,N]");
    require(k.size(2) > 0 && H % k.size(2) == 0, "H must be a multiple of Hk");
    require(N >= 8 && N <= MAX_HEAD && N % 8 == 0, "the head size must be a multiple of 8 up to 128");
    const std::vector<int64_t> gates = {v.size(0), v.size(1), H};
    require(g.sizes() == gates && beta.sizes() == gates, "g and beta are [B,T,H]");
    const float sc = scale_of(scale, N);
    require(sc > 0.f && std::isfinite(sc), "scale must be positive");
    return sc;
}
struct Delta : Function<Delta> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, const Maybe& s0_, const Maybe& doc_, double scale,
                                 bool grad) {
        const Tensor s0 = or_none(s0_), doc = or_none(doc_);
        const int64_t B = v.size(0), T = v.size(1), H = v.size(2), N = v.size(3);
        check_side(s0, "s0", F32, {B, H, N, N}, q);
        check_side(doc, "doc", torch::kInt32, {B, T}, q);
        const Guard guard(q.device());
        rwkv_delta_args a = delta_args(q, k, v, g, beta, scale);
        const Tensor start = s0.defined() ? on_16(s0) : Tensor();
        Tensor y = at::empty({B, T, H, N}, q.options()), sT = at::empty({B, H, N, N}, q.options().dtype(F32)), saved;
        a.s0 = P(start); a.doc = P(doc); a.y = P(y); a.sT = P(sT);
        if (grad) {
            a.saved_bytes = rwkv_delta_saved_bytes(a.B, a.T, a.H, a.Hk, a.N);
            saved = bytes(q, a.saved_bytes);
            a.saved = P(saved);
        }
        a.workspace_bytes = rwkv_delta_workspace_bytes(a.B, a.T, a.H, a.Hk, a.N, 0);
        const Tensor ws = a.workspace_bytes > 0 ? bytes(q, a.workspace_bytes) : Tensor();
        a.workspace = P(ws);
        ok(rwkv_delta_forward(stream_of(q), &a));
        if (grad) ctx->save_for_backward({q, k, v, g, beta, doc, saved});
        ctx->saved_data["scale"] = scale;
        put(ctx, {{"state", s0.defined()}});
        ctx->set_materialize_grads(false);
        return {y, sT};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        once_only("gated_delta");
        const auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &gate = s[3], &beta = s[4], &saved = s[6];
        const Tensor dy = g[0].defined() ? on_16(g[0].contiguous()) : Tensor(), dsT = g[1].defined() ? on_16(g[1].contiguous()) : Tensor();
        const Guard guard(q.device());
        rwkv_delta_args a = delta_args(q, k, v, gate, beta, ctx->saved_data["scale"].toDouble());
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
        Tensor dg = at::empty(gate.sizes(), gate.options()), dbeta = at::empty(gate.sizes(), gate.options());
        Tensor ds0 = get(ctx, "state") ? at::empty({a.B, a.H, a.N, a.N}, q.options().dtype(F32)) : Tensor();
        a.doc = P(s[5]); a.saved = P(saved); a.saved_bytes = saved.numel();
        a.dy = P(dy); a.dsT = P(dsT); a.dq = P(dq); a.dk = P(dk); a.dv = P(dv); a.dg = P(dg); a.dbeta = P(dbeta); a.ds0 = P(ds0);
        a.workspace_bytes = rwkv_delta_workspace_bytes(a.B, a.T, a.H, a.Hk, a.N, 1);
        const Tensor ws = a.workspace_bytes > 0 ? bytes(q, a.workspace_bytes) : Tensor();
        a.workspace = P(ws);
        ok(rwkv_delta_backward(stream_of(q), &a));
        return {dq, dk, dv, dg, dbeta, ds0, NONE, NONE, NONE};
    }
};
std::tuple<Tensor, Tensor> delta_op(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, const Maybe& s0, const Maybe& doc, c10::optional<double> scale) {
    require(q.dim() == 4 && k.dim() == 4 && v.dim() == 4 && g.dim() == 3 && beta.dim() == 3, "q and k are [B,T,Hk,N], v is [B,T,H,N], g and beta are [B,T,H]");
    const float sc = check_delta(q, k, v, g, beta, scale);
    const Tensor s = or_none(s0);
    variable_list o = Delta::apply(q, k, v, g, beta, s0, doc, static_cast<double>(sc), wants_grad({&q, &k, &v, &g, &beta}) || (s.defined() && wants_grad({&s})));
    return {o[0], o[1]};
}
Tensor delta_step_op(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_, const Tensor& beta_, const Tensor& s, const Tensor& out, c10::optional<double> scale) {
    require(!wants_grad({&q_, &k_, &v_, &g_, &beta_, &s, &out}), "STEP has no gradients: call it under torch.no_grad()");
    require(q_.dim() == 3 && k_.dim() == 3 && v_.dim() == 3 && g_.dim() == 2 && beta_.dim() == 2, "q and k are [B,Hk,N], v is [B,H,N], g and beta are [B,H]");
    const Tensor q = q_.unsqueeze(1), k = k_.unsqueeze(1), v = v_.unsqueeze(1), g = g_.unsqueeze(1), beta = beta_.unsqueeze(1);
    const float sc = check_delta(q, k, v, g, beta, scale);
    const int64_t B = v.size(0), H = v.size(2), N = v.size(3);
    check_side(s, "s", F32, {B, H, N, N}, q);
    check_side(out, "out", F32, {B, H, N, N}, q);
    check_writable(out, "the new state");
    for (const Tensor* x : {&q_, &k_, &v_, &g_, &beta_}) require(!touch(out, *x), "out must share no memory with q, k, v, g and beta");
    require(out.data_ptr() == s.data_ptr() || !touch(out, s), "out must be s, or share no memory with it");
    const Guard guard(q.device());
    rwkv_delta_args a = delta_args(q, k, v, g, beta, sc);
    Tensor y = at::empty({B, H, N}, q.options());
    a.s0 = P(s); a.sT = P(out); a.y = P(y);
    a.workspace_bytes = rwkv_delta_workspace_bytes(a.B, a.T, a.H, a.Hk, a.N, 0);
    const Tensor ws = a.workspace_bytes > 0 ? bytes(q, a.workspace_bytes) : Tensor();
    a.workspace = P(ws);
    ok(rwkv_delta_forward(stream_of(q), &a));
    written(out);
    return y;
}

// --------------------------------------------------------------------------------------------- a paged cache in 8 bits
constexpr auto F8 = torch::kFloat8_e4m3fn;
// pages [P,page,Hk,N] in 8 bits and their scales [P,Hk], beside `first`
void check_cache8(const Tensor& kp, const Tensor& vp, const Tensor& ks, const Tensor& vs, const Tensor& first, int64_t N) {
    require(kp.dim() == 4 && vp.sizes() == kp.sizes(), "k_pages and v_pages are [P,page,Hk,N]");
    const int64_t page = kp.size(1), Hk = kp.size(2);
    for (const auto& t : std::initializer_list<std::pair<const Tensor*, const char*>>{{&kp, "k_pages"}, {&vp, "v_pages"}}) {
        const std::string n = t.second;
        require(t.first->is_cuda() && first.is_cuda(), "tensors must live on a HIP device: there is no CPU path");
        require(t.first->device() == first.device(), n + " is on " + t.first->device().str() + ", expected " + first.device().str());
        require(t.first->scalar_type() == F8, n + ".dtype must be torch.float8_e4m3fn, got " + str(t.first->scalar_type()));
        require(t.first->stride(3) == 1, n + " must be dense in its last dimension");
    }
    require(kp.size(3) == N && Hk > 0, "the head size must be that of the pages");
    require(N >= 16 && N <= MAX_HEAD && N % 16 == 0, "the head size must be a multiple of 16 up to 128");
    require(page > 0 && (page & (page - 1)) == 0, "page must be a power of two");
    check_side(ks, "k_scales", F32, {kp.size(0), Hk}, first);
    check_side(vs, "v_scales", F32, {kp.size(0), Hk}, first);
}
void cache8_write_op(const Tensor& k, const Tensor& v, const Tensor& kp, const Tensor& vp, const Tensor& ks, const Tensor& vs, const Tensor& slots) {
    require(!wants_grad({&k, &v}), "WRITE has no gradients: call it under torch.no_grad()");
    require(k.dim() == 3 && v.sizes() == k.sizes(), "k and v are [n,Hk,N]");
    check_rows({{&k, "k"}, {&v, "v"}}, k);
    check_cache8(kp, vp, ks, vs, k, k.size(2));
    require(kp.size(2) == k.size(1), "k, v and the pages have the same heads");
    check_side(slots, "slots", torch::kInt32, {k.size(0)}, k);
    check_writable(kp, "k_pages"), check_writable(vp, "v_pages"), check_writable(ks, "k_scales"), check_writable(vs, "v_scales");
    for (const Tensor* x : {&kp, &vp})
        for (int64_t d = 0; d < 3; ++d) require(x->size(d) <= 1 || x->stride(d) != 0, "pages are written: no place of theirs may stand for several (as in an expanded tensor)");
    rwkv_cache8_args a{};
    a.dtype = dtype_of(k, "k", false);
    if (k.size(0) == 0) return;
    require(kp.numel() == 0 || (kp.data_ptr() != vp.data_ptr() && !touch(ks, vs)), "keys and values need pages and scales of their own");
    for (const Tensor* x : {&kp, &vp, &ks, &vs})
        for (const Tensor* y : {&k, &v, &slots}) require(!touch(*x, *y), "pages and scales must share no memory with k, v and slots");
    const Guard guard(k.device());
    a.n = i32(k.size(0)); a.Hk = i32(k.size(1)); a.N = i32(k.size(2)); a.P = i32(kp.size(0)); a.page = i32(kp.size(1));
    a.k = P(k); a.v = P(v); a.k_st = stride_of(k, 0); a.k_sh = stride_of(k, 1); a.v_st = stride_of(v, 0); a.v_sh = stride_of(v, 1);
    a.k_pages = P(kp); a.v_pages = P(vp);
    a.kp_sp = stride_of(kp, 0); a.kp_st = stride_of(kp, 1); a.kp_sh = stride_of(kp, 2);
    a.vp_sp = stride_of(vp, 0); a.vp_st = stride_of(vp, 1); a.vp_sh = stride_of(vp, 2);
    a.k_scales = P(ks); a.v_scales = P(vs); a.slots = P(slots);
    ok(rwkv_cache8_write(stream_of(k), &a));
    written(kp), written(vp), written(ks), written(vs);
}
Tensor paged8_op(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& ks, const Tensor& vs, const Tensor& table, const Tensor& lens, const Maybe& slopes_, double cap,
                 c10::optional<double> scale) {
    const Tensor slopes = or_none(slopes_);
    require(!wants_grad({&q}), "paged_attention8 has no gradients: call it under torch.no_grad()");
    require(q.dim() == 3, "q is [B,H,N]");
    const int64_t B = q.size(0), H = q.size(1), N = q.size(2);
    check({{&q, "q"}}, q.scalar_type(), q);
    check_cache8(kp, vp, ks, vs, q, N);
    const int64_t page = kp.size(1), Hk = kp.size(2);
    require(H % Hk == 0, "H must be a multiple of Hk");
    require(table.dim() == 2, "table is [B,M]");
    check_side(table, "table", torch::kInt32, {B, table.size(1)}, q);
    check_side(lens, "lens", torch::kInt32, {B}, q);
    check_side(slopes, "slopes", F32, {H}, q);
    require(cap == 0.0 || (cap >= 0x1p-20 && cap <= 4096.0), "cap must be 0, or from 2^-20 to 4096");
    const Guard guard(q.device());
    rwkv_paged8_args a{};
    a.dtype = dtype_of(q, "q", false);
    a.B = i32(B); a.H = i32(H); a.Hk = i32(Hk); a.N = i32(N); a.P = i32(kp.size(0)); a.page = i32(page); a.M = i32(table.size(1));
    a.scale = scale_of(scale, N); a.cap = static_cast<float>(cap);
    require(a.scale > 0.f && std::isfinite(a.scale), "scale must be positive");
    a.k_sp = stride_of(kp, 0); a.k_st = stride_of(kp, 1); a.k_sh = stride_of(kp, 2);
    a.v_sp = stride_of(vp, 0); a.v_st = stride_of(vp, 1); a.v_sh = stride_of(vp, 2);
    const Tensor qq = on_16(q);
    Tensor y = at::empty({B, H, N}, q.options());
    a.q = P(qq); a.k_pages = P(kp); a.v_pages = P(vp); a.k_scales = P(ks); a.v_scales = P(vs); a.table = P(table); a.lens = P(lens); a.slopes = P(slopes); a.y = P(y);
    a.workspace_bytes = rwkv_paged8_workspace_bytes(a.B, a.H, a.Hk, a.N, a.page, a.M);
    const Tensor ws = a.workspace_bytes > 0 ? bytes(q, a.workspace_bytes) : Tensor();
    a.workspace = P(ws);
    ok(rwkv_paged8_attn(stream_of(q), &a));
    return y;
}

// --------------------------------------------------------------------------------------------- page tables
std::tuple<Tensor, Tensor, Tensor, Tensor> tables_op(const Tensor& lens, const Tensor& more, const Tensor& table, const Tensor& pool, const Tensor& taken, int64_t page, int64_t n) {
    require(lens.dim() == 1 && table.dim() == 2 && pool.dim() == 1, "lens and more are [B], table is [B,M], pool is [F], taken is [1]");
    constexpr auto I32 = torch::kInt32;
    check({{&lens, "lens"}, {&table, "table"}, {&pool, "pool"}}, I32, lens);
    const int64_t B = lens.size(0);
    check_side(more, "more", I32, {B}, lens);
    check_side(taken, "taken", I32, {1}, lens);
    require(table.size(0) == B, "table is [B,M]");
    require(page > 0 && page <= (1 << 30) && (page & (page - 1)) == 0, "page must be a power of two");
    require(n >= 0 && n <= std::numeric_limits<int>::max(), "n must be from 0 to 2147483647");
    check_writable(table, "table");
    for (const Tensor* x : {&lens, &more, &pool, &taken}) require(!touch(table, *x), "table must share no memory with lens, more, pool and taken");
    const Guard guard(lens.device());
    rwkv_tables_args a{};
    a.B = i32(B); a.M = i32(table.size(1)); a.F = i32(pool.size(0)); a.page = static_cast<int>(page); a.n = static_cast<int>(n);
    Tensor slots = at::empty({n}, lens.options()), starts = at::empty({B + 1}, lens.options()), held = at::empty({B}, lens.options()), out = at::empty({1}, lens.options());
    a.lens = P(lens); a.more = P(more); a.table = P(table); a.pool = P(pool); a.taken = P(taken);
    a.slots = n > 0 ? slots.data_ptr<int>() : nullptr; a.starts = P(starts); a.held = P(held); a.taken_out = P(out);
    ok(rwkv_tables_extend(stream_of(lens), &a));
    written(table);
    return {slots, starts, held, out};
}

}  // namespace

void bind_autograd(py::module_& m) {
    auto ops = m.def_submodule("ops");
    ops.def("wkv4", &wkv4_op);
    ops.def("timex", &timex_op);
    ops.def("wkv5_f32", &wkv5_f32_op);
    ops.def("wkv5a", &wkv5a_op);
    ops.def("wkv5_bf16", &wkv5_bf16_op);
    ops.def("wkv6", &wkv6_op);
    ops.def("wkv6_state", &wkv6_state_op);
    ops.def("rwkv7_passing", &rwkv7_passing_op);
    ops.def("rwkv7_state", &rwkv7_state_op);
    ops.def("rwkv7", &rwkv7_op);
    ops.def("gated_recurrence", &grec_op);
    ops.def("gated_recurrence_step", &grec_step_op);
    ops.def("attention", &attention_op);
    ops.def("paged_attention", &paged_op);
    ops.def("gated_delta", &delta_op);
    ops.def("gated_delta_step", &delta_step_op);
    ops.def("cache8_write", &cache8_write_op);
    ops.def("paged_attention8", &paged8_op);
    ops.def("tables_extend", &tables_op);
}
