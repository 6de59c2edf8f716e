// The host side of the Python layer's calls, native: argument checks, output
// and scratch allocation, argument blocks and the call into libmamba_ss.so.
//
// A scan step's two calls fill about 130 fields of the C ABI's argument
// blocks; from Python, through ctypes, they and the checks ahead of them took
// 251 us per forward + backward of a 2 x 64 x 256 scan whose kernels run for
// 45 us (now 130, most of it torch's autograd engine); a block's decode step
// took 95 us (now 42), RMSNorm forward + backward at 32768 x 768 155 to 164 (92;
// figures bound by the host vary by a quarter between runs there).  The functions
// here take the tensors, the raw stream handle and flags, and raise the same
// exceptions with the same messages.  They hold no state.  The GIL is released
// around the calls into the library.
#include <torch/extension.h>

#include <optional>
#include <string>
#include <vector>

#include "../../include/mamba_ss.h"

namespace py = pybind11;
using at::Tensor;
using OptT = std::optional<Tensor>;

namespace {

[[noreturn]] void value_error(const std::string& msg) { throw py::value_error(msg); }

std::string shape_str(at::IntArrayRef s) {            // as Python prints a tuple
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + (s.size() == 1 ? ",)" : ")");
}
std::string dtype_str(at::ScalarType t) {
    const py::gil_scoped_acquire gil;                 // (a backward's checks run without it)
    return std::string(py::str(py::cast(t)));
}

// what: the module's prefix of its messages
#define REQUIRE(what, cond, msg)                                                   \
    do {                                                                           \
        if (!(cond)) value_error(std::string(what) + ": " + (msg));                \
    } while (0)

void check(int rc, const char* what) {
    if (rc == SS_OK) return;
    const std::string msg = std::string(what) + ": " + ss_last_error();
    if (rc == SS_ERR_INVALID || rc == SS_ERR_UNSUPPORTED) value_error(msg);
    throw std::runtime_error(msg);
}

template <typename F>
void launch(const at::Device& dev, const char* what, F&& f) {
    int rc;
    {
        std::optional<py::gil_scoped_release> nogil;
        if (PyGILState_Check()) nogil.emplace();       // (autograd's thread does not hold it)
        const c10::OptionalDeviceGuard guard(dev);
        rc = f();
    }
    check(rc, what);                 // (the message is this thread's)
}

// The stream that is current for the device.  A node's backward takes its
// forward's (kept in the node): autograd makes that one current for it, and its
// thread need not take the GIL to ask.
void* current_stream(const at::Device& dev) {
    if (!dev.is_cuda()) return nullptr;                // (refused by the call)
    const py::gil_scoped_acquire gil;
    static const py::handle get = py::object(py::module_::import("torch._C").attr("_cuda_getCurrentRawStream")).release();
    return reinterpret_cast<void*>(get(int(dev.index())).cast<int64_t>());
}
// whether an operator's node will be asked for a backward
bool wants_grad(std::initializer_list<const Tensor*> inputs) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : inputs)
        if (t && t->defined() && t->requires_grad()) return true;
    return false;
}
// A forward-mode tangent would be lost: the operators have none.
void no_tangents(const char* what, std::initializer_list<const Tensor*> inputs) {
    for (const Tensor* t : inputs)
        REQUIRE(what, !t || !t->defined() || !t->_fw_grad(0).defined(), "forward-mode derivatives are not implemented");
}
const Tensor* at_opt(const OptT& t) { return t ? &*t : nullptr; }
// A tensor that the library wrote in place: autograd then refuses a backward that
// saved what it held (tensors made in inference mode are never saved).
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Tensor given(const OptT& t) { return t ? *t : Tensor(); }
OptT maybe(const Tensor& t) { return t.defined() ? OptT(t) : OptT(); }
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
// The operators' gradients have no derivative of their own.  With create_graph they
// come out of a node that says so when a second backward reaches it; the values are of
// use as they are.
struct FinalGrads : torch::autograd::Function<FinalGrads> {
    static variable_list forward(AutogradContext* ctx, const Tensor&, const variable_list& grads, const std::string& what) {
        ctx->saved_data["what"] = what;
        variable_list r;
        for (const Tensor& g : grads) r.push_back(g.variable_data());
        return r;
    }
    static variable_list backward(AutogradContext* ctx, variable_list) {
        throw std::runtime_error(ctx->saved_data["what"].toStringRef() + ": second derivatives are not implemented");
    }
};
variable_list final_grads(const char* what, variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list some;
    for (const Tensor& g : grads)
        if (g.defined()) some.push_back(g);
    if (some.empty()) return grads;
    // (a node needs an input that requires a gradient)
    const Tensor anchor = at::empty({0}, some[0].options().dtype(at::kFloat)).requires_grad_();
    const variable_list r = FinalGrads::apply(anchor, some, std::string(what));
    size_t at = 0;
    for (Tensor& g : grads)
        if (g.defined()) g = r[at++];
    return grads;
}
std::vector<OptT> final_grads_py(const std::string& what, const std::vector<OptT>& grads) {
    variable_list r;
    for (const OptT& g : grads) r.push_back(given(g));
    std::vector<OptT> out;
    for (const Tensor& g : final_grads(what.c_str(), r)) out.push_back(maybe(g));
    return out;
}
void* node_stream(AutogradContext* ctx) { return reinterpret_cast<void*>(ctx->saved_data["stream"].toInt()); }

bool itype_of(at::ScalarType t, int32_t* out) {
    switch (t) {
        case at::kFloat: *out = SS_F32; return true;
        case at::kBFloat16: *out = SS_BF16; return true;
        case at::kHalf: *out = SS_F16; return true;
        default: return false;
    }
}
bool unit(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }
void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const OptT& t) { return t ? t->data_ptr() : nullptr; }
template <typename T> T* fptr(const OptT& t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }
Tensor f32_like(at::IntArrayRef shape, const Tensor& like) {
    return at::empty(shape, like.options().dtype(at::kFloat).memory_format(c10::nullopt));
}
Tensor bytes_on(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// ------------------------------------------------------------------ scan --
constexpr const char* kScan = "selective_scan";

int64_t chunks(int64_t seqlen) { return (seqlen + ss_chunk_size() - 1) / ss_chunk_size(); }

void check_seq(const char* name, const Tensor& t, at::IntArrayRef shape, at::ScalarType dtype, const at::Device& dev) {
    REQUIRE(kScan, t.device() == dev, std::string(name) + " is on " + t.device().str() + ", expected " + dev.str());
    REQUIRE(kScan, t.sizes() == shape,
            std::string(name) + " has shape " + shape_str(t.sizes()) + ", expected " + shape_str(shape));
    REQUIRE(kScan, t.scalar_type() == dtype,
            std::string(name) + " has dtype " + dtype_str(t.scalar_type()) + ", expected " + dtype_str(dtype));
    REQUIRE(kScan, unit(t), std::string(name) + " must have unit stride along seqlen");
}

void fill_fwd(ss_fwd_args& a, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
              const OptT& D, const OptT& bias, bool softplus, const OptT& z, const OptT& out, const OptT& x,
              const OptT& y) {
    REQUIRE(kScan, u.dim() == 3, "u must be (batch, dim, seqlen), got shape " + shape_str(u.sizes()));
    const at::Device dev = u.device();
    REQUIRE(kScan, dev.is_cuda(), "tensors must be on a ROCm GPU device (no CPU path)");
    int32_t itype = 0;
    REQUIRE(kScan, itype_of(u.scalar_type(), &itype), "unsupported dtype " + dtype_str(u.scalar_type()));
    const at::ScalarType dt = u.scalar_type();
    const int64_t batch = u.size(0), dim = u.size(1), seqlen = u.size(2);
    check_seq("delta", delta, u.sizes(), dt, dev);
    REQUIRE(kScan, A.dim() == 2 && A.size(0) == dim, "A must be (dim, dstate), got " + shape_str(A.sizes()));
    REQUIRE(kScan, A.scalar_type() == at::kFloat && A.device() == dev, "A must be fp32 on the same device");
    const int64_t dstate = A.size(1);
    const bool vb = B.dim() >= 3, vc = C.dim() >= 3;
    const int64_t groups = vb ? B.size(1) : vc ? C.size(1) : 1;
    for (int i = 0; i < 2; ++i) {
        const Tensor& M = i ? C : B;
        const std::string name = i ? "C" : "B";
        REQUIRE(kScan, M.device() == dev, name + " is on " + M.device().str() + ", expected " + dev.str());
        if (i ? vc : vb) {
            REQUIRE(kScan, M.dim() == 4 && M.size(0) == batch && M.size(1) == groups && M.size(2) == dstate &&
                               M.size(3) == seqlen,
                    name + " must be (batch, n_groups, dstate, seqlen), got " + shape_str(M.sizes()));
            REQUIRE(kScan, M.scalar_type() == dt,
                    name + " has dtype " + dtype_str(M.scalar_type()) + ", expected " + dtype_str(dt));
            REQUIRE(kScan, seqlen <= 1 || M.stride(3) == 1, name + " must have unit stride along seqlen");
        } else {
            REQUIRE(kScan, M.dim() == 2 && M.size(0) == dim && M.size(1) == dstate,
                    "constant " + name + " must be (dim, dstate), got " + shape_str(M.sizes()));
            REQUIRE(kScan, M.scalar_type() == at::kFloat, "constant " + name + " must be fp32");
        }
    }
    for (int i = 0; i < 2; ++i) {
        const OptT& v = i ? bias : D;
        if (v)
            REQUIRE(kScan, v->dim() == 1 && v->size(0) == dim && v->scalar_type() == at::kFloat && v->device() == dev &&
                               v->is_contiguous(),
                    std::string(i ? "delta_bias" : "D") + " must be a contiguous fp32 (" + std::to_string(dim) +
                        ",) tensor");
    }
    if (z) check_seq("z", *z, u.sizes(), dt, dev);
    a = ss_fwd_args{};
    a.batch = batch; a.dim = dim; a.seqlen = seqlen; a.dstate = dstate; a.n_groups = groups;
    a.itype = itype;
    a.is_var_B = vb; a.is_var_C = vc;
    a.has_D = D.has_value(); a.has_delta_bias = bias.has_value(); a.has_z = z.has_value();
    a.delta_softplus = softplus;
    a.n_chunks = chunks(seqlen);
    a.u_batch_stride = u.stride(0); a.u_dim_stride = u.stride(1);
    a.delta_batch_stride = delta.stride(0); a.delta_dim_stride = delta.stride(1);
    if (z) a.z_batch_stride = z->stride(0), a.z_dim_stride = z->stride(1);
    if (out) a.out_batch_stride = out->stride(0), a.out_dim_stride = out->stride(1);
    if (y) a.y_batch_stride = y->stride(0), a.y_dim_stride = y->stride(1);
    a.A_dim_stride = A.stride(0); a.A_dstate_stride = A.stride(1);
    if (vb) a.B_batch_stride = B.stride(0), a.B_group_stride = B.stride(1), a.B_dstate_stride = B.stride(2);
    else a.B_group_stride = B.stride(0), a.B_dstate_stride = B.stride(1);
    if (vc) a.C_batch_stride = C.stride(0), a.C_group_stride = C.stride(1), a.C_dstate_stride = C.stride(2);
    else a.C_group_stride = C.stride(0), a.C_dstate_stride = C.stride(1);
    a.u = ptr(u); a.delta = ptr(delta); a.A = static_cast<float*>(ptr(A)); a.B = ptr(B); a.C = ptr(C);
    a.D = fptr<float>(D); a.delta_bias = fptr<float>(bias); a.z = ptr(z);
    a.out = ptr(out); a.x = fptr<float>(x); a.y = ptr(y);
}

bool same_shape(const Tensor& t, std::initializer_list<int64_t> s) { return t.sizes() == at::IntArrayRef(s); }

// As forward_into's checks: the outputs, then everything fill_fwd looks at.
void fill_fwd_into(ss_fwd_args& a, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B,
                   const Tensor& C, const OptT& D, const OptT& bias, bool softplus, const OptT& out, const OptT& x,
                   const OptT& z, const OptT& y, const OptT& last) {
    REQUIRE(kScan, out.has_value(), "out is required");
    check_seq("out", *out, u.sizes(), delta.scalar_type(), u.device());
    REQUIRE(kScan, u.dim() == 3, "u must be (batch, dim, seqlen), got shape " + shape_str(u.sizes()));
    const int64_t batch = u.size(0), dim = u.size(1), seqlen = u.size(2), n = A.dim() == 2 ? A.size(1) : -1;
    if (x)
        REQUIRE(kScan, x->scalar_type() == at::kFloat && x->is_contiguous() && x->device() == u.device() &&
                           same_shape(*x, {batch, chunks(seqlen), dim, n}),
                "x must be a contiguous fp32 (batch, n_chunks, dim, dstate) tensor");
    if (y) check_seq("y", *y, u.sizes(), delta.scalar_type(), u.device());
    if (last)
        REQUIRE(kScan, last->scalar_type() == at::kFloat && last->is_contiguous() && last->device() == u.device() &&
                           same_shape(*last, {batch, dim, n}),
                "last_state must be a contiguous fp32 (batch, dim, dstate) tensor");
    fill_fwd(a, u, delta, A, B, C, D, bias, softplus, z, out, x, y);
    a.last_state = fptr<float>(last);
}

void scan_fwd(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const OptT& D,
              const OptT& bias, bool softplus, const OptT& out, const OptT& x, const OptT& z, const OptT& y,
              const OptT& last, bool auto_ws, OptT ws, int64_t stream) {
    ss_fwd_args a;
    fill_fwd_into(a, u, delta, A, B, C, D, bias, softplus, out, x, z, y, last);
    if (auto_ws) {
        const int64_t n = ss_fwd_workspace_bytes(&a);
        if (n < 0) check(SS_ERR_INVALID, "selective_scan.forward");
        if (n > 0) ws = bytes_on(n, u);
    }
    if (ws) {
        REQUIRE(kScan, ws->is_cuda() && ws->is_contiguous(), "workspace must be a contiguous GPU tensor");
        a.workspace = ptr(*ws);
        a.workspace_bytes = ws->numel() * ws->element_size();
    }
    // (a workspace made here is freed to the stream's caching allocator, which
    // keeps it valid for the work queued on the stream)
    launch(u.device(), "selective_scan.forward", [&] { return ss_fwd(&a, reinterpret_cast<void*>(stream)); });
}

Tensor seq_unit(const Tensor& t) { return unit(t) ? t : t.contiguous(); }
Tensor f32c(const Tensor& t) { return t.to(at::kFloat).contiguous(); }

// SelectiveScanZFn's forward: (out, last_state, saved tensors, B squeezed, C squeezed).
py::tuple scan_z_fwd(const Tensor& u_, const Tensor& delta_, const Tensor& A_, const Tensor& B_, const Tensor& C_,
                     const OptT& D_, const OptT& z_, const OptT& bias_, bool softplus, bool need_bwd, bool want_last,
                     int64_t stream) {
    const Tensor u = seq_unit(u_), delta = seq_unit(delta_);
    const OptT z = z_ ? OptT(seq_unit(*z_)) : OptT();
    const bool sqB = B_.dim() == 3, sqC = C_.dim() == 3;
    Tensor B = sqB ? B_.unsqueeze(1) : B_, C = sqC ? C_.unsqueeze(1) : C_;
    B = B.dim() < 3 ? f32c(B) : seq_unit(B);
    C = C.dim() < 3 ? f32c(C) : seq_unit(C);
    const Tensor A = A_.to(at::kFloat);
    const OptT D = D_ ? OptT(f32c(*D_)) : OptT(), bias = bias_ ? OptT(f32c(*bias_)) : OptT();
    REQUIRE(kScan, u.dim() == 3, "u must be (batch, dim, seqlen), got shape " + shape_str(u.sizes()));
    REQUIRE(kScan, A.dim() == 2, "A must be (dim, dstate), got " + shape_str(A.sizes()));
    const int64_t batch = u.size(0), dim = u.size(1), seqlen = u.size(2), n = A.size(1);
    const Tensor out = at::empty_like(delta, delta.options(), at::MemoryFormat::Contiguous);
    // the checkpoints x and the pre-gate output y exist for the backward:
    // without a gradient to compute they are neither allocated nor written
    OptT x, y, last;
    if (need_bwd) x = f32_like({batch, chunks(seqlen), dim, n}, u);
    if (need_bwd && z) y = at::empty_like(out);
    if (want_last) {
        last = f32_like({batch, dim, n}, u);
        if (seqlen == 0) last->zero_();
    }
    scan_fwd(u, delta, A, B, C, D, bias, softplus, out, x, z, y, last, true, OptT(), stream);
    return py::make_tuple(out, last, py::make_tuple(u, delta, A, B, C, D, bias, z, x, y), sqB, sqC);
}

void fill_bwd(ss_bwd_args& b, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
              const OptT& D, const OptT& bias, const Tensor& dout, const OptT& x, bool softplus, const Tensor& du,
              const Tensor& ddelta, const OptT& dA, const OptT& dB, const OptT& dC, const OptT& dD, const OptT& dbias,
              const OptT& z, const OptT& y, const OptT& dz) {
    REQUIRE(kScan, x.has_value(), "x (the forward's checkpoints) is required");
    REQUIRE(kScan, !z || (y && dz), "y from the forward and dz are required with z");
    REQUIRE(kScan, u.dim() == 3, "u must be (batch, dim, seqlen), got shape " + shape_str(u.sizes()));
    const int64_t batch = u.size(0), dim = u.size(1), seqlen = u.size(2), n = A.dim() == 2 ? A.size(1) : -1;
    const at::Device dev = u.device();
    REQUIRE(kScan, x->scalar_type() == at::kFloat && same_shape(*x, {batch, chunks(seqlen), dim, n}) &&
                       x->is_contiguous() && x->device() == dev,
            "x does not come from forward");
    const at::ScalarType ddt = delta.scalar_type();
    check_seq("dout", dout, u.sizes(), ddt, dev);
    check_seq("du", du, u.sizes(), u.scalar_type(), dev);
    check_seq("ddelta", ddelta, u.sizes(), ddt, dev);
    if (y) check_seq("y", *y, u.sizes(), ddt, dev);
    if (dz) check_seq("dz", *dz, u.sizes(), ddt, dev);
    const struct { const char* name; const OptT& g; const Tensor* ref; } gs[] = {
        {"dA", dA, &A}, {"dB", dB, &B}, {"dC", dC, &C}, {"dD", dD, D ? &*D : nullptr},
        {"ddelta_bias", dbias, bias ? &*bias : nullptr}};
    for (const auto& e : gs)
        if (e.ref)
            REQUIRE(kScan, e.g && e.g->scalar_type() == at::kFloat && e.g->is_contiguous() &&
                               e.g->sizes() == e.ref->sizes() && e.g->device() == dev,
                    std::string(e.name) + " must be a contiguous fp32 tensor of shape " + shape_str(e.ref->sizes()));
    b = ss_bwd_args{};
    fill_fwd(b.f, u, delta, A, B, C, D, bias, softplus, z, OptT(), x, y);
    b.dout_batch_stride = dout.stride(0); b.dout_dim_stride = dout.stride(1);
    b.du_batch_stride = du.stride(0); b.du_dim_stride = du.stride(1);
    b.ddelta_batch_stride = ddelta.stride(0); b.ddelta_dim_stride = ddelta.stride(1);
    if (dz) b.dz_batch_stride = dz->stride(0), b.dz_dim_stride = dz->stride(1);
    b.dout = ptr(dout); b.du = ptr(du); b.ddelta = ptr(ddelta); b.dz = ptr(dz);
    b.dA = fptr<float>(dA); b.dB = fptr<float>(dB); b.dC = fptr<float>(dC); b.dD = fptr<float>(dD);
    b.ddelta_bias = fptr<float>(dbias);
}

// The backward of a filled block; auto_ws allocates the scratch it asks for.
void run_bwd(ss_bwd_args& b, const Tensor& u, bool auto_ws, OptT ws, bool zero, int64_t stream) {
    if (auto_ws) {
        const int64_t n = ss_bwd_workspace_bytes(&b);
        if (n < 0) check(SS_ERR_INVALID, "selective_scan.backward");
        if (n > 0) ws = bytes_on(n, u);
    }
    if (ws) {
        REQUIRE(kScan, ws->device() == u.device() && ws->is_contiguous(),
                "workspace must be a contiguous tensor on the inputs' device");
        b.workspace = ptr(*ws);
        b.workspace_bytes = ws->numel() * ws->element_size();
    }
    b.zero_grads = zero;
    launch(u.device(), "selective_scan.backward", [&] { return ss_bwd(&b, reinterpret_cast<void*>(stream)); });
}

void scan_bwd(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const OptT& D,
              const OptT& bias, const Tensor& dout, const OptT& x, bool softplus, const Tensor& du,
              const Tensor& ddelta, const OptT& dA, const OptT& dB, const OptT& dC, const OptT& dD, const OptT& dbias,
              const OptT& z, const OptT& y, const OptT& dz, bool auto_ws, OptT ws, bool zero, bool deterministic,
              int64_t stream) {
    ss_bwd_args b;
    fill_bwd(b, u, delta, A, B, C, D, bias, dout, x, softplus, du, ddelta, dA, dB, dC, dD, dbias, z, y, dz);
    b.deterministic = deterministic;
    run_bwd(b, u, auto_ws, std::move(ws), zero, stream);
}

// backward(): gradients allocated here, cleared by the library.
py::tuple scan_bwd_new(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
                       const OptT& D, const OptT& bias, const Tensor& dout, const OptT& x, bool softplus,
                       const OptT& z, const OptT& y, bool deterministic, int64_t stream) {
    const auto like = [](const Tensor& t) { return at::empty_like(t, t.options(), at::MemoryFormat::Contiguous); };
    const Tensor du = like(u), ddelta = like(delta);
    const Tensor dA = f32_like(A.sizes(), A), dB = f32_like(B.sizes(), B), dC = f32_like(C.sizes(), C);
    const OptT dD = D ? OptT(f32_like(D->sizes(), *D)) : OptT();
    const OptT dbias = bias ? OptT(f32_like(bias->sizes(), *bias)) : OptT(), dz = z ? OptT(like(*z)) : OptT();
    scan_bwd(u, delta, A, B, C, D, bias, dout, x, softplus, du, ddelta, dA, dB, dC, dD, dbias, z, y, dz, true, OptT(),
             true, deterministic, stream);
    return py::make_tuple(du, ddelta, dA, dB, dC, dD, dbias, dz);
}

// ------------------------------------------------------------------ conv --
Tensor weight2d(const Tensor& w_, int64_t dim) {
    const Tensor w = w_.dim() == 3 ? w_.reshape({w_.size(0), w_.size(-1)}) : w_;
    REQUIRE(kScan, w.dim() == 2 && w.size(0) == dim, "weight must be (dim, width), got " + shape_str(w_.sizes()));
    return w;
}
// The weight as (dim, width) and the bias as the library reads them: in the
// rows' type where both are, else in fp32.
std::pair<Tensor, OptT> conv_params(const Tensor& weight, const OptT& bias, int64_t dim, const at::Device& dev,
                                    at::ScalarType rows = at::kFloat) {
    const bool io = weight.scalar_type() == rows && (!bias || bias->scalar_type() == rows);
    const at::ScalarType ty = io ? rows : at::kFloat;
    const Tensor w = weight2d(weight, dim).to(dev, ty);
    OptT b;
    if (bias) {
        b = bias->to(dev, ty).contiguous();
        REQUIRE(kScan, same_shape(*b, {dim}),
                "bias must be (" + std::to_string(dim) + ",), got " + shape_str(bias->sizes()));
    }
    return {w, b};
}
int32_t dtype_code(const Tensor& t) {
    int32_t c = SS_F32;
    itype_of(t.scalar_type(), &c);
    return c;
}
void fill_conv(ss_conv1d_args& a, const Tensor& x, const Tensor& w, const OptT& b, bool silu, const OptT& out) {
    REQUIRE(kScan, x.dim() == 3, "x must be (batch, dim, seqlen), got " + shape_str(x.sizes()));
    REQUIRE(kScan, x.is_cuda(), "tensors must be on a ROCm GPU device (no CPU path)");
    a = ss_conv1d_args{};
    REQUIRE(kScan, itype_of(x.scalar_type(), &a.itype), "unsupported dtype " + dtype_str(x.scalar_type()));
    REQUIRE(kScan, unit(x), "x must have unit stride along seqlen");
    a.batch = x.size(0); a.dim = x.size(1); a.seqlen = x.size(2); a.width = w.size(1);
    a.has_bias = b.has_value(); a.silu = silu;
    a.x_batch_stride = x.stride(0); a.x_dim_stride = x.stride(1);
    if (out) a.out_batch_stride = out->stride(0), a.out_dim_stride = out->stride(1);
    a.w_dim_stride = w.stride(0); a.w_width_stride = w.stride(1);
    // (weight and bias of the type passed beside the block)
    a.x = ptr(x); a.weight = static_cast<float*>(ptr(w)); a.bias = fptr<float>(b); a.out = ptr(out);
}
Tensor conv_fwd(const Tensor& x, const Tensor& weight, const OptT& bias, bool silu, OptT out, int64_t stream) {
    REQUIRE(kScan, x.dim() == 3, "x must be (batch, dim, seqlen), got " + shape_str(x.sizes()));
    const auto [w, b] = conv_params(weight, bias, x.size(1), x.device(), x.scalar_type());
    const int32_t wd = dtype_code(w);
    if (!out) out = at::empty(x.sizes(), x.options());
    REQUIRE(kScan, out->sizes() == x.sizes() && out->scalar_type() == x.scalar_type() && unit(*out),
            "out must match x in shape and dtype, with unit stride along seqlen");
    ss_conv1d_args a;
    fill_conv(a, x, w, b, silu, out);
    launch(x.device(), "causal_conv1d_fwd", [&] { return ss_conv1d_fwd_typed(&a, wd, reinterpret_cast<void*>(stream)); });
    return *out;
}
// (dx, dweight (dim, width), dbias): in fp32, summed by atomics or, when
// deterministic, in a fixed order; with `typed`, of the weight's and bias's
// own types where the library writes them (fixed order, one launch for both).
py::tuple conv_bwd(const Tensor& x, const Tensor& weight, const OptT& bias, const Tensor& dout_, bool silu, OptT dx,
                   bool deterministic, bool typed, int64_t stream) {
    REQUIRE(kScan, x.dim() == 3, "x must be (batch, dim, seqlen), got " + shape_str(x.sizes()));
    const auto [w, b] = typed ? conv_params(weight, bias, x.size(1), x.device(), x.scalar_type())
                              : conv_params(weight, bias, x.size(1), x.device());
    const int32_t wd = dtype_code(w);
    REQUIRE(kScan, dout_.sizes() == x.sizes() && dout_.scalar_type() == x.scalar_type(),
            "dout must match x in shape and dtype");
    const Tensor dout = seq_unit(dout_);
    if (!dx) dx = at::empty(x.sizes(), x.options());
    const bool zero = !typed || x.numel() == 0;
    const Tensor dw = at::empty(w.sizes(), w.options());
    const OptT db = b ? OptT(at::empty(b->sizes(), b->options())) : OptT();
    if (zero) {
        dw.zero_();
        if (db) db->zero_();
    }
    ss_conv1d_bwd_args g{};
    fill_conv(g.f, x, w, b, silu, OptT());
    g.dout_batch_stride = dout.stride(0); g.dout_dim_stride = dout.stride(1);
    g.dx_batch_stride = dx->stride(0); g.dx_dim_stride = dx->stride(1);
    g.dout = ptr(dout); g.dx = ptr(*dx); g.dweight = static_cast<float*>(ptr(dw)); g.dbias = fptr<float>(db);
    OptT ws;
    if (deterministic || typed) {
        const int64_t n = ss_conv1d_bwd_workspace_bytes(&g);
        REQUIRE(kScan, n >= 0, "invalid conv1d sizes");
        ws = f32_like({std::max<int64_t>(n / 4, 1)}, x);
        g.workspace = static_cast<float*>(ptr(*ws));
        g.workspace_bytes = ws->numel() * 4;
    }
    launch(x.device(), "causal_conv1d_bwd", [&] {
        void* st = reinterpret_cast<void*>(stream);
        return typed ? ss_conv1d_bwd_typed(&g, wd, st) : ss_conv1d_bwd(&g, st);
    });
    return py::make_tuple(*dx, dw, db);
}

// --------------------------------------------------------------- RMSNorm --
constexpr const char* kNorm = "rms_norm";

// (rows, dim) view with unit column stride (a copy only when no such view exists)
Tensor norm_rows(const Tensor& t_, int64_t dim) {
    const Tensor t = dim > 1 && t_.stride(-1) != 1 ? t_.contiguous() : t_;
    const Tensor v = t.dim() == 2 && dim > 0 && t.size(1) == dim ? t : t.reshape({-1, dim});
    return dim > 1 && v.stride(1) != 1 ? v.contiguous() : v;
}
Tensor norm_weight(const Tensor& w, const Tensor& x) {
    REQUIRE(kNorm, w.dim() == 1 && w.size(0) == x.size(-1),
            "weight must be (" + std::to_string(x.size(-1)) + ",), got " + shape_str(w.sizes()));
    REQUIRE(kNorm, w.device() == x.device(), "weight is on " + w.device().str() + ", x on " + x.device().str());
    return (w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat ? w : w.to(at::kFloat)).contiguous();
}
py::tuple norm_fwd(const Tensor& x, const Tensor& weight, const OptT& residual, double eps, bool want_rstd, bool want_s,
                   int64_t stream) {
    REQUIRE(kNorm, x.is_cuda(), "tensors must be on a ROCm GPU device (no CPU path)");
    ss_rmsnorm_args a{};
    REQUIRE(kNorm, itype_of(x.scalar_type(), &a.dtype), "unsupported dtype " + dtype_str(x.scalar_type()));
    REQUIRE(kNorm, x.dim() >= 1, "x must have at least one dimension");
    const int64_t dim = x.size(-1);
    const Tensor w = norm_weight(weight, x), x2 = norm_rows(x, dim);
    itype_of(w.scalar_type(), &a.w_dtype);
    OptT r2, rout, rstd;
    if (residual) {
        REQUIRE(kNorm, residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() &&
                           residual->device() == x.device(),
                "residual must match x in shape, dtype and device");
        r2 = norm_rows(*residual, dim);
    }
    const Tensor out = at::empty(x2.sizes(), x.options());
    if (r2 && want_s) rout = at::empty_like(out);
    if (want_rstd) rstd = f32_like({x2.size(0)}, x);
    a.rows = x2.size(0); a.dim = dim;
    a.eps = float(eps);
    a.x_row_stride = x2.stride(0); a.out_row_stride = out.stride(0);
    if (r2) {
        a.residual_row_stride = r2->stride(0);
        if (rout) a.residual_out_row_stride = rout->stride(0);
    }
    a.x = ptr(x2); a.residual = ptr(r2); a.weight = ptr(w);
    a.out = ptr(out); a.residual_out = ptr(rout); a.rstd = fptr<float>(rstd);
    launch(x.device(), "rms_norm forward", [&] { return ss_rmsnorm_fwd(&a, reinterpret_cast<void*>(stream)); });
    return py::make_tuple(out, rout, rstd);
}
py::tuple norm_bwd(const Tensor& s, const Tensor& weight, const Tensor& rstd, const Tensor& dout,
                   const OptT& dresidual_out, int64_t stream) {
    const int64_t dim = s.size(-1);
    const Tensor w = norm_weight(weight, s), s2 = norm_rows(s, dim), dy = norm_rows(dout.to(s.scalar_type()), dim);
    const OptT dr = dresidual_out ? OptT(norm_rows(dresidual_out->to(s.scalar_type()), dim)) : OptT();
    const int64_t rows = s2.size(0);
    REQUIRE(kNorm, dy.sizes() == s2.sizes() && (!dr || dr->sizes() == s2.sizes()), "dout must match s");
    REQUIRE(kNorm, rstd.scalar_type() == at::kFloat && same_shape(rstd, {rows}) && rstd.is_contiguous(),
            "rstd must be fp32 (rows,) contiguous");
    const Tensor dx = at::empty(s2.sizes(), s.options()), dw = at::empty({dim}, w.options());
    const int64_t n = ss_rmsnorm_bwd_workspace_bytes(rows, dim);
    const Tensor ws = bytes_on(std::max<int64_t>(n, 1), s);
    ss_rmsnorm_bwd_args g{};
    g.rows = rows; g.dim = dim;
    REQUIRE(kNorm, itype_of(s.scalar_type(), &g.dtype) && itype_of(w.scalar_type(), &g.w_dtype),
            "unsupported dtype " + dtype_str(s.scalar_type()));
    g.s_row_stride = s2.stride(0); g.dout_row_stride = dy.stride(0); g.dx_row_stride = dx.stride(0);
    if (dr) g.dresidual_out_row_stride = dr->stride(0);
    g.s = ptr(s2); g.weight = ptr(w); g.rstd = static_cast<float*>(ptr(rstd)); g.dout = ptr(dy); g.dresidual_out = ptr(dr);
    g.dx = ptr(dx); g.dweight = ptr(dw); g.workspace = ptr(ws); g.workspace_bytes = n;
    launch(s.device(), "rms_norm backward", [&] { return ss_rmsnorm_bwd(&g, reinterpret_cast<void*>(stream)); });
    return py::make_tuple(dx, dw);
}

// ---------------------------------------------------------------- decode --
bool mult(const Tensor& t, int64_t stride0, size_t align) {
    return t.stride(0) % stride0 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % align == 0;
}
// the shapes ss_decode_linear takes (others run on torch's library GEMM)
bool linear_fits(const Tensor& x, const Tensor& weight, const OptT& bias, int64_t max_rows) {
    return x.is_cuda() && x.dim() == 2 && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf) &&
           weight.scalar_type() == x.scalar_type() && weight.dim() == 2 && weight.size(1) == x.size(1) &&
           x.size(1) % 16 == 0 && 0 < x.size(0) && x.size(0) <= max_rows && x.stride(1) == 1 &&
           weight.stride(1) == 1 && mult(x, 4, 8) && mult(weight, 4, 8) &&
           (!bias || ((bias->scalar_type() == x.scalar_type() || bias->scalar_type() == at::kFloat) &&
                      bias->is_contiguous()));
}
bool linear_norm_fits(const Tensor& x, const OptT& residual, const Tensor& nw) {
    const auto rows16 = [](const Tensor& t) { return t.stride(1) == 1 && mult(t, 8, 16); };
    return x.size(1) <= 1024 && rows16(x) &&
           (!residual || (residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() &&
                          rows16(*residual))) &&
           nw.dim() == 1 && nw.size(0) == x.size(1) &&
           (nw.scalar_type() == x.scalar_type() || nw.scalar_type() == at::kFloat) && nw.is_contiguous() &&
           reinterpret_cast<uintptr_t>(nw.data_ptr()) % 16 == 0;
}
// Workspace bytes of the K split for a product of these sizes.
int64_t linear_ws_bytes(int64_t batch, int64_t n_out, int64_t k_in) {
    ss_decode_linear_args a{};
    a.batch = batch; a.n_out = n_out; a.k_in = k_in;
    return ss_decode_linear_workspace_bytes(&a);
}
// The fused launch for fitting tensors: (y, s or None).
py::tuple linear(const Tensor& x, const Tensor& weight, const OptT& bias, bool has_conv, const OptT& conv_state,
                 const OptT& conv_w, const OptT& conv_b, bool silu, bool has_norm, const OptT& residual,
                 const OptT& nw, double eps, const OptT& ws, int64_t stream) {
    const int64_t batch = x.size(0), k_in = x.size(1), n_out = weight.size(0);
    const Tensor y = at::empty({batch, n_out}, x.options());
    ss_decode_linear_args a{};
    a.batch = batch; a.n_out = n_out; a.k_in = k_in;
    itype_of(x.scalar_type(), &a.dtype);
    a.bias_dtype = a.dtype;
    if (bias) itype_of(bias->scalar_type(), &a.bias_dtype);
    a.x_row_stride = x.stride(0); a.w_row_stride = weight.stride(0); a.y_row_stride = y.stride(0);
    a.x = ptr(x); a.weight = ptr(weight); a.bias = ptr(bias); a.y = ptr(y);
    ss_conv1d_update_args c{};
    Tensor w;
    OptT cb;
    if (has_conv) {
        REQUIRE(kScan, conv_state && conv_w, "conv_state and the conv weight are required");
        const int64_t dim = conv_state->size(1);
        std::tie(w, cb) = conv_params(*conv_w, conv_b, dim, x.device());
        REQUIRE(kScan, conv_state->dim() == 3 && same_shape(*conv_state, {batch, dim, w.size(1)}) &&
                           conv_state->scalar_type() == x.scalar_type() && conv_state->device() == x.device() &&
                           dim <= n_out,
                "conv_state must be (" + std::to_string(batch) + ", dim <= " + std::to_string(n_out) +
                    ", width) of x's dtype, got " + shape_str(conv_state->sizes()));
        c.batch = batch; c.dim = dim; c.width = w.size(1);
        c.itype = a.dtype; c.has_bias = cb.has_value(); c.silu = silu;
        c.state_batch_stride = conv_state->stride(0);
        c.state_dim_stride = conv_state->stride(1);
        c.state_width_stride = conv_state->stride(2);
        c.w_dim_stride = w.stride(0); c.w_width_stride = w.stride(1);
        c.conv_state = ptr(*conv_state); c.weight = static_cast<float*>(ptr(w)); c.bias = fptr<float>(cb);
        a.conv = &c;
    }
    ss_rmsnorm_args n{};
    OptT s;
    if (has_norm) {
        s = residual ? at::empty_like(x) : x;
        n.rows = batch; n.dim = k_in;
        n.dtype = a.dtype;
        itype_of(nw->scalar_type(), &n.w_dtype);
        n.eps = float(eps);
        n.x_row_stride = x.stride(0);
        if (residual) {
            n.residual_row_stride = residual->stride(0);
            n.residual_out_row_stride = s->stride(0);
            n.residual = ptr(*residual);
            n.residual_out = ptr(*s);
        }
        n.x = ptr(x); n.weight = ptr(*nw);
        a.norm = &n;
        a.x = nullptr;
        a.x_row_stride = 0;
    }
    if (ws && ss_decode_linear_workspace_bytes(&a) > 0) {
        a.workspace = ptr(*ws);
        a.workspace_bytes = ws->numel();
    }
    launch(x.device(), "decode_linear", [&] { return ss_decode_linear(&a, reinterpret_cast<void*>(stream)); });
    return py::make_tuple(y, s);
}

constexpr const char* kState = "selective_state_update";

Tensor state_update(const Tensor& state, const Tensor& x, const OptT& dt, const OptT& dt_low, const OptT& dt_w,
                    const Tensor& A, const Tensor& B_, const Tensor& C_, const OptT& D, const OptT& z,
                    const OptT& dt_bias, bool softplus, OptT out, int64_t stream) {
    REQUIRE(kState, x.dim() == 2 && x.is_cuda(), "x must be (batch, dim) on a ROCm GPU device (no CPU path)");
    ss_state_update_args a{};
    REQUIRE(kState, itype_of(x.scalar_type(), &a.itype), "unsupported dtype " + dtype_str(x.scalar_type()));
    const int64_t batch = x.size(0), dim = x.size(1);
    const at::Device dev = x.device();
    const at::ScalarType ty = x.scalar_type();
    const auto num = [](int64_t v) { return std::to_string(v); };
    REQUIRE(kState, state.dim() == 3 && state.size(0) == batch && state.size(1) == dim &&
                        state.scalar_type() == at::kFloat && state.device() == dev,
            "state must be fp32 (" + num(batch) + ", " + num(dim) + ", dstate)");
    const int64_t n = state.size(2);
    if (dt_low) {
        REQUIRE(kState, dt_low->dim() == 2 && dt_low->size(0) == batch && dt_low->scalar_type() == ty &&
                            dt_low->device() == dev,
                "dt_low must be (batch, rank) in x's dtype");
        REQUIRE(kState, dt_w.has_value(), "dt_weight is required with dt_low");
        REQUIRE(kState, same_shape(*dt_w, {dim, dt_low->size(1)}) && dt_w->scalar_type() == ty && dt_w->device() == dev,
                "dt_weight must be (dim, rank) in x's dtype");
    } else {
        REQUIRE(kState, dt.has_value(), "dt is required");
        REQUIRE(kState, dt->sizes() == x.sizes() && dt->scalar_type() == ty, "dt must match x in shape and dtype");
    }
    REQUIRE(kState, same_shape(A, {dim, n}), "A must be (" + num(dim) + ", " + num(n) + ")");
    const Tensor A32 = A.to(dev, at::kFloat);
    const Tensor B = B_.dim() == 2 ? B_.unsqueeze(1) : B_, C = C_.dim() == 2 ? C_.unsqueeze(1) : C_;
    REQUIRE(kState, B.dim() == 3 && B.size(0) == batch && B.size(2) == n && B.scalar_type() == ty,
            "B must be (batch, [n_groups,] dstate) in x's dtype");
    REQUIRE(kState, C.sizes() == B.sizes() && C.scalar_type() == ty, "C must match B");
    REQUIRE(kState, B.size(1) > 0 && dim % B.size(1) == 0,
            "dim " + num(dim) + " is not a multiple of n_groups " + num(B.size(1)));
    const OptT D32 = D ? OptT(D->to(dev, at::kFloat).contiguous()) : OptT();
    const OptT b32 = dt_bias ? OptT(dt_bias->to(dev, at::kFloat).contiguous()) : OptT();
    REQUIRE(kState, !D32 || same_shape(*D32, {dim}), "D must be (" + num(dim) + ",)");
    REQUIRE(kState, !b32 || same_shape(*b32, {dim}), "dt_bias must be (" + num(dim) + ",)");
    REQUIRE(kState, !z || (z->sizes() == x.sizes() && z->scalar_type() == ty), "z must match x");
    if (!out) out = at::empty({batch, dim}, x.options());
    a.batch = batch; a.dim = dim; a.dstate = n; a.n_groups = B.size(1);
    a.has_D = D32.has_value(); a.has_z = z.has_value(); a.has_delta_bias = b32.has_value();
    a.delta_softplus = softplus;
    a.state_batch_stride = state.stride(0); a.state_dim_stride = state.stride(1); a.state_dstate_stride = state.stride(2);
    a.x_batch_stride = x.stride(0); a.x_dim_stride = x.stride(1);
    if (dt_low) {
        a.delta_rank = dt_low->size(1);
        a.delta_low_batch_stride = dt_low->stride(0); a.delta_low_rank_stride = dt_low->stride(1);
        a.delta_weight_dim_stride = dt_w->stride(0); a.delta_weight_rank_stride = dt_w->stride(1);
        a.delta_low = ptr(*dt_low); a.delta_weight = ptr(*dt_w);
    } else {
        a.delta_batch_stride = dt->stride(0); a.delta_dim_stride = dt->stride(1);
        a.delta = ptr(*dt);
    }
    if (z) a.z_batch_stride = z->stride(0), a.z_dim_stride = z->stride(1);
    a.out_batch_stride = out->stride(0); a.out_dim_stride = out->stride(1);
    a.A_dim_stride = A32.stride(0); a.A_dstate_stride = A32.stride(1);
    a.B_batch_stride = B.stride(0); a.B_group_stride = B.stride(1); a.B_dstate_stride = B.stride(2);
    a.C_batch_stride = C.stride(0); a.C_group_stride = C.stride(1); a.C_dstate_stride = C.stride(2);
    a.state = static_cast<float*>(ptr(state)); a.x = ptr(x); a.A = static_cast<float*>(ptr(A32));
    a.B = ptr(B); a.C = ptr(C); a.D = fptr<float>(D32); a.z = ptr(z); a.delta_bias = fptr<float>(b32); a.out = ptr(*out);
    launch(dev, "selective_state_update", [&] { return ss_state_update(&a, reinterpret_cast<void*>(stream)); });
    return *out;
}

// ------------------------------------------------------ linear attention --
constexpr const char* kLin = "linear_attn";

void on_device(const char* what, const char* name, const Tensor& t, const at::Device& dev) {
    REQUIRE(what, t.device() == dev, std::string(name) + " is on " + t.device().str() + ", expected " + dev.str());
}
void of_type(const char* what, const char* name, const Tensor& t, at::ScalarType ty) {
    REQUIRE(what, t.scalar_type() == ty,
            std::string(name) + " has dtype " + dtype_str(t.scalar_type()) + ", expected " + dtype_str(ty));
}
// The log decays as the library reads them: fp32, (batch, seqlen, heads) with
// strides (0 along batch and seqlen where every head has one decay).
Tensor decays(const char* what, const Tensor& g_, int64_t batch, int64_t seqlen, int64_t heads, const Tensor& v) {
    on_device(what, "g", g_, v.device());
    REQUIRE(what, g_.scalar_type() == at::kFloat || g_.scalar_type() == v.scalar_type(),
            "g has dtype " + dtype_str(g_.scalar_type()) + ", expected float32 or v's");
    const bool per_head = g_.dim() == 1;
    const bool ok = per_head ? same_shape(g_, {heads}) : seqlen < 0 ? same_shape(g_, {batch, heads})
                                                                    : same_shape(g_, {batch, seqlen, heads});
    REQUIRE(what, ok, std::string("g must be ") + (seqlen < 0 ? "(batch, heads)" : "(batch, seqlen, heads)") +
                          " or (heads,), got " + shape_str(g_.sizes()));
    const Tensor g = g_.to(at::kFloat);
    return !per_head ? g : seqlen < 0 ? g.expand({batch, heads}) : g.expand({batch, seqlen, heads});
}
Tensor state_arg(const char* name, const Tensor& t, at::IntArrayRef shape, const at::Device& dev) {
    on_device(kLin, name, t, dev);
    of_type(kLin, name, t, at::kFloat);
    REQUIRE(kLin, t.sizes() == shape, std::string(name) + " has shape " + shape_str(t.sizes()) + ", expected " + shape_str(shape));
    return t.contiguous();
}

struct LinIn { Tensor q, k, v, g; OptT initial, lengths; };

LinIn fill_linear(ss_linear_attn_args& a, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_,
                  const OptT& initial, const OptT& lengths, double scale) {
    a = ss_linear_attn_args{};
    REQUIRE(kLin, v_.dim() == 4, "v must be (batch, seqlen, heads, d_value), got shape " + shape_str(v_.sizes()));
    const at::Device dev = v_.device();
    REQUIRE(kLin, dev.is_cuda(), "tensors must be on a ROCm GPU device (no CPU path)");
    REQUIRE(kLin, itype_of(v_.scalar_type(), &a.dtype), "unsupported dtype " + dtype_str(v_.scalar_type()));
    const int64_t B = v_.size(0), L = v_.size(1), H = v_.size(2), V = v_.size(3);
    REQUIRE(kLin, q_.dim() == 4 && q_.size(0) == B && q_.size(1) == L,
            "q must be (batch, seqlen, groups, d_key), got shape " + shape_str(q_.sizes()));
    REQUIRE(kLin, k_.sizes() == q_.sizes(), "k has shape " + shape_str(k_.sizes()) + ", expected " + shape_str(q_.sizes()));
    const int64_t G = q_.size(2), K = q_.size(3);
    REQUIRE(kLin, H == 0 || (G > 0 && H % G == 0),
            "heads " + std::to_string(H) + " is not a multiple of groups " + std::to_string(G));
    on_device(kLin, "q", q_, dev); on_device(kLin, "k", k_, dev);
    of_type(kLin, "q", q_, v_.scalar_type()); of_type(kLin, "k", k_, v_.scalar_type());
    LinIn in{seq_unit(q_), seq_unit(k_), seq_unit(v_), decays(kLin, g_, B, L, H, v_), {}, {}};
    if (initial) in.initial = state_arg("initial_state", *initial, {B, H, K, V}, dev);
    if (lengths) {
        on_device(kLin, "lengths", *lengths, dev);
        REQUIRE(kLin, same_shape(*lengths, {B}) && (lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong),
                "lengths must be a (batch,) integer tensor, got " + shape_str(lengths->sizes()) + " " + dtype_str(lengths->scalar_type()));
        in.lengths = (lengths->scalar_type() == at::kInt ? *lengths : lengths->clamp(0, L).to(at::kInt)).contiguous();
    }
    a.batch = B; a.seqlen = L; a.heads = H; a.groups = G; a.d_key = K; a.d_value = V;
    a.scale = float(scale);
    a.q_batch_stride = in.q.stride(0); a.q_len_stride = in.q.stride(1); a.q_head_stride = in.q.stride(2);
    a.k_batch_stride = in.k.stride(0); a.k_len_stride = in.k.stride(1); a.k_head_stride = in.k.stride(2);
    a.v_batch_stride = in.v.stride(0); a.v_len_stride = in.v.stride(1); a.v_head_stride = in.v.stride(2);
    a.g_batch_stride = in.g.stride(0); a.g_len_stride = in.g.stride(1); a.g_head_stride = in.g.stride(2);
    a.q = ptr(in.q); a.k = ptr(in.k); a.v = ptr(in.v); a.g = static_cast<float*>(ptr(in.g));
    a.initial_state = fptr<float>(in.initial); a.lengths = fptr<int32_t>(in.lengths);
    return in;
}

int64_t lin_segs(const ss_linear_attn_args& a) {
    const int64_t n = ss_linear_attn_segment(&a);
    if (n < 0) check(SS_ERR_INVALID, kLin);
    return std::max<int64_t>(1, (a.seqlen + n - 1) / n);
}

struct LinOut { Tensor out; OptT last, ends; LinIn in; };     // in: the tensors as read
LinOut lin_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const OptT& initial,
               const OptT& lengths, double scale, bool want_last, bool want_ends, void* stream) {
    ss_linear_attn_args a;
    const LinIn in = fill_linear(a, q, k, v, g, initial, lengths, scale);
    const Tensor out = at::empty({a.batch, a.seqlen, a.heads, a.d_value}, in.v.options());
    OptT last, ends, ws;
    if (want_last) last = f32_like({a.batch, a.heads, a.d_key, a.d_value}, in.v);
    const int64_t segs = lin_segs(a);
    if (want_ends) ends = f32_like({a.batch, a.heads, segs, a.d_key, a.d_value}, in.v);
    a.out_batch_stride = out.stride(0); a.out_len_stride = out.stride(1); a.out_head_stride = out.stride(2);
    a.out = ptr(out); a.last_state = fptr<float>(last); a.ends = fptr<float>(ends);
    const int64_t n = ss_linear_attn_fwd_workspace_bytes(&a);
    if (n < 0) check(SS_ERR_INVALID, kLin);
    if (n > 0) {
        ws = bytes_on(n, in.v);
        a.workspace = ptr(*ws); a.workspace_bytes = n;
    }
    launch(in.v.device(), "linear_attn forward", [&] { return ss_linear_attn_fwd(&a, stream); });
    return {out, last, ends, in};
}

struct LinGrads { Tensor dq, dk, dv, dg; OptT dinitial; };    // dg: fp32
LinGrads lin_bwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const OptT& initial,
                  const OptT& lengths, const Tensor& ends, double scale, bool g_per_head, const Tensor& dout_,
                  const OptT& dlast_, bool want_dinitial, void* stream) {
    ss_linear_attn_bwd_args b{};
    const LinIn in = fill_linear(b.f, q, k, v, g, initial, lengths, scale);
    const ss_linear_attn_args& a = b.f;
    const at::Device dev = in.v.device();
    REQUIRE(kLin, dout_.sizes() == in.v.sizes() && dout_.scalar_type() == in.v.scalar_type() && dout_.device() == dev,
            "dout must match v, got " + shape_str(dout_.sizes()) + " " + dtype_str(dout_.scalar_type()));
    const Tensor dout = seq_unit(dout_);
    REQUIRE(kLin, same_shape(ends, {a.batch, a.heads, lin_segs(a), a.d_key, a.d_value}) && ends.is_contiguous() &&
                      ends.scalar_type() == at::kFloat && ends.device() == dev,
            "ends does not come from the forward");
    OptT dlast, dinitial, ws;
    if (dlast_) dlast = state_arg("dlast_state", *dlast_, {a.batch, a.heads, a.d_key, a.d_value}, dev);
    if (want_dinitial) dinitial = f32_like({a.batch, a.heads, a.d_key, a.d_value}, in.v);
    const Tensor dq = at::empty(in.q.sizes(), in.q.options()), dk = at::empty(in.q.sizes(), in.q.options()),
                 dv = at::empty(in.v.sizes(), in.v.options());
    const Tensor dg = g_per_head ? f32_like({a.heads}, in.v) : f32_like({a.batch, a.seqlen, a.heads}, in.v);
    if (a.batch == 0) dg.zero_();
    if (a.heads == 0) {                                // (q and k reach no output)
        dq.zero_();
        dk.zero_();
    }
    b.f.ends = static_cast<float*>(ptr(ends));
    b.dout_batch_stride = dout.stride(0); b.dout_len_stride = dout.stride(1); b.dout_head_stride = dout.stride(2);
    b.dout = ptr(dout); b.dlast_state = fptr<float>(dlast);
    b.dq = ptr(dq); b.dk = ptr(dk); b.dv = ptr(dv); b.dg = static_cast<float*>(ptr(dg));
    b.dinitial_state = fptr<float>(dinitial);
    b.g_per_head = g_per_head;
    if (a.batch > 0 && a.heads > 0) {
        // (an empty tensor has no address; the library asks for one)
        if (!b.dg) b.dg = b.f.ends;
        const int64_t n = ss_linear_attn_bwd_workspace_bytes(&b);
        if (n < 0) check(SS_ERR_INVALID, kLin);
        if (n > 0) {
            ws = bytes_on(n, in.v);
            b.f.workspace = ptr(*ws); b.f.workspace_bytes = n;
        }
        launch(dev, "linear_attn backward", [&] { return ss_linear_attn_bwd(&b, stream); });
    }
    return {dq, dk, dv, dg, dinitial};
}

// The autograd node, native like the rest of a call's host side: a forward +
// backward of a small layer is bound by it (as a Python node, a border of 2047
// x 1001 rows took 128 us for 38 of kernels).
struct LinAttn : torch::autograd::Function<LinAttn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                                 const OptT& initial, const OptT& lengths, double scale, bool want_last, bool need) {
        void* const stream = current_stream(v.device());
        const LinOut r = lin_fwd(q, k, v, g, initial, lengths, scale, want_last, need, stream);
        if (need) {
            ctx->saved_data["stream"] = reinterpret_cast<int64_t>(stream);
            ctx->save_for_backward({r.in.q, r.in.k, r.in.v, r.in.g, given(r.in.initial), given(r.in.lengths), given(r.ends)});
            ctx->saved_data["scale"] = scale;
            ctx->saved_data["g_type"] = int64_t(g.scalar_type());
            ctx->saved_data["per_head"] = g.dim() == 1;
            ctx->set_materialize_grads(false);
        }
        variable_list out{r.out};
        if (want_last) out.push_back(*r.last);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list r(9);
        const Tensor dlast = grads.size() > 1 ? grads[1] : Tensor();
        if (!grads[0].defined() && !dlast.defined()) return r;
        const auto t = ctx->get_saved_variables();
        const Tensor dout = grads[0].defined() ? grads[0] : at::zeros_like(t[2]);
        const bool has_initial = t[4].defined();
        const LinGrads d = lin_bwd(t[0], t[1], t[2], t[3], maybe(t[4]), maybe(t[5]), t[6], ctx->saved_data["scale"].toDouble(),
                                   ctx->saved_data["per_head"].toBool(), dout, maybe(dlast),
                                   has_initial && ctx->needs_input_grad(4), node_stream(ctx));
        if (ctx->needs_input_grad(0)) r[0] = d.dq;
        if (ctx->needs_input_grad(1)) r[1] = d.dk;
        if (ctx->needs_input_grad(2)) r[2] = d.dv;
        if (ctx->needs_input_grad(3)) r[3] = d.dg.to(at::ScalarType(ctx->saved_data["g_type"].toInt()));
        r[4] = given(d.dinitial);
        return final_grads(kLin, r);
    }
};
// (out, last_state or None)
py::tuple linear_attn(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const OptT& initial,
                      const OptT& lengths, double scale, bool want_last) {
    no_tangents(kLin, {&q, &k, &v, &g, at_opt(initial)});
    const bool need = wants_grad({&q, &k, &v, &g, at_opt(initial)});
    if (!need) {
        const LinOut r = lin_fwd(q, k, v, g, initial, lengths, scale, want_last, false, current_stream(v.device()));
        return py::make_tuple(r.out, r.last);
    }
    const variable_list r = LinAttn::apply(q, k, v, g, initial, lengths, scale, want_last, need);
    return py::make_tuple(r[0], want_last ? OptT(r[1]) : OptT());
}

constexpr const char* kLinUp = "linear_attn_update";

Tensor lin_update(const Tensor& state, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_, double scale,
                  OptT out, int64_t stream) {
    REQUIRE(kLinUp, v_.dim() == 3 && v_.is_cuda(), "v must be (batch, heads, d_value) on a ROCm GPU device (no CPU path)");
    ss_linear_attn_update_args a{};
    REQUIRE(kLinUp, itype_of(v_.scalar_type(), &a.dtype), "unsupported dtype " + dtype_str(v_.scalar_type()));
    const at::Device dev = v_.device();
    const int64_t B = v_.size(0), H = v_.size(1), V = v_.size(2);
    REQUIRE(kLinUp, q_.dim() == 3 && q_.size(0) == B, "q must be (batch, groups, d_key), got shape " + shape_str(q_.sizes()));
    REQUIRE(kLinUp, k_.sizes() == q_.sizes(), "k has shape " + shape_str(k_.sizes()) + ", expected " + shape_str(q_.sizes()));
    const int64_t G = q_.size(1), K = q_.size(2);
    REQUIRE(kLinUp, H == 0 || (G > 0 && H % G == 0),
            "heads " + std::to_string(H) + " is not a multiple of groups " + std::to_string(G));
    no_tangents(kLinUp, {&state, &q_, &k_, &v_, &g_});
    REQUIRE(kLinUp, !wants_grad({&state, &q_, &k_, &v_, &g_}),
            "a token's update has no backward; call it under torch.no_grad(), or linear_attn_fn for gradients");
    on_device(kLinUp, "q", q_, dev); on_device(kLinUp, "k", k_, dev); on_device(kLinUp, "state", state, dev);
    of_type(kLinUp, "q", q_, v_.scalar_type()); of_type(kLinUp, "k", k_, v_.scalar_type());
    of_type(kLinUp, "state", state, at::kFloat);
    REQUIRE(kLinUp, same_shape(state, {B, H, K, V}),
            "state has shape " + shape_str(state.sizes()) + ", expected " + shape_str({B, H, K, V}));
    REQUIRE(kLinUp, state.numel() == 0 || ((V <= 1 || state.stride(3) == 1) && (K <= 1 || state.stride(2) == V)),
            "state must be contiguous along its last two dims (it is updated in place)");
    const Tensor q = seq_unit(q_), k = seq_unit(k_), v = seq_unit(v_), g = decays(kLinUp, g_, B, -1, H, v_);
    const bool own_out = out.has_value();
    if (own_out)
        REQUIRE(kLinUp, out->sizes() == v.sizes() && out->scalar_type() == v.scalar_type() && out->device() == dev && unit(*out),
                "out must match v, with unit stride along the last dim");
    else out = at::empty({B, H, V}, v.options());
    a.batch = B; a.heads = H; a.groups = G; a.d_key = K; a.d_value = V;
    a.scale = float(scale);
    a.state_batch_stride = state.stride(0); a.state_head_stride = state.stride(1);
    a.q_batch_stride = q.stride(0); a.q_head_stride = q.stride(1);
    a.k_batch_stride = k.stride(0); a.k_head_stride = k.stride(1);
    a.v_batch_stride = v.stride(0); a.v_head_stride = v.stride(1);
    a.out_batch_stride = out->stride(0); a.out_head_stride = out->stride(1);
    a.g_batch_stride = g.stride(0); a.g_head_stride = g.stride(1);
    a.state = static_cast<float*>(ptr(state)); a.q = ptr(q); a.k = ptr(k); a.v = ptr(v);
    a.g = static_cast<float*>(ptr(g)); a.out = ptr(*out);
    launch(dev, kLinUp, [&] { return ss_linear_attn_update(&a, reinterpret_cast<void*>(stream)); });
    written(state);
    if (own_out) written(*out);
    return *out;
}

// ------------------------------------------------------------ block norms --
constexpr const char* kBlockNorm = "block_norm";
constexpr const char* kGatedNorm = "gated_rms_norm";

// as norm_rows, rows of no elements too
Tensor any_rows(const Tensor& t) {
    const int64_t dim = t.size(-1);
    if (dim > 0) return norm_rows(t, dim);
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
    return t.reshape({rows, 0});
}
// rows of x's shape and type
Tensor like_rows(const char* what, const char* name, const Tensor& t, const Tensor& x) {
    REQUIRE(what, t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && t.device() == x.device(),
            std::string(name) + " must match x in shape, dtype and device, got " + shape_str(t.sizes()) + " " +
                dtype_str(t.scalar_type()));
    return any_rows(t);
}
// weights as the library reads them: all of x's type, or all fp32
struct Weights { std::vector<OptT> w; int32_t dtype; };
Weights weights_of(const char* what, const Tensor& x, std::initializer_list<std::pair<const char*, const OptT*>> ws) {
    Weights r{{}, 0};
    bool same = true;
    for (const auto& [name, w] : ws) {
        if (!*w) continue;
        const Tensor& t = **w;
        REQUIRE(what, t.dim() == 1 && t.size(0) == x.size(-1),
                std::string(name) + " must be (" + std::to_string(x.size(-1)) + ",), got " + shape_str(t.sizes()));
        REQUIRE(what, t.device() == x.device(), std::string(name) + " is on " + t.device().str() + ", x on " + x.device().str());
        REQUIRE(what, at::isFloatingType(t.scalar_type()), std::string(name) + " must be a float tensor");
        same = same && t.scalar_type() == x.scalar_type();
    }
    const at::ScalarType ty = same ? x.scalar_type() : at::kFloat;
    for (const auto& [name, w] : ws) r.w.push_back(*w ? OptT((*w)->to(ty).contiguous()) : OptT());
    itype_of(ty, &r.dtype);
    return r;
}
void norm_x(const char* what, const Tensor& x, int32_t* dtype) {
    REQUIRE(what, x.is_cuda(), "tensors must be on a ROCm GPU device (no CPU path)");
    REQUIRE(what, itype_of(x.scalar_type(), dtype), "unsupported dtype " + dtype_str(x.scalar_type()));
    REQUIRE(what, x.dim() >= 1, "x must have at least one dimension");
}

// (out, s: of x's shape; read: x, residual, gate, post, pre, scale_vec, rows as (rows, dim))
struct BorderOut { Tensor out, s; OptT rstd; variable_list read; };
BorderOut block_norm_fwd(const Tensor& x_, const Tensor& residual_, const OptT& gate_, const Tensor& post, const Tensor& pre,
                         const OptT& scale_vec, double scale, double eps, bool want_rstd, void* stream) {
    ss_block_norm_args a{};
    norm_x(kBlockNorm, x_, &a.dtype);
    const Tensor x = any_rows(x_), residual = like_rows(kBlockNorm, "residual", residual_, x_);
    const OptT gate = gate_ ? OptT(like_rows(kBlockNorm, "gate", *gate_, x_)) : OptT(), opost = post, opre = pre;
    const Weights w = weights_of(kBlockNorm, x_, {{"post", &opost}, {"pre", &opre}, {"scale", &scale_vec}});
    a.w_dtype = w.dtype;
    a.rows = x.size(0); a.dim = x.size(1);
    a.eps = float(eps); a.scale = float(scale);
    // (of x's shape, not views: what autograd returns can then be changed in place)
    const Tensor out = at::empty(x_.sizes(), x.options()), s = at::empty(x_.sizes(), x.options());
    OptT rstd;
    if (want_rstd) rstd = f32_like({a.rows, 2}, x);
    a.x_row_stride = x.stride(0); a.residual_row_stride = residual.stride(0);
    if (gate) a.gate_row_stride = gate->stride(0);
    a.out_row_stride = a.residual_out_row_stride = a.dim;
    a.x = ptr(x); a.residual = ptr(residual); a.gate = ptr(gate);
    a.post = ptr(w.w[0]); a.pre = ptr(w.w[1]); a.scale_vec = ptr(w.w[2]);
    a.out = ptr(out); a.residual_out = ptr(s); a.rstd = fptr<float>(rstd);
    launch(x.device(), "block_norm forward", [&] { return ss_block_norm_fwd(&a, stream); });
    return {out, s, rstd, {x, residual, given(gate), given(w.w[0]), given(w.w[1]), given(w.w[2])}};
}

// from the forward's tensors as read
struct BorderGrads { Tensor dx; OptT dresidual, dgate; Tensor dpost, dpre; OptT dscale; };
BorderGrads block_norm_bwd(const Tensor& x, const Tensor& residual, const OptT& gate, const Tensor& post, const Tensor& pre,
                         const OptT& scale_vec, const Tensor& rstd, double scale, const OptT& dout_, const OptT& ds_,
                         bool want_dresidual, void* stream) {
    ss_block_norm_bwd_args g{};
    norm_x(kBlockNorm, x, &g.dtype);
    REQUIRE(kBlockNorm, x.dim() == 2, "x must be (rows, dim)");
    const int64_t rows = x.size(0), dim = x.size(1);
    REQUIRE(kBlockNorm, rstd.scalar_type() == at::kFloat && same_shape(rstd, {rows, 2}) && rstd.is_contiguous(),
            "rstd must be fp32 (rows, 2) contiguous");
    REQUIRE(kBlockNorm, itype_of(post.scalar_type(), &g.w_dtype), "unsupported dtype " + dtype_str(post.scalar_type()));
    OptT dout, ds, dresidual, dgate, dscale;
    if (dout_) dout = like_rows(kBlockNorm, "dout", *dout_, x);
    if (ds_) ds = like_rows(kBlockNorm, "dresidual_out", *ds_, x);
    const Tensor dx = at::empty(x.sizes(), x.options()), dpost = at::empty({dim}, post.options()),
                 dpre = at::empty({dim}, post.options());
    if (want_dresidual) dresidual = at::empty(x.sizes(), x.options());
    if (gate) dgate = at::empty(x.sizes(), x.options());
    if (scale_vec) dscale = at::empty({dim}, post.options());
    const int64_t n = ss_block_norm_bwd_workspace_bytes(rows, dim);
    if (n < 0) check(SS_ERR_INVALID, kBlockNorm);
    const Tensor ws = bytes_on(std::max<int64_t>(n, 1), x);
    g.rows = rows; g.dim = dim; g.scale = float(scale);
    g.x_row_stride = x.stride(0); g.residual_row_stride = residual.stride(0);
    if (gate) g.gate_row_stride = gate->stride(0);
    if (dout) g.dout_row_stride = dout->stride(0);
    if (ds) g.dresidual_out_row_stride = ds->stride(0);
    g.x = ptr(x); g.residual = ptr(residual); g.gate = ptr(gate); g.post = ptr(post); g.pre = ptr(pre);
    g.scale_vec = ptr(scale_vec); g.rstd = static_cast<float*>(ptr(rstd)); g.dout = ptr(dout); g.dresidual_out = ptr(ds);
    g.dx = ptr(dx); g.dresidual = ptr(dresidual); g.dgate = ptr(dgate); g.dpost = ptr(dpost); g.dpre = ptr(dpre);
    g.dscale = ptr(dscale); g.workspace = ptr(ws); g.workspace_bytes = n;
    launch(x.device(), "block_norm backward", [&] { return ss_block_norm_bwd(&g, stream); });
    return {dx, dresidual, dgate, dpost, dpre, dscale};
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const Tensor& post, const Tensor& pre,
                                 const OptT& gate, const OptT& scale_vec, double scale, double eps) {
        void* const stream = current_stream(x.device());
        const BorderOut r = block_norm_fwd(x, residual, gate, post, pre, scale_vec, scale, eps, true, stream);
        ctx->saved_data["stream"] = reinterpret_cast<int64_t>(stream);
        variable_list saved = r.read;
        saved.push_back(*r.rstd);
        ctx->save_for_backward(saved);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["types"] = std::vector<int64_t>{int64_t(post.scalar_type()), int64_t(pre.scalar_type()),
                                                        scale_vec ? int64_t(scale_vec->scalar_type()) : 0};
        ctx->set_materialize_grads(false);
        return {r.out, r.s};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list r(8);
        if (!grads[0].defined() && !grads[1].defined()) return r;
        const auto t = ctx->get_saved_variables();
        const auto rows = [&](const Tensor& g) { return g.defined() ? OptT(g.reshape(t[0].sizes())) : OptT(); };
        const BorderGrads d = block_norm_bwd(t[0], t[1], maybe(t[2]), t[3], t[4], maybe(t[5]), t[6], ctx->saved_data["scale"].toDouble(),
                                             rows(grads[0]), rows(grads[1]), ctx->needs_input_grad(1), node_stream(ctx));
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const auto types = ctx->saved_data["types"].toIntVector();
        const auto typed = [&](const Tensor& w, int i) { return w.to(at::ScalarType(types[i])); };
        const size_t at_gate = 4, at_scale = t[2].defined() ? 5 : 4;      // (an absent gate is no input)
        if (ctx->needs_input_grad(0)) r[0] = d.dx.view(shape);
        if (ctx->needs_input_grad(1)) r[1] = d.dresidual->view(shape);
        if (ctx->needs_input_grad(2)) r[2] = typed(d.dpost, 0);
        if (ctx->needs_input_grad(3)) r[3] = typed(d.dpre, 1);
        if (t[2].defined() && ctx->needs_input_grad(at_gate)) r[4] = d.dgate->view(shape);
        if (t[5].defined() && ctx->needs_input_grad(at_scale)) r[5] = typed(*d.dscale, 2);
        return final_grads(kBlockNorm, r);
    }
};
// (out, s)
py::tuple block_norm(const Tensor& x, const Tensor& residual, const Tensor& post, const Tensor& pre, const OptT& gate,
                     const OptT& scale_vec, double scale, double eps) {
    no_tangents(kBlockNorm, {&x, &residual, &post, &pre, at_opt(gate), at_opt(scale_vec)});
    if (!wants_grad({&x, &residual, &post, &pre, at_opt(gate), at_opt(scale_vec)})) {
        const BorderOut r = block_norm_fwd(x, residual, gate, post, pre, scale_vec, scale, eps, false, current_stream(x.device()));
        return py::make_tuple(r.out, r.s);
    }
    const variable_list r = BlockNorm::apply(x, residual, post, pre, gate, scale_vec, scale, eps);
    return py::make_tuple(r[0], r[1]);
}

// (out of x's shape; x, gate, weight as read, rows as (rows, dim))
variable_list gated_norm_fwd(const Tensor& x_, const Tensor& gate_, const Tensor& weight, int64_t groups, double eps,
                             void* stream) {
    ss_gated_norm_args a{};
    norm_x(kGatedNorm, x_, &a.dtype);
    const Tensor x = any_rows(x_), gate = like_rows(kGatedNorm, "gate", gate_, x_);
    const OptT ow = weight;
    const Weights w = weights_of(kGatedNorm, x_, {{"weight", &ow}});
    a.w_dtype = w.dtype;
    a.rows = x.size(0); a.dim = x.size(1); a.groups = groups; a.eps = float(eps);
    const Tensor out = at::empty(x_.sizes(), x.options());
    a.x_row_stride = x.stride(0); a.gate_row_stride = gate.stride(0); a.out_row_stride = a.dim;
    a.x = ptr(x); a.gate = ptr(gate); a.weight = ptr(w.w[0]); a.out = ptr(out);
    launch(x.device(), "gated_rms_norm forward", [&] { return ss_gated_norm_fwd(&a, stream); });
    return {out, x, gate, *w.w[0]};
}

// (dx, dgate, dweight)
variable_list gated_norm_bwd(const Tensor& x, const Tensor& gate, const Tensor& weight, const Tensor& dout_, int64_t groups,
                             double eps, void* stream) {
    ss_gated_norm_bwd_args g{};
    norm_x(kGatedNorm, x, &g.dtype);
    REQUIRE(kGatedNorm, x.dim() == 2, "x must be (rows, dim)");
    const Tensor dout = like_rows(kGatedNorm, "dout", dout_, x);
    REQUIRE(kGatedNorm, itype_of(weight.scalar_type(), &g.w_dtype), "unsupported dtype " + dtype_str(weight.scalar_type()));
    const int64_t rows = x.size(0), dim = x.size(1);
    const Tensor dx = at::empty(x.sizes(), x.options()), dgate = at::empty(x.sizes(), x.options()),
                 dw = at::empty({dim}, weight.options());
    const int64_t n = ss_gated_norm_bwd_workspace_bytes(rows, dim, groups);
    if (n < 0) check(SS_ERR_INVALID, kGatedNorm);
    const Tensor ws = bytes_on(std::max<int64_t>(n, 1), x);
    g.rows = rows; g.dim = dim; g.groups = groups; g.eps = float(eps);
    g.x_row_stride = x.stride(0); g.gate_row_stride = gate.stride(0); g.dout_row_stride = dout.stride(0);
    g.x = ptr(x); g.gate = ptr(gate); g.weight = ptr(weight); g.dout = ptr(dout);
    g.dx = ptr(dx); g.dgate = ptr(dgate); g.dweight = ptr(dw); g.workspace = ptr(ws); g.workspace_bytes = n;
    launch(x.device(), "gated_rms_norm backward", [&] { return ss_gated_norm_bwd(&g, stream); });
    return {dx, dgate, dw};
}

struct GatedNorm : torch::autograd::Function<GatedNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& weight, int64_t groups, double eps) {
        void* const stream = current_stream(x.device());
        const variable_list r = gated_norm_fwd(x, gate, weight, groups, eps, stream);
        ctx->saved_data["stream"] = reinterpret_cast<int64_t>(stream);
        ctx->save_for_backward({r[1], r[2], r[3]});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["type"] = int64_t(weight.scalar_type());
        return r[0];
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto t = ctx->get_saved_variables();
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const variable_list d = gated_norm_bwd(t[0], t[1], t[2], grads[0].reshape(t[0].sizes()), ctx->saved_data["groups"].toInt(),
                                               ctx->saved_data["eps"].toDouble(), node_stream(ctx));
        variable_list r(5);
        if (ctx->needs_input_grad(0)) r[0] = d[0].view(shape);
        if (ctx->needs_input_grad(1)) r[1] = d[1].view(shape);
        if (ctx->needs_input_grad(2)) r[2] = d[2].to(at::ScalarType(ctx->saved_data["type"].toInt()));
        return final_grads(kGatedNorm, r);
    }
};
Tensor gated_norm(const Tensor& x, const Tensor& gate, const Tensor& weight, int64_t groups, double eps) {
    no_tangents(kGatedNorm, {&x, &gate, &weight});
    if (!wants_grad({&x, &gate, &weight}))
        return gated_norm_fwd(x, gate, weight, groups, eps, current_stream(x.device()))[0];
    return GatedNorm::apply(x, gate, weight, groups, eps);
}

// -------------------------------------------------------------- clipping --
constexpr const char* kClip = "clip_grads";

// Clips grads into outs (the same list: in place); returns the norm, a 0-d fp32 tensor.
Tensor clip_grads(const std::vector<Tensor>& grads, const std::vector<Tensor>& outs, double max_norm, double eps,
                  int64_t device_index, int64_t stream) {
    REQUIRE(kClip, outs.size() == grads.size(),
            "out holds " + std::to_string(outs.size()) + " tensors, expected " + std::to_string(grads.size()));
    const at::Device dev = grads.empty() ? at::Device(at::kCUDA, at::DeviceIndex(device_index)) : grads[0].device();
    REQUIRE(kClip, dev.is_cuda(), "tensors must be on a ROCm GPU device (no CPU path)");
    const size_t n = grads.size();
    std::vector<const void*> in(n);
    std::vector<void*> out(n);
    std::vector<int64_t> numels(n);
    std::vector<int32_t> dtypes(n);
    for (size_t i = 0; i < n; ++i) {
        const Tensor &g = grads[i], &o = outs[i];
        const auto at_i = [&] { return " of tensor " + std::to_string(i); };
        REQUIRE(kClip, g.device() == dev && o.device() == dev, "all tensors must be on one device");
        no_tangents(kClip, {&g, &o});
        REQUIRE(kClip, itype_of(g.scalar_type(), &dtypes[i]), "unsupported dtype " + dtype_str(g.scalar_type()) + at_i());
        REQUIRE(kClip, g.is_non_overlapping_and_dense(), "gaps or overlaps in the elements" + at_i());
        if (!o.is_same(g))
            REQUIRE(kClip, o.scalar_type() == g.scalar_type() && o.sizes() == g.sizes() && o.strides() == g.strides(),
                    "out must match the gradient in shape, strides and dtype" + at_i());
        in[i] = g.data_ptr(); out[i] = o.data_ptr(); numels[i] = g.numel();
    }
    ss_clip_grads_args a{};
    a.count = int64_t(n);
    a.grads = in.data(); a.outs = out.data(); a.numels = numels.data(); a.dtypes = dtypes.data();
    a.max_norm = float(max_norm); a.eps = float(eps);
    const auto options = at::TensorOptions().device(dev);
    const Tensor norm = at::empty({}, options.dtype(at::kFloat));
    const int64_t bytes = ss_clip_grads_workspace_bytes(&a);
    if (bytes < 0) check(SS_ERR_INVALID, kClip);
    const Tensor ws = at::empty({bytes}, options.dtype(at::kByte));
    a.norm = static_cast<float*>(ptr(norm)); a.workspace = ptr(ws); a.workspace_bytes = bytes;
    launch(dev, kClip, [&] { return ss_clip_grads(&a, reinterpret_cast<void*>(stream)); });
    for (const Tensor& o : outs) written(o);
    return norm;
}

}  // namespace

PYBIND11_MODULE(mamba_host, m) {
    // argument blocks at an address (ctypes structures of the prepared launches and queries)
    m.def("fill_fwd_into", [](uintptr_t at, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B,
                              const Tensor& C, const OptT& D, const OptT& bias, bool softplus, const OptT& out,
                              const OptT& x, const OptT& z, const OptT& y, const OptT& last) {
        fill_fwd_into(*reinterpret_cast<ss_fwd_args*>(at), u, delta, A, B, C, D, bias, softplus, out, x, z, y, last);
    });
    m.def("fill_bwd", [](uintptr_t at, const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B,
                         const Tensor& C, const OptT& D, const OptT& bias, const Tensor& dout, const OptT& x,
                         bool softplus, const Tensor& du, const Tensor& ddelta, const OptT& dA, const OptT& dB,
                         const OptT& dC, const OptT& dD, const OptT& dbias, const OptT& z, const OptT& y,
                         const OptT& dz) {
        fill_bwd(*reinterpret_cast<ss_bwd_args*>(at), u, delta, A, B, C, D, bias, dout, x, softplus, du, ddelta, dA,
                 dB, dC, dD, dbias, z, y, dz);
    });
    m.def("scan_fwd", &scan_fwd);
    m.def("scan_z_fwd", &scan_z_fwd);
    m.def("scan_bwd", &scan_bwd);
    m.def("scan_bwd_new", &scan_bwd_new);
    m.def("conv_fwd", &conv_fwd);
    m.def("conv_bwd", &conv_bwd);
    m.def("norm_fwd", &norm_fwd);
    m.def("norm_bwd", &norm_bwd);
    m.def("linear_fits", &linear_fits);
    m.def("linear_norm_fits", &linear_norm_fits);
    m.def("linear_ws_bytes", &linear_ws_bytes);
    m.def("linear", &linear);
    m.def("state_update", &state_update);
    m.def("linear_attn", &linear_attn);
    m.def("lin_update", &lin_update);
    m.def("block_norm", &block_norm);
    m.def("gated_norm", &gated_norm);
    m.def("clip_grads", &clip_grads);
    m.def("final_grads", &final_grads_py);
    m.def("abi", [] { return py::make_tuple(SS_ABI_VERSION, sizeof(ss_fwd_args), sizeof(ss_bwd_args)); });
}
