// Host side of the calls whose device time is a few microseconds: argument checks, output allocation and the parameter block
// of one C ABI call, on torch tensors, in C++.  In Python the same steps cost 25-30 us per call (a ctypes structure of some
// thirty fields, as many tensor attributes, a device context, a stream object), which is what a decode step of a small batch
// or a short prompt then waited for.  The library's functions are handed over as addresses (bind), so that this module and
// the ctypes binding drive the same loaded library; checks and messages are those of the Python wrappers (ops.py).
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/types.h>

#include <cmath>
#include <map>

#include "../../include/vortex_b200.h"

namespace py = pybind11;
using at::Tensor;
using Opt = std::optional<Tensor>;

namespace {

decltype(&vtx_decode_layer) p_decode_layer;
decltype(&vtx_fused_fir_fwd) p_fused_fir_fwd;
decltype(&vtx_fused_iir_fwd) p_fused_iir_fwd;
decltype(&vtx_fused_iir_scratch_bytes) p_fused_iir_scratch_bytes;
decltype(&vtx_last_error) p_last_error;
decltype(&vtx_qk_norm_rotary_fwd) p_rotary_fwd;
decltype(&vtx_qk_norm_rotary_bwd) p_rotary_bwd;
decltype(&vtx_qk_norm_rotary_bwd_scratch_bytes) p_rotary_bwd_scratch_bytes;
decltype(&vtx_rotary_append) p_rotary_append;
decltype(&vtx_paged_decode_attention) p_paged_decode;
decltype(&vtx_paged_decode_scratch_bytes) p_paged_decode_scratch_bytes;
decltype(&vtx_copy_pages) p_copy_pages;

// The entry points run without the GIL (see the module definition); an error is made with it.
[[noreturn]] void raise(PyObject* type, const std::string& msg) {
    const py::gil_scoped_acquire gil;
    PyErr_SetString(type, msg.c_str());
    throw py::error_already_set();
}
void check(int rc) {
    if (rc == 0) return;
    char buf[512];
    p_last_error(buf, sizeof buf);
    PyObject* type = rc == VTX_ERR_BAD_ARG || rc == VTX_ERR_ALIGNMENT ? PyExc_ValueError
                     : rc == VTX_ERR_UNSUPPORTED ? PyExc_NotImplementedError : PyExc_RuntimeError;
    raise(type, "vortex_b200: " + std::string(buf) + " (status " + std::to_string(rc) + ")");
}
void need_cuda(const Tensor& t) {
    if (!t.is_cuda()) raise(PyExc_RuntimeError, "vortex_b200 kernels need CUDA tensors (there is no CPU path)");
}
void need_cuda(const Opt& t) { if (t) need_cuda(*t); }
bool known(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
int64_t code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return VTX_F32;
        case at::kBFloat16: return VTX_BF16;
        case at::kHalf: return VTX_F16;
        default: raise(PyExc_TypeError, std::string("vortex_b200: unsupported dtype ") + c10::toString(t.scalar_type()));
    }
}
// parameters are read with their own dtype; dense and beside the activations
Tensor param(const Tensor& t, const Tensor& like) {
    if (t.device() != like.device()) raise(PyExc_RuntimeError, "vortex_b200: parameter on a different device than the activations");
    Tensor r = t;
    if (!known(r.scalar_type())) r = r.detach().to(at::kFloat);
    return r.is_contiguous() ? r : r.detach().contiguous();
}
Opt param(const Opt& t, const Tensor& like) { return t ? Opt(param(*t, like)) : Opt(); }
const void* ptr(const Tensor& t) { return t.const_data_ptr(); }
const void* ptr(const Opt& t) { return t ? t->const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.mutable_data_ptr(); }
// A tensor that the caller owns is written: autograd then sees that what it may have saved of it is gone.  (Tensors made in
// inference mode carry no version.)
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
int64_t code_or_0(const Opt& t) { return t ? code(*t) : 0; }
// (straight to the CUDA allocator: at::empty's way through the dispatcher costs another half microsecond)
Tensor empty(at::IntArrayRef size, const Tensor& like, at::ScalarType dtype) {
    return at::detail::empty_cuda(size, dtype, like.device(), std::nullopt);
}
void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
std::string str(const Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + (t.dim() == 1 ? ",)" : ")");
}

const Tensor& have(const Opt& t, const char* use) {
    if (!t) raise(PyExc_AttributeError, std::string("'NoneType' object has no attribute '") + use + "'");
    return *t;
}

// fp32 [G, S] parameter block; the tensors stay alive until the call has been issued
struct Modal {
    vtx_modal_params m{};
    Tensor lp, res;
    Opt th, ri;
    Modal(const Tensor& log_poles, const Tensor& residues, const Tensor& like, const Opt& theta, const Opt& res_im) {
        auto f32 = [&](const Tensor& t) {
            if (t.scalar_type() == at::kFloat && t.device() == like.device() && t.is_contiguous()) return t;
            return t.detach().to(like.device(), at::kFloat).contiguous();
        };
        res = f32(residues);
        if (res.dim() != 2) raise(PyExc_ValueError, "residues must be [G, S]");
        m.G = res.size(0); m.S = res.size(1);
        auto gs = [&](const Tensor& t) {
            Tensor r = f32(t);
            return r.numel() == m.G * m.S ? r : r.reshape({m.G, m.S});      // (raises as reshape does)
        };
        lp = gs(log_poles);
        if (theta) th = gs(*theta);
        if (res_im) ri = gs(*res_im);
        m.log_poles = ptr(lp); m.theta = ptr(th); m.res_re = ptr(res); m.res_im = ptr(ri);
    }
};

std::tuple<Tensor, Tensor, Tensor> decode_layer(Tensor u, const Tensor& w3_, const Opt& b3_, const Tensor& fir_state, int64_t D, const Opt& h_,
                                                const Opt& inner_state, const Opt& bias_, bool flip_filter, bool gated_bias, const Opt& log_poles,
                                                const Opt& residues, const Opt& iir_state, const Opt& theta, const Opt& res_im, int64_t layout,
                                                int64_t num_heads, bool flip) {
    need_cuda(u); need_cuda(w3_); need_cuda(fir_state);
    u = u.contiguous();
    if (u.dim() != 2) raise(PyExc_ValueError, "u must be [B, 3D]");
    const int64_t B = u.size(0), C3 = u.size(1);
    if (C3 != 3 * D) raise(PyExc_ValueError, "expected " + std::to_string(3 * D) + " packed channels, got " + std::to_string(C3));
    const Tensor w3 = param(w3_, u);
    const int64_t K3 = C3 ? w3.numel() / C3 : 0;
    if (K3 * C3 != w3.numel()) raise(PyExc_RuntimeError, "shape '[" + std::to_string(C3) + ", -1]' is invalid for input of size " + std::to_string(w3.numel()));
    const Opt b3 = param(b3_, u), bias = param(bias_, u);
    const Tensor fs = fir_state.contiguous();
    if (fs.size(-1) != K3 - 1) raise(PyExc_NotImplementedError, "decode_layer needs a full featurizer cache (prompt of at least K3-1 tokens)");
    vtx_decode_layer_params p{};
    p.io_dtype = code(u);
    Tensor fs_out = empty({B, C3, K3 - 1}, u, at::kFloat), y = empty({B, D}, u, u.scalar_type()), state;
    p.u = ptr(u); p.w3 = ptr(w3); p.w3_dtype = code(w3); p.b3 = ptr(b3); p.b3_dtype = code_or_0(b3);
    p.fir_state_in = ptr(fs); p.fir_state_dtype = code(fs); p.fir_state_out = static_cast<float*>(out(fs_out));
    p.bias = ptr(bias); p.bias_dtype = code_or_0(bias); p.y = out(y);
    p.B = B; p.D = D; p.K3 = K3; p.layout = layout; p.num_heads = num_heads; p.flip_x1x2 = flip; p.flip_filter = flip_filter;
    std::optional<Modal> modal;
    Tensor h, in;
    if (h_) {
        h = param(*h_, u);
        p.G = h.size(0);
        p.K = p.G ? h.numel() / p.G : 0;
        in = have(inner_state, "contiguous").contiguous();
        if (in.size(-1) != p.K - 1) raise(PyExc_NotImplementedError, "decode_layer needs a full inner cache (prompt of at least K-1 tokens)");
        state = empty({B, D, p.K - 1}, u, at::kFloat);
        p.h = ptr(h); p.h_dtype = code(h);
        p.inner_state_in = ptr(in); p.inner_state_dtype = code(in); p.inner_state_out = static_cast<float*>(out(state));
        p.bias_mode = bias ? (gated_bias ? VTX_BIAS_GATED : VTX_BIAS_ADD) : VTX_BIAS_NONE;
    } else {
        have(residues, "detach");
        modal.emplace(have(log_poles, "detach"), *residues, u, theta, res_im);
        in = have(iir_state, "contiguous").contiguous();
        if (in.scalar_type() != at::kFloat) in = in.to(at::kFloat);
        state = at::empty_like(in);
        p.modal = modal->m; p.K = 0; p.G = modal->m.G;
        p.iir_state_in = static_cast<const float*>(ptr(in)); p.iir_state_out = static_cast<float*>(out(state));
    }
    const c10::cuda::CUDAGuard on(u.device());
    check(p_decode_layer(&p, stream_of(u)));
    return {y, fs_out, state};
}

std::tuple<Tensor, Opt, Opt> fused_fir_fwd(Tensor u, const Tensor& w3_, const Opt& b3_, const Tensor& h_, const Opt& bias_, int64_t D, int64_t taps,
                                           int64_t bias_mode, int64_t layout, int64_t num_heads, bool flip, bool want_state, int64_t hist_rows) {
    need_cuda(u); need_cuda(w3_); need_cuda(b3_); need_cuda(h_); need_cuda(bias_);
    if (u.dim() != 3) raise(PyExc_ValueError, "u must be [B, L, 3D]");
    if (u.stride(2) != 1) {
        if (hist_rows) raise(PyExc_ValueError, "hist_rows needs u with unit channel stride (a view into the buffer that holds the history)");
        u = u.contiguous();
    }
    const int64_t B = u.size(0), L = u.size(1), C3 = u.size(2);
    if (C3 != 3 * D) raise(PyExc_ValueError, "expected " + std::to_string(3 * D) + " packed channels, got " + std::to_string(C3));
    const Tensor w3 = param(w3_, u), h = param(h_, u);
    const int64_t K3 = C3 ? w3.numel() / C3 : 0, G = h.size(0), K = G ? h.numel() / G : 0;
    if (K3 * C3 != w3.numel()) raise(PyExc_RuntimeError, "shape '[" + std::to_string(C3) + ", -1]' is invalid for input of size " + std::to_string(w3.numel()));
    const Opt b3 = param(b3_, u), bias = param(bias_, u);
    if (hist_rows && u.storage_offset() < hist_rows * u.stride(1))
        raise(PyExc_ValueError, "hist_rows=" + std::to_string(hist_rows) + ": u starts " +
                                    std::to_string(u.storage_offset() / std::max<int64_t>(u.stride(1), 1)) + " rows into its storage");
    vtx_fused_fir_params p{};
    p.io_dtype = code(u);
    Tensor y = empty({B, L, D}, u, u.scalar_type());
    Opt fs, ist;
    if (want_state) {
        fs = empty({B, C3, hist_rows ? K3 - 1 : std::min(L, K3 - 1)}, u, u.scalar_type());
        ist = empty({B, D, hist_rows ? K - 1 : std::min(L, K - 1)}, u, u.scalar_type());
        p.fir_state = fs->numel() ? out(*fs) : nullptr;
        p.inner_state = ist->numel() ? out(*ist) : nullptr;
    }
    p.u = ptr(u); p.u_stride_b = u.stride(0); p.u_stride_l = u.stride(1);
    p.w3 = ptr(w3); p.w3_dtype = code(w3); p.b3 = ptr(b3); p.b3_dtype = code_or_0(b3);
    p.h = ptr(h); p.h_dtype = code(h); p.bias = ptr(bias); p.bias_dtype = code_or_0(bias);
    p.y = out(y); p.y_stride_b = L * D; p.y_stride_l = D;
    p.B = B; p.L = L; p.D = D; p.G = G; p.K3 = K3; p.K = K;
    p.layout = layout; p.num_heads = num_heads; p.flip_x1x2 = flip;
    p.taps = taps; p.bias_mode = bias ? bias_mode : VTX_BIAS_NONE; p.u_hist_rows = hist_rows;
    const c10::cuda::CUDAGuard on(u.device());
    check(p_fused_fir_fwd(&p, stream_of(u)));
    return {y, fs, ist};
}

std::tuple<Tensor, Opt> fused_iir_fwd(Tensor u, const Tensor& w3_, const Tensor& log_poles, const Tensor& residues, const Opt& bias_, int64_t D,
                                      int64_t layout, int64_t num_heads, bool flip, const Opt& theta, const Opt& res_im, bool want_state,
                                      const Opt& b3_, Opt state_in, Opt fir_state_in, int64_t hist_rows, const Opt& out_) {
    need_cuda(u); need_cuda(w3_); need_cuda(residues); need_cuda(bias_); need_cuda(b3_); need_cuda(state_in); need_cuda(fir_state_in);
    if (u.dim() != 3) raise(PyExc_ValueError, "u must be [B, L, 3D]");
    if (u.stride(2) != 1) {
        if (hist_rows) raise(PyExc_ValueError, "hist_rows needs u with unit channel stride (a view into the buffer that holds the history)");
        u = u.contiguous();
    }
    if (hist_rows) {
        if (hist_rows < 2 || fir_state_in) raise(PyExc_ValueError, "hist_rows must be >= 2 and excludes fir_state_in");
        if (u.storage_offset() < hist_rows * u.stride(1))
            raise(PyExc_ValueError, "hist_rows=" + std::to_string(hist_rows) + ": u starts " +
                                        std::to_string(u.storage_offset() / std::max<int64_t>(u.stride(1), 1)) + " rows into its storage");
    }
    const int64_t B = u.size(0), L = u.size(1), C3 = u.size(2);
    if (C3 != 3 * D) raise(PyExc_ValueError, "expected " + std::to_string(3 * D) + " packed channels, got " + std::to_string(C3));
    const Tensor w3 = param(w3_, u);
    const int64_t K3 = C3 ? w3.numel() / C3 : 0;
    if (K3 * C3 != w3.numel()) raise(PyExc_RuntimeError, "shape '[" + std::to_string(C3) + ", -1]' is invalid for input of size " + std::to_string(w3.numel()));
    const Opt bias = param(bias_, u), b3 = param(b3_, u);
    const Modal m(log_poles, residues, u, theta, res_im);
    vtx_fused_iir_params p{};
    p.io_dtype = code(u);
    Tensor y;
    if (out_) {       // a [B, L, D] view with unit channel stride (e.g. a range of rows of a larger output)
        y = *out_;
        if (y.dim() != 3 || y.size(0) != B || y.size(1) != L || y.size(2) != D || y.scalar_type() != u.scalar_type() || y.stride(2) != 1 || y.device() != u.device())
            raise(PyExc_ValueError, "out must be a [B, L, D] tensor of u's dtype and device with unit channel stride");
    } else {
        y = empty({B, L, D}, u, u.scalar_type());
    }
    auto shape = [&] { return theta ? std::vector<int64_t>{B, D, m.m.S, 2} : std::vector<int64_t>{B, D, m.m.S}; };
    Opt st;
    if (want_state) { st = empty(shape(), u, at::kFloat); p.state = static_cast<float*>(out(*st)); }
    if (state_in) {
        if (state_in->sizes() != at::IntArrayRef(shape())) raise(PyExc_ValueError, "state_in has shape " + str(*state_in));
        state_in = state_in->to(at::kFloat).contiguous();
    }
    if (fir_state_in) {
        if (fir_state_in->sizes() != at::IntArrayRef({B, C3, 2}))
            raise(PyExc_ValueError, "fir_state_in has shape " + str(*fir_state_in) + ", expected (" + std::to_string(B) + ", " + std::to_string(C3) + ", 2)");
        fir_state_in = fir_state_in->contiguous();
    }
    p.u = ptr(u); p.u_stride_b = u.stride(0); p.u_stride_l = u.stride(1);
    p.w3 = ptr(w3); p.w3_dtype = code(w3); p.b3 = ptr(b3); p.b3_dtype = code_or_0(b3);
    p.modal = m.m; p.bias = ptr(bias); p.bias_dtype = code_or_0(bias);
    p.y = out(y); p.y_stride_b = y.stride(0); p.y_stride_l = y.stride(1);
    p.B = B; p.L = L; p.D = D; p.K3 = K3; p.layout = layout; p.num_heads = num_heads; p.flip_x1x2 = flip;
    p.state_in = static_cast<const float*>(ptr(state_in)); p.fir_state_in = ptr(fir_state_in); p.fir_state_dtype = code_or_0(fir_state_in);
    p.u_hist_rows = hist_rows;
    const int64_t need = p_fused_iir_scratch_bytes(&p);
    Tensor scratch;
    if (need > 0) { scratch = empty({need}, u, at::kByte); p.scratch = out(scratch); }
    const c10::cuda::CUDAGuard on(u.device());
    check(p_fused_iir_fwd(&p, stream_of(u)));
    return {y, st};
}

// ---- attention layers ----------------------------------------------------------------------------------------------------
[[noreturn]] void bad(const std::string& msg) { raise(PyExc_ValueError, msg); }
void same_device(const Tensor& t, const Tensor& like) {
    need_cuda(t);
    if (t.device() != like.device()) raise(PyExc_RuntimeError, "vortex_b200: tensors on different devices");
}
// [B, L, H, D] view of [T, H, D] or [B, L, H, D] rows, unit stride over D
struct Rows4 {
    Tensor t;
    int64_t B, L, H, D, sb, sl, sh;
    Rows4(const Tensor& x, const char* name) : t(x) {
        if (t.dim() != 3 && t.dim() != 4) bad(std::string(name) + " must be [T, H, D] or [B, L, H, D], got " + str(t));
        if (t.size(-1) != 1 && t.stride(-1) != 1) t = t.contiguous();
        const bool four = t.dim() == 4;
        B = four ? t.size(0) : 1; L = t.size(four ? 1 : 0); H = t.size(-2); D = t.size(-1);
        sb = four ? t.stride(0) : 0; sl = t.stride(four ? 1 : 0); sh = t.stride(-2);
    }
    bool tokens_as(const Rows4& o) const { return t.dim() == o.t.dim() && B == o.B && L == o.L && D == o.D; }
};

struct Rotary {
    vtx_rotary_params p{};
    std::vector<Tensor> keep;
    Rotary(const Rows4& q, const Rows4* k, const Opt& positions_, const Opt& inv_freq_, const Opt& qw, const Opt& kw, double eps, bool interleaved, double scale) {
        p.io_dtype = code(q.t);
        p.B = q.B; p.L = q.L; p.D = q.D; p.Hq = q.H;
        p.q = ptr(q.t); p.q_stride_b = q.sb; p.q_stride_l = q.sl; p.q_stride_h = q.sh;
        if (k) {
            same_device(k->t, q.t);
            if (!k->tokens_as(q) || k->t.scalar_type() != q.t.scalar_type())
                bad("k must have the tokens, head size and dtype of q: " + str(k->t) + " beside " + str(q.t));
            p.Hk = k->H;
            p.k = ptr(k->t); p.k_stride_b = k->sb; p.k_stride_l = k->sl; p.k_stride_h = k->sh;
        }
        if (positions_) {
            Tensor pos = *positions_;
            same_device(pos, q.t);
            if (pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong) raise(PyExc_TypeError, "positions must be int32 or int64");
            p.positions_i64 = pos.scalar_type() == at::kLong;
            if (q.t.dim() == 4 && pos.dim() == 2 && pos.size(0) == q.B && pos.size(1) == q.L) {
                p.pos_stride_b = pos.stride(0); p.pos_stride_l = pos.stride(1);
            } else if (pos.dim() == 1 && pos.size(0) == q.L) {          // [T], or [L] for every batch element
                p.pos_stride_l = pos.stride(0);
            } else {
                bad("positions have shape " + str(pos) + " for tokens of " + str(q.t));
            }
            p.positions = ptr(pos);
            keep.push_back(pos);
        }
        if (inv_freq_) {
            Tensor f = *inv_freq_;
            same_device(f, q.t);
            if (f.scalar_type() != at::kDouble && f.scalar_type() != at::kFloat) raise(PyExc_TypeError, "inv_freq must be float64 or float32");
            if (f.dim() != 1 || 2 * f.size(0) > q.D) bad("inv_freq must be [rot / 2] with rot <= " + std::to_string(q.D) + ", got " + str(f));
            f = f.contiguous();
            p.inv_freq = ptr(f); p.inv_freq_f64 = f.scalar_type() == at::kDouble; p.rot = 2 * f.size(0);
            keep.push_back(f);
        }
        auto weight = [&](const Opt& w, const char* name, const void*& at, int64_t& dt) {
            if (!w) return;
            need_cuda(*w);
            Tensor t = param(*w, q.t);
            if (t.dim() != 1 || t.size(0) != q.D) bad(std::string(name) + " must be [" + std::to_string(q.D) + "], got " + str(t));
            at = ptr(t); dt = code(t);
            keep.push_back(t);
        };
        weight(qw, "q_weight", p.q_weight, p.q_weight_dtype);
        weight(kw, "k_weight", p.k_weight, p.k_weight_dtype);
        p.eps = eps; p.interleaved = interleaved; p.scale = scale;
    }
    void q_to(const Tensor& t) { const Rows4 r(t, "q"); p.q_out = out(t); p.q_out_stride_b = r.sb; p.q_out_stride_l = r.sl; p.q_out_stride_h = r.sh; }
    void k_to(const Tensor& t) { const Rows4 r(t, "k"); p.k_out = out(t); p.k_out_stride_b = r.sb; p.k_out_stride_l = r.sl; p.k_out_stride_h = r.sh; }
};

std::tuple<Tensor, Opt> qk_norm_rotary(const Tensor& q_, const Opt& k_, const Tensor& positions, const Tensor& inv_freq, const Opt& qw, const Opt& kw,
                                       double eps, bool interleaved, double scale) {
    need_cuda(q_);
    const Rows4 q(q_, "q");
    std::optional<Rows4> k;
    if (k_) { need_cuda(*k_); k.emplace(*k_, "k"); }
    else if (kw) bad("k_weight without k");
    Rotary r(q, k ? &*k : nullptr, positions, inv_freq, qw, kw, eps, interleaved, scale);
    Tensor qo = empty(q.t.sizes(), q.t, q.t.scalar_type());
    Opt ko;
    r.q_to(qo);
    if (k) { ko = empty(k->t.sizes(), q.t, q.t.scalar_type()); r.k_to(*ko); }
    const c10::cuda::CUDAGuard on(q.t.device());
    check(p_rotary_fwd(&r.p, stream_of(q.t)));
    return {qo, ko};
}

std::tuple<Tensor, Opt, Opt, Opt> qk_norm_rotary_bwd(const Tensor& dq_, const Opt& dk_, const Tensor& q_, const Opt& k_, const Tensor& positions,
                                                     const Tensor& inv_freq, const Opt& qw, const Opt& kw, double eps, bool interleaved, double scale) {
    need_cuda(q_);
    const Rows4 q(q_, "q"), dq(dq_, "dq");
    std::optional<Rows4> k, dk;
    if (k_) {
        need_cuda(*k_);
        k.emplace(*k_, "k");
        dk.emplace(have(dk_, "shape"), "dk");
    }
    Rotary r(q, k ? &*k : nullptr, positions, inv_freq, qw, kw, eps, interleaved, scale);
    vtx_rotary_bwd_params p{};
    auto grad = [&](const Rows4& d, const Rows4& x, const void*& at, int64_t& sb, int64_t& sl, int64_t& sh) {
        same_device(d.t, q.t);
        if (d.t.sizes() != x.t.sizes() || d.t.scalar_type() != x.t.scalar_type()) bad("a gradient has shape " + str(d.t) + " or dtype other than its tensor's");
        at = ptr(d.t); sb = d.sb; sl = d.sl; sh = d.sh;
    };
    grad(dq, q, p.dq_out, p.dq_out_stride_b, p.dq_out_stride_l, p.dq_out_stride_h);
    if (k) grad(*dk, *k, p.dk_out, p.dk_out_stride_b, p.dk_out_stride_l, p.dk_out_stride_h);
    Tensor gq = empty(q.t.sizes(), q.t, q.t.scalar_type()), scratch;
    Opt gk, gqw, gkw;
    r.q_to(gq);
    if (k) { gk = empty(k->t.sizes(), q.t, q.t.scalar_type()); r.k_to(*gk); }
    auto dtype_of = [](int64_t c) { return c == VTX_F32 ? at::kFloat : c == VTX_BF16 ? at::kBFloat16 : at::kHalf; };
    if (qw) { gqw = empty({q.D}, q.t, dtype_of(r.p.q_weight_dtype)); p.dq_weight = out(*gqw); }
    if (kw) { gkw = empty({q.D}, q.t, dtype_of(r.p.k_weight_dtype)); p.dk_weight = out(*gkw); }
    p.fwd = r.p;
    const int64_t need = p_rotary_bwd_scratch_bytes(&p.fwd);
    if (need > 0) { scratch = empty({need}, q.t, at::kByte); p.scratch = out(scratch); }
    const c10::cuda::CUDAGuard on(q.t.device());
    check(p_rotary_bwd(&p, stream_of(q.t)));
    return {gq, gk, gqw, gkw};
}

// The differentiable call.  In C++ because a small step of training waits for the host: as a Python function forward and
// backward of 1003 tokens took 109 us, 15 of them on the GPU.
struct QkNormRotary : torch::autograd::Function<QkNormRotary> {
    using List = torch::autograd::variable_list;
    static List forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Opt& k, const Tensor& positions, const Tensor& inv_freq,
                        const Opt& qw, const Opt& kw, double eps, bool interleaved, double scale) {
        auto [qo, ko] = qk_norm_rotary(q, k, positions, inv_freq, qw, kw, eps, interleaved, scale);
        const bool norm = qw || kw;
        auto or_none = [](const Opt& t) { return t ? *t : Tensor(); };
        // (a rotation's gradient is the rotation back: it needs neither q nor k)
        ctx->save_for_backward({norm ? q : Tensor(), norm ? or_none(k) : Tensor(), positions, inv_freq, or_none(qw), or_none(kw)});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["scale"] = scale;
        return ko ? List{qo, *ko} : List{qo};
    }
    // The gradients of a tensor and its weight, as functions of what they were formed from: the output's gradient dy, and behind
    // a norm the tensor x and its weight w (without one the gradient is linear in dy).  There are no second derivatives, and a
    // node with edges to all of these says so on whichever of them a second differentiation goes through; one without them
    // would be passed over where only some inputs' gradients are asked for, and its part left out of the sum.
    static void once(Tensor& gx, Tensor& gw, const Tensor& dy, const Tensor& x, const Tensor& w) {
        List in{gx};
        if (w.defined()) {
            in.push_back(gw);
            in.push_back(x);
            in.push_back(w);
        }
        in.push_back(dy);
        const int64_t n = (int64_t)in.size();
        const auto node = std::make_shared<torch::autograd::DelayedError>(
            "qk_norm_rotary can be differentiated once: its gradients must not have been used in what is differentiated again", n);
        const List made = (*node)(std::move(in));
        gx = made[0];
        if (w.defined()) gw = made[1];
    }
    static List backward(torch::autograd::AutogradContext* ctx, const List& grads) {
        const List saved = ctx->get_saved_variables();
        auto opt = [](const Tensor& t) { return t.defined() ? Opt(t) : Opt(); };
        const Opt qw = opt(saved[4]), kw = opt(saved[5]);
        const bool norm = qw || kw;
        const Tensor &dq = grads[0], &q = norm ? saved[0] : dq;
        const Opt dk = grads.size() > 1 ? Opt(grads[1]) : Opt(), k = norm ? opt(saved[1]) : dk;
        List out(9);
        {
            const at::AutoGradMode off(false);
            auto [gq, gk, gqw, gkw] = qk_norm_rotary_bwd(dq, dk, q, k, saved[2], saved[3], qw, kw, ctx->saved_data["eps"].toDouble(),
                                                         ctx->saved_data["interleaved"].toBool(), ctx->saved_data["scale"].toDouble());
            out[0] = gq;
            if (gk) out[1] = *gk;
            if (gqw) out[4] = *gqw;
            if (gkw) out[5] = *gkw;
        }
        if (at::GradMode::is_enabled()) {                // (create_graph)
            once(out[0], out[4], grads[0], saved[0], saved[4]);
            if (dk) once(out[1], out[5], grads[1], saved[1], saved[5]);
        }
        return out;
    }
};

std::tuple<Tensor, Opt> qk_norm_rotary_grad(const Tensor& q, const Opt& k, const Tensor& positions, const Tensor& inv_freq, const Opt& qw, const Opt& kw,
                                            double eps, bool interleaved, double scale) {
    auto dual = [](const Opt& t) { return t && t->_fw_grad(/*level=*/0).defined(); };
    if (dual(q) || dual(k) || dual(inv_freq) || dual(qw) || dual(kw))            // (the kernel would drop the tangent)
        raise(PyExc_NotImplementedError, "qk_norm_rotary has no forward-mode derivative");
    auto wants = [](const Opt& t) { return t && t->requires_grad(); };
    if (!at::GradMode::is_enabled() || !(q.requires_grad() || wants(k) || wants(qw) || wants(kw)))
        return qk_norm_rotary(q, k, positions, inv_freq, qw, kw, eps, interleaved, scale);
    auto out = QkNormRotary::apply(q, k, positions, inv_freq, qw, kw, eps, interleaved, scale);
    return {out[0], out.size() > 1 ? Opt(out[1]) : Opt()};
}

struct Pool {
    int64_t pages, size, sp, ss, sh;
    Pool(const Tensor& t, const char* name, const Tensor& like, int64_t Hk, int64_t D) {
        same_device(t, like);
        if (t.dim() != 4 || t.size(2) != Hk || t.size(3) != D || t.scalar_type() != like.scalar_type())
            bad(std::string(name) + " must be [pages, page_size, " + std::to_string(Hk) + ", " + std::to_string(D) + "] of q's dtype, got " + str(t));
        if (D != 1 && t.stride(3) != 1) bad(std::string(name) + " must have unit stride over the head's values");
        pages = t.size(0); size = t.size(1); sp = t.stride(0); ss = t.stride(1); sh = t.stride(2);
    }
};
void int32_on(const Tensor& t, const char* name, const Tensor& like, int64_t dims) {
    same_device(t, like);
    if (t.scalar_type() != at::kInt) raise(PyExc_TypeError, std::string(name) + " must be int32");
    if (t.dim() != dims || (t.size(-1) > 1 && t.stride(-1) != 1)) bad(std::string(name) + " must be a dense " + std::to_string(dims) + "-dimensional tensor, got " + str(t));
}

Tensor rotary_append(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& positions, const Tensor& k_pages, const Tensor& v_pages,
                     const Tensor& table, const Opt& inv_freq, const Opt& qw, const Opt& kw, const Opt& seq_ids, double eps, bool interleaved,
                     double scale) {
    need_cuda(q_); need_cuda(k_); need_cuda(v_);
    const Rows4 q(q_, "q"), k(k_, "k"), v(v_, "v");
    Rotary r(q, &k, positions, inv_freq, qw, kw, eps, interleaved, scale);
    same_device(v.t, q.t);
    if (v.t.sizes() != k.t.sizes() || v.t.scalar_type() != k.t.scalar_type()) bad("v must have the shape and dtype of k");
    const Pool kp(k_pages, "k_pages", q.t, k.H, k.D), vp(v_pages, "v_pages", q.t, k.H, k.D);
    if (kp.pages != vp.pages || kp.size != vp.size || kp.size < 1) bad("k_pages and v_pages must have the same pages, of at least one token");
    for (const Tensor* t : {&k_pages, &v_pages})
        for (int i = 0; i < 4; ++i)
            if (t->size(i) > 1 && t->stride(i) == 0) bad("the pools are written: no dimension of theirs may be expanded");
    int32_on(table, "block_table", q.t, 2);
    vtx_rotary_append_params p{};
    Tensor qo = empty(q.t.sizes(), q.t, q.t.scalar_type());
    r.q_to(qo);
    p.rot = r.p;
    p.v = ptr(v.t); p.v_stride_b = v.sb; p.v_stride_l = v.sl; p.v_stride_h = v.sh;
    p.k_pages = out(k_pages); p.k_stride_page = kp.sp; p.k_stride_slot = kp.ss; p.k_stride_head = kp.sh;
    p.v_pages = out(v_pages); p.v_pages_stride_page = vp.sp; p.v_pages_stride_slot = vp.ss; p.v_pages_stride_head = vp.sh;
    p.block_table = static_cast<const int32_t*>(ptr(table)); p.table_stride = table.stride(0); p.table_width = table.size(1);
    p.num_seqs = table.size(0); p.num_pages = kp.pages; p.page_size = kp.size;
    if (seq_ids) {
        int32_on(*seq_ids, "seq_ids", q.t, 1);
        if (seq_ids->size(0) != q.B * q.L) bad("seq_ids must name a row of the block table for each of the " + std::to_string(q.B * q.L) + " tokens");
        p.seq_ids = static_cast<const int32_t*>(ptr(*seq_ids));
    } else if (q.B * q.L != p.num_seqs) {
        bad("without seq_ids there is one token for every row of the block table: " + std::to_string(q.B * q.L) + " tokens, " +
            std::to_string(p.num_seqs) + " rows");
    }
    const c10::cuda::CUDAGuard on(q.t.device());
    check(p_rotary_append(&p, stream_of(q.t)));
    written(k_pages); written(v_pages);
    return qo;
}

std::tuple<Tensor, Opt> paged_decode_attention(const Tensor& q_, const Tensor& k_pages, const Tensor& v_pages, const Opt& table, const Tensor& seqlens,
                                               std::optional<double> softmax_scale, int64_t window, bool want_lse) {
    need_cuda(q_);
    if (q_.dim() != 3) bad("q must be [B, H, D], got " + str(q_));
    const Tensor q = q_.size(2) != 1 && q_.stride(2) != 1 ? q_.contiguous() : q_;
    if (k_pages.dim() != 4) bad("k_pages must be [pages, page_size, H, D], got " + str(k_pages));
    vtx_paged_decode_params p{};
    p.io_dtype = code(q);
    p.B = q.size(0); p.Hq = q.size(1); p.D = q.size(2); p.Hk = k_pages.size(2);
    const Pool kp(k_pages, "k_pages", q, p.Hk, p.D), vp(v_pages, "v_pages", q, p.Hk, p.D);
    if (kp.pages != vp.pages || kp.size != vp.size) bad("k_pages and v_pages must have the same pages");
    int32_on(seqlens, "seqlens", q, 1);
    if (seqlens.size(0) != p.B) bad("seqlens must be [" + std::to_string(p.B) + "], got " + str(seqlens));
    if (table) {
        int32_on(*table, "block_table", q, 2);
        if (table->size(0) != p.B || table->size(1) < 1) bad("block_table must be [" + std::to_string(p.B) + ", pages of a sequence], got " + str(*table));
        p.block_table = static_cast<const int32_t*>(ptr(*table)); p.table_stride = table->stride(0); p.table_width = table->size(1);
    } else if (kp.pages != p.B) {
        bad("without a block_table the caches must be [B, keys, H, D]");
    }
    Tensor o = empty(q.sizes(), q, q.scalar_type()), scratch;
    Opt lse;
    if (want_lse) { lse = empty({p.B, p.Hq}, q, at::kFloat); p.lse = static_cast<float*>(out(*lse)); }
    p.q = ptr(q); p.q_stride_b = q.stride(0); p.q_stride_h = q.stride(1);
    p.k_pages = ptr(k_pages); p.k_stride_page = kp.sp; p.k_stride_slot = kp.ss; p.k_stride_head = kp.sh;
    p.v_pages = ptr(v_pages); p.v_stride_page = vp.sp; p.v_stride_slot = vp.ss; p.v_stride_head = vp.sh;
    p.seqlens = static_cast<const int32_t*>(ptr(seqlens));
    p.out = out(o); p.out_stride_b = o.stride(0); p.out_stride_h = o.stride(1);
    p.softmax_scale = softmax_scale ? *softmax_scale : 1.0 / std::sqrt((double)p.D);
    p.window = window; p.num_pages = kp.pages; p.page_size = kp.size;
    const c10::cuda::CUDAGuard on(q.device());
    const int64_t need = p_paged_decode_scratch_bytes(&p);
    if (need > 0) { scratch = empty({need}, q, at::kByte); p.scratch = out(scratch); }
    check(p_paged_decode(&p, stream_of(q)));
    return {o, lse};
}

void copy_pages(const std::vector<Tensor>& pools, const std::vector<int64_t>& src, const std::vector<int64_t>& dst) {
    if (src.size() != dst.size()) bad("copy_pages: " + std::to_string(src.size()) + " sources for " + std::to_string(dst.size()) + " destinations");
    if (pools.empty()) return;
    vtx_copy_pages_params p{};
    const Tensor& first = pools[0];
    std::vector<void*> at;
    for (const Tensor& t : pools) {
        same_device(t, first);
        if (t.dim() < 1 || t.sizes() != first.sizes() || t.strides() != first.strides() || t.scalar_type() != first.scalar_type())
            bad("copy_pages: the pools must have one shape, layout and dtype");
        at.push_back(out(t));
    }
    const int64_t n = first.size(0), es = first.element_size();
    int64_t page = 1;
    for (int64_t i = first.dim() - 1; i > 0; --i) {
        if (first.size(i) > 1 && first.stride(i) != page) bad("copy_pages: a page must be contiguous");
        page *= first.size(i);
    }
    p.pool_ptrs = at.data(); p.src = src.data(); p.dst = dst.data();
    p.pools = (int64_t)pools.size(); p.pairs = (int64_t)src.size(); p.num_pages = n;
    p.page_bytes = page * es; p.page_stride_bytes = n > 1 ? first.stride(0) * es : page * es;
    const c10::cuda::CUDAGuard on(first.device());
    check(p_copy_pages(&p, stream_of(first)));
    if (p.pairs) for (const Tensor& t : pools) written(t);
}

}  // namespace

PYBIND11_MODULE(_vtx_host, m) {
    m.def("abi_version", [] { return VTX_ABI_VERSION; });
    m.def("bind", [](uintptr_t decode, uintptr_t fir, uintptr_t iir, uintptr_t iir_scratch, uintptr_t last_error) {
        p_decode_layer = reinterpret_cast<decltype(p_decode_layer)>(decode);
        p_fused_fir_fwd = reinterpret_cast<decltype(p_fused_fir_fwd)>(fir);
        p_fused_iir_fwd = reinterpret_cast<decltype(p_fused_iir_fwd)>(iir);
        p_fused_iir_scratch_bytes = reinterpret_cast<decltype(p_fused_iir_scratch_bytes)>(iir_scratch);
        p_last_error = reinterpret_cast<decltype(p_last_error)>(last_error);
    });
    // the attention layers' functions, by name
    m.def("bind_attention", [](const std::map<std::string, uintptr_t>& f) {
        p_rotary_fwd = reinterpret_cast<decltype(p_rotary_fwd)>(f.at("vtx_qk_norm_rotary_fwd"));
        p_rotary_bwd = reinterpret_cast<decltype(p_rotary_bwd)>(f.at("vtx_qk_norm_rotary_bwd"));
        p_rotary_bwd_scratch_bytes = reinterpret_cast<decltype(p_rotary_bwd_scratch_bytes)>(f.at("vtx_qk_norm_rotary_bwd_scratch_bytes"));
        p_rotary_append = reinterpret_cast<decltype(p_rotary_append)>(f.at("vtx_rotary_append"));
        p_paged_decode = reinterpret_cast<decltype(p_paged_decode)>(f.at("vtx_paged_decode_attention"));
        p_paged_decode_scratch_bytes = reinterpret_cast<decltype(p_paged_decode_scratch_bytes)>(f.at("vtx_paged_decode_scratch_bytes"));
        p_copy_pages = reinterpret_cast<decltype(p_copy_pages)>(f.at("vtx_copy_pages"));
    });
    // Without the GIL, as torch's own calls and calls through ctypes are: an allocation or a launch into a full queue can
    // block, and the process's other threads go on meanwhile.
    m.def("decode_layer", &decode_layer, py::call_guard<py::gil_scoped_release>());
    m.def("fused_fir_fwd", &fused_fir_fwd, py::call_guard<py::gil_scoped_release>());
    m.def("fused_iir_fwd", &fused_iir_fwd, py::call_guard<py::gil_scoped_release>());
    m.def("qk_norm_rotary", &qk_norm_rotary_grad, py::call_guard<py::gil_scoped_release>());
    m.def("qk_norm_rotary_bwd", &qk_norm_rotary_bwd, py::call_guard<py::gil_scoped_release>());
    m.def("rotary_append", &rotary_append, py::call_guard<py::gil_scoped_release>());
    m.def("paged_decode_attention", &paged_decode_attention, py::call_guard<py::gil_scoped_release>());
    m.def("copy_pages", &copy_pages, py::call_guard<py::gil_scoped_release>());
}
