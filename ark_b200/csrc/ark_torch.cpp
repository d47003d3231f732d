// ark_torch.cpp -- torch binding of the activation operators (section 4 of
// ark_opt.h): checks of arguments, outputs and workspaces from torch's
// allocator, torch's current stream, and the call into libark_cuda.so.
//
// These calls are a few microseconds of GPU time each at small sizes, which the
// same checks in Python did not keep up with (23 us of host time for a rotation
// of 64 tokens that runs 3.5 us).
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <string>
#include <tuple>
#include <utility>

#include "../../include/ark_opt.h"

namespace py = pybind11;
using at::Tensor;
using MaybeTensor = std::optional<Tensor>;
using Outputs = std::pair<Tensor, MaybeTensor>;

namespace {

[[noreturn]] void bad_value(const std::string& s) { throw py::value_error(s); }
[[noreturn]] void bad_type(const std::string& s) { throw py::type_error(s); }

// ArkError(fn, code) for a status that is not success
void check(const char* fn, int code) {
    if (code == ARK_OK) return;
    const py::object cls = py::module_::import("ark_b200._lib").attr("ArkError");
    PyErr_SetObject(cls.ptr(), cls(fn, code).ptr());
    throw py::error_already_set();
}

std::string shape_of(const Tensor& t) {
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}

int type_code(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return ARK_TYPE_F16;
        case at::kBFloat16: return ARK_TYPE_BF16;
        case at::kFloat: return ARK_TYPE_F32;
        case at::kInt: return ARK_TYPE_I32;
        case at::kLong: return ARK_TYPE_I64;
        default: return -1;
    }
}
bool is_float(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16 || t == at::kFloat; }

void need_float(const Tensor& t, const char* what, bool half_only = false) {
    if (!is_float(t.scalar_type()) || (half_only && t.scalar_type() == at::kFloat))
        bad_type(std::string(what) + ": unsupported type " + toString(t.scalar_type()));
    if (!t.is_cuda()) bad_value(std::string(what) + ": buffers must be CUDA tensors (device memory)");
}
void need_like(const Tensor& t, const Tensor& like, const char* what) {
    if (t.scalar_type() != like.scalar_type() || t.device() != like.device())
        bad_value(std::string(what) + ": expected " + toString(like.scalar_type()) + " on " +
                  like.device().str() + ", got " + toString(t.scalar_type()) + " on " + t.device().str());
}
void need_device(at::Device a, at::Device b) {
    if (a != b) bad_value("buffers on " + a.str() + " and " + b.str());
}

// a [rows, cols] tensor with contiguous rows; returns its row stride
uint64_t rows_of(const Tensor& t, const char* what, int64_t rows = -1, int64_t cols = -1,
                 bool written = false) {
    need_float(t, what);
    if (t.dim() != 2 || (rows >= 0 && t.size(0) != rows) || (cols >= 0 && t.size(1) != cols))
        bad_value(std::string(what) + ": expected [" + (rows < 0 ? "rows" : std::to_string(rows)) + ", " +
                  (cols < 0 ? "cols" : std::to_string(cols)) + "], got " + shape_of(t));
    if (t.size(1) > 1 && t.stride(1) != 1) bad_value(std::string(what) + ": rows must be contiguous");
    if (written && t.size(0) > 1 && t.stride(0) < t.size(1))
        bad_value(std::string(what) + ": rows of an output may not overlap");
    return (uint64_t)t.stride(0);
}

// The tensors' device as the current one, and torch's current stream there.
struct On {
    c10::cuda::CUDAGuard guard;
    void* stream;
    explicit On(at::Device d)
        : guard(d), stream(c10::cuda::getCurrentCUDAStream(d.index()).stream()) {}
};

Tensor fresh(at::IntArrayRef size, at::ScalarType type, at::Device d) {
    return at::detail::empty_cuda(size, type, d, std::nullopt);
}

// ------------------------------------------------------------ Act8
int kind_code(const std::string& kind) {
    if (kind == "e4m3") return ARK_ACT8_E4M3;
    if (kind == "int8") return ARK_ACT8_INT8;
    bad_value("kind: expected 'e4m3' or 'int8', got '" + kind + "'");
}

class Act8 {
public:
    // tensors that a caller holds
    Act8(const py::object& data, const py::object& scale, int64_t cols, const std::string& kind, bool wide)
        : cols_(cols), kind_(kind_code(kind)) {
        if (cols < 0) bad_value("cols: expected a length");
        const int64_t pitch = (int64_t)ark_cuda_act8_pitch((uint64_t)cols);
        data_ = bytes(data, "data");
        scale_ = bytes(scale, "scale");
        rows_ = data_.dim() == 2 ? data_.size(0) : -1;
        shaped(data_, "data", pitch);
        shaped(scale_, "scale", pitch / 32);
        need_device(data_.device(), scale_.device());
        c_ = ark_act8{data_.data_ptr<uint8_t>(), scale_.data_ptr<uint8_t>(), (uint64_t)rows_,
                      (uint64_t)cols_, kind_, wide};
    }
    // room for one, in one allocation
    Act8(int64_t rows, int64_t cols, int kind, at::Device d, at::ScalarType from) : rows_(rows), cols_(cols), kind_(kind) {
        if (rows < 0 || cols < 0) bad_value("rows, cols: expected lengths");
        if (!d.is_cuda()) bad_value("buffers must be CUDA tensors (device memory)");
        const int64_t pitch = (int64_t)ark_cuda_act8_pitch((uint64_t)cols);
        whole_ = fresh({rows * (pitch + pitch / 32)}, at::kByte, d);
        uint8_t* p = whole_.data_ptr<uint8_t>();
        c_ = ark_act8{p, p + rows * pitch, (uint64_t)rows, (uint64_t)cols, kind, 0};
        hold(from);
    }
    // what it is packed from
    void hold(at::ScalarType from) { c_.wide = from != at::kHalf; }
    bool wide() const { return c_.wide != 0; }
    const ark_act8* c() const { return &c_; }
    at::Device device() const { return whole_.defined() ? whole_.device() : data_.device(); }
    int64_t rows() const { return rows_; }
    int64_t cols() const { return cols_; }
    int kind() const { return kind_; }
    std::string kind_name() const { return kind_ == ARK_ACT8_E4M3 ? "e4m3" : "int8"; }
    int64_t pitch() const { return (int64_t)ark_cuda_act8_pitch((uint64_t)cols_); }
    int64_t nbytes() const { return rows_ * (pitch() + pitch() / 32); }
    Tensor data() {
        if (!data_.defined()) data_ = whole_.narrow(0, 0, rows_ * pitch()).view({rows_, pitch()});
        return data_;
    }
    Tensor scale() {
        if (!scale_.defined())
            scale_ = whole_.narrow(0, rows_ * pitch(), rows_ * (pitch() / 32)).view({rows_, pitch() / 32});
        return scale_;
    }
    void need(const char* what, int64_t rows, int64_t cols) const {
        if (rows_ != rows || cols_ != cols)
            bad_value(std::string(what) + ": expected a checkpoint of [" + std::to_string(rows) + ", " +
                      std::to_string(cols) + "], got [" + std::to_string(rows_) + ", " +
                      std::to_string(cols_) + "]");
    }

private:
    static Tensor bytes(const py::object& o, const char* what) {
        if (!THPVariable_Check(o.ptr()) || THPVariable_Unpack(o.ptr()).scalar_type() != at::kByte)
            bad_type(std::string(what) + ": expected a uint8 CUDA tensor");
        const Tensor t = THPVariable_Unpack(o.ptr());
        if (!t.is_cuda()) bad_value(std::string(what) + ": buffers must be CUDA tensors (device memory)");
        return t;
    }
    void shaped(const Tensor& t, const char* what, int64_t width) const {
        if (t.dim() != 2 || t.size(0) != rows_ || t.size(1) != width || !t.is_contiguous())
            bad_value(std::string(what) + ": expected contiguous [rows, " + std::to_string(width) +
                      "], got " + shape_of(t));
    }
    Tensor whole_, data_, scale_;
    int64_t rows_ = 0, cols_ = 0;
    int kind_;
    ark_act8 c_;
};

// ------------------------------------------------------------ checkpoints
Act8 act8_pack(const Tensor& x, const std::optional<std::string>& kind, Act8* out) {
    const uint64_t ld = rows_of(x, "x");
    const int code = kind ? kind_code(*kind) : out ? out->kind() : ARK_ACT8_E4M3;
    if (out && code != out->kind()) bad_value("out: expected a checkpoint of " + *kind + ", got " + out->kind_name());
    const On on(x.device());
    if (out) {
        out->need("out", x.size(0), x.size(1));
        need_device(x.device(), out->device());
    }
    const Act8 c = out ? *out : Act8(x.size(0), x.size(1), code, x.device(), x.scalar_type());
    check("ark_cuda_act8_pack",
          ark_cuda_act8_pack(x.data_ptr(), type_code(x.scalar_type()), ld, c.c(), on.stream));
    if (!out) return c;
    out->hold(x.scalar_type());
    return *out;
}

Tensor act8_unpack(const Act8& c, at::ScalarType dtype, const MaybeTensor& out) {
    const On on(c.device());
    Tensor y;
    if (out) {
        rows_of(*out, "out", c.rows(), c.cols(), true);
        need_device(c.device(), out->device());
        y = *out;
    } else {
        if (!is_float(dtype)) bad_type(std::string("unsupported type ") + toString(dtype));
        y = fresh({c.rows(), c.cols()}, dtype, c.device());
    }
    check("ark_cuda_act8_unpack", ark_cuda_act8_unpack(c.c(), y.data_ptr(), type_code(y.scalar_type()),
                                                       (uint64_t)y.stride(0), on.stream));
    return y;
}

Tensor weight_grad(const Act8& x, const Tensor& dy, const MaybeTensor& out, bool accumulate,
                   const std::optional<at::ScalarType>& dtype) {
    need_float(dy, "dy", true);
    const uint64_t ld = rows_of(dy, "dy", x.rows());
    if (accumulate && !out) bad_value("accumulate needs out");
    need_device(x.device(), dy.device());
    const On on(dy.device());
    const int64_t n = dy.size(1);
    Tensor w;
    if (out) {
        rows_of(*out, "out", x.cols(), n, true);
        need_device(dy.device(), out->device());
        if (dtype && out->scalar_type() != *dtype)
            bad_value(std::string("out: expected ") + toString(*dtype) + ", got " + toString(out->scalar_type()));
        w = *out;
    } else {
        if (dtype && !is_float(*dtype)) bad_type(std::string("unsupported type ") + toString(*dtype));
        w = fresh({x.cols(), n}, dtype ? *dtype : dy.scalar_type(), dy.device());
    }
    const int type = type_code(w.scalar_type());
    const uint64_t ldw = (uint64_t)w.stride(0);
    ark_act8 c = *x.c();
    if (dy.scalar_type() != at::kHalf) c.wide = 0;   // BF16 has the range
    const uint64_t need = ark_cuda_weight_grad_workspace(&c, dy.data_ptr(), ld, (uint64_t)n);
    Tensor ws;
    if (need) ws = fresh({(int64_t)need}, at::kByte, dy.device());
    check("ark_cuda_weight_grad",
          ark_cuda_weight_grad(&c, dy.data_ptr(), type_code(dy.scalar_type()), ld, (uint64_t)n,
                               w.data_ptr(), type, ldw, accumulate, need ? ws.data_ptr() : nullptr, need,
                               on.stream));
    return w;
}

// ------------------------------------------------------------ SwiGLU
py::object swiglu(const Tensor& a, const Tensor& b, const std::optional<std::string>& checkpoint,
                  const MaybeTensor& out) {
    const uint64_t la = rows_of(a, "a");
    const int64_t rows = a.size(0), cols = a.size(1);
    const uint64_t lb = rows_of(b, "b", rows, cols);
    need_like(b, a, "b");
    const On on(a.device());
    if (out) {
        rows_of(*out, "out", rows, cols, true);
        need_like(*out, a, "out");
    }
    const Tensor y = out ? *out : fresh({rows, cols}, a.scalar_type(), a.device());
    std::optional<Act8> ca, cb;
    if (checkpoint) {
        const int kind = kind_code(*checkpoint);
        ca.emplace(rows, cols, kind, a.device(), a.scalar_type());
        cb.emplace(rows, cols, kind, a.device(), a.scalar_type());
    }
    check("ark_cuda_swiglu",
          ark_cuda_swiglu(a.data_ptr(), la, b.data_ptr(), lb, type_code(a.scalar_type()), (uint64_t)rows,
                          (uint64_t)cols, y.data_ptr(), (uint64_t)y.stride(0), ca ? ca->c() : nullptr,
                          cb ? cb->c() : nullptr, on.stream));
    return ca ? py::object(py::make_tuple(y, *ca, *cb)) : py::cast(y);
}

py::tuple swiglu_backward(const Tensor& dy, const Act8& ca, const Act8& cb,
                          const std::optional<std::string>& checkpoint,
                          const std::optional<std::pair<Tensor, Tensor>>& out) {
    const int64_t rows = ca.rows(), cols = ca.cols();
    cb.need("cb", rows, cols);
    if (cb.kind() != ca.kind() || (checkpoint && kind_code(*checkpoint) != ca.kind()))
        bad_value("checkpoints of one call are of one kind");
    const uint64_t lg = rows_of(dy, "dy", rows, cols);
    need_device(dy.device(), ca.device());
    need_device(dy.device(), cb.device());
    const On on(dy.device());
    Tensor da, db;
    if (out) {
        rows_of(out->first, "da", rows, cols, true);
        rows_of(out->second, "db", rows, cols, true);
        need_like(out->first, dy, "da");
        need_like(out->second, dy, "db");
        da = out->first, db = out->second;
    } else {
        da = fresh({rows, cols}, dy.scalar_type(), dy.device());
        db = fresh({rows, cols}, dy.scalar_type(), dy.device());
    }
    std::optional<Act8> cy;
    if (checkpoint) cy.emplace(rows, cols, ca.kind(), dy.device(), dy.scalar_type());
    check("ark_cuda_swiglu_backward",
          ark_cuda_swiglu_backward(dy.data_ptr(), lg, type_code(dy.scalar_type()), ca.c(), cb.c(),
                                   da.data_ptr(), (uint64_t)da.stride(0), db.data_ptr(),
                                   (uint64_t)db.stride(0), cy ? cy->c() : nullptr, on.stream));
    return cy ? py::make_tuple(da, db, *cy) : py::make_tuple(da, db);
}

// ------------------------------------------------------------ rotary positions
struct RopePlan {
    ark_rope_plan c;
    RopePlan(int64_t rotary_dim, double base, const std::string& layout,
             const std::optional<std::string>& scaling, double factor, double original, double fast,
             double slow) {
        if (layout != "half" && layout != "interleaved")
            bad_value("layout: expected 'half' or 'interleaved', got '" + layout + "'");
        const std::string s = scaling ? *scaling : "none";
        const char* names[] = {"none", "linear", "base", "parts", "wave"};
        int code = -1;
        for (int i = 0; i < 5; ++i)
            if (s == names[i]) code = i;
        if (code < 0)
            bad_value("scaling: expected 'linear', 'base', 'parts', 'wave' or None, got '" + s + "'");
        if (rotary_dim < 2 || rotary_dim > ARK_ROPE_MAX_DIM || rotary_dim % 2)
            bad_value("rotary_dim: expected an even number from 2 to " + std::to_string(ARK_ROPE_MAX_DIM) +
                      ", got " + std::to_string(rotary_dim));
        check("ark_cuda_rope_plan",
              ark_cuda_rope_plan(&c, (uint32_t)rotary_dim, layout == "interleaved", base, (uint32_t)code,
                                 factor, original, fast, slow));
    }
    std::vector<double> frequencies() const {
        std::vector<double> f;
        for (uint32_t i = 0; i < c.rotary_dim / 2; ++i)
            f.push_back(std::ldexp((double)c.turns[i], -64) * 6.283185307179586476925);
        return f;
    }
};

struct Positions {
    const void* p = nullptr;
    int type = 0;
    uint64_t seq = 0;
    Positions(const MaybeTensor& positions, const std::optional<int64_t>& seq_len, const Tensor& q) {
        const int64_t tokens = q.size(0);
        if (!positions) {
            const int64_t n = seq_len ? *seq_len : tokens;
            if (n < 0 || (n == 0 && tokens)) bad_value("seq_len: expected a positive length");
            seq = n ? (uint64_t)n : 1;
            return;
        }
        if (seq_len) bad_value("positions or seq_len, not both");
        const Tensor& t = *positions;
        if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong)
            bad_type("positions: expected an int32 or int64 CUDA tensor");
        if (t.device() != q.device())
            bad_value("positions: expected on " + q.device().str() + ", got " + t.device().str());
        if (t.dim() != 1 || t.size(0) != tokens || !t.is_contiguous())
            bad_value("positions: expected contiguous [" + std::to_string(tokens) + "], got " + shape_of(t));
        p = t.data_ptr();
        type = type_code(t.scalar_type());
        if (!p) seq = 1;   // no tokens: torch gives no memory, and the call takes no positions for a length
    }
};

ark_heads heads_of(const Tensor& t, const char* what) {
    need_float(t, what);
    if (t.dim() != 3) bad_value(std::string(what) + ": expected [tokens, heads, dim], got " + shape_of(t));
    if (t.size(2) > 1 && t.stride(2) != 1)
        bad_value(std::string(what) + ": the last dimension must be contiguous");
    return ark_heads{t.data_ptr(), (uint64_t)t.size(1), (uint64_t)t.stride(0), (uint64_t)t.stride(1)};
}

// q and k of a call and their outputs
struct Pair {
    Tensor oq, ok;
    ark_heads q, k, out_q, out_k;
    bool two;
    Pair(const Tensor& tq, const MaybeTensor& tk, const RopePlan& plan, const std::optional<Outputs>& out,
         const char* nq = "q", const char* nk = "k")
        : two(tk.has_value()) {
        q = heads_of(tq, nq);
        const int64_t t = tq.size(0), d = tq.size(2);
        if (d < (int64_t)plan.c.rotary_dim)
            bad_value(std::string(nq) + ": heads of " + std::to_string(d) + " are shorter than the rotated " +
                      std::to_string(plan.c.rotary_dim));
        if (d > ARK_ROPE_MAX_DIM)
            bad_value(std::string(nq) + ": heads of " + std::to_string(d) + ": at most " +
                      std::to_string(ARK_ROPE_MAX_DIM) + " are supported");
        if (two) {
            k = heads_of(*tk, nk);
            need_like(*tk, tq, nk);
            if (tk->size(0) != t || tk->size(2) != d)
                bad_value(std::string(nk) + ": expected [" + std::to_string(t) + ", heads, " +
                          std::to_string(d) + "], got " + shape_of(*tk));
        }
        if (out) {
            oq = out->first;
            out_q = same(oq, tq, "out q");
            if (two != out->second.has_value()) bad_value("out: one tensor for each of q and k");
            if (two) ok = *out->second, out_k = same(ok, *tk, "out k");
        } else {
            oq = fresh(tq.sizes(), tq.scalar_type(), tq.device());
            out_q = heads_of(oq, "out q");
            if (two) ok = fresh(tk->sizes(), tk->scalar_type(), tk->device()), out_k = heads_of(ok, "out k");
        }
    }
    const ark_heads* pk() const { return two ? &k : nullptr; }
    const ark_heads* pok() const { return two ? &out_k : nullptr; }
    py::object k_out() const { return two ? py::cast(ok) : py::none(); }

private:
    static ark_heads same(const Tensor& o, const Tensor& t, const char* what) {
        const ark_heads h = heads_of(o, what);
        need_like(o, t, what);
        if (o.sizes() != t.sizes())
            bad_value(std::string(what) + ": expected " + shape_of(t) + ", got " + shape_of(o));
        return h;
    }
};

const void* gain_of(const Tensor& g, const char* what, const Tensor& q) {
    need_float(g, what);
    if (g.dim() != 1 || g.size(0) != q.size(2) || !g.is_contiguous() || g.device() != q.device())
        bad_value(std::string(what) + ": expected contiguous [" + std::to_string(q.size(2)) + "] on " +
                  q.device().str() + ", got " + shape_of(g) + " on " + g.device().str());
    return g.data_ptr();
}
struct Gains {
    const void *q, *k = nullptr;
    int type;
    Gains(const Tensor& t, bool two, const Tensor& gq, const MaybeTensor& gk, const char* nq, const char* nk)
        : q(gain_of(gq, nq, t)), type(type_code(gq.scalar_type())) {
        if (!two) return;
        if (!gk) bad_value(std::string(nk) + ": expected a tensor");
        k = gain_of(*gk, nk, t);
        if (gk->scalar_type() != gq.scalar_type())
            bad_value(std::string(nq) + " and " + nk + " are of different types");
    }
};

py::tuple rope(const Tensor& q, const MaybeTensor& k, const RopePlan& plan, const MaybeTensor& positions,
               const std::optional<int64_t>& seq_len, bool inverse, const std::optional<Outputs>& out) {
    need_float(q, "q");
    const On on(q.device());
    const Pair p(q, k, plan, out);
    const Positions pos(positions, seq_len, q);
    check("ark_cuda_rope",
          ark_cuda_rope(&plan.c, &p.q, p.pk(), &p.out_q, p.pok(), type_code(q.scalar_type()),
                        (uint64_t)q.size(0), (uint64_t)q.size(2), pos.p, pos.type, pos.seq, inverse,
                        on.stream));
    return py::make_tuple(p.oq, p.k_out());
}

py::tuple qk_norm_rope(const Tensor& q, const MaybeTensor& k, const Tensor& gain_q, const MaybeTensor& gain_k,
                       const RopePlan& plan, const MaybeTensor& positions,
                       const std::optional<int64_t>& seq_len, double eps,
                       const std::optional<std::string>& checkpoint, const std::optional<Outputs>& out) {
    need_float(q, "q");
    const On on(q.device());
    const Pair p(q, k, plan, out);
    const Gains g(q, p.two, gain_q, gain_k, "gain_q", "gain_k");
    const Positions pos(positions, seq_len, q);
    std::optional<Act8> cq, ck;
    if (checkpoint) {
        const int kind = kind_code(*checkpoint);
        cq.emplace(q.size(0), q.size(1) * q.size(2), kind, q.device(), q.scalar_type());
        if (k) ck.emplace(k->size(0), k->size(1) * k->size(2), kind, q.device(), q.scalar_type());
    }
    check("ark_cuda_qk_norm_rope",
          ark_cuda_qk_norm_rope(&plan.c, &p.q, p.pk(), &p.out_q, p.pok(), type_code(q.scalar_type()),
                                (uint64_t)q.size(0), (uint64_t)q.size(2), g.q, g.k, g.type, (float)eps,
                                pos.p, pos.type, pos.seq, cq ? cq->c() : nullptr, ck ? ck->c() : nullptr,
                                on.stream));
    if (!cq) return py::make_tuple(p.oq, p.k_out());
    return py::make_tuple(p.oq, p.k_out(), *cq, ck ? py::cast(*ck) : py::none());
}

// x of the backward: a checkpoint, or the tensor itself
struct Source {
    const ark_act8* held = nullptr;
    const ark_heads* tensor = nullptr;
    ark_heads h;
    int kind = -1;
    Source(const py::object& x, const Tensor& d, const char* what) {
        if (py::isinstance<Act8>(x)) {
            const Act8& c = x.cast<const Act8&>();
            need_device(d.device(), c.device());
            c.need(what, d.size(0), d.size(1) * d.size(2));
            held = c.c();
            kind = c.kind();
            return;
        }
        if (!THPVariable_Check(x.ptr())) bad_type(std::string(what) + ": expected an Act8 or a CUDA tensor");
        const Tensor& t = THPVariable_Unpack(x.ptr());
        h = heads_of(t, what);
        need_like(t, d, what);
        if (t.sizes() != d.sizes())
            bad_value(std::string(what) + ": expected " + shape_of(d) + ", got " + shape_of(t));
        tensor = &h;
    }
    Source() {}
    Source(const Source&) = delete;
};

py::tuple qk_norm_rope_backward(const Tensor& dq, const MaybeTensor& dk, const py::object& q,
                                const py::object& k, const Tensor& gain_q, const MaybeTensor& gain_k,
                                const RopePlan& plan, const MaybeTensor& positions,
                                const std::optional<int64_t>& seq_len, double eps,
                                const std::optional<Outputs>& out, const std::optional<Outputs>& out_gains,
                                bool accumulate) {
    if (accumulate && !out_gains) bad_value("accumulate needs out_gains");
    need_float(dq, "dq");
    const On on(dq.device());
    const Pair p(dq, dk, plan, out, "dq", "dk");
    const Gains g(dq, p.two, gain_q, gain_k, "gain_q", "gain_k");
    const Positions pos(positions, seq_len, dq);
    const Source sq(q, dq, "q");
    std::optional<Source> sk;
    if (p.two) {
        sk.emplace(k, *dk, "k");
        if (sk->kind != sq.kind) bad_value("q and k: both checkpoints of one kind, or both tensors");
    }
    Tensor gq, gk;
    if (out_gains) {
        gq = out_gains->first;
        if (p.two && !out_gains->second) bad_value("out_gains: one tensor for each of q and k");
        if (p.two) gk = *out_gains->second;
    } else {
        gq = fresh(gain_q.sizes(), gain_q.scalar_type(), dq.device());
        if (p.two) gk = fresh(gain_k->sizes(), gain_k->scalar_type(), dq.device());
    }
    const Gains dg(dq, p.two, gq, p.two ? MaybeTensor(gk) : MaybeTensor(), "dgain_q", "dgain_k");
    const uint64_t need = ark_cuda_qk_norm_rope_workspace((uint64_t)dq.size(2));
    const Tensor ws = fresh({(int64_t)(need / 4)}, at::kFloat, dq.device());
    check("ark_cuda_qk_norm_rope_backward",
          ark_cuda_qk_norm_rope_backward(
              &plan.c, &p.q, p.pk(), &p.out_q, p.pok(), type_code(dq.scalar_type()), (uint64_t)dq.size(0),
              (uint64_t)dq.size(2), sq.held, sk ? sk->held : nullptr, sq.tensor, sk ? sk->tensor : nullptr,
              g.q, g.k, g.type, (float)eps, pos.p, pos.type, pos.seq, const_cast<void*>(dg.q),
              const_cast<void*>(dg.k), dg.type, accumulate, ws.data_ptr(), need, on.stream));
    return py::make_tuple(p.oq, p.k_out(), gq, p.two ? py::cast(gk) : py::none());
}

}  // namespace

PYBIND11_MODULE(_ark_torch, m) {
    using py::arg;
    const auto none = py::none();
    py::class_<Act8>(m, "Act8", R"(An 8-bit checkpoint of a [rows, cols] activation.

data:  uint8 [rows, cols rounded up to 128], one byte per element;
scale: uint8 [rows, data.shape[1] / 32], the power-of-two scale of 32 columns as
       its exponent + 127 (255: the block held an infinity or a NaN and reads
       back as NaN).
kind:  "e4m3" (4 significant bits at every size) or "int8" (a fixed step of 1/127
       to 1/64 of the block's largest).
wide:  whether it may hold values that FP16 cannot: true of one packed from BF16 or
       FP32 here; of bytes that a caller holds, the caller says so.)")
        .def(py::init<const py::object&, const py::object&, int64_t, const std::string&, bool>(), arg("data"),
             arg("scale"), arg("cols"), arg("kind") = "e4m3", arg("wide") = false)
        .def_static(
            "empty",
            [](int64_t rows, int64_t cols, const std::string& kind, const std::optional<at::Device>& device) {
                const int code = kind_code(kind);
                at::Device d = device ? *device : at::Device(at::kCUDA);
                if (d.is_cuda() && !d.has_index()) d = at::Device(at::kCUDA, c10::cuda::current_device());
                return Act8(rows, cols, code, d, at::kHalf);
            },
            arg("rows"), arg("cols"), arg("kind") = "e4m3", arg("device") = none,
            "Room for a checkpoint (its contents are whatever was there), in one allocation; data and\n"
            "scale are views of it.")
        .def_property_readonly("data", &Act8::data)
        .def_property_readonly("scale", &Act8::scale)
        .def_property_readonly("device", &Act8::device)
        .def_property_readonly("rows", &Act8::rows)
        .def_property_readonly("cols", &Act8::cols)
        .def_property_readonly("pitch", &Act8::pitch)
        .def_property_readonly("kind", &Act8::kind_name)
        .def_property_readonly("wide", &Act8::wide)
        .def_property_readonly("nbytes", &Act8::nbytes);

    py::class_<RopePlan>(m, "RopePlan", R"(The rotation of the first rotary_dim elements of each head.

layout:  "half" (pairs i, i + rotary_dim/2) or "interleaved" (2i, 2i + 1).
base:    pair i turns base^(-2i/rotary_dim) radians per position.
scaling: for contexts longer than the trained one: None; "linear" (every
         frequency / factor); "base" (base * factor^(d/(d-2))); "parts"
         (frequencies above `fast` turns over the `original` length kept, below
         `slow` divided by factor, a ramp over the pairs between, and cos and sin
         times 0.1 ln(factor) + 1); "wave" (the same ends, a ramp over the number
         of turns).
Host memory only: made once, usable on every device and in graphs.)")
        .def(py::init<int64_t, double, const std::string&, const std::optional<std::string>&, double, double,
                      double, double>(),
             arg("rotary_dim"), arg("base") = 10000.0, arg("layout") = "half", arg("scaling") = none,
             arg("factor") = 1.0, arg("original") = 0.0, arg("fast") = 32.0, arg("slow") = 1.0)
        .def_property_readonly("rotary_dim", [](const RopePlan& p) { return p.c.rotary_dim; })
        .def_property_readonly("layout",
                               [](const RopePlan& p) { return p.c.interleaved ? "interleaved" : "half"; })
        .def_property_readonly("gain", [](const RopePlan& p) { return p.c.gain; })
        .def("frequencies", &RopePlan::frequencies, "Radians per position of each pair.");

    m.doc() = "The activation operators.  None of them makes an autograd node: what they return\n"
              "requires no gradient, whatever their inputs do.";
    m.def("act8_pack", &act8_pack, arg("x"), arg("kind") = none, arg("out") = none,
          "Checkpoint x [rows, cols] (FP16, BF16 or FP32) in 8 bits.  kind: that of out, or \"e4m3\".\n"
          "No autograd node is made.");
    m.def("act8_unpack", &act8_unpack, arg("checkpoint"), arg("dtype") = at::kHalf, arg("out") = none,
          "The activation that a checkpoint stands for; a finite value that the type cannot\n"
          "hold saturates at its largest.");
    m.def("weight_grad", &weight_grad, arg("x"), arg("dy"), arg("out") = none, arg("accumulate") = false,
          arg("dtype") = none, R"(dW [in, out_features] = X^T dY of y = x W, X [tokens, in] read from its
checkpoint, dY [tokens, out_features] FP16 or BF16.  The products are of dY's type;
FP16 dY with a checkpoint that is `wide` takes two products of BF16 (dY as the sum of
two) and so keeps the checkpoint's range.  With FP16 dY and one that is not, a value
above FP16's range becomes an infinity in dW.

out: where to write (FP16, BF16 or FP32; for example a range of the gradient
     buffer viewed as [in, out_features]); default: a new tensor of `dtype`
     (default: dY's).
accumulate: add to what is in `out`.)");
    m.def("swiglu", &swiglu, arg("a"), arg("b"), arg("checkpoint") = none, arg("out") = none,
          R"(y = silu(a) * b for a, b [rows, cols].  With checkpoint ("e4m3" or "int8")
returns (y, Act8 of a, Act8 of b), made in the same pass.  out may be a or b.

No autograd node is made: the backward is swiglu_backward, by the caller.)");
    m.def("swiglu_backward", &swiglu_backward, arg("dy"), arg("ca"), arg("cb"), arg("checkpoint") = none,
          arg("out") = none, R"((da, db) of swiglu from the checkpoints of a and b.  With checkpoint, returns
(da, db, Act8 of the remade product) for the weight gradient of the projection
that reads it; its kind is that of ca.  out: (da, db), one of which may be dy.)");
    m.def("rope", &rope, arg("q"), arg("k"), arg("plan"), arg("positions") = none, arg("seq_len") = none,
          arg("inverse") = false, arg("out") = none, R"(Rotate q [tokens, heads, dim] and k [tokens, kv heads, dim] (or None).

positions: int32 / int64 [tokens], any non-negative value; a negative one marks a
           padding token, whose outputs are zero.  None: token index modulo
           seq_len (default: one sequence).
inverse:   the opposite rotation, which is the backward.
out:       (q, k) to write to, for example q and k themselves.
Any strides with contiguous heads' elements.  Returns (q, k).

No autograd node is made: the backward is the inverse rotation, by the caller.)");
    m.def("qk_norm_rope", &qk_norm_rope, arg("q"), arg("k"), arg("gain_q"), arg("gain_k"), arg("plan"),
          arg("positions") = none, arg("seq_len") = none, arg("eps") = 1e-6, arg("checkpoint") = none,
          arg("out") = none, R"(RMS norm of each head of q and k (k may be None) with its gain [dim], then the
rotation, in one pass.  With checkpoint ("e4m3" or "int8") q and k as they come
in are checkpointed too: returns (q, k, Act8 of q, Act8 of k), each of
[tokens, heads * dim], else (q, k).

No autograd node is made: the backward is qk_norm_rope_backward, by the caller.)");
    m.def("qk_norm_rope_backward", &qk_norm_rope_backward, arg("dq"), arg("dk"), arg("q"), arg("k"),
          arg("gain_q"), arg("gain_k"), arg("plan"), arg("positions") = none, arg("seq_len") = none,
          arg("eps") = 1e-6, arg("out") = none, arg("out_gains") = none, arg("accumulate") = false,
          R"(Backward of qk_norm_rope: (dq, dk, dgain_q, dgain_k).

dq, dk:  gradients of the outputs (dk may be None).
q, k:    the inputs' checkpoints (Act8), or the inputs themselves.
out:     (dq, dk) to write to, for example dq and dk themselves.
out_gains: (dgain_q, dgain_k) [dim] to write to, for example ranges of the
         gradient buffer; default: new tensors of the gains' type.
accumulate: add the gains' gradients to what is in out_gains.)");
}
