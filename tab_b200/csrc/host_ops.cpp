// tab_b200._host: the bodies of tab_b200.ops' operators - checks, output and scratch allocation, one C-ABI call - in native code.
//
// A small convolution takes the device less time than the interpreter needs to check sixteen arguments, allocate two tensors
// and convert twenty values for a foreign call (about 20 us); here that is 2-3 us.  Every function returns None for arguments
// that are anything but plainly valid (wrong device, dtype, size; an empty result; an error code of the C ABI): the caller
// then runs its own body, which names what is wrong or does the rare case, so that there is one set of messages.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include "../../include/tab_b200.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

bool plain(const Tensor& t, at::ScalarType dtype) { return t.defined() && t.is_cuda() && t.is_contiguous() && t.scalar_type() == dtype; }
tab_stream_t stream_of(const Tensor& t) { return reinterpret_cast<tab_stream_t>(at::cuda::getCurrentCUDAStream(t.get_device()).stream()); }
Tensor make(const Tensor& like, at::IntArrayRef size, at::ScalarType dtype) { return at::empty(size, like.options().dtype(dtype)); }

// n elements are the product of the sizes.  Sizes come from the caller one by one: their product may leave 64 bits, and a wrapped
// one must not pass for the size of a small tensor.
bool holds(int64_t n, std::initializer_list<int64_t> sizes) {
    int64_t product = 1;
    for (const int64_t s : sizes)
        if (__builtin_mul_overflow(product, s, &product)) return false;
    return n == product;
}

struct Conv {
    int type, p1, p2, s1, s2, N, H, W, C, KN, KH, KW;
    int64_t OH = 0, OW = 0, PC = 0;
    // Valid sizes with a result that is not empty.
    bool good() {
        if (type < 0 || type > 3 || N < 1 || H < 1 || W < 1 || C < 1 || KN < 1 || KH < 1 || KW < 1 || p1 < 0 || p2 < 0 || s1 < 1 || s2 < 1) return false;
        OH = ((int64_t)H + 2 * (int64_t)p1 - KH + 1) / s1;
        OW = ((int64_t)W + 2 * (int64_t)p2 - KW + 1) / s2;
        PC = ((int64_t)C + 63) / 64;
        return OH > 0 && OW > 0;
    }
    // n elements are `per_word` for each packed word of the weights, `per_pixel` for each pixel of the activations, the results.
    bool weights(int64_t n, int64_t per_word) const { return holds(n, {KN, KH, KW, PC, per_word}); }
    bool activations(int64_t n, int64_t per_pixel) const { return holds(n, {N, H, W, per_pixel}); }
    bool results(int64_t n) const { return holds(n, {N, KN, OH, OW}); }
};

py::object quantize(const Tensor& X, const Tensor& ths, int bitwidth, int N, int H, int W, int C) {
    Tensor QX, BTN;
    {
        py::gil_scoped_release nogil;
        if (plain(X, at::kFloat) && plain(ths, at::kFloat) && N >= 1 && H >= 1 && W >= 1 && C >= 1 && bitwidth >= 1 &&
            holds(X.numel(), {N, H, W, C}) && ths.numel() == N) {
            const c10::cuda::CUDAGuard guard(X.device());
            QX = make(X, {N, H, W, ((int64_t)C + 63) / 64, bitwidth == 1 ? 1 : 2}, at::kLong);
            BTN = make(X, {N}, at::kInt);
            if (tab_quantize_launch(X.data_ptr<float>(), ths.data_ptr<float>(), QX.data_ptr<int64_t>(), BTN.data_ptr<int32_t>(),
                                    bitwidth, N, H, W, C, stream_of(X)) != TAB_OK) QX.reset();
        }
    }
    if (!QX.defined()) return py::none();
    py::list out(2);
    out[0] = QX; out[1] = BTN;
    return out;
}

py::object conv2d(const Tensor& X, const Tensor& QW, const Tensor& ths, const Tensor& btn, int type, int p1, int p2, int s1, int s2,
                  int N, int H, int W, int C, int KN, int KH, int KW) {
    Tensor Y;
    {
        py::gil_scoped_release nogil;
        Conv g{type, p1, p2, s1, s2, N, H, W, C, KN, KH, KW};
        if (g.good() && plain(X, at::kFloat) && plain(QW, at::kLong) && plain(ths, at::kFloat) && plain(btn, at::kInt) &&
            g.weights(QW.numel(), type == 1 || type == 3 ? 1 : 2) && (type != 2 || btn.numel() == KN) &&
            g.activations(X.numel(), C) && ths.numel() == N) {
            const c10::cuda::CUDAGuard guard(X.device());
            Y = make(X, {N, KN, g.OH, g.OW}, at::kFloat);
            const size_t bytes = tab_conv2d_workspace_bytes(type, p1, p2, s1, s2, N, H, W, C, KN, KH, KW);
            Tensor ws = make(X, {(int64_t)std::max<size_t>(bytes, 256)}, at::kByte);
            if (tab_conv2d_launch(X.data_ptr<float>(), QW.data_ptr<int64_t>(), ths.data_ptr<float>(), btn.data_ptr<int32_t>(), Y.data_ptr<float>(),
                                  ws.data_ptr(), (size_t)ws.numel(), type, p1, p2, s1, s2, N, H, W, C, KN, KH, KW, stream_of(X)) != TAB_OK) Y.reset();
        }
    }
    return Y.defined() ? py::cast(Y) : py::none();
}

// state: zeroed, of tab_conv2d_state_bytes(N) bytes.
py::object quantize_auto(const Tensor& X, double scale, int bitwidth, int N, int H, int W, int C, const Tensor& state) {
    Tensor QX, ths;
    {
        py::gil_scoped_release nogil;
        if (plain(X, at::kFloat) && N >= 1 && H >= 1 && W >= 1 && C >= 1 && bitwidth >= 1 && holds(X.numel(), {N, H, W, C}) &&
            state.defined() && state.is_cuda()) {
            const c10::cuda::CUDAGuard guard(X.device());
            QX = make(X, {N, H, W, ((int64_t)C + 63) / 64, bitwidth == 1 ? 1 : 2}, at::kLong);
            ths = make(X, {N}, at::kFloat);
            if (tab_quantize_auto_launch(X.data_ptr<float>(), (float)scale, state.data_ptr(), ths.data_ptr<float>(), QX.data_ptr<int64_t>(), bitwidth,
                                         N, H, W, C, stream_of(X)) != TAB_OK) QX.reset();
        }
    }
    if (!QX.defined()) return py::none();
    return py::make_tuple(QX, ths);
}

// Byte weights of several layers -> their 4-bit operands, parts of one allocation.
py::object pack_weights(const std::vector<Tensor>& W8) {
    std::vector<Tensor> W4;
    {
        py::gil_scoped_release nogil;
        std::vector<int64_t> sizes;
        int64_t total = 0;
        for (const Tensor& w : W8) {
            if (!plain(w, at::kChar) || w.numel() == 0 || w.numel() % 64 != 0 || w.device() != W8[0].device()) break;
            sizes.push_back(w.numel() / 2);
            total += w.numel() / 2;
        }
        if (!W8.empty() && sizes.size() == W8.size()) {
            const c10::cuda::CUDAGuard guard(W8[0].device());
            W4 = make(W8[0], {total}, at::kByte).split_with_sizes(sizes);
            std::vector<const int8_t*> from;
            std::vector<uint8_t*> to;
            std::vector<long long> words;
            for (size_t i = 0; i < W8.size(); i++) {
                from.push_back(W8[i].data_ptr<int8_t>());
                to.push_back(W4[i].data_ptr<uint8_t>());
                words.push_back(sizes[i] / 32);
            }
            if (tab_pack_weights_many_launch((int)W8.size(), from.data(), to.data(), words.data(), stream_of(W8[0])) != TAB_OK) W4.clear();
        }
    }
    if (W4.empty()) return py::none();
    return py::cast(W4);
}

// The GEMM stage on 4-bit weights (ops.conv2d_bits with uint8 weights), or on byte weights that the call packs first.
py::object conv2d_packed4(const Tensor& QX, const Tensor& weights, int type, int p1, int p2, int s1, int s2, int N, int H, int W, int C, int KN, int KH, int KW,
                          const OptTensor& residual, c10::optional<double> threshold_scale, const OptTensor& state, bool out_int16,
                          c10::optional<int> next_bitwidth) {
    Tensor Y, nxt, QN;
    int rc = TAB_OK;
    {
        py::gil_scoped_release nogil;
        Conv g{type, p1, p2, s1, s2, N, H, W, C, KN, KH, KW};
        const bool want = threshold_scale.has_value();
        if (g.good() && plain(QX, at::kLong) && (plain(weights, at::kByte) || (plain(weights, at::kChar) && weights.device() == QX.device())) && g.activations(QX.numel(), g.PC * (type == 2 || type == 3 ? 1 : 2)) &&
            g.weights(weights.numel(), weights.scalar_type() == at::kByte ? 32 : 64) && (!residual.has_value() || ((plain(*residual, at::kShort) || (!out_int16 && plain(*residual, at::kFloat))) && g.results(residual->numel()))) &&
            (!want || (state.has_value() && state->defined() && state->is_cuda())) && (!next_bitwidth.has_value() || want)) {
            const c10::cuda::CUDAGuard guard(QX.device());
            const int nb = next_bitwidth.has_value() ? (*next_bitwidth == 1 ? 1 : 2) : 0;
            Y = make(QX, {N, KN, g.OH, g.OW}, out_int16 ? at::kShort : at::kFloat);
            if (want) nxt = make(QX, {N}, at::kFloat);
            if (nb) QN = make(QX, {N, g.OH, g.OW, ((int64_t)KN + 63) / 64, nb}, at::kLong);
            Tensor W4 = weights;
            if (weights.scalar_type() == at::kChar) {
                W4 = make(weights, {weights.numel() / 2}, at::kByte);
                rc = tab_pack_weights_launch(weights.data_ptr<int8_t>(), W4.data_ptr<uint8_t>(), KN, KH, KW, C, stream_of(QX));
            }
            if (rc == TAB_OK) rc = tab_conv2d_packed4_launch(QX.data_ptr<int64_t>(), W4.data_ptr<uint8_t>(), Y.data_ptr(), out_int16 ? 1 : 0, type, p1, p2, s1, s2,
                                          N, H, W, C, KN, KH, KW, residual.has_value() ? residual->data_ptr() : nullptr, residual.has_value() && residual->scalar_type() == at::kShort ? 1 : 0,
                                          want ? state->data_ptr() : nullptr, want ? nxt.data_ptr<float>() : nullptr,
                                          want ? (float)*threshold_scale : 0.f, nb ? QN.data_ptr<int64_t>() : nullptr, nb, stream_of(QX));
            if (rc != TAB_OK) Y.reset();
        }
    }
    if (rc == TAB_E_TOO_LARGE) return py::int_(rc);                         // the caller need not find that out again
    if (!Y.defined()) return py::none();
    py::object th = nxt.defined() ? py::cast(nxt) : py::none();
    if (QN.defined()) return py::make_tuple(Y, th, QN);
    return py::make_tuple(Y, th);
}

// Both launches of a layer kept as byte weights: quantiser (against the thresholds given, or against those it finds) with the
// weights packed on the side, then the GEMM stage.
py::object layer(const Tensor& X, const Tensor& W8, int type, int p1, int p2, int s1, int s2, int N, int H, int W, int C, int KN, int KH, int KW,
                 const OptTensor& thresholds, double scale, const OptTensor& state) {
    Tensor Y;
    {
        py::gil_scoped_release nogil;
        Conv g{type, p1, p2, s1, s2, N, H, W, C, KN, KH, KW};
        if (g.good() && plain(X, at::kFloat) && plain(W8, at::kChar) && W8.device() == X.device() && g.activations(X.numel(), C) && g.weights(W8.numel(), 64) &&
            (thresholds.has_value() ? plain(*thresholds, at::kFloat) && thresholds->numel() == N : state.has_value() && state->defined() && state->is_cuda())) {
            const c10::cuda::CUDAGuard guard(X.device());
            if (tab_conv2d_packed4_covers(type, p1, p2, s1, s2, N, H, W, C, KN, KH, KW)) {
                const int bits = type == 2 || type == 3 ? 1 : 2;
                const bool find = !thresholds.has_value();
                Tensor QX = make(X, {N, H, W, g.PC, bits}, at::kLong), W4 = make(X, {W8.numel() / 2}, at::kByte), found;
                if (find) found = make(X, {N}, at::kFloat);
                Y = make(X, {N, KN, g.OH, g.OW}, at::kFloat);
                int rc = tab_quantize_pack_launch(X.data_ptr<float>(), find ? nullptr : thresholds->data_ptr<float>(), (float)scale, find ? state->data_ptr() : nullptr,
                                                  find ? found.data_ptr<float>() : nullptr, QX.data_ptr<int64_t>(), bits, N, H, W, C, W8.data_ptr<int8_t>(),
                                                  W4.data_ptr<uint8_t>(), W8.numel() / 64, stream_of(X));
                if (rc == TAB_OK) rc = tab_conv2d_packed4_launch(QX.data_ptr<int64_t>(), W4.data_ptr<uint8_t>(), Y.data_ptr(), 0, type, p1, p2, s1, s2, N, H, W, C,
                                                                 KN, KH, KW, nullptr, 0, nullptr, nullptr, 0.f, nullptr, 0, stream_of(X));
                if (rc != TAB_OK) Y.reset();
            }
        }
    }
    return Y.defined() ? py::cast(Y) : py::none();
}

// ---- 8-bit blocks and the residual stream ---------------------------------------------------------------------------------------
int type_of(const Tensor& t) {
    const auto s = t.scalar_type();
    return s == at::kFloat ? TAB_FP32 : s == at::kBFloat16 ? TAB_BF16 : s == at::kHalf ? TAB_FP16 : -1;
}
int type_of(at::ScalarType s) { return s == at::kFloat ? TAB_FP32 : s == at::kBFloat16 ? TAB_BF16 : s == at::kHalf ? TAB_FP16 : -1; }
int format_of(at::ScalarType s) { return s == at::kFloat8_e4m3fn ? TAB_E4M3 : s == at::kFloat8_e5m2 ? TAB_E5M2 : -1; }
bool on_cuda(const Tensor& t) { return t.defined() && t.is_cuda() && !t.is_neg(); }      // (a negated view's memory is not its values)
int64_t blocks(int64_t n) { return (n + 127) / 128; }

// The dimensions before the last one as one axis: its length and the distance of its places, which stays as it is where there is at most one.  A
// distance of 0 (a broadcast dimension) is one like any other, hence the word of its own for having met a dimension.
bool leading_axis(const Tensor& t, int64_t& length, int64_t& distance) {
    bool met = false;
    int64_t step = 0;                                                      // what the next (outer) dimension must be apart
    const auto sizes = t.sizes(), strides = t.strides();
    length = 1;
    for (int64_t i = t.dim() - 2; i >= 0; i--) {
        const int64_t size = sizes[i], stride = strides[i];
        if (size == 1) continue;
        if (!met) distance = stride;
        else if (stride != step) return false;
        met = true;
        step = stride * size;
        length *= size;
    }
    return true;
}

// Leading dimensions that are one axis of evenly spaced rows without gaps in them, none of them empty.
struct Rows {
    int64_t M = 1, K = 0, pitch = 0;
    bool of(const Tensor& t) {
        const int64_t d = t.dim();
        if (d == 0 || t.numel() == 0) return false;
        K = t.sizes()[d - 1];
        if (K > 1 && t.strides()[d - 1] != 1) return false;
        pitch = K;
        return leading_axis(t, M, pitch) && pitch >= K && M < (1LL << 31) && K < (1LL << 31) - 256;
    }
};

// Rows::of for the tests, which need no device: (rows, row length, pitch), or None for what it does not take.
py::object row_layout(const Tensor& t) {
    Rows r;
    return r.of(t) ? py::object(py::make_tuple(r.M, r.K, r.pitch)) : py::none();
}

// An uninitialised tensor, past the dispatcher (two or three of them are most of what a small call costs the host).
Tensor fresh(const Tensor& like, at::IntArrayRef size, at::IntArrayRef strides, at::ScalarType dtype) {
    return Tensor(at::detail::empty_strided_cuda(size, strides, like.options().dtype(dtype)));
}
Tensor fresh(const Tensor& like, at::IntArrayRef size, at::ScalarType dtype) { return Tensor(at::detail::empty_cuda(size, like.options().dtype(dtype))); }
using Strides = c10::SmallVector<int64_t, 6>;

// 8-bit values of `shape` (rows x n), every row starting on 16 bytes.
Tensor new_blocks(const Tensor& like, at::IntArrayRef shape, int64_t n, at::ScalarType dtype) {
    const int64_t pitch = (n + 15) / 16 * 16;
    if (pitch == n) return fresh(like, shape, dtype);
    Strides strides(shape.size(), 1);
    int64_t step = pitch;
    for (int64_t i = (int64_t)shape.size() - 2; i >= 0; i--) {
        strides[i] = step;
        step *= shape[i];
    }
    return fresh(like, shape, strides, dtype);
}
Strides with_last(const Tensor& t, int64_t n) {
    Strides s(t.sizes().begin(), t.sizes().end());
    s.back() = n;
    return s;
}

// Scales `shape` that lie block by block.
Tensor new_scales(const Tensor& like, at::IntArrayRef shape, int64_t rows) {
    Strides strides(shape.size());
    int64_t step = 1;
    for (int64_t i = (int64_t)shape.size() - 2; i >= 0; i--) {
        strides[i] = step;
        step *= shape[i];
    }
    strides.back() = (rows + 15) / 16 * 16;
    return fresh(like, shape, strides, at::kFloat8_e8m0fnu);
}

struct Quantized { Tensor q, s, qt, st; };
bool quantize_any(const Tensor& x, at::ScalarType dtype, bool both, bool square, Quantized& o) {
    Rows r;
    const int format = format_of(dtype);
    if (!on_cuda(x) || type_of(x) < 0 || format < 0 || (square && x.dim() != 2) || !r.of(x)) return false;
    const c10::cuda::CUDAGuard guard(x.device());
    o.q = new_blocks(x, x.sizes(), r.K, dtype);
    o.s = square ? fresh(x, {blocks(r.M), blocks(r.K)}, at::kFloat8_e8m0fnu) : new_scales(x, with_last(x, blocks(r.K)), r.M);
    if (both) {
        o.qt = new_blocks(x, {r.K, r.M}, r.M, dtype);
        o.st = square ? fresh(x, {blocks(r.K), blocks(r.M)}, at::kFloat8_e8m0fnu) : new_scales(x, {r.K, blocks(r.M)}, r.K);
    }
    const int64_t pk = (r.K + 15) / 16 * 16, pm = (r.M + 15) / 16 * 16;
    return tab_quantize_blocks_launch(x.data_ptr(), type_of(x), r.pitch, r.M, (int)r.K, format, square, o.q.data_ptr(), pk, static_cast<uint8_t*>(o.s.data_ptr()),
                                      square ? blocks(r.K) : pm, both ? o.qt.data_ptr() : nullptr, pm, both ? static_cast<uint8_t*>(o.st.data_ptr()) : nullptr,
                                      square ? blocks(r.M) : pk, stream_of(x)) == TAB_OK;
}
py::object quantized(const Tensor& x, at::ScalarType dtype, bool both, bool square) {
    Quantized o;
    bool ok;
    {
        py::gil_scoped_release nogil;
        ok = quantize_any(x, dtype, both, square, o);
    }
    if (!ok) return py::none();
    return both ? py::make_tuple(o.q, o.s, o.qt, o.st) : py::make_tuple(o.q, o.s);
}
py::object quantize_blocks(const Tensor& x, at::ScalarType dtype, bool columns) { return quantized(x, dtype, columns, false); }
py::object quantize_blocks2d(const Tensor& w, at::ScalarType dtype, bool transposed) { return quantized(w, dtype, transposed, true); }

struct Operand {
    Rows r;
    int share = 1;
    int64_t sr = 0, sk = 0;
    bool of(const Tensor& q, const Tensor& s) {
        return on_cuda(q) && on_cuda(s) && s.device() == q.device() && format_of(q.scalar_type()) >= 0 && s.scalar_type() == at::kFloat8_e8m0fnu && r.of(q) && scales(s);
    }
    // The scales of r's values.
    bool scales(const Tensor& s) {
        if (s.dim() == 0 || s.size(-1) != blocks(r.K)) return false;
        sk = s.stride(-1);
        int64_t rows = 1;
        if (!leading_axis(s, rows, sr)) return false;
        if (rows != r.M && rows != blocks(r.M)) return false;
        share = rows == r.M ? 1 : 128;
        return true;
    }
};
// Operand::scales for the tests, which need no device: (rows to a scale, distance of rows, of blocks), or None for what it does not take.
py::object scale_layout(const Tensor& q, const Tensor& s) {
    Operand o;
    return o.r.of(q) && o.scales(s) ? py::object(py::make_tuple(o.share, o.sr, o.sk)) : py::none();
}
bool matmul_any(const Tensor& a, const Tensor& as, const Tensor& b, const Tensor& bs, at::ScalarType dtype, Tensor& y) {
    Operand A, B;
    const int type = type_of(dtype);
    if (type < 0 || !A.of(a, as) || !B.of(b, bs) || b.dim() != 2 || A.r.K != B.r.K || a.device() != b.device()) return false;
    const c10::cuda::CUDAGuard guard(a.device());
    y = fresh(a, with_last(a, B.r.M), dtype);
    return tab_matmul_blocks_launch(a.data_ptr(), format_of(a.scalar_type()), A.r.pitch, static_cast<const uint8_t*>(as.data_ptr()), A.share, A.sr, A.sk,
                                    b.data_ptr(), format_of(b.scalar_type()), B.r.pitch, static_cast<const uint8_t*>(bs.data_ptr()), B.share, B.sr, B.sk,
                                    y.data_ptr(), type, B.r.M, (int)A.r.M, (int)B.r.M, (int)A.r.K, stream_of(a)) == TAB_OK;
}
py::object matmul_blocks(const Tensor& a, const Tensor& as, const Tensor& b, const Tensor& bs, at::ScalarType dtype) {
    Tensor y;
    bool ok;
    {
        py::gil_scoped_release nogil;
        ok = matmul_any(a, as, b, bs, dtype, y);
    }
    return ok ? py::cast(y) : py::none();
}

// Gradients of gradients are refused when somebody asks for them, not before.
void differentiable_once(torch::autograd::variable_list& grads) {
    if (!at::GradMode::is_enabled()) return;
    auto error = std::make_shared<torch::autograd::DelayedError>("tab_b200: this operator is differentiable once", 1);
    for (auto& g : grads)
        if (g.defined()) g = (*error)({g.detach().requires_grad_()})[0];
}
Tensor even_rows(const Tensor& g) {
    Rows r;
    if (g.defined() && g.is_neg()) return g.resolve_neg().contiguous();
    return !g.defined() || g.numel() == 0 || r.of(g) ? g : g.contiguous();
}

// Kept values as matmul_any takes them: hooks on saved tensors (which keep them on the host, say) may hand them back without the bytes between rows.
Tensor aligned_rows(const Tensor& q) {
    Rows r;
    if (!q.defined() || !r.of(q) || ((r.M == 1 || r.pitch % 16 == 0) && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0)) return q;
    Tensor o = new_blocks(q, q.sizes(), r.K, q.scalar_type());
    o.view(at::kByte).copy_(q.view(at::kByte));
    return o;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// nn.block_linear; x and weight have passed quantize_any's conditions, so that only an error of the CUDA runtime is left to report.
struct BlockLinear : torch::autograd::Function<BlockLinear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, int64_t out_type, int64_t grad_type, bool need_x, bool need_w) {
        Quantized xq, wq;
        Tensor y;
        TORCH_CHECK(quantize_any(x, at::kFloat8_e4m3fn, need_w, false, xq) && quantize_any(weight, at::kFloat8_e4m3fn, need_x, true, wq) &&
                        matmul_any(xq.q, xq.s, wq.q, wq.s, (at::ScalarType)out_type, y),
                    "block_linear: a launch failed [cudaError ", tab_last_cuda_error(), ", status ", tab_device_status(), "]");
        ctx->save_for_backward({xq.qt, xq.st, wq.qt, wq.st});
        ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)x.scalar_type(), (int64_t)weight.scalar_type(), grad_type};
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const auto types = ctx->saved_data["types"].toIntVector();
        variable_list out(6);
        // what this pass is asked for, of what was kept for any
        const bool need_w = saved[0].defined() && ctx->needs_input_grad(1), need_x = saved[2].defined() && ctx->needs_input_grad(0);
        if (!grads[0].defined() || (!need_x && !need_w)) return out;
        const Tensor g = even_rows(grads[0].detach());
        Quantized q;
        bool ok = quantize_any(g, (at::ScalarType)types[2], need_w, false, q);
        if (ok && need_x) ok = matmul_any(q.q, q.s, aligned_rows(saved[2]), saved[3], (at::ScalarType)types[0], out[0]);
        if (ok && need_w) ok = matmul_any(q.qt, q.st, aligned_rows(saved[0]), saved[1], (at::ScalarType)types[1], out[1]);
        TORCH_CHECK(ok, "block_linear: a launch of the backward pass failed [cudaError ", tab_last_cuda_error(), "]");
        differentiable_once(out);
        return out;
    }
};
py::object block_linear(const Tensor& x, const Tensor& weight, at::ScalarType out_type, at::ScalarType grad_type) {
    Tensor y;
    {
        py::gil_scoped_release nogil;
        Rows r, w;
        if (on_cuda(x) && on_cuda(weight) && x.device() == weight.device() && type_of(x) >= 0 && type_of(weight) >= 0 && type_of(out_type) >= 0 && format_of(grad_type) >= 0 &&
            weight.dim() == 2 && r.of(x) && w.of(weight) && r.K == w.K) {
            const bool grad = at::GradMode::is_enabled();
            y = BlockLinear::apply(x, weight, (int64_t)out_type, (int64_t)grad_type, grad && x.requires_grad(), grad && weight.requires_grad());
        }
    }
    return y.defined() ? py::cast(y) : py::none();
}

// The inputs of residual_norm as the C ABI takes them; false for anything the interpreter's body has to look at.
struct Norm {
    tab_norm_t a = {};
    Rows r;
    bool of(const Tensor& y, const Tensor& x, const Tensor& w2, const Tensor& b2, const Tensor& w1, const Tensor& b1, const Tensor& gate, double alpha, int64_t layer, double eps) {
        if (!on_cuda(y) || type_of(y) < 0 || layer < 0 || layer > 1 || !r.of(y)) return false;
        a.y = y.data_ptr(); a.ldy = r.pitch; a.type = type_of(y); a.layer = (int)layer; a.alpha = (float)alpha; a.eps = (float)eps; a.M = r.M; a.C = (int)r.K;
        Rows q;
        if (x.defined()) {
            if (!on_cuda(x) || x.device() != y.device() || x.scalar_type() != y.scalar_type() || x.sizes() != y.sizes() || !q.of(x)) return false;
            a.x = x.data_ptr(); a.ldx = q.pitch;
        }
        int ptype = -1;
        const struct { const Tensor& t; const void** p; } weights[4] = {{w1, &a.w1}, {b1, &a.b1}, {w2, &a.w2}, {b2, &a.b2}};
        for (const auto& w : weights) {
            if (!w.t.defined()) continue;
            const int type = type_of(w.t);
            if (!on_cuda(w.t) || w.t.device() != y.device() || (type != TAB_FP32 && type != a.type) || w.t.dim() != 1 || w.t.size(0) != r.K || !w.t.is_contiguous() ||
                (ptype >= 0 && ptype != type)) return false;
            *w.p = w.t.data_ptr();
            a.ptype = ptype = type;
        }
        if ((a.b1 && !a.w1) || (a.b2 && !a.w2) || (!layer && (a.b1 || a.b2))) return false;
        if (gate.defined()) {
            a.gtype = type_of(gate);
            if (!on_cuda(gate) || gate.device() != y.device() || (a.gtype != TAB_FP32 && a.gtype != a.type)) return false;
            a.gate = gate.data_ptr();
            if (gate.dim() == 1 && gate.size(0) == r.K && (gate.is_contiguous() || r.K == 1)) {
                a.gkind = TAB_GATE_CHANNEL;
            } else if (gate.dim() == y.dim() && gate.sizes().slice(0, y.dim() - 1) == y.sizes().slice(0, y.dim() - 1) && (gate.size(-1) == 1 || gate.size(-1) == r.K)) {
                Rows g;
                if (!g.of(gate)) return false;
                a.gkind = gate.size(-1) == 1 ? TAB_GATE_TOKEN : TAB_GATE_FULL;
                a.ldg = g.pitch;
            } else {
                return false;
            }
        }
        return true;
    }
    bool plain() const { return !a.x && !a.w1 && !a.gate; }                // r is y
};
// r (undefined where it is y), h or its blocks, statistics where asked for.
bool norm_any(Norm& n, const Tensor& y, c10::optional<at::ScalarType> quantize, bool stats, Tensor& r, Tensor& h, Tensor& s, Tensor& st) {
    const c10::cuda::CUDAGuard guard(y.device());
    if (!n.plain()) { r = fresh(y, y.sizes(), y.scalar_type()); n.a.r = r.data_ptr(); n.a.ldr = n.r.K; }
    if (quantize.has_value()) {
        n.a.format = format_of(*quantize);
        if (n.a.format < 0 || !n.a.w2) return false;
        h = new_blocks(y, y.sizes(), n.r.K, *quantize);
        s = new_scales(y, with_last(y, blocks(n.r.K)), n.r.M);
        n.a.q = h.data_ptr(); n.a.ldq = (n.r.K + 15) / 16 * 16; n.a.lds = (n.r.M + 15) / 16 * 16; n.a.s = static_cast<uint8_t*>(s.data_ptr());
    } else if (n.a.w2) {
        h = fresh(y, y.sizes(), y.scalar_type());
        n.a.h = h.data_ptr(); n.a.ldh = n.r.K;
    }
    if (stats) { st = fresh(y, {n.r.M, 4}, at::kFloat); n.a.stats = st.data_ptr<float>(); }
    return tab_residual_norm_launch(&n.a, stream_of(y)) == TAB_OK;
}
const Tensor& given(const OptTensor& t) {
    static const Tensor none;
    return t.has_value() ? *t : none;
}
py::object residual_norm(const Tensor& y, const OptTensor& x, const OptTensor& w2, const OptTensor& b2, const OptTensor& w1, const OptTensor& b1, const OptTensor& gate, double alpha,
                         const std::string& kind, double eps, c10::optional<at::ScalarType> quantize) {
    Norm n;
    Tensor r, h, s, st;
    bool ok;
    {
        py::gil_scoped_release nogil;
        ok = (kind == "rms" || kind == "layer") && n.of(y, given(x), given(w2), given(b2), given(w1), given(b1), given(gate), alpha, kind == "layer", eps) &&
             norm_any(n, y, quantize, false, r, h, s, st);
    }
    if (!ok) return py::none();
    py::object first = n.plain() ? py::cast(y) : py::cast(r), second = h.defined() ? py::cast(h) : py::none();
    return quantize.has_value() ? py::make_tuple(first, second, s) : py::make_tuple(first, second);
}

// nn.residual_norm.  Returns r, then h, those that there are.
struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& y, const OptTensor& ox, const OptTensor& ow2, const OptTensor& ob2, const OptTensor& ow1, const OptTensor& ob1,
                                 const OptTensor& ogate, double alpha, int64_t layer, double eps) {
        const Tensor &x = given(ox), &w2 = given(ow2), &b2 = given(ob2), &w1 = given(ow1), &b1 = given(ob1), &gate = given(ogate);
        Norm n;
        Tensor r, h, s, st;
        TORCH_CHECK(n.of(y, x, w2, b2, w1, b1, gate, alpha, layer, eps) && norm_any(n, y, c10::nullopt, true, r, h, s, st),
                    "residual_norm: the launch failed [cudaError ", tab_last_cuda_error(), "]");
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({y, n.plain() ? Tensor() : r, st, w2, b2, w1, b1, gate});
        ctx->saved_data["residual"] = x.defined();
        ctx->saved_data["alpha"] = alpha; ctx->saved_data["layer"] = layer; ctx->saved_data["eps"] = eps;
        variable_list out;
        if (r.defined()) out.push_back(r);
        if (h.defined()) out.push_back(h);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto v = ctx->get_saved_variables();
        const Tensor &w2 = v[3], &b2 = v[4], &w1 = v[5], &b1 = v[6];
        const bool plain = !v[1].defined(), residual = ctx->saved_data["residual"].toBool();
        variable_list out(10);
        const Tensor gr = plain ? Tensor() : even_rows(grads[0].defined() ? grads[0].detach() : grads[0]);
        const Tensor gh = w2.defined() ? even_rows(grads.back().defined() ? grads.back().detach() : grads.back()) : Tensor();
        if (!gr.defined() && !gh.defined()) return out;
        // Hooks on kept tensors may hand them back with other strides; in another type, shape or place they are not what the gradients belong to.
        const Tensor y = even_rows(v[0]), r = even_rows(v[1]), st = v[2].contiguous(), gate = v[7].defined() && v[7].dim() > 1 ? even_rows(v[7]) : v[7];
        auto fits = [&](const Tensor& t) { return !t.defined() || (on_cuda(t) && t.device() == y.device() && t.scalar_type() == y.scalar_type() && t.sizes() == y.sizes()); };
        TORCH_CHECK(fits(y) && fits(r) && fits(gr) && fits(gh) && on_cuda(st) && st.device() == y.device() && st.scalar_type() == at::kFloat && y.dim() > 0 &&
                        st.numel() * y.size(-1) == 4 * y.numel() && reinterpret_cast<uintptr_t>(st.data_ptr()) % 16 == 0,
                    "residual_norm: the backward pass needs the kept tensors in the type, shape and place in which the forward pass kept them");
        Norm n;
        bool ok = n.of(y, Tensor(), w2, b2, w1, b1, gate, ctx->saved_data["alpha"].toDouble(), ctx->saved_data["layer"].toInt(), ctx->saved_data["eps"].toDouble());
        if (ok) {
            const c10::cuda::CUDAGuard guard(y.device());
            tab_norm_backward_t b = {};
            Rows q;
            n.a.r = const_cast<void*>(static_cast<const void*>((plain ? y : r).data_ptr()));
            n.a.ldr = n.r.pitch;
            if (!plain) { ok = q.of(r); n.a.ldr = q.pitch; q = Rows(); }
            n.a.stats = st.data_ptr<float>();
            b.f = n.a;
            if (gr.defined()) { ok = ok && q.of(gr); b.gr = gr.data_ptr(); b.ldgr = q.pitch; }
            q = Rows();
            if (gh.defined()) { ok = ok && q.of(gh); b.gh = gh.data_ptr(); b.ldgh = q.pitch; }
            const struct { const Tensor& like; void** p; } grads_of[7] = {{y, &b.dy}, {residual ? y : st, &b.dx}, {w2, &b.dw2}, {b2, &b.db2}, {w1, &b.dw1}, {b1, &b.db1}, {gate, &b.dgate}};
            bool sums = false;
            size_t input = 0;                                              // autograd numbers the tensors that there are
            for (size_t i = 0; i < 7; i++) {
                if (!grads_of[i].like.defined() || (i == 1 && !residual) || !ctx->needs_input_grad(input++)) continue;
                out[i] = fresh(grads_of[i].like, grads_of[i].like.sizes(), grads_of[i].like.scalar_type());
                *grads_of[i].p = out[i].data_ptr();
                sums = sums || i > 1;
            }
            b.lddy = b.lddx = n.r.K;
            Tensor partial;
            if (sums) { partial = fresh(y, {(int64_t)(tab_residual_norm_workspace_bytes(n.r.M, (int)n.r.K) / 4)}, at::kFloat); b.partial = partial.data_ptr<float>(); }
            ok = ok && tab_residual_norm_backward_launch(&b, stream_of(y)) == TAB_OK;
        }
        TORCH_CHECK(ok, "residual_norm: a launch of the backward pass failed [cudaError ", tab_last_cuda_error(), "]");
        differentiable_once(out);
        return out;
    }
};
py::object residual_norm_grad(const Tensor& y, const OptTensor& x, const OptTensor& w2, const OptTensor& b2, const OptTensor& w1, const OptTensor& b1, const OptTensor& gate, double alpha,
                              const std::string& kind, double eps) {
    Norm n;
    variable_list out;
    bool ok;
    {
        py::gil_scoped_release nogil;
        ok = (kind == "rms" || kind == "layer") && n.of(y, given(x), given(w2), given(b2), given(w1), given(b1), given(gate), alpha, kind == "layer", eps) && (n.a.w2 || !n.plain()) &&
             n.r.K <= 16384;
        if (ok) out = ResidualNorm::apply(y, x, w2, b2, w1, b1, gate, alpha, (int64_t)(kind == "layer"), eps);
    }
    if (!ok) return py::none();
    py::object r = n.plain() ? py::cast(y) : py::cast(out[0]), h = n.a.w2 ? py::cast(out.back()) : py::none();
    return py::make_tuple(r, h);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("quantize", &quantize);
    m.def("conv2d", &conv2d);
    m.def("quantize_auto", &quantize_auto);
    m.def("layer", &layer);
    m.def("pack_weights", &pack_weights);
    m.def("conv2d_packed4", &conv2d_packed4);
    m.def("row_layout", &row_layout);
    m.def("scale_layout", &scale_layout);
    m.def("quantize_blocks", &quantize_blocks);
    m.def("quantize_blocks2d", &quantize_blocks2d);
    m.def("matmul_blocks", &matmul_blocks);
    m.def("residual_norm", &residual_norm);
    m.def("block_linear", &block_linear);
    m.def("residual_norm_grad", &residual_norm_grad);
}
