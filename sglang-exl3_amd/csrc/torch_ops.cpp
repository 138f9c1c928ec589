// Native entry of the operators that programs call eagerly, one per layer:
// exl3_gemv, exl3_linear_cat, exl3_linear_part, exl3_gate_up_swiglu and the
// block-scaled FP8 operators.
//
// A one-token call is bound by its host path: from Python (operator wrapper,
// checks, two ctypes calls, stream and device queries) exl3_gemv took 20.5 us
// on the host for a kernel of 12 (4096 x 14336) or 4 us (512 x 512), three shards
// through exl3_linear_cat 29.2.  Here the usual call - dense tensors of the
// current device, a workspace that is large enough, no graph capture - goes
// from the dispatcher to the C ABI: 5.4 and 6.6 us.  Every other call
// (autograd inputs, strided or misaligned tensors, the first call of a shape,
// capture, and whatever is refused) goes to the operator's *_general twin, the
// Python implementation, so its checks, messages and bookkeeping stay the only ones.
//
// The operators are defined in Python; this file adds the kernels of two
// dispatch keys.  The library that holds the C ABI is bound by address, so that it
// is loaded once.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/InferenceMode.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/library.h>

#include <map>
#include <mutex>
#include <utility>

#include "../../include/sglang_exl3_amd.h"

namespace {

struct Abi {
    decltype(&exl3_gemv) gemv;
    decltype(&exl3_gemv_workspace_size) gemv_ws;
    decltype(&exl3_linear_cat_part) cat;
    decltype(&exl3_linear_cat_workspace_size) cat_ws;
    decltype(&exl3_gate_up_swiglu) gate_up;
    decltype(&exl3_gate_up_workspace_size) gate_up_ws;
    decltype(&exl3_fp8_quant_rows) quant;
    decltype(&exl3_fp8_norm_quant) norm;
    decltype(&exl3_fp8_swiglu_quant) swiglu;
    decltype(&exl3_fp8_linear) fp8;
    decltype(&exl3_fp8_linear_workspace_size) fp8_ws;
} abi;

// The buffers of ops.workspace(), by (device, stream); never destroyed (the
// allocator may be gone before this library at exit).
std::mutex& ws_lock() {
    static std::mutex* m = new std::mutex;
    return *m;
}
std::map<std::pair<int64_t, int64_t>, at::Tensor>& ws_map() {
    static auto* m = new std::map<std::pair<int64_t, int64_t>, at::Tensor>;
    return *m;
}

void keep_workspace(const at::Tensor& ws, int64_t stream) {
    std::lock_guard<std::mutex> g(ws_lock());
    ws_map()[{ws.get_device(), stream}] = ws;
}

// Stream and workspace of a call on `dev`; false: the general path.
struct Launch {
    hipStream_t stream;
    at::Tensor ws;
    bool get(int64_t dev, size_t need) {
        const auto s = c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev);
        stream = s.stream();
        hipStreamCaptureStatus cap;
        if (hipStreamIsCapturing(stream, &cap) != hipSuccess || cap != hipStreamCaptureStatusNone) return false;
        std::lock_guard<std::mutex> g(ws_lock());
        const auto it = ws_map().find({dev, (int64_t)reinterpret_cast<intptr_t>(stream)});
        if (it == ws_map().end() || (size_t)it->second.numel() < need) return false;
        ws = it->second;
        return true;
    }
};

bool on_current(const at::Tensor& x) {
    int dev = -1;
    return x.is_cuda() && hipGetDevice(&dev) == hipSuccess && dev == x.get_device();
}
const uint16_t* u16(const at::Tensor& t) { return static_cast<const uint16_t*>(t.const_data_ptr()); }
bool at_bytes(const at::Tensor& t, uintptr_t a) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % a == 0; }

// A half vector of at least `len` elements, packed and dword-aligned.
bool half_vec(const at::Tensor& t, int64_t dev, int64_t len) {
    return t.is_cuda() && t.get_device() == dev && t.scalar_type() == at::kHalf && t.is_contiguous() &&
           t.numel() >= len && at_bytes(t, 4);
}
// Trellis words [k/16, n/16, 16 K], packed and 16-byte aligned.
bool trellis_ok(const at::Tensor& t, int64_t dev, int64_t k, int64_t K) {
    return t.is_cuda() && t.get_device() == dev && t.scalar_type() == at::kShort && t.dim() == 3 &&
           t.is_contiguous() && t.size(0) * 16 == k && t.size(1) > 0 && t.size(1) < (1 << 24) && t.size(2) == 16 * K && at_bytes(t, 16);
}
// Rows of x (m x k); 0: the general path.
int64_t rows_of(const at::Tensor& x, bool bf16_too) {
    if (x.dim() < 2 || !on_current(x) || !x.is_contiguous() || !at_bytes(x, 4)) return 0;
    if (x.scalar_type() != at::kHalf && !(bf16_too && x.scalar_type() == at::kBFloat16)) return 0;
    const int64_t k = x.size(-1);
    const int64_t m = k > 0 ? x.numel() / k : 0;
    return k <= (1 << 24) && m <= (1 << 24) ? m : 0;
}
// A failed call may have left counters behind: clean the buffer, then let the
// general path raise (or run).
bool done(int rc, Launch& l) {
    if (rc == EXL3_OK) return true;
    l.ws.zero_();
    return false;
}

// ------------------------------------------------------------------ exl3_gemv

using GemvFn = at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, c10::SymInt,
                          bool, c10::SymInt);
struct Gemv {
    static constexpr const char *name = "sglang_exl3::exl3_gemv", *general = "sglang_exl3::exl3_gemv_general";
};

at::Tensor gemv(const at::Tensor& x, const at::Tensor& trellis, const at::Tensor& suh, const at::Tensor& svh,
                int64_t K, bool mcg, int64_t mmode) {
    const int64_t m = rows_of(x, false), k = m ? x.size(-1) : 0, dev = m ? x.get_device() : -1;
    if (m >= 1 && m <= 64 && (mmode == 0 || mmode == 1) && K >= 1 && K <= 8 && trellis_ok(trellis, dev, k, K) &&
        half_vec(suh, dev, k) && half_vec(svh, dev, trellis.size(1) * 16)) {
        const int64_t n = trellis.size(1) * 16;
        Launch l;
        if (l.get(dev, abi.gemv_ws((int)m, (int)k, (int)n, (int)K, 1))) {
            at::Tensor y = at::empty({m, n}, x.options());
            if (done(abi.gemv(u16(x), trellis.const_data_ptr<int16_t>(), u16(suh), u16(svh),
                              static_cast<uint16_t*>(y.mutable_data_ptr()), (int)m, (int)k, (int)n, (int)K,
                              mcg ? 1 : 2, l.ws.mutable_data_ptr(), l.ws.numel(), l.stream),
                     l))
                return y;
        }
    }
    static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow(Gemv::general, "").typed<GemvFn>();
    return h.call(x, trellis, suh, svh, K, mcg, mmode);
}

// ------------------------------------------------------------ exl3_linear_cat

using CatFn = at::Tensor(const at::Tensor&, at::TensorList, at::TensorList, at::TensorList, c10::SymInt, c10::SymInt,
                         bool);
struct Cat {
    static constexpr const char *name = "sglang_exl3::exl3_linear_cat",
                                *general = "sglang_exl3::exl3_linear_cat_general";
};
using PartFn = at::Tensor(const at::Tensor&, at::TensorList, at::TensorList, at::TensorList, c10::SymInt, c10::SymInt,
                          bool, c10::SymInt);
struct Part {
    static constexpr const char *name = "sglang_exl3::exl3_linear_part",
                                *general = "sglang_exl3::exl3_linear_part_general";
};

// Weights from `first` on, side by side [m, n] or (apart) packed one after the
// other [m * n]; an undefined tensor: the general path.
at::Tensor linear_weights(const at::Tensor& x, at::TensorList trellis, at::TensorList suh, at::TensorList svh,
                          int64_t K, int64_t codebook, bool out_bf16, int64_t first, bool apart) {
    const int64_t m = rows_of(x, true), k = m ? x.size(-1) : 0, dev = m ? x.get_device() : -1;
    const size_t count = trellis.size();
    bool ok = m >= 1 && count >= 1 && count <= 4 && suh.size() == count && svh.size() == count && K >= 1 && K <= 8 &&
              codebook >= 0 && codebook <= 2 && first >= 0 && first < (int64_t)count;
    const int16_t* tr[4];
    const uint16_t *su[4], *sv[4];
    int ns[4];
    int64_t n = 0;
    for (size_t j = 0; ok && j < count; ++j) {
        ok = trellis_ok(trellis[j], dev, k, K) && half_vec(suh[j], dev, k) &&
             half_vec(svh[j], dev, trellis[j].size(1) * 16);
        if (!ok) break;
        tr[j] = trellis[j].const_data_ptr<int16_t>();
        su[j] = u16(suh[j]);
        sv[j] = u16(svh[j]);
        ns[j] = (int)(trellis[j].size(1) * 16);
        if ((int64_t)j >= first) n += ns[j];
    }
    Launch l;
    if (ok && l.get(dev, abi.cat_ws((int)m, (int)k, ns, (int)count, (int)K))) {
        const auto options = x.options().dtype(out_bf16 ? at::kBFloat16 : at::kHalf);
        at::Tensor y = apart ? at::empty({m * n}, options) : at::empty({m, n}, options);
        if (done(abi.cat(x.const_data_ptr(), x.scalar_type() == at::kBFloat16 ? 1 : 0, tr, su, sv, ns, (int)count,
                         (int)first, apart ? 1 : 0, y.mutable_data_ptr(), out_bf16 ? 1 : 0, (int)m, (int)k, (int)K,
                         (int)codebook, l.ws.mutable_data_ptr(), l.ws.numel(), l.stream),
                 l))
            return y;
    }
    return {};
}

at::Tensor linear_cat(const at::Tensor& x, at::TensorList trellis, at::TensorList suh, at::TensorList svh, int64_t K,
                      int64_t codebook, bool out_bf16) {
    at::Tensor y = linear_weights(x, trellis, suh, svh, K, codebook, out_bf16, 0, false);
    if (y.defined()) return y;
    static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow(Cat::general, "").typed<CatFn>();
    return h.call(x, trellis, suh, svh, K, codebook, out_bf16);
}

at::Tensor linear_part(const at::Tensor& x, at::TensorList trellis, at::TensorList suh, at::TensorList svh, int64_t K,
                       int64_t codebook, bool out_bf16, int64_t first) {
    at::Tensor y = linear_weights(x, trellis, suh, svh, K, codebook, out_bf16, first, true);
    if (y.defined()) return y;
    static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow(Part::general, "").typed<PartFn>();
    return h.call(x, trellis, suh, svh, K, codebook, out_bf16, first);
}

// -------------------------------------------------------- exl3_gate_up_swiglu

using GateUpFn = at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                            const at::Tensor&, const at::Tensor&, c10::SymInt, c10::SymInt, double);
struct GateUp {
    static constexpr const char *name = "sglang_exl3::exl3_gate_up_swiglu",
                                *general = "sglang_exl3::exl3_gate_up_swiglu_general";
};

at::Tensor gate_up(const at::Tensor& x, const at::Tensor& suh, const at::Tensor& gt, const at::Tensor& gsv,
                   const at::Tensor& ut, const at::Tensor& usv, int64_t K, int64_t codebook, double limit) {
    const int64_t m = rows_of(x, false), k = m ? x.size(-1) : 0, dev = m ? x.get_device() : -1;

    if (m >= 1 && K >= 1 && K <= 8 && codebook >= 0 && codebook <= 2 && limit >= 0.0 && trellis_ok(gt, dev, k, K) &&
        trellis_ok(ut, dev, k, K) && gt.size(1) == ut.size(1) && half_vec(suh, dev, k) &&
        half_vec(gsv, dev, gt.size(1) * 16) && half_vec(usv, dev, gt.size(1) * 16)) {
        const int64_t n = gt.size(1) * 16;
        Launch l;
        if (l.get(dev, abi.gate_up_ws((int)m, (int)k, (int)n, (int)K))) {
            at::Tensor y = at::empty({m, n}, x.options());
            if (done(abi.gate_up(u16(x), u16(suh), gt.const_data_ptr<int16_t>(), u16(gsv),
                                 ut.const_data_ptr<int16_t>(), u16(usv), static_cast<uint16_t*>(y.mutable_data_ptr()),
                                 (int)m, (int)k, (int)n, (int)K, (int)codebook, (float)limit, l.ws.mutable_data_ptr(),
                                 l.ws.numel(), l.stream),
                     l))
                return y;
        }
    }
    static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow(GateUp::general, "").typed<GateUpFn>();
    return h.call(x, suh, gt, gsv, ut, usv, K, codebook, limit);
}

// ------------------------------------------------------- block-scaled FP8 rows

using Two = std::tuple<at::Tensor, at::Tensor>;
using OptTensor = std::optional<at::Tensor>;

int fp8_groups(int64_t k) { return (int)((k + 127) / 128); }
hipStream_t stream_of(int64_t dev) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream(); }

// Dense 16-bit rows of the current device as (rows, stride) that the kernels
// take as they are; false: the general path.
struct Fp8Rows {
    int64_t m, k, stride;
    int dtype;
    bool get(const at::Tensor& x) {
        if (x.dim() < 1 || !on_current(x) || !at_bytes(x, 16)) return false;
        if (x.scalar_type() != at::kHalf && x.scalar_type() != at::kBFloat16) return false;
        k = x.size(-1);
        if (k <= 0 || k > (1 << 24) || x.numel() == 0) return false;
        m = x.numel() / k;
        if (m > (1 << 24) || m * fp8_groups(k) > 0x7fffffff) return false;
        if (x.dim() == 2 && m > 1) {
            stride = x.stride(0);
            if (x.stride(1) != 1 || stride < k) return false;
        } else {
            if (!x.is_contiguous()) return false;
            stride = k;
        }
        dtype = x.scalar_type() == at::kBFloat16 ? EXL3_DTYPE_BF16 : EXL3_DTYPE_F16;
        return stride % 8 == 0;
    }
};

// A new tensor on x's device, straight from the allocator (at::empty goes through the dispatcher: 0.15 us more).
at::Tensor fresh(const at::Tensor& x, at::IntArrayRef size, at::ScalarType type) {
    return at::detail::empty_cuda(size, type, x.device(), std::nullopt);
}

// q and its scales for rows like x's of k columns.
Two fp8_out(const at::Tensor& x, int64_t k) {
    at::DimVector q(x.sizes().begin(), x.sizes().end()), s = q;
    q.back() = k;
    s.back() = fp8_groups(k);
    return {fresh(x, q, at::kFloat8_e4m3fn), fresh(x, s, at::kFloat)};
}
uint8_t* bytes_of(at::Tensor& t) { return static_cast<uint8_t*>(t.mutable_data_ptr()); }
float* floats_of(at::Tensor& t) { return static_cast<float*>(t.mutable_data_ptr()); }

using QuantFn = Two(const at::Tensor&);
struct Quant {
    static constexpr const char *name = "sglang_exl3::fp8_quant_rows", *general = "sglang_exl3::fp8_quant_rows_general";
};

Two fp8_quant_rows(const at::Tensor& x) {
    Fp8Rows r;
    if (r.get(x) && r.k % 16 == 0) {
        Two out = fp8_out(x, r.k);
        if (abi.quant(x.const_data_ptr(), r.stride, bytes_of(std::get<0>(out)), floats_of(std::get<1>(out)), r.dtype,
                      (int)r.m, (int)r.k, stream_of(x.get_device())) == EXL3_OK)
            return out;
    }
    static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow(Quant::general, "").typed<QuantFn>();
    return h.call(x);
}

using NormFn = std::vector<at::Tensor>(const at::Tensor&, const at::Tensor&, double, const OptTensor&, bool);
struct Norm {
    static constexpr const char *name = "sglang_exl3::fp8_norm_quant", *general = "sglang_exl3::fp8_norm_quant_general";
};

std::vector<at::Tensor> fp8_norm_quant(const at::Tensor& x, const at::Tensor& weight, double eps,
                                       const OptTensor& residual, bool rows) {
    Fp8Rows r, s;
    const bool add = residual.has_value();
    if (r.get(x) && r.k % 16 == 0 && r.k <= 32768 && eps >= 0.0 && weight.is_cuda() &&
        weight.get_device() == x.get_device() && weight.scalar_type() == x.scalar_type() && weight.dim() == 1 &&
        weight.size(0) == r.k && weight.is_contiguous() && at_bytes(weight, 16) &&
        (!add || (s.get(*residual) && s.dtype == r.dtype && residual->sizes() == x.sizes() &&
                  residual->get_device() == x.get_device()))) {
        Two q = fp8_out(x, r.k);
        std::vector<at::Tensor> out = {std::get<0>(q), std::get<1>(q)};
        if (add) out.push_back(fresh(x, x.sizes(), x.scalar_type()));
        if (rows) out.push_back(fresh(x, x.sizes(), x.scalar_type()));
        if (abi.norm(x.const_data_ptr(), r.stride, add ? residual->const_data_ptr() : nullptr, add ? s.stride : 0,
                     weight.const_data_ptr(), (float)eps, add ? out[2].mutable_data_ptr() : nullptr,
                     rows ? out.back().mutable_data_ptr() : nullptr, bytes_of(out[0]), floats_of(out[1]), r.dtype,
                     (int)r.m, (int)r.k, stream_of(x.get_device())) == EXL3_OK)
            return out;
    }
    static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow(Norm::general, "").typed<NormFn>();
    return h.call(x, weight, eps, residual, rows);
}

using SwigluFn = Two(const at::Tensor&, double);
struct Swiglu {
    static constexpr const char *name = "sglang_exl3::fp8_swiglu_quant",
                                *general = "sglang_exl3::fp8_swiglu_quant_general";
};

Two fp8_swiglu_quant(const at::Tensor& x, double limit) {
    Fp8Rows r;
    if (r.get(x) && r.k % 32 == 0 && (limit == 0.0 || limit >= 1.17549435e-38)) {
        Two out = fp8_out(x, r.k / 2);
        if (abi.swiglu(x.const_data_ptr(), r.stride, (float)limit, bytes_of(std::get<0>(out)),
                       floats_of(std::get<1>(out)), r.dtype, (int)r.m, (int)(r.k / 2),
                       stream_of(x.get_device())) == EXL3_OK)
            return out;
    }
    static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow(Swiglu::general, "").typed<SwigluFn>();
    return h.call(x, limit);
}

using LinearFn = at::Tensor(const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&,
                            const OptTensor&, bool);
struct Linear {
    static constexpr const char *name = "sglang_exl3::fp8_linear", *general = "sglang_exl3::fp8_linear_general";
};

at::Tensor fp8_linear(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& weight_scale,
                      const OptTensor& x_scale, const OptTensor& bias, bool out_bf16) {
    const auto out = out_bf16 ? at::kBFloat16 : at::kHalf;
    const int64_t n = weight.dim() == 2 ? weight.size(0) : 0, k = weight.dim() == 2 ? weight.size(1) : 0;
    const auto here = [&](const at::Tensor& t, at::ScalarType type) {
        return t.is_cuda() && t.get_device() == x.get_device() && t.scalar_type() == type && t.is_contiguous();
    };
    bool ok = on_current(x) && n > 0 && n <= (1 << 24) && k > 0 && k % 16 == 0 && k <= (1 << 22) && x.dim() >= 1 &&
              x.size(-1) == k && x.numel() > 0 && x.is_contiguous() && at_bytes(x, 16) && here(weight, at::kFloat8_e4m3fn) &&
              at_bytes(weight, 16) && here(weight_scale, at::kFloat) && weight_scale.dim() == 2 &&
              weight_scale.size(0) == fp8_groups(n) && weight_scale.size(1) == fp8_groups(k);
    int type = EXL3_DTYPE_E4M3;
    if (ok && x.scalar_type() == at::kFloat8_e4m3fn)
        ok = x_scale.has_value() && here(*x_scale, at::kFloat) && x_scale->dim() == x.dim() &&
             x_scale->size(-1) == fp8_groups(k) && x_scale->sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1);
    else if (ok) {
        type = x.scalar_type() == at::kBFloat16 ? EXL3_DTYPE_BF16 : EXL3_DTYPE_F16;
        ok = !x_scale.has_value() && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf);
    }
    if (ok && bias.has_value()) ok = here(*bias, out) && bias->dim() == 1 && bias->size(0) == n;
    const int64_t m = ok ? x.numel() / k : 0;
    if (ok && m <= (1 << 24) && m * fp8_groups(k) <= 0x7fffffff) {
        const size_t need = abi.fp8_ws(type, (int)m, (int)k, (int)n);
        Launch l;
        if (need == 0) l.stream = stream_of(x.get_device());
        if (need == 0 || l.get(x.get_device(), need)) {
            at::Tensor y = fresh(x, {m, n}, out);
            const int rc = abi.fp8(x.const_data_ptr(), type, x_scale.has_value() ? x_scale->const_data_ptr<float>() : nullptr,
                                   static_cast<const uint8_t*>(weight.const_data_ptr()),
                                   weight_scale.const_data_ptr<float>(),
                                   bias.has_value() ? bias->const_data_ptr() : nullptr, y.mutable_data_ptr(),
                                   out_bf16 ? EXL3_DTYPE_BF16 : EXL3_DTYPE_F16, (int)m, (int)k, (int)n,
                                   need ? l.ws.mutable_data_ptr() : nullptr, need ? l.ws.numel() : 0, l.stream);
            if (need ? done(rc, l) : rc == EXL3_OK) return y;
        }
    }
    static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow(Linear::general, "").typed<LinearFn>();
    return h.call(x, weight, weight_scale, x_scale, bias, out_bf16);
}

// -------------------------------------------------------------------- autograd

bool wants_grad(const at::Tensor& t) { return t.requires_grad(); }
bool wants_grad(at::TensorList ts) {
    for (const auto& t : ts)
        if (t.requires_grad()) return true;
    return false;
}
bool wants_grad(const OptTensor& t) { return t.has_value() && t->requires_grad(); }
bool wants_grad(const c10::SymInt&) { return false; }
bool wants_grad(bool) { return false; }
bool wants_grad(double) { return false; }

// Inputs that require grad take the general operator (its autograd kernel);
// others go below autograd, to the modes and keys that follow.
template <class Op, class F>
struct Autograd;
template <class Op, class R, class... A>
struct Autograd<Op, R(A...)> {
    static R call(c10::DispatchKeySet ks, A... a) {
        if (c10::GradMode::is_enabled() && (wants_grad(a) || ...)) {
            static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow(Op::general, "").template typed<R(A...)>();
            return h.call(a...);
        }
        static const auto h = c10::Dispatcher::singleton().findSchemaOrThrow(Op::name, "").template typed<R(A...)>();
        at::AutoDispatchBelowAutograd below;
        return h.redispatch(ks & c10::after_autograd_keyset, a...);
    }
};

}  // namespace

TORCH_LIBRARY_IMPL(sglang_exl3, CUDA, m) {
    m.impl("exl3_gemv", gemv);
    m.impl("exl3_linear_cat", linear_cat);
    m.impl("exl3_linear_part", linear_part);
    m.impl("exl3_gate_up_swiglu", gate_up);
    m.impl("fp8_quant_rows", fp8_quant_rows);
    m.impl("fp8_norm_quant", fp8_norm_quant);
    m.impl("fp8_swiglu_quant", fp8_swiglu_quant);
    m.impl("fp8_linear", fp8_linear);
    m.impl("keep_workspace", keep_workspace);
}

TORCH_LIBRARY_IMPL(sglang_exl3, AutogradCUDA, m) {
    m.impl("exl3_gemv", Autograd<Gemv, GemvFn>::call);
    m.impl("exl3_linear_cat", Autograd<Cat, CatFn>::call);
    m.impl("exl3_linear_part", Autograd<Part, PartFn>::call);
    m.impl("exl3_gate_up_swiglu", Autograd<GateUp, GateUpFn>::call);
    m.impl("fp8_quant_rows", Autograd<Quant, QuantFn>::call);
    m.impl("fp8_norm_quant", Autograd<Norm, NormFn>::call);
    m.impl("fp8_swiglu_quant", Autograd<Swiglu, SwigluFn>::call);
    m.impl("fp8_linear", Autograd<Linear, LinearFn>::call);
}

// The PyTorch that this was built for (EXL3_TORCH_VERSION), looked up in the file
// before it is loaded: another one's ABI need not fit.
extern "C" __attribute__((used)) const char exl3_ops_torch[] = "exl3-ops-torch:" EXL3_TORCH_VERSION;

// Addresses of the C ABI, in the order of _lib.py's _OPS_BOUND.
extern "C" void exl3_ops_bind(void* const* fn) {
    abi.gemv = reinterpret_cast<decltype(abi.gemv)>(fn[0]);
    abi.gemv_ws = reinterpret_cast<decltype(abi.gemv_ws)>(fn[1]);
    abi.cat = reinterpret_cast<decltype(abi.cat)>(fn[2]);
    abi.cat_ws = reinterpret_cast<decltype(abi.cat_ws)>(fn[3]);
    abi.gate_up = reinterpret_cast<decltype(abi.gate_up)>(fn[4]);
    abi.gate_up_ws = reinterpret_cast<decltype(abi.gate_up_ws)>(fn[5]);
    abi.quant = reinterpret_cast<decltype(abi.quant)>(fn[6]);
    abi.norm = reinterpret_cast<decltype(abi.norm)>(fn[7]);
    abi.swiglu = reinterpret_cast<decltype(abi.swiglu)>(fn[8]);
    abi.fp8 = reinterpret_cast<decltype(abi.fp8)>(fn[9]);
    abi.fp8_ws = reinterpret_cast<decltype(abi.fp8_ws)>(fn[10]);
}
