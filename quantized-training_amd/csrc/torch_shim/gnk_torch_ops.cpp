// gnk_torch_ops.cpp -- device ("CUDA" key = HIP on ROCm) implementations of the hot gn_kernels operators, registered from C++.
//
// The operator SCHEMAS live in Python (gn_kernels/mm.py, quantize.py: the reference's own strings, triton_mm.py:112,345-346); this
// file only replaces the per-call host path dispatcher -> Python -> ctypes -> C ABI (13-22 us per call) by
// dispatcher -> C++ -> C ABI (~3 us): the reference's CUTLASS ops are registered the same way (csrc/cutlass_sm89_fp8.cu:187-190,
// TORCH_LIBRARY_IMPL(gn_kernels, CUDA, m)).  No arithmetic happens here: every function validates, allocates the output as the
// reference does (at::empty) and calls the extern "C" entry point of libgnk_hip.so declared in include/gnk.h.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>   // PyTorch-ROCm: HIP devices carry DeviceType CUDA
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include "../../../include/gnk.h"

namespace {

int dtype_code(at::ScalarType t, const char *op) {
    switch (t) {
        case at::kBFloat16: return GNK_BF16;
        case at::kHalf: return GNK_F16;
        case at::kFloat: return GNK_F32;
        case at::kChar: return GNK_I8;
        case at::kFloat8_e4m3fn: return GNK_E4M3;
        case at::kFloat8_e5m2: return GNK_E5M2;
        case at::kInt: return GNK_I32;
        default: TORCH_CHECK(false, "gn_kernels::", op, ": unsupported dtype ", t);
    }
}

bool is_float(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf || t == at::kFloat; }

void check(int rc, const char *op) { TORCH_CHECK(rc == 0, "gn_kernels::", op, " failed (status ", rc, "): ", gnk_last_error()); }

void *stream_of(const at::Tensor &t) { return (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream(); }

// ---------------------------------------------------------------------------------------------- GEMMs
at::Tensor int8_mm(const at::Tensor &A, const at::Tensor &B) {
    const int64_t M = A.size(0), K = A.size(1), N = B.size(1);
    at::Tensor C = at::empty({M, N}, A.options().dtype(at::kInt));
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(A.device());
    check(gnk_int8_mm((const int8_t *)A.data_ptr(), (const int8_t *)B.data_ptr(), (int32_t *)C.data_ptr(), M, N, K, A.stride(0), A.stride(1),
                      B.stride(0), B.stride(1), stream_of(A)),
          "int8_mm");
    return C;
}

at::Tensor scaled_mm_impl(const at::Tensor &A, const at::Tensor &B, const at::Tensor &rs, const at::Tensor &cs, at::ScalarType out, int order,
                          const char *op) {
    const int64_t M = A.size(0), K = A.size(1), N = B.size(1);
    TORCH_CHECK(is_float(rs.scalar_type()), "gn_kernels::", op, ": scale dtype ", rs.scalar_type(), " is not bf16 / fp16 / fp32");
    at::Tensor C = at::empty({M, N}, A.options().dtype(out));
    const int ad = dtype_code(A.scalar_type(), op), bd = dtype_code(B.scalar_type(), op);
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(A.device());
    // long K, small output (grad-weight shapes): offer the library a split-K workspace if it wants one
    const int64_t ws_bytes = (K >= 2048 && A.scalar_type() == at::kChar) ? gnk_scaled_mm_workspace_bytes(ad, bd, M, N, K) : 0;
    int rc;
    if (ws_bytes > 0) {
        at::Tensor ws = at::empty({ws_bytes}, A.options().dtype(at::kByte));
        rc = gnk_scaled_mm_ws(A.data_ptr(), ad, B.data_ptr(), bd, C.data_ptr(), dtype_code(out, op), rs.data_ptr(), cs.data_ptr(),
                              dtype_code(rs.scalar_type(), op), cs.numel() == 1, order, M, N, K, A.stride(0), A.stride(1), B.stride(0), B.stride(1),
                              ws.data_ptr(), ws_bytes, stream_of(A));
    } else {
        rc = gnk_scaled_mm(A.data_ptr(), ad, B.data_ptr(), bd, C.data_ptr(), dtype_code(out, op), rs.data_ptr(), cs.data_ptr(),
                           dtype_code(rs.scalar_type(), op), cs.numel() == 1, order, M, N, K, A.stride(0), A.stride(1), B.stride(0), B.stride(1),
                           stream_of(A));
    }
    check(rc, op);
    return C;
}

// (f32(acc) * row) * col, output dtype = scale dtype (reference triton_mm.py:382-407)
at::Tensor scaled_mm(const at::Tensor &A, const at::Tensor &B, const at::Tensor &rs, const at::Tensor &cs) {
    return scaled_mm_impl(A, B, rs, cs, rs.scalar_type(), 0, "scaled_mm");
}

// == scaled_mm(A, B, sA, sB).T as a contiguous tensor (gn_kernels/mm.py:scaled_mm_t): operand roles and multiply order swapped together
at::Tensor scaled_mm_t(const at::Tensor &A, const at::Tensor &B, const at::Tensor &sA, const at::Tensor &sB) {
    return scaled_mm_impl(B.t(), A.t(), sB, sA, sA.scalar_type(), 1, "scaled_mm_t");
}

// block sizes from integer shape ratios (reference triton_mm.py:419,434-436); ragged tilings are refused (see gn_kernels/mm.py)
at::Tensor tile_scaled_mm(const at::Tensor &A, const at::Tensor &B, const at::Tensor &sA, const at::Tensor &sB) {
    const int64_t M = A.size(0), K = A.size(1), N = B.size(1);
    TORCH_CHECK(is_float(sA.scalar_type()), "gn_kernels::tile_scaled_mm: scale dtype ", sA.scalar_type(), " is not bf16 / fp16 / fp32");
    TORCH_CHECK(sA.size(0) > 0 && sA.size(1) > 0 && sB.size(1) > 0, "gn_kernels::tile_scaled_mm: empty scale tensor");
    const int64_t QM = M / sA.size(0), QK = K / sA.size(1), QN = N / sB.size(1);
    TORCH_CHECK(QM >= 1 && QN >= 1 && QK >= 1 && M % sA.size(0) == 0 && N % sB.size(1) == 0 && K % sA.size(1) == 0,
                "gn_kernels::tile_scaled_mm: scale shapes ", sA.sizes(), ", ", sB.sizes(), " do not tile a (", M, ", ", K, ") x (", K, ", ", N,
                ") product evenly");
    at::Tensor C = at::empty({M, N}, A.options().dtype(sA.scalar_type()));
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(A.device());
    check(gnk_tile_scaled_mm(A.data_ptr(), dtype_code(A.scalar_type(), "tile_scaled_mm"), B.data_ptr(), dtype_code(B.scalar_type(), "tile_scaled_mm"),
                             C.data_ptr(), dtype_code(sA.scalar_type(), "tile_scaled_mm"), sA.data_ptr(), sB.data_ptr(),
                             dtype_code(sA.scalar_type(), "tile_scaled_mm"), M, N, K, A.stride(0), A.stride(1), B.stride(0), B.stride(1), sA.stride(0),
                             sA.stride(1), sB.stride(0), sB.stride(1), QM, QN, QK, stream_of(A)),
          "tile_scaled_mm");
    return C;
}

// ---------------------------------------------------------------------------------------------- quantize
bool dense2d(const at::Tensor &x) { return x.is_contiguous() || x.t().is_contiguous(); }

void sr_args(bool sr, const c10::optional<at::Tensor> &rng, uint64_t &seed) {
    seed = 0;
    if (!sr) return;
    // the Python wrappers always pass the call's Philox key (a 0-dim int64 HOST tensor drawn from torch's CPU generator); an op called
    // directly without one draws here, the same way
    const at::Tensor r = rng.has_value() ? *rng : at::randint(0, (int64_t)1 << 62, {}, at::TensorOptions().dtype(at::kLong));
    seed = (uint64_t)r.item<int64_t>();
}

std::tuple<at::Tensor, at::Tensor> quantize_int8(const at::Tensor &x, int64_t dim, bool sr, double eps, const c10::optional<at::Tensor> &rng) {
    const int64_t nd = x.dim();
    TORCH_CHECK(is_float(x.scalar_type()) && nd >= 1, "gn_kernels::quantize_int8: unsupported input (dtype ", x.scalar_type(), ", ", nd, " dims)");
    const int64_t d = ((dim % nd) + nd) % nd;
    TORCH_CHECK(nd == 2 || (d == nd - 1 && x.is_contiguous()), "gn_kernels::quantize_int8: unsupported input (shape ", x.sizes(), ", strides ",
                x.strides(), ", dim ", dim, ")");
    int64_t R, C, sxr, sxc, sqr, sqc;
    at::Tensor q;
    if (nd == 2) {
        q = dense2d(x) ? at::empty_strided(x.sizes(), x.strides(), x.options().dtype(at::kChar)) : at::empty_like(x, x.options().dtype(at::kChar));
        const int64_t o = 1 - d;
        R = x.size(o); C = x.size(d); sxr = x.stride(o); sxc = x.stride(d); sqr = q.stride(o); sqc = q.stride(d);
    } else {
        C = x.size(nd - 1);
        R = C > 0 ? x.numel() / C : 0;
        sxr = C; sxc = 1; sqr = C; sqc = 1;
        q = at::empty(x.sizes(), x.options().dtype(at::kChar));
    }
    auto sshape = x.sizes().vec();
    sshape[d] = 1;
    at::Tensor scale = at::empty(sshape, x.options());
    if (x.numel() == 0) return {q, scale.zero_()};
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    const int64_t ws_bytes = gnk_quantize_int8_workspace_bytes(R, C, sxr, sxc);
    at::Tensor ws;
    if (ws_bytes > 0) ws = at::empty({ws_bytes}, x.options().dtype(at::kByte));
    uint64_t seed;
    sr_args(sr, rng, seed);
    check(gnk_quantize_int8(x.data_ptr(), dtype_code(x.scalar_type(), "quantize_int8"), R, C, sxr, sxc, (int8_t *)q.data_ptr(), sqr, sqc,
                            scale.data_ptr(), (float)eps, sr, seed, 0, ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes, stream_of(x)),
          "quantize_int8");
    return {q, scale};
}

bool rows16(const at::Tensor &x) {   // shape / stride part of supports_rowwise_colmax / supports_colwise_given (gn_kernels/quantize.py)
    return x.dim() == 2 && is_float(x.scalar_type()) && x.numel() > 0 && x.stride(1) == 1 && x.stride(0) >= x.size(1) &&
           (x.stride(0) * (int64_t)x.element_size()) % 16 == 0 && x.size(1) % (16 / (int64_t)x.element_size()) == 0;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> quantize_int8_rowwise_colmax(const at::Tensor &x_in, bool sr, double eps,
                                                                           const c10::optional<at::Tensor> &rng) {
    const int code = rows16(x_in) ? dtype_code(x_in.scalar_type(), "quantize_int8_rowwise_colmax") : -1;
    TORCH_CHECK(code >= 0 && gnk_quantize_int8_rowwise_colmax_workspace_bytes(code, x_in.size(0), x_in.size(1)) > 0,
                "gn_kernels::quantize_int8_rowwise_colmax: unsupported input (shape ", x_in.sizes(), ", strides ", x_in.strides(), ", dtype ",
                x_in.scalar_type(), ")");
    const at::Tensor x = ((uintptr_t)x_in.data_ptr() % 16 == 0) ? x_in : x_in.clone(at::MemoryFormat::Contiguous);   // fresh allocations are aligned
    const int64_t R = x.size(0), C = x.size(1);
    at::Tensor q = at::empty_like(x, x.options().dtype(at::kChar));
    if (q.stride(1) != 1) q = at::empty({R, C}, x.options().dtype(at::kChar));
    at::Tensor scale = at::empty({R, 1}, x.options());
    at::Tensor colmax = at::empty({C}, x.options().dtype(at::kFloat));
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    const int64_t ws_bytes = gnk_quantize_int8_rowwise_colmax_workspace_bytes(code, R, C);
    at::Tensor ws = at::empty({ws_bytes}, x.options().dtype(at::kByte));
    uint64_t seed;
    sr_args(sr, rng, seed);
    check(gnk_quantize_int8_rowwise_colmax(x.data_ptr(), code, R, C, x.stride(0), (int8_t *)q.data_ptr(), q.stride(0), scale.data_ptr(),
                                           (float *)colmax.data_ptr(), (float)eps, sr, seed, 0, ws.data_ptr(), ws_bytes, stream_of(x)),
          "quantize_int8_rowwise_colmax");
    return {q, scale, colmax};
}

std::tuple<at::Tensor, at::Tensor> quantize_int8_colwise_given(const at::Tensor &x_in, const at::Tensor &absmax, bool sr, double eps,
                                                              const c10::optional<at::Tensor> &rng) {
    TORCH_CHECK(rows16(x_in), "gn_kernels::quantize_int8_colwise_given: unsupported input (shape ", x_in.sizes(), ", strides ", x_in.strides(),
                ", dtype ", x_in.scalar_type(), ")");
    const at::Tensor x = ((uintptr_t)x_in.data_ptr() % 16 == 0) ? x_in : x_in.clone(at::MemoryFormat::Contiguous);
    const int64_t P = x.size(0), Q = x.size(1);
    TORCH_CHECK(absmax.is_cuda() && absmax.scalar_type() == at::kFloat && absmax.numel() == Q && absmax.is_contiguous(),
                "gn_kernels::quantize_int8_colwise_given: absmax must be a contiguous fp32 device tensor with one value per column");
    at::Tensor q = at::empty_like(x, x.options().dtype(at::kChar));
    if (q.stride(1) != 1) q = at::empty({P, Q}, x.options().dtype(at::kChar));
    at::Tensor scale = at::empty({1, Q}, x.options());
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    uint64_t seed;
    sr_args(sr, rng, seed);
    check(gnk_quantize_int8_colwise_given_absmax(x.data_ptr(), dtype_code(x.scalar_type(), "quantize_int8_colwise_given"), P, Q, x.stride(0),
                                                 (int8_t *)q.data_ptr(), q.stride(0), scale.data_ptr(), (const float *)absmax.data_ptr(), (float)eps,
                                                 sr, seed, 0, stream_of(x)),
          "quantize_int8_colwise_given");
    return {q, scale};
}

// ---------------------------------------------------------------------------------------------- products grouped by expert (gn_kernels/grouped.py)
void grouped_args(const at::Tensor &A, const at::Tensor &B, const at::Tensor &sA, const at::Tensor &sB, const at::Tensor &ends, const char *op) {
    TORCH_CHECK(is_float(sA.scalar_type()) && sB.scalar_type() == sA.scalar_type(), "gn_kernels::", op, ": scale dtypes ", sA.scalar_type(), ", ",
                sB.scalar_type(), " are not one of bf16 / fp16 / fp32");
    TORCH_CHECK(sA.is_contiguous() && sB.is_contiguous(), "gn_kernels::", op, ": scales must be contiguous");
    TORCH_CHECK(ends.scalar_type() == at::kInt && ends.dim() == 1 && ends.is_contiguous(), "gn_kernels::", op, ": offs must be a contiguous 1-D int32 tensor");
    TORCH_CHECK(B.device() == A.device() && sA.device() == A.device() && sB.device() == A.device() && ends.device() == A.device(), "gn_kernels::", op,
                ": all tensors must be on one device");
}

at::Tensor workspace_for(const at::Tensor &A, int64_t bytes) { return bytes > 0 ? at::empty({bytes}, A.options().dtype(at::kByte)) : at::Tensor(); }

at::Tensor grouped_scaled_mm(const at::Tensor &A, const at::Tensor &B, const at::Tensor &sA, const at::Tensor &sB, const at::Tensor &ends) {
    const char *op = "grouped_scaled_mm";
    grouped_args(A, B, sA, sB, ends, op);
    TORCH_CHECK(A.dim() == 2 && B.dim() == 3 && B.size(1) == A.size(1) && ends.size(0) == B.size(0) && sA.numel() == A.size(0) &&
                (sB.numel() == B.size(0) * B.size(2) || sB.numel() == B.size(0)), "gn_kernels::", op, ": shapes ", A.sizes(), ", ", B.sizes(), ", ", sA.sizes(),
                ", ", sB.sizes(), ", ", ends.sizes(), " do not go together");
    const int64_t T = A.size(0), K = A.size(1), E = B.size(0), N = B.size(2);
    at::Tensor C = at::empty({T, N}, sA.options());
    const int ad = dtype_code(A.scalar_type(), op), bd = dtype_code(B.scalar_type(), op), sd = dtype_code(sA.scalar_type(), op);
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(A.device());
    const int64_t nws = gnk_grouped_scaled_mm_rows_workspace_bytes(A.data_ptr(), B.data_ptr(), T, E, N, K, A.stride(0), A.stride(1), B.stride(0), B.stride(1),
                                                                   B.stride(2));
    const at::Tensor ws = workspace_for(A, nws);
    check(gnk_grouped_scaled_mm_rows(A.data_ptr(), ad, B.data_ptr(), bd, C.data_ptr(), sd, sA.data_ptr(), sB.data_ptr(), sd, sB.size(2) == 1 && N != 1,
                                     (const int32_t *)ends.data_ptr(), T, E, N, K, A.stride(0), A.stride(1), B.stride(0), B.stride(1), B.stride(2),
                                     nws > 0 ? ws.data_ptr() : nullptr, nws, stream_of(A)),
          op);
    return C;
}

at::Tensor grouped_scaled_mm_depth(const at::Tensor &A, const at::Tensor &B, const at::Tensor &sA, const at::Tensor &sB, const at::Tensor &ends) {
    const char *op = "grouped_scaled_mm_depth";
    grouped_args(A, B, sA, sB, ends, op);
    const int64_t E = ends.size(0), M = A.size(0), T = A.size(1), N = B.size(1);
    TORCH_CHECK(A.dim() == 2 && B.dim() == 2 && B.size(0) == T && sA.numel() == E * M && (sB.numel() == E * N || sB.numel() == E), "gn_kernels::", op,
                ": shapes ", A.sizes(), ", ", B.sizes(), ", ", sA.sizes(), ", ", sB.sizes(), ", ", ends.sizes(), " do not go together");
    at::Tensor C = at::empty({E, M, N}, sA.options());
    const int ad = dtype_code(A.scalar_type(), op), bd = dtype_code(B.scalar_type(), op), sd = dtype_code(sA.scalar_type(), op);
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(A.device());
    const int64_t copies = gnk_grouped_scaled_mm_depth_workspace_bytes(A.data_ptr(), B.data_ptr(), T, M, N, A.stride(0), A.stride(1), B.stride(0), B.stride(1));
    const int64_t nws = (copies + 15) / 16 * 16 + gnk_grouped_scaled_mm_depth_split_bytes(T, E, M, N);
    const at::Tensor ws = workspace_for(A, nws);
    check(gnk_grouped_scaled_mm_depth(A.data_ptr(), ad, B.data_ptr(), bd, C.data_ptr(), sd, sA.data_ptr(), sB.data_ptr(), sd, sB.size(2) == 1 && N != 1,
                                      (const int32_t *)ends.data_ptr(), T, E, M, N, A.stride(0), A.stride(1), B.stride(0), B.stride(1),
                                      nws > 0 ? ws.data_ptr() : nullptr, nws, stream_of(A)),
          op);
    return C;
}

std::tuple<at::Tensor, at::Tensor> quantize_int8_grouped(const at::Tensor &x, const at::Tensor &ends, bool sr, double eps, const c10::optional<at::Tensor> &rng) {
    const char *op = "quantize_int8_grouped";
    TORCH_CHECK(is_float(x.scalar_type()) && x.dim() == 2, "gn_kernels::", op, ": unsupported input (shape ", x.sizes(), ", dtype ", x.scalar_type(), ")");
    TORCH_CHECK(ends.scalar_type() == at::kInt && ends.dim() == 1 && ends.is_contiguous() && ends.device() == x.device(), "gn_kernels::", op,
                ": offs must be a contiguous 1-D int32 tensor on x's device");
    const int64_t T = x.size(0), C = x.size(1), E = ends.size(0);
    at::Tensor q = at::empty({T, C}, x.options().dtype(at::kChar)), scale = at::empty({E, 1, C}, x.options());
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    const int64_t nws = gnk_quantize_int8_grouped_workspace_bytes(T, E, C);
    const at::Tensor ws = workspace_for(x, nws);
    uint64_t seed;
    sr_args(sr, rng, seed);
    check(gnk_quantize_int8_grouped(x.data_ptr(), dtype_code(x.scalar_type(), op), (const int32_t *)ends.data_ptr(), T, E, C, x.stride(0), x.stride(1),
                                    (int8_t *)q.data_ptr(), scale.data_ptr(), (float)eps, sr, seed, 0, nws > 0 ? ws.data_ptr() : nullptr, nws, stream_of(x)),
          op);
    return {q, scale};
}

// F.grouped_mm on a mixed-precision weight (subclasses/mixed_precision.py), forward and backward as one call each: seven quantizations and three products
// whose host path would otherwise cost more than the kernels of a small layer.  w: (E, K, N) as grouped_mm takes it, usually a view of (E, N, K) weights.
// Temporaries are carved out of one allocation.
struct Carver {
    at::Tensor buf;
    int64_t used = 0;
    static int64_t up(int64_t n) { return (n + 255) / 256 * 256; }
    char *take(int64_t n) {
        char *const p = (char *)buf.data_ptr() + used;
        used += up(n);
        return p;
    }
};

void grouped_linear_args(const at::Tensor &x, const at::Tensor &w, const at::Tensor &ends, const char *op) {
    TORCH_CHECK(x.dim() == 2 && w.dim() == 3 && w.size(1) == x.size(1) && is_float(x.scalar_type()) && w.scalar_type() == x.scalar_type(), "gn_kernels::", op,
                ": x ", x.sizes(), " ", x.scalar_type(), " and weight ", w.sizes(), " ", w.scalar_type(), " do not go together");
    TORCH_CHECK(ends.scalar_type() == at::kInt && ends.dim() == 1 && ends.is_contiguous() && ends.size(0) == w.size(0), "gn_kernels::", op,
                ": offs must be a contiguous 1-D int32 tensor with one end per expert");
    TORCH_CHECK(w.device() == x.device() && ends.device() == x.device(), "gn_kernels::", op, ": all tensors must be on one device");
}

void quant_rows(const at::Tensor &x, int code, int64_t R, int64_t C, int64_t sr, char *q, char *s, void *st, const char *op) {
    if (R == 0) return;
    check(gnk_quantize_int8(x.data_ptr(), code, R, C, sr, 1, (int8_t *)q, C, 1, s, 1e-12f, 0, 0, 0, nullptr, 0, st), op);
}

at::Tensor grouped_linear_int8(const at::Tensor &x_in, const at::Tensor &w, const at::Tensor &ends) {
    const char *op = "grouped_linear_int8";
    grouped_linear_args(x_in, w, ends, op);
    const at::Tensor x = x_in.stride(1) == 1 || x_in.size(1) == 1 ? x_in : x_in.contiguous();
    const at::Tensor wt = w.transpose(1, 2).contiguous();                       // (E, N, K): no copy in the usual call
    const int64_t T = x.size(0), K = x.size(1), E = w.size(0), N = w.size(2), es = x.element_size();
    const int code = dtype_code(x.scalar_type(), op);
    at::Tensor y = at::empty({T, N}, x.options());
    if (K == 0) return y.zero_();
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    void *const st = stream_of(x);
    // the operand copies' size depends on alignment only through the base, which the carver aligns
    const int64_t nws = gnk_grouped_scaled_mm_rows_workspace_bytes(nullptr, nullptr, T, E, N, K, K, 1, N * K, 1, K);
    Carver c{at::empty({Carver::up(T * K) + Carver::up(T * es) + Carver::up(E * N * K) + Carver::up(E * N * es) + nws + 256}, x.options().dtype(at::kByte))};
    char *const xq = c.take(T * K), *const xs = c.take(T * es), *const wq = c.take(E * N * K), *const ws = c.take(E * N * es), *const scratch = c.take(nws);
    quant_rows(x, code, T, K, x.stride(0), xq, xs, st, op);
    quant_rows(wt, code, E * N, K, K, wq, ws, st, op);
    check(gnk_grouped_scaled_mm_rows(xq, GNK_I8, wq, GNK_I8, y.data_ptr(), code, xs, ws, code, 0, (const int32_t *)ends.data_ptr(), T, E, N, K, K, 1, N * K, 1, K,
                                     nws > 0 ? scratch : nullptr, nws, st),
          op);
    return y;
}

std::tuple<at::Tensor, at::Tensor> grouped_linear_int8_backward(const at::Tensor &g_in, const at::Tensor &x_in, const at::Tensor &w, const at::Tensor &ends, bool need_x,
                                                                bool need_w) {
    const char *op = "grouped_linear_int8_backward";
    grouped_linear_args(x_in, w, ends, op);
    TORCH_CHECK(g_in.dim() == 2 && g_in.size(0) == x_in.size(0) && g_in.size(1) == w.size(2) && g_in.scalar_type() == x_in.scalar_type() && g_in.device() == x_in.device(),
                "gn_kernels::", op, ": gradient ", g_in.sizes(), " ", g_in.scalar_type(), " does not fit");
    const at::Tensor g = g_in.contiguous(), x = x_in.contiguous();
    const int64_t T = x.size(0), K = x.size(1), E = w.size(0), N = w.size(2), es = x.element_size();
    const int code = dtype_code(x.scalar_type(), op);
    const int32_t *const end = (const int32_t *)ends.data_ptr();
    at::Tensor gx = at::empty({need_x ? T : 0, K}, x.options()), gw = at::empty({need_w ? E : 0, N, K}, x.options());
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    void *const st = stream_of(x);
    auto quant_cols = [&](const at::Tensor &t, const int32_t *e, int64_t rows, int64_t cols, char *q, char *s, char *scratch, int64_t bytes) {
        check(gnk_quantize_int8_grouped(t.data_ptr(), code, e, rows, E, cols, cols, 1, (int8_t *)q, s, 1e-12f, 0, 0, 0, bytes > 0 ? scratch : nullptr, bytes, st), op);
    };
    if (need_x && N == 0) gx.zero_();
    if (need_x && N > 0) {
        const at::Tensor wt = w.transpose(1, 2).contiguous();
        const int64_t qws = gnk_quantize_int8_grouped_workspace_bytes(E * N, E, K);
        const int64_t nws = gnk_grouped_scaled_mm_rows_workspace_bytes(nullptr, nullptr, T, E, K, N, N, 1, N * K, K, 1);
        Carver c{at::empty({Carver::up(T * N) + Carver::up(T * es) + Carver::up(E * N * K) + Carver::up(E * K * es) + Carver::up(qws) + nws + 256}, x.options().dtype(at::kByte))};
        char *const gq = c.take(T * N), *const gs = c.take(T * es), *const wq = c.take(E * N * K), *const ws = c.take(E * K * es), *const part = c.take(qws);
        char *const scratch = c.take(nws);
        quant_rows(g, code, T, N, N, gq, gs, st, op);
        quant_cols(wt, nullptr, E * N, K, wq, ws, part, qws);                   // an expert's N rows are a group
        check(gnk_grouped_scaled_mm_rows(gq, GNK_I8, wq, GNK_I8, gx.data_ptr(), code, gs, ws, code, 0, end, T, E, K, N, N, 1, N * K, K, 1,
                                         nws > 0 ? scratch : nullptr, nws, st),
              op);
    }
    if (need_w) {
        const int64_t qg = gnk_quantize_int8_grouped_workspace_bytes(T, E, N), qx = gnk_quantize_int8_grouped_workspace_bytes(T, E, K);
        const int64_t nws = (gnk_grouped_scaled_mm_depth_workspace_bytes(nullptr, nullptr, T, N, K, 1, N, K, 1) + 15) / 16 * 16 +
                            gnk_grouped_scaled_mm_depth_split_bytes(T, E, N, K);
        Carver c{at::empty({Carver::up(T * N) + Carver::up(E * N * es) + Carver::up(T * K) + Carver::up(E * K * es) + Carver::up(std::max(qg, qx)) + nws + 256},
                           x.options().dtype(at::kByte))};
        char *const gq = c.take(T * N), *const gs = c.take(E * N * es), *const xq = c.take(T * K), *const xs = c.take(E * K * es), *const part = c.take(std::max(qg, qx));
        char *const scratch = c.take(nws);
        quant_cols(g, end, T, N, gq, gs, part, qg);
        quant_cols(x, end, T, K, xq, xs, part, qx);
        check(gnk_grouped_scaled_mm_depth(gq, GNK_I8, xq, GNK_I8, gw.data_ptr(), code, gs, xs, code, 0, end, T, E, N, K, 1, N, K, 1, nws > 0 ? scratch : nullptr, nws, st),
              op);
    }
    return {gx, gw};
}

at::Tensor orthogonalize(const at::Tensor &G_in, int64_t steps, double a, double b, double c, double eps) {
    const char *op = "orthogonalize";
    TORCH_CHECK(is_float(G_in.scalar_type()) && G_in.dim() >= 2, "gn_kernels::", op, ": unsupported input (shape ", G_in.sizes(), ", dtype ", G_in.scalar_type(), ")");
    const at::Tensor G = G_in.contiguous();
    const int64_t rows = G.size(-2), cols = G.size(-1);
    int64_t batch = 1;
    for (int64_t d = 0; d < G.dim() - 2; ++d) batch *= G.size(d);
    at::Tensor out = at::empty(G.sizes(), G.options());
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(G.device());
    const int code = dtype_code(G.scalar_type(), op);
    const int64_t nws = gnk_orthogonalize_workspace_bytes_of(code, batch, rows, cols);
    const at::Tensor ws = workspace_for(G, nws);
    check(gnk_orthogonalize(G.data_ptr(), code, out.data_ptr(), code, batch, rows, cols, (int)steps, (float)a, (float)b, (float)c, (float)eps,
                            nws > 0 ? ws.data_ptr() : nullptr, nws, stream_of(G)),
          op);
    return out;
}

}  // namespace

TORCH_LIBRARY_IMPL(gn_kernels, CUDA, m) {
    m.impl("int8_mm", &int8_mm);
    m.impl("scaled_mm", &scaled_mm);
    m.impl("scaled_mm_t", &scaled_mm_t);
    m.impl("tile_scaled_mm", &tile_scaled_mm);
    m.impl("quantize_int8", &quantize_int8);
    m.impl("quantize_int8_rowwise_colmax", &quantize_int8_rowwise_colmax);
    m.impl("quantize_int8_colwise_given", &quantize_int8_colwise_given);
    m.impl("grouped_scaled_mm", &grouped_scaled_mm);
    m.impl("grouped_scaled_mm_depth", &grouped_scaled_mm_depth);
    m.impl("quantize_int8_grouped", &quantize_int8_grouped);
    m.impl("grouped_linear_int8", &grouped_linear_int8);
    m.impl("grouped_linear_int8_backward", &grouped_linear_int8_backward);
    m.impl("orthogonalize", &orthogonalize);
}
