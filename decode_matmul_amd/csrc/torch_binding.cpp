// PyTorch-ROCm operator over the C ABI of libdmm.so.  Host code only: no device code is
// compiled here, the kernels live in dmm.hip, dmm_ops.hip and the dmm_*.h files they include, behind
// include/dmm.h.
//
// Mirrors the operator boundary of the reference,
// /root/reference/decode_matmul_cuda/decode_matmul_cuda.cu:178-239: one module, a function
// `decode_matmul`, inputs checked with TORCH_CHECK (-> Python RuntimeError), output
// allocated by the op on x's device, launch on the current stream under a DeviceGuard.
// Differences, all deliberate: half precision with a scale (x half, codes 16-bit, grid half
// [256,8], scale float -> half); no shape demands beyond K % 8 == 0; no device
// synchronisation and no exit() on error (a non-zero status becomes an exception); the
// GIL is released around the launch.
#include <torch/extension.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "dmm.h"

namespace {

#define DMM_CHECK_DEVICE(t) TORCH_CHECK((t).is_cuda(), #t " must be a GPU tensor")
#define DMM_CHECK_CONTIGUOUS(t) TORCH_CHECK((t).is_contiguous(), #t " must be contiguous")
#define DMM_CHECK_INPUT(t)       \
    do {                         \
        DMM_CHECK_DEVICE(t);     \
        DMM_CHECK_CONTIGUOUS(t); \
    } while (false)

bool is_code_dtype(const torch::Tensor &t)
{
    return t.scalar_type() == torch::kInt16 || t.scalar_type() == torch::kUInt16;
}

void check_status(int st, const char *what)
{
    TORCH_CHECK(st == DMM_OK, what, " failed: ", dmm_status_string(st), " (status ", st, ")");
}

// allow_cpu: the operator and the decoder also take tensors in host memory (all of them there), which
// go to the library's host route; every other operation is GPU-only
void check_codes_grid(const torch::Tensor &codes, const torch::Tensor &grid, bool allow_cpu = false)
{
    if (allow_cpu && codes.is_cpu()) {
        DMM_CHECK_CONTIGUOUS(codes);
        DMM_CHECK_CONTIGUOUS(grid);
    } else {
        DMM_CHECK_INPUT(codes);
        DMM_CHECK_INPUT(grid);
    }
    TORCH_CHECK(is_code_dtype(codes), "codes must be int16 or uint16");
    TORCH_CHECK(grid.scalar_type() == torch::kHalf, "grid must be float16");
    TORCH_CHECK(codes.dim() == 2, "codes must be [N, K/8]");
    TORCH_CHECK(grid.dim() == 2 && grid.size(0) == 256 && grid.size(1) == 8, "grid must be [256, 8]");
    TORCH_CHECK(codes.device() == grid.device(), "codes and grid must be on the same device");
}

enum class Path { kAuto, kGemv, kGemm, kGeneric };

torch::Tensor run(const torch::Tensor &x, const torch::Tensor &codes, const torch::Tensor &grid,
                  double scale, Path path)
{
    if (x.is_cpu()) {
        DMM_CHECK_CONTIGUOUS(x);
    } else {
        DMM_CHECK_INPUT(x);
    }
    check_codes_grid(codes, grid, true);
    TORCH_CHECK(x.scalar_type() == torch::kHalf, "x must be float16");
    TORCH_CHECK(x.dim() == 2, "x must be [M, K]");
    TORCH_CHECK(x.device() == codes.device(), "x and codes must be on the same device");
    TORCH_CHECK(x.size(-1) == codes.size(-1) * 8, "x.size(-1) must be 8 * codes.size(-1)");

    const int64_t M = x.size(-2);
    const int64_t N = codes.size(-2);
    const int64_t K = x.size(-1);

    if (x.is_cpu()) {
        // tensors in host memory: the library's host route (the reference's CPU path,
        // test_decode_matmul.py:58-71, in the half-precision form); no GPU call is made
        TORCH_CHECK(path == Path::kAuto, "the named kernel paths are GPU paths; CPU tensors take path 'auto'");
        torch::Tensor y = torch::empty({M, N}, x.options().requires_grad(false));
        int st;
        {
            pybind11::gil_scoped_release nogil;
            st = dmm_decode_matmul_host_f16(x.data_ptr(), codes.data_ptr(), grid.data_ptr(), static_cast<float>(scale),
                                            y.data_ptr(), M, N, K);
        }
        check_status(st, "decode_matmul (host)");
        return y;
    }

    c10::DeviceGuard guard(x.device());
    torch::Tensor y = torch::empty({M, N}, x.options().requires_grad(false));
    hipStream_t stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
    // split-K workspace for short x, from torch's caching allocator: stream-ordered, so calls
    // on different streams never share one
    torch::Tensor workspace;
    const int64_t ws_bytes = path == Path::kAuto ? dmm_workspace_bytes(M, N, K) : 0;
    if (ws_bytes > 0) workspace = torch::empty({ws_bytes}, x.options().dtype(torch::kUInt8).requires_grad(false));

    int st;
    {
        pybind11::gil_scoped_release nogil;
        const void *xp = x.data_ptr(), *cp = codes.data_ptr(), *gp = grid.data_ptr();
        void *yp = y.data_ptr();
        const float sc = static_cast<float>(scale);
        switch (path) {
            case Path::kGemv: st = dmm_gemv_f16(xp, cp, gp, sc, yp, M, N, K, stream); break;
            case Path::kGemm: st = dmm_gemm_f16(xp, cp, gp, sc, yp, M, N, K, stream); break;
            case Path::kGeneric: st = dmm_generic_f16(xp, cp, gp, sc, yp, M, N, K, stream); break;
            default:
                st = dmm_decode_matmul_ws_f16(xp, cp, gp, sc, yp, M, N, K, ws_bytes > 0 ? workspace.data_ptr() : nullptr,
                                              ws_bytes, stream);
                break;
        }
    }
    check_status(st, "decode_matmul");
    return y;
}

torch::Tensor decode_matmul(torch::Tensor x, torch::Tensor codes, torch::Tensor grid, double scale)
{
    return run(x, codes, grid, scale, Path::kAuto);
}

torch::Tensor decode_matmul_path(torch::Tensor x, torch::Tensor codes, torch::Tensor grid, double scale,
                                 const std::string &path)
{
    Path p;
    if (path == "auto") p = Path::kAuto;
    else if (path == "gemv") p = Path::kGemv;
    else if (path == "gemm") p = Path::kGemm;
    else if (path == "generic") p = Path::kGeneric;
    else TORCH_CHECK(false, "unknown path '", path, "' (auto, gemv, gemm, generic)");
    return run(x, codes, grid, scale, p);
}

torch::Tensor decode(torch::Tensor codes, torch::Tensor grid)
{
    check_codes_grid(codes, grid, true);
    const int64_t N = codes.size(0);
    const int64_t K = codes.size(1) * 8;
    if (codes.is_cpu()) {   // host memory: the library's host decoder, no GPU call
        torch::Tensor W = torch::empty({N, K}, grid.options().requires_grad(false));
        int st;
        {
            pybind11::gil_scoped_release nogil;
            st = dmm_decode_host_f16(codes.data_ptr(), grid.data_ptr(), W.data_ptr(), N, K);
        }
        check_status(st, "decode (host)");
        return W;
    }
    c10::DeviceGuard guard(codes.device());
    torch::Tensor W = torch::empty({N, K}, grid.options().requires_grad(false));
    hipStream_t stream = c10::hip::getCurrentHIPStream(codes.device().index()).stream();
    int st;
    {
        pybind11::gil_scoped_release nogil;
        st = dmm_decode_f16(codes.data_ptr(), grid.data_ptr(), W.data_ptr(), N, K, stream);
    }
    check_status(st, "decode");
    return W;
}

// Offline repack for the batch-1 kernel: codes [N, K/8] -> packed [ceil(N/16)*16, K/8] (same
// dtype; rows past N are zero padding), and the operator on packed codes.
torch::Tensor pack_codes(torch::Tensor codes)
{
    DMM_CHECK_INPUT(codes);
    TORCH_CHECK(is_code_dtype(codes) && codes.dim() == 2, "codes must be int16 or uint16 [N, K/8]");
    const int64_t N = codes.size(0), K = codes.size(1) * 8;
    TORCH_CHECK(K >= 256 && K % 256 == 0, "packing needs K % 256 == 0");
    c10::DeviceGuard guard(codes.device());
    torch::Tensor packed = torch::empty({(N + 15) / 16 * 16, K / 8}, codes.options().requires_grad(false));
    hipStream_t stream = c10::hip::getCurrentHIPStream(codes.device().index()).stream();
    int st;
    {
        pybind11::gil_scoped_release nogil;
        st = dmm_pack_codes(codes.data_ptr(), packed.data_ptr(), N, K, stream);
    }
    check_status(st, "pack_codes");
    return packed;
}

torch::Tensor decode_matmul_packed(torch::Tensor x, torch::Tensor packed, torch::Tensor grid, double scale, int64_t N)
{
    DMM_CHECK_INPUT(x);
    check_codes_grid(packed, grid);
    TORCH_CHECK(x.scalar_type() == torch::kHalf && x.dim() == 2, "x must be float16 [M, K]");
    TORCH_CHECK(x.device() == packed.device(), "x and packed must be on the same device");
    TORCH_CHECK(x.size(-1) == packed.size(-1) * 8, "x.size(-1) must be 8 * packed.size(-1)");
    TORCH_CHECK(N >= 0 && packed.size(0) == (N + 15) / 16 * 16, "packed must have ceil(N / 16) * 16 rows");
    const int64_t M = x.size(0), K = x.size(1);
    c10::DeviceGuard guard(x.device());
    torch::Tensor y = torch::empty({M, N}, x.options().requires_grad(false));
    hipStream_t stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
    torch::Tensor workspace;
    const int64_t ws_bytes = dmm_workspace_bytes(M, N, K);
    if (ws_bytes > 0) workspace = torch::empty({ws_bytes}, x.options().dtype(torch::kUInt8).requires_grad(false));
    int st;
    {
        pybind11::gil_scoped_release nogil;
        st = dmm_decode_matmul_packed_f16(x.data_ptr(), packed.data_ptr(), grid.data_ptr(), static_cast<float>(scale),
                                          y.data_ptr(), M, N, K, ws_bytes > 0 ? workspace.data_ptr() : nullptr,
                                          ws_bytes, stream);
    }
    check_status(st, "decode_matmul_packed");
    return y;
}

// The reference's own signature: int8 x, int16 codes (tiled like its kernel reads them, or
// row-major), int64[256] table -> int32 (decode_matmul_cuda.cu:178-234).
torch::Tensor decode_matmul_int8(torch::Tensor x, torch::Tensor weights_compressed, torch::Tensor codebook_abs,
                                 bool tiled)
{
    DMM_CHECK_INPUT(x);
    DMM_CHECK_INPUT(weights_compressed);
    DMM_CHECK_INPUT(codebook_abs);
    TORCH_CHECK(x.scalar_type() == torch::kInt8, "x must be int8");
    TORCH_CHECK(is_code_dtype(weights_compressed), "weights_compressed must be int16 or uint16");
    TORCH_CHECK(codebook_abs.scalar_type() == torch::kInt64 && codebook_abs.numel() == 256,
                "codebook_abs must be int64[256]");
    TORCH_CHECK(x.dim() == 2 && weights_compressed.dim() == 2, "x must be [M, K], weights_compressed [N, K/8]");
    TORCH_CHECK(x.size(-1) == weights_compressed.size(-1) << 3, "x.size(-1) must be 8 * weights_compressed.size(-1)");
    TORCH_CHECK(x.device() == weights_compressed.device() && x.device() == codebook_abs.device(),
                "all tensors must be on the same device");
    const int64_t M = x.size(-2), N = weights_compressed.size(-2), K = x.size(-1);
    c10::DeviceGuard guard(x.device());
    torch::Tensor out = torch::empty({M, N}, x.options().dtype(torch::kInt32).requires_grad(false));
    hipStream_t stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
    int st;
    {
        pybind11::gil_scoped_release nogil;
        st = dmm_decode_matmul_i8(x.data_ptr(), weights_compressed.data_ptr(), codebook_abs.data_ptr(),
                                  out.data_ptr(), M, N, K, tiled ? 1 : 0, stream);
    }
    check_status(st, "decode_matmul_int8");
    return out;
}

// ------------------------------------------------------------------ the operators around the product
// All tensors of a call are on one device: a GPU, or the host, whose tensors take the library's host
// route.  The weights are frozen codes and no operator here has a gradient: an input that asks for one is refused.
typedef c10::optional<torch::Tensor> MaybeTensor;

#define DMM_CHECK_SAME_DEVICE(t, dev) TORCH_CHECK((t).device() == (dev), #t " must be on ", (dev), " like x")

// A gradient is asked for by requires_grad, or forward in a tangent beside the value (which lives under no_grad too).
void check_no_grad(const torch::Tensor &t, const char *what, const char *name)
{
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), what, ": ", name,
                " requires a gradient, which this operator does not compute; call it under torch.no_grad() or detach the input");
    TORCH_CHECK(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined()), what, ": ", name,
                " carries a tangent of forward-mode differentiation, a gradient which this operator does not compute; unpack or detach the input");
}

void check_device(const torch::Device &d, const char *what)
{
    TORCH_CHECK(d.is_cuda() || d.is_cpu(), what, ": tensors must be on a GPU or on the host");
}

int float_type(const torch::Tensor &t, const char *name)
{
    if (t.scalar_type() == torch::kHalf) return DMM_F16;
    TORCH_CHECK(t.scalar_type() == torch::kFloat, name, " must be float16 or float32");
    return DMM_F32;
}

int out_type_of(torch::ScalarType t)
{
    TORCH_CHECK(t == torch::kHalf || t == torch::kFloat, "out_dtype must be float16 or float32");
    return t == torch::kHalf ? DMM_F16 : DMM_F32;
}

int activation_of(const std::string &name)
{
    if (name == "none") return DMM_ACT_NONE;
    if (name == "relu") return DMM_ACT_RELU;
    if (name == "silu") return DMM_ACT_SILU;
    if (name == "gelu") return DMM_ACT_GELU;
    if (name == "gelu_tanh") return DMM_ACT_GELU_TANH;
    TORCH_CHECK(false, "unknown activation '", name, "' (none, relu, silu, gelu, gelu_tanh)");
}

hipStream_t stream_of(const torch::Device &d)
{
    return d.is_cuda() ? c10::hip::getCurrentHIPStream(d.index()).stream() : nullptr;
}

// the code matrix (or matrices) and the grid, on x's device
void check_weights(const torch::Tensor &x, const torch::Tensor &codes, const torch::Tensor &grid, int64_t dim, const char *what)
{
    check_device(x.device(), what);
    DMM_CHECK_CONTIGUOUS(x);
    DMM_CHECK_CONTIGUOUS(codes);
    DMM_CHECK_CONTIGUOUS(grid);
    DMM_CHECK_SAME_DEVICE(codes, x.device());
    DMM_CHECK_SAME_DEVICE(grid, x.device());
    TORCH_CHECK(x.scalar_type() == torch::kHalf, "x must be float16");
    TORCH_CHECK(x.dim() == 2, "x must be [rows, K]");
    TORCH_CHECK(is_code_dtype(codes), "codes must be int16 or uint16");
    TORCH_CHECK(codes.dim() == dim, dim == 2 ? "codes must be [N, K/8]" : "codes must be [E, N, K/8]");
    TORCH_CHECK(grid.scalar_type() == torch::kHalf && grid.dim() == 2 && grid.size(0) == 256 && grid.size(1) == 8,
                "grid must be float16 [256, 8]");
    TORCH_CHECK(x.size(1) == codes.size(-1) * 8, "x.size(-1) must be 8 * codes.size(-1)");
    check_no_grad(x, what, "x");
    check_no_grad(grid, what, "grid");
}

torch::Tensor decode_matmul_fused(torch::Tensor x, torch::Tensor codes, torch::Tensor grid, double scale, double scale_up,
                                  MaybeTensor bias, const std::string &activation, bool gated, MaybeTensor residual,
                                  torch::ScalarType out_dtype)
{
    check_weights(x, codes, grid, 2, "decode_matmul_fused");
    const int64_t M = x.size(0), K = x.size(1), rows = codes.size(0);
    TORCH_CHECK(!gated || rows % 2 == 0, "a gated call needs the gate's rows and as many up rows in codes");
    const int64_t N = gated ? rows / 2 : rows;
    dmm_epilogue ep{};
    ep.activation = activation_of(activation);
    ep.gated = gated;
    ep.scale = static_cast<float>(scale);
    ep.scale_up = static_cast<float>(scale_up);
    ep.out_type = out_type_of(out_dtype);
    if (bias) {
        DMM_CHECK_SAME_DEVICE(*bias, x.device());
        DMM_CHECK_CONTIGUOUS(*bias);
        TORCH_CHECK(bias->dim() == 1 && bias->size(0) == rows, "bias must have one value per row of codes");
        check_no_grad(*bias, "decode_matmul_fused", "bias");
        ep.bias_type = float_type(*bias, "bias");
        ep.bias = bias->data_ptr();
    }
    if (residual) {
        DMM_CHECK_SAME_DEVICE(*residual, x.device());
        DMM_CHECK_CONTIGUOUS(*residual);
        TORCH_CHECK(residual->dim() == 2 && residual->size(0) == M && residual->size(1) == N, "residual must be [M, N]");
        check_no_grad(*residual, "decode_matmul_fused", "residual");
        ep.residual_type = float_type(*residual, "residual");
        ep.residual = residual->data_ptr();
    }
    c10::OptionalDeviceGuard guard;
    if (x.is_cuda()) guard.reset_device(x.device());
    torch::Tensor y = torch::empty({M, N}, x.options().dtype(out_dtype).requires_grad(false));
    torch::Tensor workspace;
    const int64_t ws_bytes = x.is_cuda() ? dmm_fused_workspace_bytes(M, N, K, gated) : 0;
    if (ws_bytes > 0) workspace = torch::empty({ws_bytes}, x.options().dtype(torch::kUInt8).requires_grad(false));
    hipStream_t stream = stream_of(x.device());
    int st;
    {
        pybind11::gil_scoped_release nogil;
        st = x.is_cpu() ? dmm_decode_matmul_fused_host(x.data_ptr(), codes.data_ptr(), grid.data_ptr(), &ep, y.data_ptr(), M, N, K)
                        : dmm_decode_matmul_fused(x.data_ptr(), codes.data_ptr(), grid.data_ptr(), &ep, y.data_ptr(), M, N, K,
                                                  ws_bytes > 0 ? workspace.data_ptr() : nullptr, ws_bytes, stream);
    }
    check_status(st, "decode_matmul_fused");
    return y;
}

bool share_memory(const torch::Tensor &a, const torch::Tensor &b)   // both contiguous
{
    const char *pa = static_cast<const char *>(a.data_ptr()), *pb = static_cast<const char *>(b.data_ptr());
    return a.nbytes() > 0 && b.nbytes() > 0 && pa < pb + b.nbytes() && pb < pa + a.nbytes();
}

torch::Tensor decode_matmul_grouped(torch::Tensor x, torch::Tensor codes, torch::Tensor grid, double scale, double scale_up,
                                    MaybeTensor scales, torch::Tensor offsets, MaybeTensor rows, MaybeTensor bias, const std::string &activation,
                                    bool gated, torch::ScalarType out_dtype, MaybeTensor out)
{
    check_weights(x, codes, grid, 3, "decode_matmul_grouped");
    const int64_t T = x.size(0), K = x.size(1), E = codes.size(0), wrows = codes.size(1);
    TORCH_CHECK(!gated || wrows % 2 == 0, "a gated call needs the gate's rows and as many up rows in codes");
    const int64_t N = gated ? wrows / 2 : wrows;
    DMM_CHECK_SAME_DEVICE(offsets, x.device());
    DMM_CHECK_CONTIGUOUS(offsets);
    TORCH_CHECK(offsets.scalar_type() == torch::kInt32 && offsets.dim() == 1 && offsets.size(0) == E + 1,
                "offsets must be int32 with one more entry than codes has experts");
    int64_t R = T;
    if (rows) {
        DMM_CHECK_SAME_DEVICE(*rows, x.device());
        DMM_CHECK_CONTIGUOUS(*rows);
        TORCH_CHECK(rows->scalar_type() == torch::kInt32 && rows->dim() == 1, "rows must be int32 [R]");
        R = rows->size(0);
    }
    dmm_epilogue ep{};
    ep.activation = activation_of(activation);
    ep.gated = gated;
    ep.scale = static_cast<float>(scale);
    ep.scale_up = static_cast<float>(scale_up);
    ep.out_type = out_type_of(out_dtype);
    int scale_cols = 1;
    if (scales) {
        DMM_CHECK_SAME_DEVICE(*scales, x.device());
        DMM_CHECK_CONTIGUOUS(*scales);
        TORCH_CHECK(scales->scalar_type() == torch::kFloat &&
                        (scales->dim() == 1 || (gated && scales->dim() == 2 && scales->size(1) == 2)) && scales->size(0) == E,
                    "scale must be a number, float32 [E], or for a gated call a pair of numbers or float32 [E, 2]");
        check_no_grad(*scales, "decode_matmul_grouped", "scale");
        scale_cols = static_cast<int>(scales->dim());
    }
    if (bias) {
        DMM_CHECK_SAME_DEVICE(*bias, x.device());
        DMM_CHECK_CONTIGUOUS(*bias);
        TORCH_CHECK(bias->dim() == 2 && bias->size(0) == E && bias->size(1) == wrows, "bias must have one value per row of codes");
        check_no_grad(*bias, "decode_matmul_grouped", "bias");
        ep.bias_type = float_type(*bias, "bias");
        ep.bias = bias->data_ptr();
    }
    c10::OptionalDeviceGuard guard;
    if (x.is_cuda()) guard.reset_device(x.device());
    torch::Tensor y;
    if (out) {
        DMM_CHECK_SAME_DEVICE(*out, x.device());
        DMM_CHECK_CONTIGUOUS(*out);
        TORCH_CHECK(out->dim() == 2 && out->size(0) == R && out->size(1) == N && out->scalar_type() == out_dtype,
                    "out must be [R, N] of out_dtype");
        check_no_grad(*out, "decode_matmul_grouped", "out");
        for (const torch::Tensor *t : {&x, &codes, &grid, &offsets, rows ? &*rows : nullptr, scales ? &*scales : nullptr, bias ? &*bias : nullptr})
            TORCH_CHECK(!t || !share_memory(*out, *t), "out must not share memory with an input");
        y = *out;
    } else {
        y = torch::empty({R, N}, x.options().dtype(out_dtype).requires_grad(false));
    }
    hipStream_t stream = stream_of(x.device());
    const void *rp = rows ? rows->data_ptr() : nullptr, *sp = scales ? scales->data_ptr() : nullptr;
    int st;
    {
        pybind11::gil_scoped_release nogil;
        st = x.is_cpu() ? dmm_decode_matmul_grouped_host(x.data_ptr(), T, rp, codes.data_ptr(), grid.data_ptr(), sp, scale_cols,
                                                         offsets.data_ptr(), &ep, y.data_ptr(), R, E, N, K)
                        : dmm_decode_matmul_grouped(x.data_ptr(), T, rp, codes.data_ptr(), grid.data_ptr(), sp, scale_cols,
                                                    offsets.data_ptr(), &ep, y.data_ptr(), R, E, N, K, stream);
    }
    check_status(st, "decode_matmul_grouped");
    // what autograd may have saved of `out` has changed
    if (out && !y.is_inference()) y.unsafeGetTensorImpl()->bump_version();
    return y;
}

// A contiguous tensor over a part of buf's memory, from byte `at` on; at moves past it, to the next multiple of 16.
// (Five small results: one allocation and five of these cost the host a third of five allocations.)
torch::Tensor carve(const torch::Tensor &buf, torch::ScalarType type, c10::IntArrayRef sizes, int64_t &at)
{
    torch::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    const int64_t item = static_cast<int64_t>(c10::elementSize(type));
    t.unsafeGetTensorImpl()->set_storage_offset(at / item);
    at = (at + t.numel() * item + 15) / 16 * 16;
    return t;
}

std::vector<torch::Tensor> route_experts(torch::Tensor logits, int64_t k, const std::string &scoring, bool normalize)
{
    check_device(logits.device(), "route_experts");
    DMM_CHECK_CONTIGUOUS(logits);
    TORCH_CHECK(logits.dim() == 2, "logits must be [T, E]");
    TORCH_CHECK(scoring == "softmax" || scoring == "sigmoid", "unknown scoring '", scoring, "' (softmax, sigmoid)");
    check_no_grad(logits, "route_experts", "logits");
    const int type = logits.scalar_type() == torch::kBFloat16 ? DMM_BF16 : float_type(logits, "logits must be bfloat16, or");
    const int64_t T = logits.size(0), E = logits.size(1);
    TORCH_CHECK(k >= 1 && k <= E && k <= 64 && E <= 1024, "k must be between 1 and min(E, 64), and E at most 1024");
    TORCH_CHECK(T <= 1 << 24 && T * k <= INT32_MAX, "at most 2^24 tokens per call");
    const int sc = scoring == "sigmoid" ? DMM_SCORE_SIGMOID : DMM_SCORE_SOFTMAX;
    c10::OptionalDeviceGuard guard;
    if (logits.is_cuda()) guard.reset_device(logits.device());
    const int64_t ws_bytes = logits.is_cuda() ? dmm_route_workspace_bytes(T, E) : 0;
    torch::Tensor buf = torch::empty({16 * T * k + 4 * (E + 1) + 5 * 16 + ws_bytes}, logits.options().dtype(torch::kUInt8).requires_grad(false));
    int64_t at = 0;
    torch::Tensor weights = carve(buf, torch::kFloat, {T, k}, at), experts = carve(buf, torch::kInt32, {T, k}, at),
                  offsets = carve(buf, torch::kInt32, {E + 1}, at), rows = carve(buf, torch::kInt32, {T * k}, at),
                  slots = carve(buf, torch::kInt32, {T, k}, at);
    void *workspace = static_cast<char *>(buf.data_ptr()) + at;   // behind the results
    hipStream_t stream = stream_of(logits.device());
    int st;
    {
        pybind11::gil_scoped_release nogil;
        st = logits.is_cpu() ? dmm_route_experts_host(logits.data_ptr(), type, T, E, k, sc, normalize, weights.data_ptr(),
                                                      experts.data_ptr(), offsets.data_ptr(), rows.data_ptr(), slots.data_ptr())
                             : dmm_route_experts(logits.data_ptr(), type, T, E, k, sc, normalize, weights.data_ptr(), experts.data_ptr(),
                                                 offsets.data_ptr(), rows.data_ptr(), slots.data_ptr(),
                                                 ws_bytes > 0 ? workspace : nullptr, ws_bytes, stream);
    }
    check_status(st, "route_experts");
    return {weights, experts, offsets, rows, slots};
}

torch::Tensor combine_experts(torch::Tensor y, torch::Tensor slots, torch::Tensor weights, MaybeTensor residual,
                              torch::ScalarType out_dtype)
{
    check_device(y.device(), "combine_experts");
    DMM_CHECK_CONTIGUOUS(y);
    DMM_CHECK_CONTIGUOUS(slots);
    DMM_CHECK_CONTIGUOUS(weights);
    TORCH_CHECK(slots.device() == y.device() && weights.device() == y.device(), "y, slots and weights must be on the same device");
    TORCH_CHECK(y.dim() == 2, "y must be [R, N]");
    TORCH_CHECK(slots.scalar_type() == torch::kInt32 && slots.dim() == 2, "slots must be int32 [T, k]");
    TORCH_CHECK(weights.scalar_type() == torch::kFloat && weights.sizes() == slots.sizes(), "weights must be float32 [T, k]");
    check_no_grad(y, "combine_experts", "y");
    check_no_grad(weights, "combine_experts", "weights");
    const int y_type = float_type(y, "y"), out_type = out_type_of(out_dtype);
    const int64_t R = y.size(0), N = y.size(1), T = slots.size(0), k = slots.size(1);
    const void *rp = nullptr;
    int r_type = DMM_F16;
    if (residual) {
        TORCH_CHECK(residual->device() == y.device(), "residual must be on the same device as y");
        DMM_CHECK_CONTIGUOUS(*residual);
        TORCH_CHECK(residual->dim() == 2 && residual->size(0) == T && residual->size(1) == N, "residual must be [T, N]");
        check_no_grad(*residual, "combine_experts", "residual");
        r_type = float_type(*residual, "residual");
        rp = residual->data_ptr();
    }
    c10::OptionalDeviceGuard guard;
    if (y.is_cuda()) guard.reset_device(y.device());
    torch::Tensor out = torch::empty({T, N}, y.options().dtype(out_dtype).requires_grad(false));
    hipStream_t stream = stream_of(y.device());
    int st;
    {
        pybind11::gil_scoped_release nogil;
        st = y.is_cpu() ? dmm_combine_experts_host(y.data_ptr(), y_type, slots.data_ptr(), weights.data_ptr(), rp, r_type, out.data_ptr(),
                                                   out_type, R, T, k, N)
                        : dmm_combine_experts(y.data_ptr(), y_type, slots.data_ptr(), weights.data_ptr(), rp, r_type, out.data_ptr(),
                                              out_type, R, T, k, N, stream);
    }
    check_status(st, "combine_experts");
    return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("decode_matmul", &decode_matmul, "Fused decode + matrix multiplication (half precision)",
          pybind11::arg("x"), pybind11::arg("codes"), pybind11::arg("grid"), pybind11::arg("scale"));
    m.def("decode_matmul_path", &decode_matmul_path, "decode_matmul through one named kernel path",
          pybind11::arg("x"), pybind11::arg("codes"), pybind11::arg("grid"), pybind11::arg("scale"),
          pybind11::arg("path"));
    m.def("decode_matmul_int8", &decode_matmul_int8,
          "The reference's integer operator: int8 x, int16 codes, int64[256] table -> int32",
          pybind11::arg("x"), pybind11::arg("weights_compressed"), pybind11::arg("codebook_abs"),
          pybind11::arg("tiled") = true);
    m.def("pack_codes", &pack_codes, "codes [N, K/8] -> the batch-1 kernel's packed layout", pybind11::arg("codes"));
    m.def("decode_matmul_packed", &decode_matmul_packed, "decode_matmul on packed codes (K % 256 == 0)",
          pybind11::arg("x"), pybind11::arg("packed"), pybind11::arg("grid"), pybind11::arg("scale"), pybind11::arg("N"));
    m.def("decode", &decode, "Decode codes [N, K/8] to the dense half matrix [N, K]",
          pybind11::arg("codes"), pybind11::arg("grid"));
    m.def("check_no_grad", [](const torch::Tensor &t, const std::string &what, const std::string &name) { check_no_grad(t, what.c_str(), name.c_str()); },
          "RuntimeError if t asks for a gradient", pybind11::arg("t"), pybind11::arg("what"), pybind11::arg("name"));
    m.def("decode_matmul_fused", &decode_matmul_fused, "decode_matmul with bias, activation, gate and residual in its epilogue",
          pybind11::arg("x"), pybind11::arg("codes"), pybind11::arg("grid"), pybind11::arg("scale"), pybind11::arg("scale_up"),
          pybind11::arg("bias"), pybind11::arg("activation"), pybind11::arg("gated"), pybind11::arg("residual"),
          pybind11::arg("out_dtype"));
    m.def("decode_matmul_grouped", &decode_matmul_grouped, "decode_matmul_fused per expert, rows grouped by expert",
          pybind11::arg("x"), pybind11::arg("codes"), pybind11::arg("grid"), pybind11::arg("scale"), pybind11::arg("scale_up"), pybind11::arg("scales"),
          pybind11::arg("offsets"), pybind11::arg("rows"), pybind11::arg("bias"), pybind11::arg("activation"), pybind11::arg("gated"),
          pybind11::arg("out_dtype"), pybind11::arg("out"));
    m.def("route_experts", &route_experts, "The k largest logits per row, their weights, and the rows sorted by expert",
          pybind11::arg("logits"), pybind11::arg("k"), pybind11::arg("scoring"), pybind11::arg("normalize"));
    m.def("combine_experts", &combine_experts, "Weighted sum of the experts' rows", pybind11::arg("y"), pybind11::arg("slots"),
          pybind11::arg("weights"), pybind11::arg("residual"), pybind11::arg("out_dtype"));
}
