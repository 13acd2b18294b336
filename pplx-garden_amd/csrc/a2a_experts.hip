// Host side of the experts' products: the checks, and what a call hands to the kernels.
#include "a2a_experts.h"

#include <atomic>

#include "a2a_host.h"

namespace a2a {
namespace {

constexpr uint64_t kRowLimit = 1ull << 24;      // bytes from row to row: offsets inside a tile are 32-bit numbers
constexpr uint64_t kWeightLimit = 1ull << 32;   // bytes of an expert's weight, likewise
constexpr uint32_t kRowsLimit = 1u << 25;       // rows of a buffer: 64 experts' counts of so many add up in 32 bits (expert_table)

int refuse(int code, const char *call, const char *what) { return fail_call(code, "%s: %s", call, what); }

bool aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Rows of `columns` entries of `size` bytes.
int check_rows(const char *call, const char *name, const void *p, uint64_t stride, uint64_t columns, uint64_t size) {
    if (p == nullptr) return fail_call(A2A_ERR_INVALID_ARGUMENT, "%s: null %s", call, name);
    if (!aligned(p) || stride % 16 != 0)
        return fail_call(A2A_ERR_UNSUPPORTED, "%s: %s and its row stride (%llu bytes) must be multiples of 16 bytes", call, name,
                         (unsigned long long)stride);
    if (stride < columns * size)
        return fail_call(A2A_ERR_INVALID_ARGUMENT, "%s: the row stride of %s (%llu bytes) is shorter than a row of %llu", call, name,
                         (unsigned long long)stride, (unsigned long long)(columns * size));
    if (stride >= kRowLimit)
        return fail_call(A2A_ERR_UNSUPPORTED, "%s: the row stride of %s is %llu bytes, must be below %llu", call, name,
                         (unsigned long long)stride, (unsigned long long)kRowLimit);
    return A2A_OK;
}

int check_weight(const char *call, const char *name, const void *p, uint64_t stride, uint64_t expert_stride, uint64_t experts,
                 uint64_t rows, uint64_t k, uint64_t size) {
    if (int rc = check_rows(call, name, p, stride, k, size)) return rc;
    if (expert_stride % 16 != 0)
        return fail_call(A2A_ERR_UNSUPPORTED, "%s: the stride from expert to expert of %s must be a multiple of 16 bytes", call, name);
    if (rows * stride >= kWeightLimit)
        return fail_call(A2A_ERR_UNSUPPORTED, "%s: an expert's %s spans %llu bytes, must be below 4 GiB", call, name,
                         (unsigned long long)(rows * stride));
    if (experts > 1 && expert_stride < (rows - 1) * stride + k * size)
        return fail_call(A2A_ERR_INVALID_ARGUMENT, "%s: the experts' %s overlap", call, name);
    return A2A_OK;
}

int check_sizes(const char *call, uint32_t experts, uint32_t padding, uint32_t rows, uint32_t n, uint32_t k, uint32_t n_step,
                uint32_t size, const int32_t *num_tokens) {
    if (experts == 0 || experts > A2A_MAX_EXPERTS)
        return fail_call(A2A_ERR_UNSUPPORTED, "%s: num_experts %u not in [1, %d]", call, experts, A2A_MAX_EXPERTS);
    if (padding == 0 || padding > 0x7FFFFFFFu)
        return fail_call(A2A_ERR_INVALID_ARGUMENT, "%s: expert_padding %u not in [1, 2^31)", call, padding);
    if (rows >= kRowsLimit) return fail_call(A2A_ERR_UNSUPPORTED, "%s: too many rows (%u, fewer than %u are supported)", call, rows, kRowsLimit);
    if (num_tokens == nullptr && experts != 1)
        return refuse(A2A_ERR_INVALID_ARGUMENT, call, "without num_tokens there is one expert that has all rows");
    if (n == 0 || n % n_step != 0 || n > 0x3FFFFFFFu)
        return fail_call(A2A_ERR_UNSUPPORTED, "%s: n %u is not a positive multiple of %u", call, n, n_step);
    if (k == 0 || (uint64_t)k * size % 16 != 0)
        return fail_call(A2A_ERR_UNSUPPORTED, "%s: k %u: a row must be a multiple of 16 bytes", call, k);
    return A2A_OK;
}

// Compute units of a device, asked for once.
int units_of(const char *call, int device, uint32_t *units) {
    constexpr int kDevices = 64;
    static std::atomic<uint32_t> known[kDevices];
    if (device < 0 || device >= kDevices) return fail_call(A2A_ERR_INVALID_ARGUMENT, "%s: device %d not in [0, %d)", call, device, kDevices);
    *units = known[device].load(std::memory_order_relaxed);
    if (*units != 0) return A2A_OK;
    int count = 0;
    const hipError_t e = hipDeviceGetAttribute(&count, hipDeviceAttributeMultiprocessorCount, device);
    if (e != hipSuccess) return fail_call((int)e, "%s: hipDeviceGetAttribute: %s", call, hipGetErrorString(e));
    if (count <= 0) return fail_call(A2A_ERR_UNSUPPORTED, "%s: device %d has %d compute units", call, device, count);
    known[device].store((uint32_t)count, std::memory_order_relaxed);
    *units = (uint32_t)count;
    return A2A_OK;
}

int launched(const char *call, hipError_t e) {
    return e == hipSuccess ? A2A_OK : fail_call((int)e, "%s: launch: %s", call, hipGetErrorString(e));
}

int forward(const char *call, bool gated, const a2a_expert_args *args, void *stream) {
    if (args == nullptr) return refuse(A2A_ERR_INVALID_ARGUMENT, call, "null args");
    const a2a_expert_args &a = *args;
    if (a.struct_size != sizeof(a2a_expert_args))
        return fail_call(A2A_ERR_INVALID_ARGUMENT, "%s: struct_size is %u, expected %zu", call, a.struct_size, sizeof(a2a_expert_args));
    const bool fp8 = a.in_dtype == A2A_F8_E4M3;
    if (!fp8 && a.in_dtype != A2A_BF16 && a.in_dtype != A2A_F16)
        return fail_call(A2A_ERR_UNSUPPORTED, "%s: in_dtype %u: F8_E4M3, BF16 and F16 are supported", call, a.in_dtype);
    const bool out_known = !fp8 ? a.out_dtype == a.in_dtype
                           : gated ? a.out_dtype == A2A_F8_E4M3
                                   : a.out_dtype == A2A_BF16 || a.out_dtype == A2A_F16 || a.out_dtype == A2A_F32;
    if (!out_known) return fail_call(A2A_ERR_UNSUPPORTED, "%s: out_dtype %u with in_dtype %u", call, a.out_dtype, a.in_dtype);
    const uint32_t size = fp8 ? 1 : 2, out_size = a.out_dtype == A2A_F8_E4M3 ? 1 : a.out_dtype == A2A_F32 ? 4 : 2;
    const uint32_t width = gated ? 2 * a.n : a.n;
    if (int rc = check_sizes(call, a.num_experts, a.expert_padding, a.rows, a.n, a.k, fp8 && gated ? 16 : 8, size, a.num_tokens))
        return rc;
    if ((a.x_scale != nullptr) != fp8 || (a.weight_scale != nullptr) != fp8) {
        if (!fp8 || a.rows != 0)
            return refuse(A2A_ERR_INVALID_ARGUMENT, call, "scales of x and of the weights go with fp8, and with nothing else");
    }
    if ((a.out_scale != nullptr) != (fp8 && gated) && (a.rows != 0 || !(fp8 && gated)))
        return refuse(A2A_ERR_INVALID_ARGUMENT, call, "out_scale goes with an fp8 output, and with nothing else");
    if (a.projections != nullptr && (fp8 || !gated))
        return refuse(A2A_ERR_UNSUPPORTED, call, "projections are those of a gated product of bf16 or f16");
    if (a.workspace != nullptr && !aligned(a.workspace)) return refuse(A2A_ERR_UNSUPPORTED, call, "workspace must be a multiple of 16 bytes");
    if (a.rows == 0) return A2A_OK;
    if (int rc = check_rows(call, "x", a.x, a.x_stride, a.k, size)) return rc;
    if (int rc = check_weight(call, "weight", a.weight, a.weight_stride, a.weight_stride_expert, a.num_experts, width, a.k, size))
        return rc;
    if (int rc = check_rows(call, "out", a.out, a.out_stride, a.n, out_size)) return rc;
    if (a.projections != nullptr) {
        if (int rc = check_rows(call, "projections", a.projections, a.projections_stride, width, size)) return rc;
    }
    DeviceGuard guard(a.device);
    if (!guard.ok) return fail_call(A2A_ERR_INVALID_ARGUMENT, "%s: cannot select device %d", call, a.device);
    uint32_t units;
    if (int rc = units_of(call, a.device, &units)) return rc;
    ProductArgs p = {};
    p.left = static_cast<const uint8_t *>(a.x);
    p.left_stride = a.x_stride;
    p.right = static_cast<const uint8_t *>(a.weight);
    p.right_stride = a.weight_stride;
    p.right_expert = a.weight_stride_expert;
    p.out = static_cast<uint8_t *>(a.out);
    p.out_stride = a.out_stride;
    p.projections = static_cast<uint8_t *>(a.projections);
    p.projections_stride = a.projections_stride;
    p.left_scale = a.x_scale;
    p.left_scale_elem = a.x_scale_stride_elem;
    p.left_scale_row = a.x_scale_stride_token;
    p.right_scale = a.weight_scale;
    p.right_scale_expert = a.weight_scale_stride_expert;
    p.right_scale_row = a.weight_scale_stride_row;
    p.right_scale_elem = a.weight_scale_stride_elem;
    p.out_scale = a.out_scale;
    p.out_scale_elem = a.out_scale_stride_elem;
    p.out_scale_row = a.out_scale_stride_token;
    p.num_tokens = a.num_tokens;
    p.experts = a.num_experts;
    p.padding = a.expert_padding;
    p.rows = a.rows;
    p.n = a.n;
    p.k = a.k;
    p.out_type = a.out_dtype;
    const uint32_t expected = a.rows_per_expert != 0 ? a.rows_per_expert : (a.rows - 1) / a.num_experts + 1;
    const int type = fp8 ? kFp8 : a.in_dtype == A2A_BF16 ? kBf16 : kF16;
    const int end = !gated ? kPlain : fp8 ? kGatedFp8 : kGated;
    return launched(call, launch_forward(type, end, p, expected, units, static_cast<float *>(a.workspace),
                                        a.workspace_bytes, static_cast<hipStream_t>(stream)));
}

int gradient(const char *call, bool gated, const a2a_expert_grad_args *args, void *stream) {
    if (args == nullptr) return refuse(A2A_ERR_INVALID_ARGUMENT, call, "null args");
    const a2a_expert_grad_args &a = *args;
    if (a.struct_size != sizeof(a2a_expert_grad_args))
        return fail_call(A2A_ERR_INVALID_ARGUMENT, "%s: struct_size is %u, expected %zu", call, a.struct_size,
                         sizeof(a2a_expert_grad_args));
    if (a.dtype != A2A_BF16 && a.dtype != A2A_F16)
        return fail_call(A2A_ERR_UNSUPPORTED, "%s: dtype %u: BF16 and F16 are supported", call, a.dtype);
    const uint32_t width = gated ? 2 * a.n : a.n;
    if (int rc = check_sizes(call, a.num_experts, a.expert_padding, a.rows, a.n, a.k, 8, 2, a.num_tokens)) return rc;
    if (a.grad_weight != nullptr) {
        if (int rc = check_weight(call, "grad_weight", a.grad_weight, a.grad_weight_stride, a.grad_weight_stride_expert, a.num_experts,
                                  width, a.k, 2))
            return rc;
    }
    if (a.rows != 0) {
        if (int rc = check_rows(call, "grad_out", a.grad_out, a.grad_out_stride, a.n, 2)) return rc;
        if (gated) {
            if (int rc = check_rows(call, "projections", a.projections, a.projections_stride, width, 2)) return rc;
            if (int rc = check_rows(call, "grad_projections", a.grad_projections, a.grad_projections_stride, width, 2)) return rc;
        }
        if (a.grad_x != nullptr) {
            if (int rc = check_rows(call, "grad_x", a.grad_x, a.grad_x_stride, a.k, 2)) return rc;
            if (int rc = check_weight(call, "weight", a.weight, a.weight_stride, a.weight_stride_expert, a.num_experts, width, a.k, 2))
                return rc;
        }
        if (a.grad_weight != nullptr) {
            if (int rc = check_rows(call, "x", a.x, a.x_stride, a.k, 2)) return rc;
        }
    }
    DeviceGuard guard(a.device);
    if (!guard.ok) return fail_call(A2A_ERR_INVALID_ARGUMENT, "%s: cannot select device %d", call, a.device);
    uint32_t units;
    if (int rc = units_of(call, a.device, &units)) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int type = a.dtype == A2A_BF16 ? kBf16 : kF16;
    ProductArgs p = {};
    p.num_tokens = a.num_tokens;
    p.experts = a.num_experts;
    p.padding = a.expert_padding;
    p.rows = a.rows;
    p.out_type = a.dtype;
    const uint32_t expected = a.rows != 0 ? (a.rows - 1) / a.num_experts + 1 : 0;
    p.left = static_cast<const uint8_t *>(gated ? a.grad_projections : a.grad_out);
    p.left_stride = gated ? a.grad_projections_stride : a.grad_out_stride;
    if (gated && a.rows != 0) {
        GateGradientArgs g = {};
        g.grad_out = static_cast<const uint8_t *>(a.grad_out);
        g.projections = static_cast<const uint8_t *>(a.projections);
        g.grad_projections = static_cast<uint8_t *>(a.grad_projections);
        g.grad_out_stride = a.grad_out_stride;
        g.projections_stride = a.projections_stride;
        g.grad_projections_stride = a.grad_projections_stride;
        g.num_tokens = a.num_tokens;
        g.experts = a.num_experts;
        g.padding = a.expert_padding;
        g.rows = a.rows;
        g.n = a.n;
        if (int rc = launched(call, launch_gate_gradient(type, g, units, s))) return rc;
    }
    if (a.grad_x != nullptr && a.rows != 0) {
        p.right = static_cast<const uint8_t *>(a.weight);
        p.right_stride = a.weight_stride;
        p.right_expert = a.weight_stride_expert;
        p.out = static_cast<uint8_t *>(a.grad_x);
        p.out_stride = a.grad_x_stride;
        p.n = a.k;
        p.k = width;
        if (int rc = launched(call, launch_gradient(type, kRowGradient, p, expected, units, s))) return rc;
    }
    if (a.grad_weight != nullptr) {
        p.right = static_cast<const uint8_t *>(a.x);
        p.right_stride = a.x_stride;
        p.right_expert = 0;
        p.out = static_cast<uint8_t *>(a.grad_weight);
        p.out_stride = a.grad_weight_stride;
        p.out_expert = a.grad_weight_stride_expert;
        p.m = width;
        p.n = a.k;
        p.k = 0;
        if (int rc = launched(call, launch_gradient(type, kWeightGradient, p, expected, units, s))) return rc;
    }
    return A2A_OK;
}

}  // namespace
}  // namespace a2a

extern "C" {

int a2a_expert_matmul(const a2a_expert_args *args, void *stream) {
    a2a::ProfilerRange range("expert_matmul");
    return a2a::forward("a2a_expert_matmul", false, args, stream);
}

int a2a_expert_gated(const a2a_expert_args *args, void *stream) {
    a2a::ProfilerRange range("expert_gated");
    return a2a::forward("a2a_expert_gated", true, args, stream);
}

int a2a_expert_matmul_grad(const a2a_expert_grad_args *args, void *stream) {
    a2a::ProfilerRange range("expert_matmul_grad");
    return a2a::gradient("a2a_expert_matmul_grad", false, args, stream);
}

int a2a_expert_gated_grad(const a2a_expert_grad_args *args, void *stream) {
    a2a::ProfilerRange range("expert_gated_grad");
    return a2a::gradient("a2a_expert_gated_grad", true, args, stream);
}

}  // extern "C"
