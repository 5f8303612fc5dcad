// token_api.cu — the token-row entry points of include/fenix_b200.h: argument checks, the device of the
// call's pointers, the launch. Every check of sizes, types and nulls comes before the first CUDA call, so
// refusals answer the same on a machine without a GPU.
#include "fenix_b200.h"
#include "token.cuh"
#include "w4.cuh"

#include <cuda_runtime.h>

#include <atomic>
#include <initializer_list>
#include <string>

namespace fxh {
fx_status abi_error(int code, const std::string& msg);
fx_status abi_exception();
}  // namespace fxh

namespace fxk {

int sm_count() {
    static std::atomic<int> count[64];
    int dev = 0;
    cudaGetDevice(&dev);
    int c = dev < 64 ? count[dev].load(std::memory_order_relaxed) : 0;
    if (!c) {
        cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev);
        if (dev < 64) count[dev].store(c, std::memory_order_relaxed);
    }
    return c;
}

}  // namespace fxk

namespace {

constexpr int64_t kMaxExtent = int64_t{1} << 30;  // rows, columns and strides: byte offsets stay below 2^62
constexpr uint64_t kWaitNs = 2000000000;          // limit of a wait inside a 4-bit linear kernel
constexpr int64_t kMaxInner = int64_t{1} << 24;   // k of a 4-bit layer: 32-bit offsets inside 128 of its rows

fx_status bad(const char* fn, const char* what) {
    return fxh::abi_error(FX_INVALID_ARGUMENT, std::string(fn) + ": " + what);
}

bool is_float(int t) { return t == FX_F32 || t == FX_F16 || t == FX_BF16; }
int64_t type_size(int t) { return t == FX_F32 ? 4 : t == FX_E4M3 ? 1 : 2; }
bool aligned(const void* p, int64_t to) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(to) == 0; }

// Packed rows for a stride of 0; false when the stride is out of range.
bool fix_stride(int64_t& stride, int64_t len) {
    if (stride == 0) stride = len;
    return stride >= len && stride < kMaxExtent;
}

// Makes the device of a call's pointers current for the call, and the caller's device again after it.
class OnDevice {
  public:
    ~OnDevice() {
        if (back_ >= 0) cudaSetDevice(back_);
    }
    // The pointers (nulls are skipped) must be memory of one sm_100 device.
    fx_status enter(const char* fn, std::initializer_list<const void*> ptrs) {
        int dev = -1;
        for (const void* p : ptrs) {
            if (!p) continue;
            cudaPointerAttributes at{};
            if (cudaError_t e = cudaPointerGetAttributes(&at, p); e != cudaSuccess) {
                cudaGetLastError();
                return fxh::abi_error(FX_UNSUPPORTED, std::string(fn) + ": " + cudaGetErrorString(e));
            }
            if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
                return bad(fn, "a pointer is not device memory");
            if (dev >= 0 && at.device != dev) return bad(fn, "pointers of different devices");
            dev = at.device;
        }
        static std::atomic<int> major[64];  // compute capability by device, 0: not asked yet
        int m = dev < 64 ? major[dev].load(std::memory_order_relaxed) : 0;
        if (!m) {
            cudaDeviceGetAttribute(&m, cudaDevAttrComputeCapabilityMajor, dev);
            if (dev < 64) major[dev].store(m, std::memory_order_relaxed);
        }
        if (m != 10) return fxh::abi_error(FX_UNSUPPORTED, std::string(fn) + ": needs an sm_100 GPU");
        int cur = -1;
        cudaGetDevice(&cur);
        if (cur != dev) {
            if (cudaError_t e = cudaSetDevice(dev); e != cudaSuccess)
                return fxh::abi_error(FX_INTERNAL, std::string(fn) + ": " + cudaGetErrorString(e));
            back_ = cur;
        }
        return FX_OK;
    }

  private:
    int back_ = -1;
};

fx_status done(const char* fn, cudaError_t e) {
    if (e == cudaSuccess) return FX_OK;
    cudaGetLastError();  // a refused launch leaves no error behind for the caller's next call
    return fxh::abi_error(FX_INTERNAL, std::string(fn) + ": " + cudaGetErrorString(e));
}

template <class F>
fx_status guarded(F&& f) {
    try {
        fxh::abi_error(FX_OK, "");
        return f();
    } catch (...) {
        return fxh::abi_exception();
    }
}

// The weights' side of a call: everything that needs no device.
fx_status check_w4(const char* fn, const uint8_t* codes, const void* scales, int scale_type, int64_t n, int64_t k,
                   int64_t group) {
    if (!is_float(scale_type)) return bad(fn, "scales are f32, f16 or bf16");
    if (n < 0 || n >= kMaxExtent || k < 1 || k >= kMaxInner) return bad(fn, "n or k out of range");
    if (group < 32 || group % 32 || k % group) return bad(fn, "group must be a multiple of 32 that divides k");
    if (n == 0) return FX_OK;
    if (!codes || !scales) return bad(fn, "null codes or scales");
    if (!aligned(codes, 16)) return bad(fn, "codes must be 16-byte aligned");
    if (!aligned(scales, type_size(scale_type))) return bad(fn, "scales are not aligned to their type");
    return FX_OK;
}

fxk::W4Args w4_args(const uint8_t* codes, const void* scales, int scale_type, const uint8_t* zeros, int64_t n,
                    int64_t k, int64_t group) {
    fxk::W4Args a{};
    a.codes = codes;
    a.scales = scales;
    a.zeros = zeros;
    a.n = static_cast<int>(n);
    a.k = static_cast<int>(k);
    a.group = static_cast<int>(group);
    a.scale_type = scale_type;
    return a;
}

}  // namespace

extern "C" {

fx_status fx_rms_norm(const void* dev_x, fx_dtype x_type, int64_t rows, int64_t cols, int64_t x_stride,
                      const void* dev_residual, fx_dtype residual_type, int64_t residual_stride, void* dev_sum,
                      int64_t sum_stride, const void* dev_weight, fx_dtype weight_type, float eps, void* dev_y,
                      fx_dtype y_type, int64_t y_stride, float* dev_scale, fx_scale scale_mode, void* stream) {
    static const char* const fn = "fx_rms_norm";
    return guarded([&]() -> fx_status {
        if (rows < 0 || rows >= kMaxExtent) return bad(fn, "rows out of range");
        if (cols < 1 || cols > fxk::kRmsMaxCols) return bad(fn, "cols must be 1..32768");
        if (!(eps > 0.f) || eps > 3.0e38f) return bad(fn, "eps must be positive and finite");
        if (!is_float(x_type) || !is_float(residual_type) || !is_float(weight_type))
            return bad(fn, "x, residual and weight are f32, f16 or bf16");
        if (!is_float(y_type) && y_type != FX_E4M3) return bad(fn, "y is f32, f16, bf16 or e4m3");
        if (y_type == FX_E4M3 ? (scale_mode != FX_SCALE_TENSOR && scale_mode != FX_SCALE_ROW)
                              : scale_mode != FX_SCALE_NONE)
            return bad(fn, "an e4m3 y takes a tensor or a row scale, another y none");
        if (!fix_stride(x_stride, cols) || !fix_stride(residual_stride, cols) || !fix_stride(sum_stride, cols) ||
            !fix_stride(y_stride, cols))
            return bad(fn, "a stride is shorter than a row or out of range");
        if (rows == 0) return FX_OK;
        if (!dev_x || !dev_y) return bad(fn, "null x or y");
        if (y_type == FX_E4M3 && !dev_scale) return bad(fn, "an e4m3 y needs dev_scale");
        if (!aligned(dev_x, type_size(x_type)) || !aligned(dev_y, type_size(y_type)) ||
            !aligned(dev_residual, type_size(residual_type)) || !aligned(dev_sum, type_size(residual_type)) ||
            !aligned(dev_weight, type_size(weight_type)) || !aligned(dev_scale, 4))
            return bad(fn, "a pointer is not aligned to its type");
        if (dev_y == dev_x && (y_type != x_type || (rows > 1 && y_stride != x_stride)))
            return bad(fn, "y in place of x needs x's type and stride");
        if (dev_sum && dev_sum == dev_x && (residual_type != x_type || (rows > 1 && sum_stride != x_stride)))
            return bad(fn, "sum in place of x needs x's type and stride");
        if (dev_sum && dev_sum == dev_residual && rows > 1 && sum_stride != residual_stride)
            return bad(fn, "sum in place of residual needs its stride");
        if (dev_y == dev_sum || dev_y == dev_residual) return bad(fn, "y may not be sum or residual");
        if (scale_mode == FX_SCALE_NONE) dev_scale = nullptr;
        OnDevice on;
        if (fx_status r = on.enter(fn, {dev_x, dev_y, dev_residual, dev_sum, dev_weight, dev_scale})) return r;
        fxk::RmsNormArgs a{};
        a.x = dev_x;
        a.residual = dev_residual;
        a.sum = dev_sum;
        a.weight = dev_weight;
        a.y = dev_y;
        a.scale = dev_scale;
        a.x_stride = x_stride;
        a.residual_stride = residual_stride;
        a.sum_stride = sum_stride;
        a.y_stride = y_stride;
        a.rows = static_cast<int>(rows);
        a.cols = static_cast<int>(cols);
        a.x_type = x_type;
        a.residual_type = residual_type;
        a.weight_type = weight_type;
        a.y_type = y_type;
        a.scale_mode = scale_mode;
        a.eps = eps;
        return done(fn, fxk::launch_rms_norm(a, static_cast<cudaStream_t>(stream)));
    });
}

fx_status fx_w4_linear(const void* dev_x, fx_dtype x_type, int64_t rows, int64_t x_stride, const float* dev_x_scale,
                       fx_scale x_scale_mode, const uint8_t* dev_codes, const void* dev_scales, fx_dtype scale_type,
                       const uint8_t* dev_zeros, int64_t n, int64_t k, int64_t group, const float* dev_bias,
                       void* dev_y, fx_dtype y_type, int64_t y_stride, void* stream) {
    static const char* const fn = "fx_w4_linear";
    return guarded([&]() -> fx_status {
        if (rows < 0 || rows >= kMaxExtent) return bad(fn, "rows out of range");
        if (x_type != FX_F16 && x_type != FX_BF16 && x_type != FX_E4M3) return bad(fn, "x is f16, bf16 or e4m3");
        if (y_type != FX_F16 && y_type != FX_BF16) return bad(fn, "y is f16 or bf16");
        if (x_type == FX_E4M3 ? (x_scale_mode != FX_SCALE_TENSOR && x_scale_mode != FX_SCALE_ROW)
                              : x_scale_mode != FX_SCALE_NONE)
            return bad(fn, "an e4m3 x takes a tensor or a row scale, another x none");
        if (fx_status r = check_w4(fn, dev_codes, dev_scales, scale_type, n, k, group)) return r;
        if (!fix_stride(x_stride, k) || !fix_stride(y_stride, n))
            return bad(fn, "a stride is shorter than a row or out of range");
        if (rows == 0 || n == 0) return FX_OK;
        if (!dev_x || !dev_y) return bad(fn, "null x or y");
        if (x_type == FX_E4M3 && !dev_x_scale) return bad(fn, "an e4m3 x needs dev_x_scale");
        if (!aligned(dev_x, type_size(x_type)) || !aligned(dev_y, 2) || !aligned(dev_x_scale, 4) ||
            !aligned(dev_bias, 4))
            return bad(fn, "a pointer is not aligned to its type");
        if (dev_y == dev_x) return bad(fn, "y may not be x");
        if (x_scale_mode == FX_SCALE_NONE) dev_x_scale = nullptr;
        OnDevice on;
        if (fx_status r = on.enter(fn, {dev_x, dev_y, dev_codes, dev_scales, dev_zeros, dev_x_scale, dev_bias}))
            return r;
        fxk::W4LinearArgs a{};
        a.w = w4_args(dev_codes, dev_scales, scale_type, dev_zeros, n, k, group);
        a.x = dev_x;
        a.x_scale = dev_x_scale;
        a.bias = dev_bias;
        a.y = dev_y;
        a.x_stride = x_stride;
        a.y_stride = y_stride;
        a.rows = static_cast<int>(rows);
        a.x_type = x_type;
        a.x_scale_mode = x_scale_mode;
        a.y_type = y_type;
        a.wait_ns = kWaitNs;
        return done(fn, fxk::launch_w4_linear(a, static_cast<cudaStream_t>(stream)));
    });
}

fx_status fx_w4_device_status(int device) {
    static const char* const fn = "fx_w4_device_status";
    return guarded([&]() -> fx_status {
        int count = 0, cur = 0;
        if (cudaGetDeviceCount(&count) != cudaSuccess || device < 0 || device >= count) {
            cudaGetLastError();
            return bad(fn, "no such device");
        }
        cudaGetDevice(&cur);
        if (cudaError_t e = cudaSetDevice(device); e != cudaSuccess) return done(fn, e);
        uint32_t few = 0, bf16 = 0, f16 = 0;
        cudaError_t e = cudaDeviceSynchronize();
        if (e == cudaSuccess) e = fxk::w4_few_status(&few);
        if (e == cudaSuccess) e = fxk::w4_many_bf16_status(&bf16);
        if (e == cudaSuccess) e = fxk::w4_many_f16_status(&f16);
        cudaSetDevice(cur);
        if (e != cudaSuccess) return done(fn, e);
        if (few || bf16 || f16)
            return fxh::abi_error(FX_INTERNAL, std::string(fn) + ": a bounded wait gave up, code " +
                                                   std::to_string(few ? few : bf16 ? bf16 : f16));
        return FX_OK;
    });
}

fx_status fx_selftest_w4_wait_timeout(int device, fx_dtype x_type, int rows, uint64_t wait_ns) {
    static const char* const fn = "fx_selftest_w4_wait_timeout";
    return guarded([&]() -> fx_status {
        int count = 0;
        if (x_type != FX_F16 && x_type != FX_BF16 && x_type != FX_E4M3) return bad(fn, "x is f16, bf16 or e4m3");
        if (rows < 1 || rows > 4096 || wait_ns == 0) return bad(fn, "rows must be 1..4096 and the limit positive");
        if (cudaGetDeviceCount(&count) != cudaSuccess || device < 0 || device >= count) {
            cudaGetLastError();
            return bad(fn, "no such device");
        }
        constexpr int kOut = 1024, kIn = 4096, kGroup = 128;
        struct Scratch {  // zeros: the layer's operands and results
            int back = -1;
            void* p = nullptr;
            ~Scratch() {
                cudaFree(p);
                if (back >= 0) cudaSetDevice(back);
            }
        } sc;
        cudaGetDevice(&sc.back);
        const size_t codes = size_t{kOut} * kIn / 2, scales = size_t{kOut} * kIn / kGroup * 2, x = size_t(rows) * kIn * 2,
                     y = size_t(rows) * kOut * 2, all = codes + scales + x + y + 256;
        cudaError_t e = cudaSetDevice(device);
        if (e == cudaSuccess) e = cudaMalloc(&sc.p, all);
        if (e == cudaSuccess) e = cudaMemset(sc.p, 0, all);
        if (e != cudaSuccess) return done(fn, e);
        uint8_t* const at = static_cast<uint8_t*>(sc.p);
        fxk::W4LinearArgs a{};
        a.w = w4_args(at, at + codes, FX_F16, nullptr, kOut, kIn, kGroup);
        a.x = at + codes + scales;
        a.y = at + codes + scales + x;
        a.x_scale = x_type == FX_E4M3 ? reinterpret_cast<const float*>(at + codes + scales + x + y) : nullptr;
        a.x_scale_mode = x_type == FX_E4M3 ? FX_SCALE_TENSOR : FX_SCALE_NONE;
        a.x_stride = kIn;
        a.y_stride = kOut;
        a.rows = rows;
        a.x_type = x_type;
        a.y_type = x_type == FX_BF16 ? FX_BF16 : FX_F16;
        a.hold_codes = true;
        a.wait_ns = wait_ns;
        e = fxk::launch_w4_linear(a, nullptr);
        if (e == cudaSuccess) e = cudaDeviceSynchronize();
        return done(fn, e);
    });
}

fx_status fx_w4_quantize(const void* dev_w, fx_dtype w_type, int64_t n, int64_t k, int64_t w_stride, int64_t group,
                         uint8_t* dev_codes, void* dev_scales, fx_dtype scale_type, uint8_t* dev_zeros, void* stream) {
    static const char* const fn = "fx_w4_quantize";
    return guarded([&]() -> fx_status {
        if (!is_float(w_type)) return bad(fn, "w is f32, f16 or bf16");
        if (fx_status r = check_w4(fn, dev_codes, dev_scales, scale_type, n, k, group)) return r;
        if (!fix_stride(w_stride, k)) return bad(fn, "a stride is shorter than a row or out of range");
        if (n == 0) return FX_OK;
        if (!dev_w) return bad(fn, "null w");
        if (!aligned(dev_w, type_size(w_type))) return bad(fn, "a pointer is not aligned to its type");
        OnDevice on;
        if (fx_status r = on.enter(fn, {dev_w, dev_codes, dev_scales, dev_zeros})) return r;
        return done(fn, fxk::launch_w4_quantize(dev_w, w_type, w_stride,
                                                w4_args(dev_codes, dev_scales, scale_type, dev_zeros, n, k, group),
                                                static_cast<cudaStream_t>(stream)));
    });
}

fx_status fx_w4_dequantize(const uint8_t* dev_codes, const void* dev_scales, fx_dtype scale_type,
                           const uint8_t* dev_zeros, int64_t n, int64_t k, int64_t group, void* dev_w, fx_dtype w_type,
                           int64_t w_stride, void* stream) {
    static const char* const fn = "fx_w4_dequantize";
    return guarded([&]() -> fx_status {
        if (!is_float(w_type)) return bad(fn, "w is f32, f16 or bf16");
        if (fx_status r = check_w4(fn, dev_codes, dev_scales, scale_type, n, k, group)) return r;
        if (!fix_stride(w_stride, k)) return bad(fn, "a stride is shorter than a row or out of range");
        if (n == 0) return FX_OK;
        if (!dev_w) return bad(fn, "null w");
        if (!aligned(dev_w, type_size(w_type))) return bad(fn, "a pointer is not aligned to its type");
        OnDevice on;
        if (fx_status r = on.enter(fn, {dev_codes, dev_scales, dev_zeros, dev_w})) return r;
        return done(fn, fxk::launch_w4_dequantize(w4_args(dev_codes, dev_scales, scale_type, dev_zeros, n, k, group),
                                                  dev_w, w_type, w_stride, static_cast<cudaStream_t>(stream)));
    });
}

}  // extern "C"
