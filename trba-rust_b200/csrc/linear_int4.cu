// Linear layer with 4-bit weights and group scales for the few rows of a
// decoding step (include/trba_ops.h, LinearInt4).  No counterpart in the
// reference; the quantisation rule is LinearInt8's (src/linear.rs:53-59) for
// 4 bits and groups.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <new>

#include "common.cuh"
#include "trba_decode.h"
#include "trba_ops.h"

struct trba_linear_int4 {
    int in = 0, out = 0, group = 0, groups = 0, device = 0, scale_dtype = 0;
    uint8_t *base = nullptr;    // one allocation: codes, scales, bias
    uint8_t *codes = nullptr;   // [out][pitch] natural order
    i64 pitch = 0;
    void *scales = nullptr;     // [out][groups]
    float *bias = nullptr;      // [out]
};

namespace trba {
namespace {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float ld_f32(const float *p) { return *p; }
__device__ __forceinline__ float ld_f32(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float ld_f32(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ void st_f32(float *p, float v) { *p = v; }
__device__ __forceinline__ void st_f32(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void st_f32(__half *p, float v) { *p = __float2half_rn(v); }

// One warp a group: scale = max |w| / 7, code = 8 + round(w / scale).
__global__ void __launch_bounds__(256) int4_quantize_kernel(const float *__restrict__ w, int in, int out, int group,
                                                            int groups, uint8_t *__restrict__ codes, i64 pitch,
                                                            float *__restrict__ scales) {
    const int lane = threadIdx.x & 31;
    const i64 total = (i64)out * groups, step = (i64)gridDim.x * (blockDim.x >> 5);
    for (i64 e = (i64)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); e < total; e += step) {
        const i64 n = e / groups;
        const int k0 = (int)(e - n * groups) * group, k1 = min(in, k0 + group);
        const float *row = w + n * in;
        float mx = 0.0f;
        for (int k = k0 + lane; k < k1; k += 32) mx = fmaxf(mx, fabsf(row[k]));
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o));
        const float s = mx > 0.0f ? fdiv(mx, 7.0f) : 1.0f;
        if (lane == 0) scales[e] = s;
        for (int k = k0 + 2 * lane; k < k1; k += 64) {
            unsigned byte = 0;
            for (int h = 0; h < 2; ++h) {
                const float v = k + h < k1 ? fminf(fmaxf(fdiv(row[k + h], s), -7.0f), 7.0f) : 0.0f;
                byte |= (unsigned)((int)roundf(v) + 8) << (4 * h);
            }
            codes[n * pitch + (k >> 1)] = (uint8_t)byte;
        }
    }
}

// One warp an output, a row of x at a time.
template <class T, class S>
__global__ void __launch_bounds__(256) int4_forward_kernel(const uint8_t *__restrict__ codes, i64 pitch,
                                                           const S *__restrict__ scales, int groups, int group,
                                                           const float *__restrict__ bias, const T *__restrict__ x,
                                                           i64 ldx, int rows, int in, int out, T *__restrict__ y,
                                                           i64 ldy) {
    const int lane = threadIdx.x & 31, n = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (n >= out) return;
    for (int r = 0; r < rows; ++r) {
        float sum = 0.0f;
        for (int g = 0; g < groups; ++g) {
            float part = 0.0f;
            const int k1 = min(in, (g + 1) * group);
            for (int k = g * group + lane; k < k1; k += 32) {
                const int q = (codes[n * pitch + (k >> 1)] >> (4 * (k & 1))) & 15;
                part = fmaf((float)(q - 8), ld_f32(x + r * ldx + k), part);
            }
            sum = fmaf(part, ld_f32(scales + (i64)n * groups + g), sum);
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
        if (lane == 0) st_f32(y + r * ldy + n, sum + bias[n]);
    }
}

int launched() {
    count_launch();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) report_error(__FILE__, __LINE__, cudaGetErrorString(e), (int)e);
    return (int)e;
}

template <class T, class S>
int forward(const trba_linear_int4 *l, const void *x, i64 ldx, int rows, void *y, i64 ldy, cudaStream_t st) {
    int4_forward_kernel<T, S><<<(l->out + 7) / 8, 256, 0, st>>>(
        l->codes, l->pitch, static_cast<const S *>(l->scales), l->groups, l->group, l->bias,
        static_cast<const T *>(x), ldx, rows, l->in, l->out, static_cast<T *>(y), ldy);
    return launched();
}

template <class T>
int forward(const trba_linear_int4 *l, const void *x, i64 ldx, int rows, void *y, i64 ldy, cudaStream_t st) {
    return l->scale_dtype == TRBA_F16 ? forward<T, __half>(l, x, ldx, rows, y, ldy, st)
                                      : forward<T, float>(l, x, ldx, rows, y, ldy, st);
}

bool sizes_ok(int in, int out, int group) {
    return in > 0 && out > 0 && (group == 32 || group == 64 || (group >= 128 && group % 128 == 0));
}

trba_linear_int4 *allocate(int in, int out, int group, int scale_dtype) {
    auto *l = new (std::nothrow) trba_linear_int4;
    if (!l) return nullptr;
    l->in = in, l->out = out, l->group = group, l->groups = (in - 1) / group + 1;
    l->scale_dtype = scale_dtype;
    l->pitch = ((i64)(in + 1) / 2 + 15) & ~15ll;
    const size_t nc = (size_t)out * l->pitch;
    const size_t ns = ((size_t)out * l->groups * (scale_dtype == TRBA_F32 ? 4 : 2) + 15) & ~(size_t)15;
    if (cudaGetDevice(&l->device) != cudaSuccess ||
        cudaMalloc(&l->base, nc + ns + (size_t)out * 4) != cudaSuccess) {
        cudaGetLastError();
        report_error(__FILE__, __LINE__, "LinearInt4: device allocation failed", -1);
        delete l;
        return nullptr;
    }
    l->codes = l->base;
    l->scales = l->base + nc;
    l->bias = reinterpret_cast<float *>(l->base + nc + ns);
    return l;
}

}  // namespace
}  // namespace trba

using namespace trba;

extern "C" {

trba_linear_int4 *trba_linear_int4_create(int in_features, int out_features, int group, const float *weight_f32,
                                          const float *bias) {
    TRBA_REQUIRE_RET(sizes_ok(in_features, out_features, group) && weight_f32, "trba_linear_int4_create: bad arguments",
                     nullptr);
    trba_linear_int4 *l = allocate(in_features, out_features, group, TRBA_F32);
    if (!l) return nullptr;
    const size_t nw = (size_t)in_features * out_features;
    float *w = nullptr;
    bool ok = cudaMalloc(&w, nw * 4) == cudaSuccess &&
              cudaMemcpy(w, weight_f32, nw * 4, cudaMemcpyHostToDevice) == cudaSuccess;
    ok = ok && (bias ? cudaMemcpy(l->bias, bias, (size_t)out_features * 4, cudaMemcpyHostToDevice)
                     : cudaMemset(l->bias, 0, (size_t)out_features * 4)) == cudaSuccess;
    if (ok) {
        int4_quantize_kernel<<<grid_for((i64)out_features * l->groups * 32), 256>>>(
            w, in_features, out_features, group, l->groups, l->codes, l->pitch, static_cast<float *>(l->scales));
        ok = launched() == 0 && cudaStreamSynchronize(nullptr) == cudaSuccess;
    }
    if (w) cudaFree(w);
    if (!ok) {
        report_error(__FILE__, __LINE__, "trba_linear_int4_create: allocation, copy or quantisation failed", -1);
        trba_linear_int4_destroy(l);
        return nullptr;
    }
    return l;
}

trba_linear_int4 *trba_linear_int4_create_codes(int in_features, int out_features, int group, const uint8_t *codes,
                                                long long ld_codes, const void *scales, int scale_dtype,
                                                long long ld_scales, const float *bias, void *stream) {
    TRBA_REQUIRE_RET(sizes_ok(in_features, out_features, group) && codes && scales &&
                         (scale_dtype == TRBA_F32 || scale_dtype == TRBA_F16) && ld_codes >= (in_features + 1ll) / 2 &&
                         ld_scales >= (in_features - 1) / group + 1,
                     "trba_linear_int4_create_codes: bad arguments", nullptr);
    trba_linear_int4 *l = allocate(in_features, out_features, group, scale_dtype);
    if (!l) return nullptr;
    cudaStream_t st = as_stream(stream);
    const size_t es = scale_dtype == TRBA_F32 ? 4 : 2;
    bool ok = cudaMemcpy2DAsync(l->codes, l->pitch, codes, ld_codes, ((size_t)in_features + 1) / 2, out_features,
                                cudaMemcpyDeviceToDevice, st) == cudaSuccess &&
              cudaMemcpy2DAsync(l->scales, l->groups * es, scales, ld_scales * es, l->groups * es, out_features,
                                cudaMemcpyDeviceToDevice, st) == cudaSuccess;
    ok = ok && (bias ? cudaMemcpyAsync(l->bias, bias, (size_t)out_features * 4, cudaMemcpyDeviceToDevice, st)
                     : cudaMemsetAsync(l->bias, 0, (size_t)out_features * 4, st)) == cudaSuccess;
    if (cudaStreamSynchronize(st) != cudaSuccess) ok = false;
    if (!ok) {
        report_error(__FILE__, __LINE__, "trba_linear_int4_create_codes: copying the weights failed", -1);
        trba_linear_int4_destroy(l);
        return nullptr;
    }
    return l;
}

void trba_linear_int4_destroy(trba_linear_int4 *l) {
    if (!l) return;
    cudaFree(l->base);
    delete l;
}

int trba_linear_int4_forward(const trba_linear_int4 *l, const void *x, int dtype, long long ldx, int rows, void *y,
                             long long ldy, void *stream) {
    TRBA_REQUIRE_RET(l && rows >= 0, "trba_linear_int4_forward: bad arguments", -1);
    if (rows == 0) return 0;
    TRBA_REQUIRE_RET(x && y && ldx >= l->in && ldy >= l->out, "trba_linear_int4_forward: bad arguments", -1);
    TRBA_REQUIRE_RET(dtype == TRBA_F32 || dtype == TRBA_BF16 || dtype == TRBA_F16,
                     "trba_linear_int4_forward: unknown element type", -1);
    const uintptr_t es = dtype == TRBA_F32 ? 4 : 2;
    TRBA_REQUIRE_RET(reinterpret_cast<uintptr_t>(x) % es == 0 && reinterpret_cast<uintptr_t>(y) % es == 0,
                     "trba_linear_int4_forward: x or y is not aligned to its elements", -1);
    int dev = -1;
    cudaGetDevice(&dev);
    TRBA_REQUIRE_RET(dev == l->device, "trba_linear_int4_forward: the layer is on another device", -1);
    cudaStream_t st = as_stream(stream);
    if (dtype == TRBA_F32) return forward<float>(l, x, ldx, rows, y, ldy, st);
    if (dtype == TRBA_BF16) return forward<__nv_bfloat16>(l, x, ldx, rows, y, ldy, st);
    return forward<__half>(l, x, ldx, rows, y, ldy, st);
}

int trba_linear_int4_get(const trba_linear_int4 *l, uint8_t *codes, float *scales, float *bias) {
    if (!l) return -1;
    TRBA_CHECK(cudaDeviceSynchronize());
    const size_t row = ((size_t)l->in + 1) / 2, ns = (size_t)l->out * l->groups;
    if (codes) TRBA_CHECK(cudaMemcpy2D(codes, row, l->codes, l->pitch, row, l->out, cudaMemcpyDeviceToHost));
    if (bias) TRBA_CHECK(cudaMemcpy(bias, l->bias, (size_t)l->out * 4, cudaMemcpyDeviceToHost));
    if (scales && l->scale_dtype == TRBA_F32) {
        TRBA_CHECK(cudaMemcpy(scales, l->scales, ns * 4, cudaMemcpyDeviceToHost));
    } else if (scales) {
        __half *tmp = new (std::nothrow) __half[ns];
        TRBA_REQUIRE_RET(tmp, "trba_linear_int4_get: out of host memory", -1);
        TRBA_CHECK(cudaMemcpy(tmp, l->scales, ns * 2, cudaMemcpyDeviceToHost));
        for (size_t i = 0; i < ns; ++i) scales[i] = __half2float(tmp[i]);
        delete[] tmp;
    }
    return 0;
}

long long trba_linear_int4_param_count(const trba_linear_int4 *l) {
    return l ? (long long)l->in * l->out + l->out : -1;
}

}  // extern "C"
