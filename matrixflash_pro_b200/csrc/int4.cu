// 4-bit weights: w = (q - z) * s with a scale s and zero point z per row and group of 32, 64 or 128
// columns. Quantising, reading back, and the product with a few rows (decoding).
#include "mfb_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mfb {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

struct Int4Params {
    unsigned char* packed;
    void* scales;
    unsigned char* zeros;
    long long rows;  // experts * n
    int n, k, group, groups, row_bytes, experts;
};

// ------------------------------------------------------------------------------------
// Quantising
// ------------------------------------------------------------------------------------
// The integer nearest to w / s, ties to even, |result| <= 64. The FP32 quotient decides except next to a
// border between two codes, where the remainder w - q s does: it is exact in FP32 there, since w and q s
// agree to within s.
__device__ __forceinline__ float nearest_code(float w, float s, float inv) {
    const float t = fminf(fmaxf(w * inv, -64.0f), 64.0f);
    float q = rintf(t);
    if (fabsf(t - q) > 0.499f) {
        const float r = fmaf(-q, s, w);
        const float half = 0.5f * s;
        if (r > half || (r == half && (static_cast<int>(q) & 1))) q += 1.0f;
        else if (r < -half || (r == -half && (static_cast<int>(q) & 1))) q -= 1.0f;
    }
    return q;
}

template <typename TS>
__device__ __forceinline__ TS saturated_scale(double s);
template <>
__device__ __forceinline__ float saturated_scale<float>(double s) {
    return static_cast<float>(fmin(s, 3.4028234663852886e38));
}
template <>
__device__ __forceinline__ __half saturated_scale<__half>(double s) {
    return __float2half_rn(static_cast<float>(fmin(s, 65504.0)));
}
template <>
__device__ __forceinline__ __nv_bfloat16 saturated_scale<__nv_bfloat16>(double s) {
    return __float2bfloat16_rn(static_cast<float>(fmin(s, 3.3895313892515355e38)));
}

// One warp per row and group.
template <typename T, typename TS>
__global__ void __launch_bounds__(256) quantize_int4_kernel(const Int4Params p, const T* __restrict__ w,
                                                            long long ldw, long long stride_w) {
    const long long unit = (blockIdx.x * 256ll + threadIdx.x) / 32;
    const int lane = threadIdx.x % 32;
    if (unit >= p.rows * p.groups) return;
    const long long row = unit / p.groups;
    const int g = static_cast<int>(unit - row * p.groups);
    const T* src = w + (row / p.n) * stride_w + (row % p.n) * ldw;
    const int per = p.group / 32;  // 1, 2 or 4 consecutive columns per lane
    const int j0 = g * p.group + lane * per;
    float v[4];
    float lo = 0.0f, hi = 0.0f;
    for (int i = 0; i < per; ++i) {
        v[i] = j0 + i < p.k ? to_f32(src[j0 + i]) : 0.0f;
        lo = fminf(lo, v[i]);
        hi = fmaxf(hi, v[i]);
    }
    for (int d = 16; d; d /= 2) {
        lo = fminf(lo, __shfl_xor_sync(~0u, lo, d));
        hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, d));
    }
    const double range = p.zeros ? (static_cast<double>(hi) - lo) / 15.0 : fmax(-static_cast<double>(lo), hi) / 7.0;
    TS scale = saturated_scale<TS>(range);
    if (to_f32(scale) == 0.0f) scale = from_f32<TS>(1.0f);
    const float s = to_f32(scale), inv = 1.0f / s;
    float z = 8.0f;
    if (p.zeros) z = fminf(fmaxf(nearest_code(-lo, s, inv), 0.0f), 15.0f);
    if (lane == 0) {
        static_cast<TS*>(p.scales)[unit] = scale;
        if (p.zeros) p.zeros[unit] = static_cast<unsigned char>(z);
    }
    unsigned codes = 0;
    for (int i = 0; i < per; ++i) {
        const float q = fminf(fmaxf(nearest_code(v[i], s, inv) + z, 0.0f), 15.0f);
        codes |= static_cast<unsigned>(q) << (4 * i);
    }
    if (per == 1) codes |= __shfl_down_sync(~0u, codes, 1) << 4;  // lanes pair up: two codes per byte
    unsigned char* dst = p.packed + row * p.row_bytes;
    if (per == 1 && (lane & 1)) return;
    for (int i = 0; i < (per + 1) / 2; ++i)
        if (j0 / 2 + i < p.row_bytes) dst[j0 / 2 + i] = static_cast<unsigned char>(codes >> (8 * i));
}

template <typename TS, typename T>
__global__ void __launch_bounds__(256) dequantize_int4_kernel(const Int4Params p, T* __restrict__ out, long long ldo,
                                                              long long stride_o) {
    const long long total = p.rows * p.row_bytes;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const long long row = i / p.row_bytes;
        const int j = 2 * static_cast<int>(i - row * p.row_bytes);
        if (j >= p.k) continue;
        const long long at = row * p.groups + j / p.group;
        const float s = to_f32(static_cast<const TS*>(p.scales)[at]);
        const float z = p.zeros ? static_cast<float>(p.zeros[at]) : 8.0f;
        const unsigned b = p.packed[i];
        T* dst = out + (row / p.n) * stride_o + (row % p.n) * ldo + j;
        dst[0] = from_f32<T>((static_cast<float>(b & 15u) - z) * s);
        if (j + 1 < p.k) dst[1] = from_f32<T>((static_cast<float>(b >> 4) - z) * s);
    }
}

// ------------------------------------------------------------------------------------
// A few rows
// ------------------------------------------------------------------------------------
// One warp per output.
template <typename TS, typename T>
__global__ void __launch_bounds__(256) gemv_int4_kernel(const Int4Params p, int rows, const T* __restrict__ x,
                                                        long long ldx, const int* __restrict__ ids, T* __restrict__ y,
                                                        long long ldy) {
    const int r = blockIdx.y, lane = threadIdx.x % 32;
    const int i = blockIdx.x * 8 + threadIdx.x / 32;
    if (i >= p.n) return;
    const int e = ids ? ids[r] : 0;
    float sum = 0.0f;
    if (e >= p.experts && lane == 0) atomicOr(&g_status, kStatusBadIndex);
    if (e >= 0 && e < p.experts) {
        const long long row = static_cast<long long>(e) * p.n + i;
        for (int j = lane; j < p.k; j += 32) {
            const long long at = row * p.groups + j / p.group;
            const float s = to_f32(static_cast<const TS*>(p.scales)[at]);
            const float z = p.zeros ? static_cast<float>(p.zeros[at]) : 8.0f;
            const unsigned q = (p.packed[row * p.row_bytes + j / 2] >> (4 * (j % 2))) & 15u;
            sum = fmaf((static_cast<float>(q) - z) * s, to_f32(x[r * ldx + j]), sum);
        }
    }
    for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(~0u, sum, d);
    if (lane == 0) y[r * ldy + i] = from_f32<T>(sum);
}

mfb_status_t validate_int4(const mfb_int4_matrix* m, Int4Params* p) {
    if (!m) return fail(MFB_EINVAL, "null 4-bit matrix");
    if (m->experts < 0 || m->n < 0 || m->k < 0) return fail(MFB_EINVAL, "4-bit matrix dimensions must be non-negative");
    if (m->group != 32 && m->group != 64 && m->group != 128)
        return fail(MFB_EINVAL, "the group size of a 4-bit matrix is 32, 64 or 128");
    if (m->scale_dtype < MFB_DTYPE_F32 || m->scale_dtype > MFB_DTYPE_BF16)
        return fail(MFB_EINVAL, "invalid scale type of a 4-bit matrix");
    const long long row_bytes = (m->k + 31ll) / 32 * 16;
    *p = Int4Params{m->packed,
                    m->scales,
                    m->zeros,
                    static_cast<long long>(m->experts) * m->n,
                    m->n,
                    m->k,
                    m->group,
                    static_cast<int>((m->k + static_cast<long long>(m->group) - 1) / m->group),
                    static_cast<int>(row_bytes),
                    m->experts};
    if (p->rows == 0 || m->k == 0) return MFB_OK;
    if (!m->packed || !m->scales) return fail(MFB_EINVAL, "null codes or scales of a 4-bit matrix");
    if (!aligned16(m->packed)) return fail(MFB_EINVAL, "packed codes must start on a 16-byte boundary");
    if (reinterpret_cast<uintptr_t>(m->scales) % dtype_bytes(m->scale_dtype))
        return fail(MFB_EINVAL, "scales must be aligned to their type");
    return MFB_OK;
}

mfb_status_t validate_dtype(int dtype) {
    if (dtype < MFB_DTYPE_F32 || dtype > MFB_DTYPE_BF16) return fail(MFB_EINVAL, "invalid element type");
    return MFB_OK;
}

// Calls f with a value of the C++ type of `dtype` (validated).
template <typename F>
mfb_status_t with_dtype(int dtype, F&& f) {
    if (dtype == MFB_DTYPE_F32) return f(float{});
    if (dtype == MFB_DTYPE_F16) return f(__half{});
    return f(__nv_bfloat16{});
}

// `m`'s rows in a caller's matrix with these strides: every row in place, none over another where written.
mfb_status_t validate_rows(const Int4Params& p, const void* w, int dtype, long long ld, long long stride, bool written) {
    if (!w) return fail(MFB_EINVAL, "null matrix");
    if (reinterpret_cast<uintptr_t>(w) % dtype_bytes(dtype)) return fail(MFB_EINVAL, "matrix must be aligned to its type");
    if (ld < 0 || stride < 0) return fail(MFB_EINVAL, "strides must be non-negative");
    if (written && p.n > 1 && ld < p.k) return fail(MFB_EINVAL, "the row stride is smaller than a row");
    if (written && p.experts > 1 && stride < (p.n - 1ll) * ld + p.k)
        return fail(MFB_EINVAL, "the matrix stride is smaller than a matrix");
    return MFB_OK;
}

}  // namespace
}  // namespace mfb

using namespace mfb;

extern "C" {

MFB_API mfb_status_t mfb_quantize_int4(int device, mfb_stream_t stream, const void* w, int dtype, long long ldw,
                                       long long stride_w, const mfb_int4_matrix* out) {
    clear_error();
    Int4Params p;
    MFB_TRY(validate_int4(out, &p));
    MFB_TRY(validate_dtype(dtype));
    if (p.rows == 0 || p.k == 0) return MFB_OK;
    MFB_TRY(validate_rows(p, w, dtype, ldw, stride_w, false));
    DeviceGuard guard;
    MFB_TRY(select_device(device));
    const long long blocks = (p.rows * p.groups + 7) / 8;
    if (blocks > 0x7fffffffLL) return fail(MFB_EINVAL, "4-bit matrix has too many groups");
    return with_dtype(dtype, [&](auto t) {
        return with_dtype(out->scale_dtype, [&](auto ts) {
            using T = decltype(t);
            quantize_int4_kernel<T, decltype(ts)><<<static_cast<unsigned>(blocks), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                p, static_cast<const T*>(w), ldw, stride_w);
            MFB_CUDA_TRY(cudaGetLastError(), "quantize_int4 launch");
            return MFB_OK;
        });
    });
}

MFB_API mfb_status_t mfb_dequantize_int4(int device, mfb_stream_t stream, const mfb_int4_matrix* m, void* out,
                                         int dtype, long long ldo, long long stride_o) {
    clear_error();
    Int4Params p;
    MFB_TRY(validate_int4(m, &p));
    MFB_TRY(validate_dtype(dtype));
    if (p.rows == 0 || p.k == 0) return MFB_OK;
    MFB_TRY(validate_rows(p, out, dtype, ldo, stride_o, true));
    DeviceGuard guard;
    MFB_TRY(select_device(device));
    return with_dtype(m->scale_dtype, [&](auto ts) {
        return with_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            dequantize_int4_kernel<decltype(ts), T><<<8 * current_sm_count(), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                p, static_cast<T*>(out), ldo, stride_o);
            MFB_CUDA_TRY(cudaGetLastError(), "dequantize_int4 launch");
            return MFB_OK;
        });
    });
}

MFB_API mfb_status_t mfb_gemv_int4(int device, mfb_stream_t stream, const mfb_int4_matrix* m, int rows, const void* x,
                                   long long ldx, int dtype, const int* expert_ids, void* y, long long ldy) {
    clear_error();
    Int4Params p;
    MFB_TRY(validate_int4(m, &p));
    MFB_TRY(validate_dtype(dtype));
    if (rows < 0 || rows > MFB_INT4_GEMV_ROWS)
        return fail(MFB_EINVAL, "mfb_gemv_int4 serves 0 to " + std::to_string(MFB_INT4_GEMV_ROWS) + " rows");
    if (!expert_ids && p.experts != 1) return fail(MFB_EINVAL, "a stack of matrices needs an expert per row");
    if (rows == 0 || p.n == 0) return MFB_OK;
    if (!y || (!x && p.k > 0)) return fail(MFB_EINVAL, "null x or y pointer");
    if (reinterpret_cast<uintptr_t>(x) % dtype_bytes(dtype) || reinterpret_cast<uintptr_t>(y) % dtype_bytes(dtype))
        return fail(MFB_EINVAL, "x and y must be aligned to their type");
    if (ldx < 0 || (rows > 1 && ldy < p.n)) return fail(MFB_EINVAL, "the row stride of y is smaller than n");
    const char* xs = static_cast<const char*>(x);
    const char* ys = static_cast<const char*>(y);
    if (p.k > 0 && ys < xs + ((rows - 1) * ldx + p.k) * dtype_bytes(dtype) &&
        xs < ys + ((rows - 1) * ldy + p.n) * dtype_bytes(dtype))
        return fail(MFB_EINVAL, "GEMV output cannot alias x");
    DeviceGuard guard;
    MFB_TRY(select_device(device));
    return with_dtype(m->scale_dtype, [&](auto ts) {
        return with_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            gemv_int4_kernel<decltype(ts), T><<<dim3((p.n + 7) / 8, rows), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                p, rows, static_cast<const T*>(x), ldx, expert_ids, static_cast<T*>(y), ldy);
            MFB_CUDA_TRY(cudaGetLastError(), "gemv_int4 launch");
            return MFB_OK;
        });
    });
}

}  // extern "C"
