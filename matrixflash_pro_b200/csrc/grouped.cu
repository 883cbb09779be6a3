// Products grouped by expert: C[t] = A[t] op(B_e) for the rows t of group e, and the gradient by the
// groups' matrices C_e = sum_t A[t]^T B[t]. Group sizes are device data (row offsets), read by the
// kernels, so nothing here waits for the host.
#include "mfb_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mfb {
namespace {

constexpr int kMaxGroups = 4096;

struct GroupedParams {
    const int* offsets;
    int groups, rows, n, k;
    long long lda, ldb, ldc, stride;
    int trans_b, zero_rest;
    const void* a;
    const void* b;
    void* c;
};

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

// Offset e, clamped to [previous, rows]; anything else is reported.
__device__ __forceinline__ int checked_offset(const GroupedParams& p, int e, int previous) {
    const int v = p.offsets[e];
    const int c = min(max(v, previous), p.rows);
    if (c != v) atomicOr(&g_status, kStatusBadIndex);
    return c;
}

// 64 x 64 tiles of C, 16 x 16 threads of 4 x 4 sums. blockIdx.y counts the 64-row tiles of the groups in
// turn (each group starts a tile of its own, so at most ceil(rows / 64) + groups are used).
template <typename T, typename TO>
__global__ void __launch_bounds__(256) grouped_simple_kernel(const GroupedParams p) {
    __shared__ float as[16][65], bs[16][65];
    __shared__ int s_e, s_t0, s_t1;
    if (threadIdx.x == 0) {
        int tile = blockIdx.y, start = checked_offset(p, 0, 0);
        s_e = -1;
        for (int e = 0; e < p.groups; ++e) {
            const int end = checked_offset(p, e + 1, start);
            const int tiles = (end - start + 63) / 64;
            if (tile < tiles) {
                s_e = e;
                s_t0 = start + tile * 64;
                s_t1 = min(end, s_t0 + 64);
                break;
            }
            tile -= tiles;
            start = end;
        }
    }
    __syncthreads();
    if (s_e < 0) return;
    const int t0 = s_t0, t1 = s_t1, j0 = blockIdx.x * 64;
    const T* a = static_cast<const T*>(p.a);
    const T* b = static_cast<const T*>(p.b) + p.stride * s_e;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float sum[4][4] = {}, part[4][4] = {};  // a chain of 64 products at a time, then the chains' sum
    for (int k0 = 0; k0 < p.k; k0 += 16) {
        for (int i = threadIdx.x; i < 1024; i += 256) {
            const int r = i / 16, c = i % 16;
            as[c][r] = t0 + r < t1 && k0 + c < p.k ? to_f32(a[(t0 + r) * p.lda + k0 + c]) : 0.0f;
            const int kk = p.trans_b ? i % 16 : i / 64, jj = p.trans_b ? i / 16 : i % 64;
            const bool in = j0 + jj < p.n && k0 + kk < p.k;
            const long long at = p.trans_b ? (j0 + jj) * p.ldb + k0 + kk : (k0 + kk) * p.ldb + j0 + jj;
            bs[kk][jj] = in ? to_f32(b[at]) : 0.0f;
        }
        __syncthreads();
        for (int kk = 0; kk < 16; ++kk)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) part[i][j] = fmaf(as[kk][ty * 4 + i], bs[kk][tx * 4 + j], part[i][j]);
        if ((k0 / 16) % 4 == 3 || k0 + 16 >= p.k)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) {
                    sum[i][j] += part[i][j];
                    part[i][j] = 0.0f;
                }
        __syncthreads();
    }
    TO* c = static_cast<TO*>(p.c);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int t = t0 + ty * 4 + i, col = j0 + tx * 4 + j;
            if (t < t1 && col < p.n) c[t * p.ldc + col] = from_f32<TO>(sum[i][j]);
        }
}

// C_e (k x n) = sum over the group's rows of A[t]^T B[t]; blockIdx.z = group.
template <typename T, typename TO>
__global__ void __launch_bounds__(256) grouped_right_simple_kernel(const GroupedParams p) {
    __shared__ float as[16][65], bs[16][65];
    __shared__ int s_t0, s_t1;
    if (threadIdx.x == 0) {
        int start = checked_offset(p, 0, 0), end = start;
        for (int e = 0; e <= static_cast<int>(blockIdx.z); ++e) {
            start = end;
            end = checked_offset(p, e + 1, start);
        }
        s_t0 = start;
        s_t1 = end;
    }
    __syncthreads();
    const int t0 = s_t0, t1 = s_t1, i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
    const T* a = static_cast<const T*>(p.a);
    const T* b = static_cast<const T*>(p.b);
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float sum[4][4] = {}, part[4][4] = {};
    for (int t = t0; t < t1; t += 16) {
        for (int i = threadIdx.x; i < 1024; i += 256) {
            const int r = i / 64, c = i % 64;
            as[r][c] = t + r < t1 && i0 + c < p.k ? to_f32(a[(t + r) * p.lda + i0 + c]) : 0.0f;
            bs[r][c] = t + r < t1 && j0 + c < p.n ? to_f32(b[(t + r) * p.ldb + j0 + c]) : 0.0f;
        }
        __syncthreads();
        for (int kk = 0; kk < 16; ++kk)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) part[i][j] = fmaf(as[kk][ty * 4 + i], bs[kk][tx * 4 + j], part[i][j]);
        if (((t - t0) / 16) % 4 == 3 || t + 16 >= t1)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) {
                    sum[i][j] += part[i][j];
                    part[i][j] = 0.0f;
                }
        __syncthreads();
    }
    TO* c = static_cast<TO*>(p.c) + p.stride * blockIdx.z;
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int row = i0 + ty * 4 + i, col = j0 + tx * 4 + j;
            if (row < p.k && col < p.n) c[row * p.ldc + col] = from_f32<TO>(sum[i][j]);
        }
}

// Zeros in the rows that belong to no group.
template <typename TO>
__global__ void __launch_bounds__(256) grouped_rest_kernel(const GroupedParams p) {
    __shared__ int s_first, s_last;
    if (threadIdx.x == 0) {
        int last = s_first = checked_offset(p, 0, 0);
        for (int e = 1; e <= p.groups; ++e) last = checked_offset(p, e, last);
        s_last = last;
    }
    __syncthreads();
    TO* c = static_cast<TO*>(p.c);
    for (int t = blockIdx.x; t < p.rows; t += gridDim.x)
        if (t < s_first || t >= s_last)
            for (int j = threadIdx.x; j < p.n; j += 256) c[t * p.ldc + j] = from_f32<TO>(0.0f);
}

int dtype_bytes(int dtype) { return dtype == MFB_DTYPE_F32 ? 4 : 2; }

// Checks that both entry points share. `right`: the gradient by the groups' matrices.
mfb_status_t validate_grouped(const mfb_grouped_desc* d, const int* offsets, const void* a, const void* b,
                              const void* c, bool right) {
    if (!d) return fail(MFB_EINVAL, "null grouped descriptor");
    if (d->groups < 0 || d->rows < 0 || d->n < 0 || d->k < 0)
        return fail(MFB_EINVAL, "grouped product dimensions must be non-negative");
    if (d->groups > kMaxGroups)
        return fail(MFB_EINVAL, "at most " + std::to_string(kMaxGroups) + " groups are supported");
    if (d->dtype < MFB_DTYPE_F32 || d->dtype > MFB_DTYPE_BF16) return fail(MFB_EINVAL, "invalid grouped operand type");
    if (d->out_dtype != d->dtype && d->out_dtype != MFB_DTYPE_F32)
        return fail(MFB_EINVAL, "the output of a grouped product has the operands' type or FP32");
    if (d->precision != MFB_PRECISION_FP32 && d->precision != MFB_PRECISION_TF32)
        return fail(MFB_EINVAL, "Invalid GEMM precision policy");
    if ((d->trans_b != 0 && d->trans_b != 1) || (d->zero_rest != 0 && d->zero_rest != 1))
        return fail(MFB_EINVAL, "trans_b and zero_rest must be 0 or 1");
    if (right && (d->trans_b || d->zero_rest))
        return fail(MFB_EINVAL, "mfb_grouped_gemm_bwd_right takes neither trans_b nor zero_rest");
    const int b_cols = right ? d->n : d->trans_b ? d->k : d->n;
    if (d->lda < std::max(1, d->k)) return fail(MFB_EINVAL, "lda is smaller than the stored row length of A");
    if (d->ldb < std::max(1, b_cols)) return fail(MFB_EINVAL, "ldb is smaller than the stored row length of B");
    if (d->ldc < std::max(1, d->n)) return fail(MFB_EINVAL, "ldc is smaller than n");
    if (d->stride < 0) return fail(MFB_EINVAL, "the stride between group matrices must be non-negative");
    if (!offsets) return fail(MFB_EINVAL, "null group offsets");
    const long long c_rows = right ? d->k : d->rows;
    if (c_rows == 0 || d->n == 0 || (right && d->groups == 0)) return MFB_OK;
    if (right && d->groups > 1 && d->stride < (c_rows - 1) * d->ldc + d->n)
        return fail(MFB_EINVAL, "stride makes the groups' outputs overlap");
    if (!c) return fail(MFB_EINVAL, "null C pointer");
    // Extents in bytes: the output may not overlap an operand.
    const long long b_rows = right ? d->rows : d->trans_b ? d->n : d->k;
    const bool reads = d->rows > 0 && d->k > 0 && d->groups > 0;
    if (!reads) return MFB_OK;
    if (!a || !b) return fail(MFB_EINVAL, "null A or B pointer");
    auto extent = [](long long r, long long ld, long long cols, long long count, long long stride, int bytes) {
        return r == 0 ? 0ll : ((r - 1) * ld + cols + (count - 1) * stride) * bytes;
    };
    const char* cs = static_cast<const char*>(c);
    const char* as = static_cast<const char*>(a);
    const char* bs = static_cast<const char*>(b);
    const int size = dtype_bytes(d->dtype);
    const char* c_end = cs + extent(c_rows, d->ldc, d->n, right ? d->groups : 1, right ? d->stride : 0,
                                    dtype_bytes(d->out_dtype));
    const char* a_end = as + extent(d->rows, d->lda, d->k, 1, 0, size);
    const char* b_end = bs + extent(b_rows, d->ldb, b_cols, right ? 1 : d->groups, right ? 0 : d->stride, size);
    if ((cs < a_end && as < c_end) || (cs < b_end && bs < c_end))
        return fail(MFB_EINVAL, "the output of a grouped product cannot alias an input");
    if (reinterpret_cast<uintptr_t>(a) % size || reinterpret_cast<uintptr_t>(b) % size ||
        reinterpret_cast<uintptr_t>(c) % dtype_bytes(d->out_dtype))
        return fail(MFB_EINVAL, "grouped operands must be aligned to their element size");
    return MFB_OK;
}

GroupedParams grouped_params(const mfb_grouped_desc& d, const int* offsets, const void* a, const void* b, void* c) {
    return GroupedParams{offsets, d.groups, d.rows,    d.n,         d.k, d.lda, d.ldb,
                         d.ldc,   d.stride, d.trans_b, d.zero_rest, a,   b,     c};
}

template <typename T, typename TO>
mfb_status_t launch_simple(const GroupedParams& p, cudaStream_t stream, bool right) {
    const unsigned nx = static_cast<unsigned>((p.n + 63) / 64);
    if (right) {
        grouped_right_simple_kernel<T, TO><<<dim3(nx, (p.k + 63) / 64, p.groups), 256, 0, stream>>>(p);
    } else {
        if (p.groups > 0)
            grouped_simple_kernel<T, TO><<<dim3(nx, (p.rows + 63) / 64 + p.groups), 256, 0, stream>>>(p);
        if (p.zero_rest) grouped_rest_kernel<TO><<<4 * current_sm_count(), 256, 0, stream>>>(p);
    }
    MFB_CUDA_TRY(cudaGetLastError(), "grouped product launch");
    return MFB_OK;
}

mfb_status_t launch_grouped(const mfb_grouped_desc& d, const GroupedParams& p, cudaStream_t stream, bool right) {
    if (d.dtype == MFB_DTYPE_F32) return launch_simple<float, float>(p, stream, right);
    if (d.dtype == MFB_DTYPE_F16)
        return d.out_dtype == MFB_DTYPE_F32 ? launch_simple<__half, float>(p, stream, right)
                                            : launch_simple<__half, __half>(p, stream, right);
    return d.out_dtype == MFB_DTYPE_F32 ? launch_simple<__nv_bfloat16, float>(p, stream, right)
                                        : launch_simple<__nv_bfloat16, __nv_bfloat16>(p, stream, right);
}

}  // namespace
}  // namespace mfb

using namespace mfb;

extern "C" {

MFB_API mfb_status_t mfb_grouped_gemm(int device, mfb_stream_t stream, const mfb_grouped_desc* desc,
                                      const int* offsets, const void* a, const void* b, void* c) {
    clear_error();
    MFB_TRY(validate_grouped(desc, offsets, a, b, c, false));
    if (desc->rows == 0 || desc->n == 0) return MFB_OK;
    DeviceGuard guard;
    MFB_TRY(select_device(device));
    return launch_grouped(*desc, grouped_params(*desc, offsets, a, b, c), reinterpret_cast<cudaStream_t>(stream),
                          false);
}

MFB_API mfb_status_t mfb_grouped_gemm_bwd_right(int device, mfb_stream_t stream, const mfb_grouped_desc* desc,
                                                const int* offsets, const void* a, const void* b, void* c) {
    clear_error();
    MFB_TRY(validate_grouped(desc, offsets, a, b, c, true));
    if (desc->groups == 0 || desc->k == 0 || desc->n == 0) return MFB_OK;
    DeviceGuard guard;
    MFB_TRY(select_device(device));
    return launch_grouped(*desc, grouped_params(*desc, offsets, a, b, c), reinterpret_cast<cudaStream_t>(stream),
                          true);
}

}  // extern "C"
