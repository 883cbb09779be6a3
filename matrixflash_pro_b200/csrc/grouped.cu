// Products grouped by expert: C[t] = A[t] op(B_e) for the rows t of group e, and the gradient by the
// groups' matrices C_e = sum_t A[t]^T B[t]. Group sizes are device data (row offsets), read by the
// kernels, so nothing here waits for the host.
#include "grouped_tc.cuh"
#include "mfb_internal.h"

#include <algorithm>
#include <map>
#include <mutex>

namespace mfb {
namespace {

int dtype_bytes(int dtype) { return dtype == MFB_DTYPE_F32 ? 4 : 2; }

// Bytes from the first to behind the last element of `count` matrices of r rows.
long long extent(long long r, long long ld, long long cols, long long count, long long stride, int bytes) {
    return r == 0 || count == 0 ? 0 : ((r - 1) * ld + cols + (count - 1) * stride) * bytes;
}

// Checks that both entry points share. `right`: the gradient by the groups' matrices.
mfb_status_t validate_grouped(const mfb_grouped_desc* d, const int* offsets, const void* a, const void* b,
                              const void* c, bool right) {
    if (!d) return fail(MFB_EINVAL, "null grouped descriptor");
    if (d->groups < 0 || d->rows < 0 || d->n < 0 || d->k < 0)
        return fail(MFB_EINVAL, "grouped product dimensions must be non-negative");
    if (std::max({d->rows, d->n, d->k}) > INT32_MAX - 65536)
        return fail(MFB_EINVAL, "grouped product dimension exceeds the 32-bit limit");
    if (d->groups > kGroupedMaxGroups)
        return fail(MFB_EINVAL, "at most " + std::to_string(kGroupedMaxGroups) + " groups are supported");
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
    // (before the calls that read nothing return: they still write zeros)
    if (reinterpret_cast<uintptr_t>(c) % dtype_bytes(d->out_dtype))
        return fail(MFB_EINVAL, "the output of a grouped product must be aligned to its element size");
    const long long b_rows = right ? d->rows : d->trans_b ? d->n : d->k;
    // Extents in bytes: the output may not overlap what the kernel reads.
    const char* cs = static_cast<const char*>(c);
    const char* c_end = cs + extent(c_rows, d->ldc, d->n, right ? d->groups : 1, right ? d->stride : 0,
                                    dtype_bytes(d->out_dtype));
    const char* os = reinterpret_cast<const char*>(offsets);
    if (cs < os + 4 * (d->groups + 1ll) && os < c_end)
        return fail(MFB_EINVAL, "the output of a grouped product cannot alias the offsets");
    if (reinterpret_cast<uintptr_t>(offsets) % 4) return fail(MFB_EINVAL, "offsets must be aligned to 4 bytes");
    const bool reads = d->rows > 0 && d->k > 0 && d->groups > 0;
    if (!reads) return MFB_OK;
    if (!a || !b) return fail(MFB_EINVAL, "null A or B pointer");
    const char* as = static_cast<const char*>(a);
    const char* bs = static_cast<const char*>(b);
    const int size = dtype_bytes(d->dtype);
    const char* a_end = as + extent(d->rows, d->lda, d->k, 1, 0, size);
    const char* b_end = bs + extent(b_rows, d->ldb, b_cols, right ? 1 : d->groups, right ? 0 : d->stride, size);
    if ((cs < a_end && as < c_end) || (cs < b_end && bs < c_end))
        return fail(MFB_EINVAL, "the output of a grouped product cannot alias an input");
    if (reinterpret_cast<uintptr_t>(a) % size || reinterpret_cast<uintptr_t>(b) % size)
        return fail(MFB_EINVAL, "grouped operands must be aligned to their element size");
    return MFB_OK;
}

// One instance of the kernel.
struct GroupedEntry {
    const void* fn;
    int smem, threads, nt, cg;
};

template <class Cfg>
GroupedEntry entry() {
    return GroupedEntry{reinterpret_cast<const void*>(&grouped_tc_kernel<Cfg>), Cfg::kSmem, Cfg::kThreads, Cfg::NT, Cfg::CG};
}

// Wide tiles on SM pairs, narrow ones on single SMs.
template <int PLANES, bool RIGHT, bool M_MN, bool TMA>
GroupedEntry entry_for(bool wide) {
    if constexpr (TMA)
        return wide ? entry<GroupedConfig<256, 2, 1, RIGHT, M_MN, true, 2, 3>>() : entry<GroupedConfig<64, 1, 1, RIGHT, M_MN, true, 2, 4>>();
    else if constexpr (PLANES == 1)
        return wide ? entry<GroupedConfig<256, 2, 1, RIGHT, M_MN, false, 1, 6>>() : entry<GroupedConfig<64, 1, 1, RIGHT, M_MN, false, 1, 8>>();
    else
        return wide ? entry<GroupedConfig<128, 2, PLANES, RIGHT, M_MN, false, 1, 3>>()
                    : entry<GroupedConfig<64, 1, PLANES, RIGHT, M_MN, false, 1, 3>>();
}

template <int PLANES, bool TMA>
GroupedEntry entry_of(bool right, bool m_mn, bool wide) {
    if (right) return entry_for<PLANES, true, true, TMA>(wide);
    return m_mn ? entry_for<PLANES, false, true, TMA>(wide) : entry_for<PLANES, false, false, TMA>(wide);
}

// Raises the kernel's shared-memory limit once per device, and says how many of its workers (SMs or SM
// pairs) fit on the device at once.
mfb_status_t grouped_workers(const GroupedEntry& e, int device, int* out) {
    static std::mutex mutex;
    static std::map<std::pair<int, const void*>, int> cache;
    std::lock_guard<std::mutex> lock(mutex);
    auto it = cache.find({device, e.fn});
    if (it != cache.end()) {
        *out = it->second;
        return MFB_OK;
    }
    MFB_CUDA_TRY(cudaFuncSetAttribute(e.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, e.smem),
                 "cudaFuncSetAttribute(grouped product)");
    int workers = sm_count(device);
    if (e.cg == 2) {
        cudaLaunchConfig_t lc{};
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {2, 1, 1};
        lc.gridDim = dim3(static_cast<unsigned>(2 * (workers / 2)));
        lc.blockDim = dim3(static_cast<unsigned>(e.threads));
        lc.dynamicSmemBytes = static_cast<size_t>(e.smem);
        lc.attrs = &attr;
        lc.numAttrs = 1;
        MFB_CUDA_TRY(cudaOccupancyMaxActiveClusters(&workers, e.fn, &lc), "cudaOccupancyMaxActiveClusters");
        if (workers <= 0) return fail(MFB_EUNSUPPORTED, "no SM pair can host the grouped product");
    }
    cache[{device, e.fn}] = workers;
    *out = workers;
    return MFB_OK;
}

// Tensor map over `count` matrices of 16-bit elements: boxes of 64 columns x box_rows, or with `wide` boxes > 0 (cols
// a multiple of 64) `wide` such boxes side by side, the columns as an axis of 64 and one of boxes.
mfb_status_t encode_16bit(CUtensorMap* map, const void* base, long long rows, int cols, long long ld, long long count,
                          long long stride, int box_rows, int wide = 0) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(MFB_ECUDA, "cuTensorMapEncodeTiled entry point unavailable");
    const cuuint64_t row_bytes = static_cast<cuuint64_t>(ld) * 2;
    const cuuint64_t matrix_bytes = static_cast<cuuint64_t>(count > 1 ? stride : ld) * 2;
    const cuuint64_t r = static_cast<cuuint64_t>(rows), n = static_cast<cuuint64_t>(count);
    const cuuint32_t br = static_cast<cuuint32_t>(box_rows), step[4] = {1, 1, 1, 1};
    const cuuint64_t dims3[3] = {static_cast<cuuint64_t>(cols), r, n}, strides3[2] = {row_bytes, matrix_bytes};
    const cuuint64_t dims4[4] = {64, r, static_cast<cuuint64_t>(cols / 64), n}, strides4[3] = {row_bytes, 128, matrix_bytes};
    const cuuint32_t box3[3] = {64, br, 1}, box4[4] = {64, br, static_cast<cuuint32_t>(wide), 1};
    // The bits are copied as they are, FP16 or BF16.
    const CUresult result =
        fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, wide ? 4 : 3, const_cast<void*>(base), wide ? dims4 : dims3,
           wide ? strides4 : strides3, wide ? box4 : box3, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (result != CUDA_SUCCESS)
        return fail(MFB_ECUDA, "cuTensorMapEncodeTiled failed (code " + std::to_string(static_cast<int>(result)) + ")");
    return MFB_OK;
}

// The largest power of two up to 32 that divides the address and every stride in bytes.
int common_alignment(const void* p, long long s0, long long s1) {
    const unsigned long long v = reinterpret_cast<uintptr_t>(p) | static_cast<unsigned long long>(s0) |
                                 static_cast<unsigned long long>(s1) | 32u;
    return static_cast<int>(v & (~v + 1));
}

mfb_status_t launch_grouped(int device, const mfb_grouped_desc& d, cudaStream_t stream, const int* offsets,
                            const void* a, const void* b, void* c, bool right) {
    const int size = dtype_bytes(d.dtype);
    const bool shared = right || d.groups <= 1 || d.stride == 0;  // B is one matrix
    GroupedParams p{};
    p.offsets = offsets;
    p.groups = d.groups;
    p.rows = d.rows;
    p.n = d.n;
    p.k = d.k;
    p.ldc = d.ldc;
    p.stride_c = right ? d.stride : 0;
    p.c = c;
    p.out_f32 = d.out_dtype == MFB_DTYPE_F32;
    p.bf16 = d.dtype == MFB_DTYPE_BF16;
    p.zero_rest = d.zero_rest;
    p.wait_limit_ns = wait_limit_ns();
    p.m_base = static_cast<const char*>(b);
    p.n_base = static_cast<const char*>(a);
    p.m_ld = d.ldb * static_cast<long long>(size);
    p.n_ld = d.lda * static_cast<long long>(size);
    p.m_stride = shared ? 0 : d.stride * size;
    p.m_align = common_alignment(b, p.m_ld, p.m_stride);
    p.n_align = common_alignment(a, p.n_ld, 0);
    p.m_shared = shared;

    const bool m_mn = !d.trans_b;
    const bool tma = size == 2 && p.m_align >= 16 && p.n_align >= 16 && d.groups > 0 && d.k > 0 && d.rows > 0;
    // Wide tiles take up to 256 rows of C (FP32: 128) per SM pair, narrow ones 64 per SM. 8 experts of 2048x4096, us,
    // narrow / wide, by rows per group: 16 27.0 / 28.2, 48 28.3 / 29.9, 64 37.7 / 30.3, 128 55.7 / 32.3 (bf16);
    // 16 127 / 128, 48 128 / 130, 64 177 / 131 (FP32): a group of more than 64 rows reads its weights twice in narrow
    // tiles. Gradient by the matrices, 8 groups of 256 rows, n = 2048, by k: 64 7.0 / 9.0, 128 8.8 / 9.0, 256 12.7 / 9.8.
    // The host knows the mean alone, and skewed groups want wide tiles at smaller means. 8 experts of 2048x4096, one of 340
    // rows and seven of 6: 35.5 / 31.1 (bf16), 159 / 165 (FP32); 32 of 2048x1024, eight of 100 and the others of 2: 36.8 /
    // 32.1, 161 / 119; 64 of 512x1024, four of 470 and the others of 2: 21.1 / 21.3, 75 / 83 (even groups of 31: 18.8 / 21.1,
    // 65 / 70). So the rule loses up to a sixth (FP32: a third) on skewed groups, and would lose as much on even ones at 30.
    const bool wide = right ? d.k > 64 : d.rows / std::max(1, d.groups) > 48;
    const GroupedEntry e = size == 2 ? (tma ? entry_of<1, true>(right, m_mn, wide) : entry_of<1, false>(right, m_mn, wide))
                           : d.precision == MFB_PRECISION_FP32 ? entry_of<3, false>(right, m_mn, wide)
                                                               : entry_of<2, false>(right, m_mn, wide);
    p.m_tiles = (d.n + 128 * e.cg - 1) / (128 * e.cg);
    // An upper bound of the tiles: each group may have one that its rows do not fill.
    const long long row_tiles = right ? static_cast<long long>(d.groups) * ((d.k + e.nt - 1) / e.nt)
                                      : (d.rows + e.nt - 1) / e.nt + std::min(d.groups, d.rows);
    if (row_tiles * p.m_tiles > 0x7fffffffLL) return fail(MFB_EINVAL, "problem has too many output tiles");

    CUtensorMap maps[4] = {};
    if (tma) {
        p.m_wide = m_mn && d.n % 64 == 0;
        p.n_wide = right && d.k % 64 == 0;
        const int m_wide = p.m_wide ? 2 : 0, n_box = e.nt / e.cg;
        if (right) {
            MFB_TRY(encode_16bit(&maps[0], b, d.rows, d.n, d.ldb, 1, 0, 64, m_wide));
            MFB_TRY(encode_16bit(&maps[1], a, d.rows, d.k, d.lda, 1, 0, 64, p.n_wide ? n_box / 64 : 0));
        } else {
            const long long b_rows = d.trans_b ? d.n : d.k;
            const int b_cols = d.trans_b ? d.k : d.n;
            MFB_TRY(encode_16bit(&maps[0], b, b_rows, b_cols, d.ldb, shared ? 1 : d.groups, d.stride, m_mn ? 64 : 128, m_wide));
            MFB_TRY(encode_16bit(&maps[1], a, d.rows, d.k, d.lda, 1, 0, n_box));
            MFB_TRY(encode_16bit(&maps[2], a, d.rows, d.k, d.lda, 1, 0, 32));
            MFB_TRY(encode_16bit(&maps[3], a, d.rows, d.k, d.lda, 1, 0, 16));
        }
    }
    int workers = 0;
    MFB_TRY(grouped_workers(e, device, &workers));
    // Without tiles the launch still clears the rows of no group.
    const long long useful = std::max(row_tiles * p.m_tiles, d.zero_rest ? (d.rows + 7ll) / 8 : 1ll);
    workers = static_cast<int>(std::min<long long>(workers, useful));
    void* args[] = {&maps[0], &maps[1], &maps[2], &maps[3], &p};
    cudaLaunchConfig_t lc{};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {2, 1, 1};
    lc.gridDim = dim3(static_cast<unsigned>(e.cg * workers));
    lc.blockDim = dim3(static_cast<unsigned>(e.threads));
    lc.dynamicSmemBytes = static_cast<size_t>(e.smem);
    lc.stream = stream;
    lc.attrs = &attr;
    lc.numAttrs = e.cg == 2 ? 1 : 0;
    MFB_CUDA_TRY(cudaLaunchKernelExC(&lc, e.fn, args), "grouped product launch");
    return MFB_OK;
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
    return launch_grouped(device, *desc, reinterpret_cast<cudaStream_t>(stream), offsets, a, b, c, false);
}

MFB_API mfb_status_t mfb_grouped_gemm_bwd_right(int device, mfb_stream_t stream, const mfb_grouped_desc* desc,
                                                const int* offsets, const void* a, const void* b, void* c) {
    clear_error();
    MFB_TRY(validate_grouped(desc, offsets, a, b, c, true));
    if (desc->groups == 0 || desc->k == 0 || desc->n == 0) return MFB_OK;
    DeviceGuard guard;
    MFB_TRY(select_device(device));
    return launch_grouped(device, *desc, reinterpret_cast<cudaStream_t>(stream), offsets, a, b, c, true);
}

}  // extern "C"
