// 4-bit weights: w = (q - z) * s with a scale s and zero point z per row and group of 32, 64 or 128
// columns. Quantising, reading back, and the product with a few rows (decoding).
#include "mfb_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

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
// y[r, i] = sum over groups of s[i, G] * sum_{j in G} (q - z)[i, j] x[r, j].
//
// The codes are read once and everything else fits beside that: a warp takes 16 output rows and 128 columns
// at a time (16 bytes of codes per row and lane, four lanes to a row), turns codes into the exact 16-bit
// integers q - z and feeds them to m16n8k16 MMAs as A, with up to 8 * RT rows of x as B. A group's sum is an
// FP32 accumulator, its scale one FMA per accumulator. FP32 rows enter as three BF16 terms (exact), added into
// the same accumulator, small ones first.
//
// Which columns meet in one MMA step is free as long as A and B agree, so a lane's word of eight codes serves two
// steps as it lies: (word >> 4 i) & 0x000f000f holds codes i and i + 4. For groups of 64 and 32 the four lanes of
// a row exchange words first, so that all columns of a step share one scale.
//
// One block of 16 warps per SM takes an even share of the 16-row tiles. Its warps split the columns (KW warps,
// every KW-th chunk each) and, where there are fewer chunks than warps, the tiles. A warp goes chunk by chunk
// through the tiles, so a chunk of x is loaded and laid out once for all of them; codes and scales of the next
// tiles are in flight in registers meanwhile. Sums wait in shared memory, a slot per tile, warp and lane, and are
// added up in a fixed order at the end.

template <typename T>
struct Int4Math {  // FP16
    static constexpr int kTerms = 1;
    __device__ __forceinline__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    // Codes i and i + 4 of a word, less z, for i = 0..3: 1024 + q (or 1024 + 16 q) has q in its low bits.
    __device__ __forceinline__ static void weights(uint32_t word, uint32_t z, uint32_t (&out)[4]) {
        const float zf = static_cast<float>(z);
        const __half2 low = __float2half2_rn(1024.0f + zf), high = __float2half2_rn(-64.0f - zf);
        const __half2 sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            uint32_t v = ((word >> (4 * i)) & 0x000f000fu) | 0x64006400u;
            uint32_t u = ((word >> (4 * i)) & 0x00f000f0u) | 0x64006400u;
            const __half2 d = __hsub2(reinterpret_cast<__half2&>(v), low);
            const __half2 e = __hfma2(reinterpret_cast<__half2&>(u), sixteenth, high);
            out[i] = reinterpret_cast<const uint32_t&>(d);
            out[i + 1] = reinterpret_cast<const uint32_t&>(e);
        }
    }
};

struct Int4MathBf16 {
    __device__ __forceinline__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    __device__ __forceinline__ static void weights(uint32_t word, uint32_t z, uint32_t (&out)[4]) {
        const __nv_bfloat162 offset = __float2bfloat162_rn(128.0f + static_cast<float>(z));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t v = ((word >> (4 * i)) & 0x000f000fu) | 0x43004300u;  // 128 + q
            const __nv_bfloat162 d = __hsub2(reinterpret_cast<__nv_bfloat162&>(v), offset);
            out[i] = reinterpret_cast<const uint32_t&>(d);
        }
    }
};
template <>
struct Int4Math<__nv_bfloat16> : Int4MathBf16 {
    static constexpr int kTerms = 1;
};
template <>
struct Int4Math<float> : Int4MathBf16 {
    static constexpr int kTerms = 3;
};

// Eight consecutive values of a row of x from column j on (0 behind column k), as 16-bit pairs per term.
template <typename T>
__device__ __forceinline__ void load_x8(const T* row, int j, int k, bool vec, uint32_t (&out)[Int4Math<T>::kTerms][4]) {
    if constexpr (sizeof(T) == 2) {
        if (vec && j + 8 <= k) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + j));
            out[0][0] = v.x, out[0][1] = v.y, out[0][2] = v.z, out[0][3] = v.w;
            return;
        }
        const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = j + 2 * i < k ? __ldg(h + j + 2 * i) : 0, hi = j + 2 * i + 1 < k ? __ldg(h + j + 2 * i + 1) : 0;
            out[0][i] = lo | hi << 16;
        }
    } else {
        float v[8];
        if (vec && j + 8 <= k) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(row + j)), b = __ldg(reinterpret_cast<const float4*>(row + j) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = j + i < k ? __ldg(reinterpret_cast<const float*>(row) + j + i) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo = v[2 * i], hi = v[2 * i + 1];
            asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(out[0][i]) : "f"(hi), "f"(lo));
#pragma unroll
            for (int t = 1; t < 3; ++t) {
                lo -= __uint_as_float(out[t - 1][i] << 16);
                hi -= __uint_as_float(out[t - 1][i] & 0xffff0000u);
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(out[t][i]) : "f"(hi), "f"(lo));
            }
        }
    }
}

// Codes, scales and zero points of one tile and chunk: rows g and g + 8 of this lane.
template <typename TS, int GROUP>
struct Int4Item {
    static constexpr int kGroups = 128 / GROUP;
    uint4 w[2];
    TS s[2][kGroups];
    uint32_t z[2];  // one byte per group

    // vec: whole chunks of groups, aligned.
    __device__ __forceinline__ void load(const Int4Params& p, long long row0, int n_left, int chunk, int lane, bool vec) {
        const int byte = chunk * 64 + lane % 4 * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long row = row0 + min(h * 8 + lane / 4, n_left - 1);  // rows past the end repeat the last
            w[h] = make_uint4(0, 0, 0, 0);
            if (byte < p.row_bytes)
                asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[h].x), "=r"(w[h].y), "=r"(w[h].z), "=r"(w[h].w)
                             : "l"(p.packed + row * p.row_bytes + byte));
            const long long at = row * p.groups + chunk * kGroups;
            const TS* sp = static_cast<const TS*>(p.scales) + at;
            z[h] = 0x08080808u;
            if (vec) {
                struct alignas(sizeof(TS) * kGroups) Vec {
                    TS v[kGroups];
                };
                const Vec v = *reinterpret_cast<const Vec*>(sp);
#pragma unroll
                for (int i = 0; i < kGroups; ++i) s[h][i] = v.v[i];
                if (p.zeros) {
                    if (kGroups == 4) z[h] = __ldg(reinterpret_cast<const uint32_t*>(p.zeros + at));
                    else if (kGroups == 2) z[h] = __ldg(reinterpret_cast<const uint16_t*>(p.zeros + at));
                    else z[h] = __ldg(p.zeros + at);
                }
            } else {
                if (p.zeros) z[h] = 0;
#pragma unroll
                for (int i = 0; i < kGroups; ++i) {
                    const bool in = chunk * kGroups + i < p.groups;
                    s[h][i] = in ? sp[i] : from_f32<TS>(0.0f);
                    if (p.zeros && in) z[h] |= static_cast<uint32_t>(__ldg(p.zeros + at + i)) << (8 * i);
                }
            }
        }
    }
};

// Exchanges words between the four lanes of a row so that word slots of one group hold codes of one group:
// slot i of lane t then starts at column slot_column(t, i) of the chunk.
template <int GROUP>
__device__ __forceinline__ void regroup(uint32_t (&w)[4], int t) {
    if (GROUP <= 64) {
        const bool upper = t >= 2;
        const uint32_t a = __shfl_xor_sync(~0u, upper ? w[0] : w[2], 2), b = __shfl_xor_sync(~0u, upper ? w[1] : w[3], 2);
        if (upper) w[0] = a, w[1] = b;
        else w[2] = a, w[3] = b;
    }
    if (GROUP == 32) {
        const bool odd = t & 1;
        const uint32_t a = __shfl_xor_sync(~0u, odd ? w[0] : w[1], 1), b = __shfl_xor_sync(~0u, odd ? w[2] : w[3], 1);
        if (odd) w[0] = a, w[2] = b;
        else w[1] = a, w[3] = b;
    }
}
template <int GROUP>
__device__ __forceinline__ int slot_column(int t, int i) {
    if (GROUP == 128) return 32 * t + 8 * i;
    if (GROUP == 64) return 32 * ((t & 1) + 2 * (i >> 1)) + 8 * ((i & 1) + 2 * (t >> 1));
    return 32 * i + 8 * t;
}

constexpr int kGemvWarps = 16;
constexpr int kGemvSlots = 128;  // 16-row tiles times warps along k whose sums one block holds at a time
constexpr int kGemvSmem = kGemvSlots * 32 * 16;

// The rows of x by expert: segment d holds rows order[begin[d]] .. order[begin[d + 1] - 1] of x.
struct GemvSegments {
    int count;
    int expert[MFB_INT4_GEMV_ROWS];
    int begin[MFB_INT4_GEMV_ROWS + 1];
    int order[MFB_INT4_GEMV_ROWS];
};

// By one warp. Rows of no expert are in no segment.
__device__ __forceinline__ void gemv_segments(const Int4Params& p, const int* ids, int rows, int lane, GemvSegments& g) {
    if (!ids) {
        if (lane == 0) g.count = 1, g.expert[0] = 0, g.begin[0] = 0, g.begin[1] = rows;
        for (int r = lane; r < rows; r += 32) g.order[r] = r;
        return;
    }
    int id[2];
    unsigned long long same[2] = {0, 0};  // the rows of this row's expert
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = lane + 32 * h;
        id[h] = r < rows ? ids[r] : -1;
        if (id[h] >= p.experts) {
            if (blockIdx.x == 0) atomicOr(&g_status, kStatusBadIndex);
            id[h] = -1;
        }
    }
    const unsigned low = __match_any_sync(~0u, id[0]), high = __match_any_sync(~0u, id[1]);
    same[0] = low;
    same[1] = static_cast<unsigned long long>(high) << 32;
    if (rows > 32)
        for (int l = 0; l < 32; ++l) {
            if (__shfl_sync(~0u, id[1], l) == id[0]) same[0] |= 1ull << (32 + l);
            if (__shfl_sync(~0u, id[0], l) == id[1]) same[1] |= 1ull << l;
        }
    int segments = 0, begin = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (h == 1 && rows <= 32) break;
        const int r = lane + 32 * h;
        const bool first = id[h] >= 0 && __ffsll(static_cast<long long>(same[h])) - 1 == r;
        const unsigned firsts = __ballot_sync(~0u, first);
        const int d = segments + __popc(firsts & ((1u << lane) - 1));
        int sum = first ? __popcll(same[h]) : 0;
        const int mine = sum;
#pragma unroll
        for (int s = 1; s < 32; s *= 2) {
            const int o = __shfl_up_sync(~0u, sum, s);
            if (lane >= s) sum += o;
        }
        if (first) {
            g.expert[d] = id[h];
            int at = begin + sum - mine;
            g.begin[d] = at;
            for (unsigned long long m = same[h]; m; m &= m - 1) g.order[at++] = __ffsll(static_cast<long long>(m)) - 1;
        }
        segments += __popc(firsts);
        begin += __shfl_sync(~0u, sum, 31);
    }
    if (lane == 0) g.count = segments, g.begin[segments] = begin;
}

// x_vec: 16-byte aligned rows of x; s_vec: aligned chunks of scales; kw_log: log2 of the warps along k.
template <typename T, typename TS, int GROUP, int RT>
__global__ void __launch_bounds__(32 * kGemvWarps, 1)
    gemv_int4_kernel(const Int4Params p, int rows, const T* __restrict__ x, long long ldx, const int* __restrict__ ids,
                     T* __restrict__ y, long long ldy, bool x_vec, bool s_vec, int kw_log) {
    using Math = Int4Math<T>;
    using Item = Int4Item<TS, GROUP>;
    constexpr int kTerms = Math::kTerms, kCols = 8 * RT;
    // Items in flight per warp, within 128 registers beside 16 * kTerms * RT of x.
    constexpr int kItemRegs = 10 + 2 * (128 / GROUP * static_cast<int>(sizeof(TS)) + 3) / 4;
    constexpr int kRoom = (88 - 16 * kTerms * RT) / kItemRegs;
    constexpr int kDepth = kRoom > 4 ? 4 : kRoom < 2 ? 2 : kRoom;
    extern __shared__ float4 sums[];  // [tile][kw][RT][lane]
    __shared__ GemvSegments seg;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, t = lane % 4;
    if (warp == 0) gemv_segments(p, ids, rows, lane, seg);
    __syncthreads();

    const int kw_count = 1 << kw_log, kw = warp & (kw_count - 1), tw = warp >> kw_log, tw_count = kGemvWarps >> kw_log;
    const int chunks = (p.k + 127) / 128, tiles = (p.n + 15) / 16;
    const int most = kGemvSlots / RT >> kw_log;
    const long long all = static_cast<long long>(seg.count) * tiles;
    long long from = all * blockIdx.x / gridDim.x;
    const long long to = all * (blockIdx.x + 1) / gridDim.x;
    while (from < to) {
        const int d = static_cast<int>(from / tiles), m0 = static_cast<int>(from - static_cast<long long>(d) * tiles);
        const int count = static_cast<int>(min(min(to - from, static_cast<long long>(tiles - m0)), static_cast<long long>(most)));
        from += count;
        const long long row0 = static_cast<long long>(seg.expert[d]) * p.n;
        const int x_first = seg.begin[d], x_count = seg.begin[d + 1] - x_first;
        for (int c0 = 0; c0 < x_count; c0 += kCols) {
            const T* xr[RT];  // the row of x in this lane's column of B
            bool live[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int c = c0 + 8 * r + lane / 4;
                live[r] = c < x_count;
                xr[r] = x + (live[r] ? seg.order[x_first + c] : 0) * ldx;
            }
            uint32_t xb[RT][kTerms][4][4];  // [slot][b0, b1 of step 0, b0, b1 of step 1]
            Item ring[kDepth];
            int load_chunk = kw, load_tile = tw;
            auto load = [&](Item& item) {
                if (load_chunk >= chunks || tw >= count) return;
                const int i = (m0 + load_tile) * 16;
                item.load(p, row0 + i, p.n - i, load_chunk, lane, s_vec);
                load_tile += tw_count;
                if (load_tile >= count) load_tile = tw, load_chunk += kw_count;
            };
#pragma unroll
            for (int i = 0; i < kDepth; ++i) load(ring[i]);
            int chunk = kw, tile = tw;
            while (chunk < chunks && tile < count) {
#pragma unroll
                for (int at = 0; at < kDepth; ++at) {
                    if (chunk >= chunks) continue;
                    if (tile == tw) {  // a new chunk: lay out its columns of x
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int r = 0; r < RT; ++r) {
                                uint32_t v[kTerms][4] = {};
                                if (live[r]) load_x8<T>(xr[r], chunk * 128 + slot_column<GROUP>(t, i), p.k, x_vec, v);
#pragma unroll
                                for (int u = 0; u < kTerms; ++u)
#pragma unroll
                                    for (int step = 0; step < 2; ++step) {
                                        xb[r][u][i][2 * step] = __byte_perm(v[u][step], v[u][step + 2], 0x5410);
                                        xb[r][u][i][2 * step + 1] = __byte_perm(v[u][step], v[u][step + 2], 0x7632);
                                    }
                            }
                    }
                    const Item item = ring[at];
                    load(ring[at]);
                    uint32_t w[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        w[h][0] = item.w[h].x, w[h][1] = item.w[h].y, w[h][2] = item.w[h].z, w[h][3] = item.w[h].w;
                        regroup<GROUP>(w[h], t);
                    }
                    float acc[RT][4] = {}, part[RT][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        constexpr int kSlots = GROUP / 32;  // word slots of a group
                        const int group = i / kSlots;
                        if (i % kSlots == 0)
#pragma unroll
                            for (int r = 0; r < RT; ++r)
#pragma unroll
                                for (int e = 0; e < 4; ++e) part[r][e] = 0.0f;
                        uint32_t lo[4], hi[4];  // rows g and g + 8, codes (i, i + 4)
                        Math::weights(w[0][i], (item.z[0] >> (8 * group)) & 15u, lo);
                        Math::weights(w[1][i], (item.z[1] >> (8 * group)) & 15u, hi);
#pragma unroll
                        for (int step = 0; step < 2; ++step) {
                            const uint32_t a[4] = {lo[2 * step], hi[2 * step], lo[2 * step + 1], hi[2 * step + 1]};
#pragma unroll
                            for (int r = 0; r < RT; ++r)
#pragma unroll
                                for (int u = kTerms - 1; u >= 0; --u)
                                    Math::mma(part[r], a, xb[r][u][i][2 * step], xb[r][u][i][2 * step + 1]);
                        }
                        if (i % kSlots == kSlots - 1) {
                            const float s0 = to_f32(item.s[0][group]), s1 = to_f32(item.s[1][group]);
#pragma unroll
                            for (int r = 0; r < RT; ++r)
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[r][e] = fmaf(e < 2 ? s0 : s1, part[r][e], acc[r][e]);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        float4& slot = sums[(((tile << kw_log) + kw) * RT + r) * 32 + lane];
                        float4 v = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
                        if (chunk != kw) {
                            const float4 o = slot;
                            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
                        }
                        slot = v;
                    }
                    tile += tw_count;
                    if (tile >= count) tile = tw, chunk += kw_count;
                }
            }
            __syncthreads();
            const int split = min(kw_count, chunks);
            for (int at = threadIdx.x; at < count * 16 * kCols; at += 32 * kGemvWarps) {
                const int i = at & 15, rest = at >> 4;  // consecutive threads: consecutive outputs
                const int c = rest % kCols, m = rest / kCols;
                const int out = (m0 + m) * 16 + i;
                if (c0 + c >= x_count || out >= p.n) continue;
                const float* v = reinterpret_cast<const float*>(sums + ((m << kw_log) * RT + c / 8) * 32) +
                                 ((i & 7) * 4 + c % 8 / 2) * 4 + (i >> 3) * 2 + (c & 1);
                float sum = 0.0f;
                for (int s = 0; s < split; ++s) sum += v[s * RT * 128];
                y[seg.order[x_first + c0 + c] * ldy + out] = from_f32<T>(sum);
            }
            __syncthreads();
        }
    }
    if (ids)  // rows of no expert
        for (int r = 0; r < rows; ++r) {
            const int e = ids[r];
            if (e >= 0 && e < p.experts) continue;
            for (int i = blockIdx.x * 32 * kGemvWarps + threadIdx.x; i < p.n; i += gridDim.x * 32 * kGemvWarps)
                y[r * ldy + i] = from_f32<T>(0.0f);
        }
}

template <typename T, typename TS, int GROUP>
mfb_status_t gemv_int4_launch(const Int4Params& p, int device, cudaStream_t stream, int rows, const T* x, long long ldx,
                              const int* ids, T* y, long long ldy) {
    const bool x_vec = (reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(ldx * sizeof(T))) % 16 == 0;
    constexpr int kGroups = 128 / GROUP;
    const bool s_vec = p.groups % kGroups == 0 && reinterpret_cast<uintptr_t>(p.scales) % (sizeof(TS) * kGroups) == 0 &&
                       reinterpret_cast<uintptr_t>(p.zeros) % kGroups == 0;
    const int chunks = (p.k + 127) / 128;
    int kw_log = 0;
    while (kw_log < 4 && (1 << kw_log) < chunks) ++kw_log;
    const long long tiles = static_cast<long long>(ids ? rows : 1) * ((p.n + 15) / 16);
    const unsigned grid = static_cast<unsigned>(std::min<long long>(tiles, sm_count(device)));
    auto go = [&](auto rt) -> mfb_status_t {
        const auto kernel = &gemv_int4_kernel<T, TS, GROUP, decltype(rt)::value>;
        static std::atomic<unsigned long long> raised{0};  // devices whose shared-memory limit is raised
        const unsigned long long bit = 1ull << (device & 63);
        if (!(raised.load(std::memory_order_acquire) & bit)) {
            MFB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemvSmem),
                         "cudaFuncSetAttribute(gemv_int4)");
            raised.fetch_or(bit, std::memory_order_release);
        }
        kernel<<<grid, 32 * kGemvWarps, kGemvSmem, stream>>>(p, rows, x, ldx, ids, y, ldy, x_vec, s_vec, kw_log);
        MFB_CUDA_TRY(cudaGetLastError(), "gemv_int4 launch");
        return MFB_OK;
    };
    // Two column tiles of x keep 16 rows in one pass over the codes; FP32 rows have no registers for that.
    if constexpr (sizeof(T) == 2)
        if (rows > 8 && !ids) return go(std::integral_constant<int, 2>());
    return go(std::integral_constant<int, 1>());
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
            using TS = decltype(ts);
            const auto launch = m->group == 32   ? &gemv_int4_launch<T, TS, 32>
                                : m->group == 64 ? &gemv_int4_launch<T, TS, 64>
                                                 : &gemv_int4_launch<T, TS, 128>;
            return launch(p, device, reinterpret_cast<cudaStream_t>(stream), rows, static_cast<const T*>(x), ldx, expert_ids,
                          static_cast<T*>(y), ldy);
        });
    });
}

}  // extern "C"
