// 4-bit weights: w = (q - z) * s with a scale s and zero point z per row and group of 32, 64 or 128
// columns. Quantising, reading back, and the product with a few rows (decoding).
#include "mfb_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
// The codes are read once and everything else fits beside that: a warp takes 16 * MT output rows and 128
// columns at a time (16 bytes of codes per row and lane, four lanes to a row), turns codes into the exact
// 16-bit integers q - z and feeds them to m16n8k16 MMAs as A, with up to 8 * RT rows of x as B. A group's sum
// is an FP32 accumulator, its scale one FMA per accumulator. FP32 rows enter as three BF16 terms (exact),
// added into the same accumulator, small ones first.
//
// Which columns meet in one MMA step is free as long as A and B agree, so a lane's word of eight codes serves two
// steps as it lies: (word >> 4 i) & 0x000f000f holds codes i and i + 4. For groups of 64 and 32 the four lanes of
// a row exchange words first, so that all columns of a step share one scale.
//
// The 8 warps of a block take every eighth chunk of the same rows and add up in shared memory in a fixed order.

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

// A chunk's codes, scales and zero points for the 2 * MT rows of a lane.
template <typename TS, int GROUP, int MT>
struct Int4Chunk {
    static constexpr int kGroups = 128 / GROUP;
    uint4 w[MT][2];
    TS s[MT][2][kGroups];
    uint32_t z[MT][2];  // one byte per group

    __device__ __forceinline__ void load(const Int4Params& p, long long row0, int n_left, int chunk, int lane, bool vec) {
        const int byte = chunk * 64 + lane % 4 * 16;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const long long row = row0 + min(mt * 16 + h * 8 + lane / 4, n_left - 1);  // rows past the end repeat the last
                const unsigned char* src = p.packed + row * p.row_bytes + byte;
                w[mt][h] = make_uint4(0, 0, 0, 0);
                if (byte < p.row_bytes)
                    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(w[mt][h].x), "=r"(w[mt][h].y), "=r"(w[mt][h].z), "=r"(w[mt][h].w)
                                 : "l"(src));
                const long long at = row * p.groups + chunk * kGroups;
                const TS* sp = static_cast<const TS*>(p.scales) + at;
                z[mt][h] = 0x08080808u;
                if (vec) {  // whole chunks of groups, aligned
                    struct alignas(sizeof(TS) * kGroups) Vec {
                        TS v[kGroups];
                    };
                    const Vec v = *reinterpret_cast<const Vec*>(sp);
#pragma unroll
                    for (int i = 0; i < kGroups; ++i) s[mt][h][i] = v.v[i];
                    if (p.zeros) {
                        if (kGroups == 4) z[mt][h] = __ldg(reinterpret_cast<const uint32_t*>(p.zeros + at));
                        else if (kGroups == 2) z[mt][h] = __ldg(reinterpret_cast<const uint16_t*>(p.zeros + at));
                        else z[mt][h] = __ldg(p.zeros + at);
                    }
                } else {
                    if (p.zeros) z[mt][h] = 0;
#pragma unroll
                    for (int i = 0; i < kGroups; ++i) {
                        const bool in = chunk * kGroups + i < p.groups;
                        s[mt][h][i] = in ? sp[i] : from_f32<TS>(0.0f);
                        if (p.zeros && in) z[mt][h] |= static_cast<uint32_t>(__ldg(p.zeros + at + i)) << (8 * i);
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

constexpr int kGemvWarps = 8;

// blockIdx.x: 16 * MT output rows. With ids, blockIdx.y is a row of x, and the block serves all rows of that row's
// expert if it is the first of them. x_vec, s_vec: 16-byte (32 for FP32) rows of x, aligned chunks of scales.
template <typename T, typename TS, int GROUP, int MT, int RT>
__global__ void __launch_bounds__(32 * kGemvWarps)
    gemv_int4_kernel(const Int4Params p, int rows, const T* __restrict__ x, long long ldx, const int* __restrict__ ids,
                     T* __restrict__ y, long long ldy, bool x_vec, bool s_vec) {
    using Math = Int4Math<T>;
    constexpr int kOut = 16 * MT, kCols = 8 * RT, kPad = kOut + 1;
    __shared__ float sums[kGemvWarps][kCols][kPad];
    __shared__ unsigned char list[MFB_INT4_GEMV_ROWS];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, t = lane % 4;
    const int i0 = blockIdx.x * kOut, n_left = p.n - i0;
    int count = rows, expert = 0;
    if (ids) {
        const int mine = blockIdx.y;
        const int a = lane < rows ? ids[lane] : -1, b = lane + 32 < rows ? ids[lane + 32] : -1;
        expert = ids[mine];
        if (expert < 0 || expert >= p.experts) {
            if (expert >= p.experts && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(&g_status, kStatusBadIndex);
            if (threadIdx.x < kOut && threadIdx.x < n_left) y[mine * ldy + i0 + threadIdx.x] = from_f32<T>(0.0f);
            return;
        }
        const unsigned low = __ballot_sync(~0u, a == expert), high = __ballot_sync(~0u, b == expert);
        const unsigned long long same = static_cast<unsigned long long>(high) << 32 | low;
        if (__ffsll(static_cast<long long>(same)) - 1 != mine) return;
        count = __popcll(same);
        if (warp == 0) {
            const unsigned below = (1u << lane) - 1;
            if (a == expert) list[__popc(low & below)] = static_cast<unsigned char>(lane);
            if (b == expert) list[__popc(low) + __popc(high & below)] = static_cast<unsigned char>(lane + 32);
        }
        __syncthreads();
    }
    const long long row0 = static_cast<long long>(expert) * p.n + i0;
    const int chunks = (p.k + 127) / 128;
    for (int first = 0; first < count; first += kCols) {
        const T* xr[RT];  // the row of x in this lane's column of B
        bool live[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int c = first + 8 * r + lane / 4;
            live[r] = c < count;
            xr[r] = x + (live[r] ? (ids ? list[c] : c) : 0) * ldx;
        }
        float acc[MT][RT][4] = {};
        Int4Chunk<TS, GROUP, MT> next;
        if (warp < chunks) next.load(p, row0, n_left, warp, lane, s_vec);
        for (int chunk = warp; chunk < chunks; chunk += kGemvWarps) {
            Int4Chunk<TS, GROUP, MT> cur = next;
            if (chunk + kGemvWarps < chunks) next.load(p, row0, n_left, chunk + kGemvWarps, lane, s_vec);
            uint32_t w[MT][2][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    w[mt][h][0] = cur.w[mt][h].x, w[mt][h][1] = cur.w[mt][h].y;
                    w[mt][h][2] = cur.w[mt][h].z, w[mt][h][3] = cur.w[mt][h].w;
                    regroup<GROUP>(w[mt][h], t);
                }
            float part[MT][RT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                constexpr int kSlots = GROUP / 32;  // word slots of a group
                if (i % kSlots == 0)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int r = 0; r < RT; ++r)
#pragma unroll
                            for (int e = 0; e < 4; ++e) part[mt][r][e] = 0.0f;
                uint32_t xv[RT][Math::kTerms][4];
                const int j = chunk * 128 + slot_column<GROUP>(t, i);
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    if (live[r]) {
                        load_x8<T>(xr[r], j, p.k, x_vec, xv[r]);
                    } else {
#pragma unroll
                        for (int u = 0; u < Math::kTerms; ++u)
#pragma unroll
                            for (int e = 0; e < 4; ++e) xv[r][u][e] = 0;
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    uint32_t lo[4], hi[4];  // rows g and g + 8, codes (i, i + 4)
                    const int group = i / kSlots;
                    Math::weights(w[mt][0][i], (cur.z[mt][0] >> (8 * group)) & 15u, lo);
                    Math::weights(w[mt][1][i], (cur.z[mt][1] >> (8 * group)) & 15u, hi);
#pragma unroll
                    for (int step = 0; step < 2; ++step) {
                        const uint32_t a[4] = {lo[2 * step], hi[2 * step], lo[2 * step + 1], hi[2 * step + 1]};
#pragma unroll
                        for (int r = 0; r < RT; ++r)
#pragma unroll
                            for (int u = Math::kTerms - 1; u >= 0; --u)
                                Math::mma(part[mt][r], a, __byte_perm(xv[r][u][step], xv[r][u][step + 2], 0x5410),
                                          __byte_perm(xv[r][u][step], xv[r][u][step + 2], 0x7632));
                    }
                    if (i % kSlots == kSlots - 1) {
                        const float s0 = to_f32(cur.s[mt][0][group]), s1 = to_f32(cur.s[mt][1][group]);
#pragma unroll
                        for (int r = 0; r < RT; ++r)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[mt][r][e] = fmaf(e < 2 ? s0 : s1, part[mt][r][e], acc[mt][r][e]);
                    }
                }
            }
        }
        if (first > 0) __syncthreads();  // the sums of the rows before have been read
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) sums[warp][8 * r + 2 * t + (e & 1)][16 * mt + lane / 4 + 8 * (e >> 1)] = acc[mt][r][e];
        __syncthreads();
        for (int at = threadIdx.x; at < kOut * kCols; at += 32 * kGemvWarps) {
            const int c = at / kOut, i = at % kOut;
            if (first + c >= count || i >= n_left) continue;
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < kGemvWarps; ++v) sum += sums[v][c][i];
            y[(ids ? list[first + c] : first + c) * ldy + i0 + i] = from_f32<T>(sum);
        }
    }
}

template <typename T, typename TS, int GROUP>
mfb_status_t gemv_int4_launch(const Int4Params& p, cudaStream_t stream, int rows, const T* x, long long ldx, const int* ids,
                              T* y, long long ldy) {
    constexpr int kVec = 8 * sizeof(T) < 16 ? 8 * sizeof(T) : 16;
    const bool x_vec = (reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(ldx * sizeof(T))) % kVec == 0;
    constexpr int kGroups = 128 / GROUP;
    const bool s_vec = p.groups % kGroups == 0 && reinterpret_cast<uintptr_t>(p.scales) % (sizeof(TS) * kGroups) == 0 &&
                       reinterpret_cast<uintptr_t>(p.zeros) % kGroups == 0;
    auto go = [&](auto mt, auto rt) {
        constexpr int MT = decltype(mt)::value, RT = decltype(rt)::value;
        const dim3 grid(static_cast<unsigned>((p.n + 16 * MT - 1) / (16 * MT)), ids ? static_cast<unsigned>(rows) : 1u);
        gemv_int4_kernel<T, TS, GROUP, MT, RT><<<grid, 32 * kGemvWarps, 0, stream>>>(p, rows, x, ldx, ids, y, ldy, x_vec, s_vec);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    if (rows <= 8) {
        if (p.n >= 32 * 148) go(Two{}, One{});
        else go(One{}, One{});
    } else {
        if (p.n >= 32 * 148) go(Two{}, Two{});
        else go(One{}, Two{});
    }
    MFB_CUDA_TRY(cudaGetLastError(), "gemv_int4 launch");
    return MFB_OK;
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
            return launch(p, reinterpret_cast<cudaStream_t>(stream), rows, static_cast<const T*>(x), ldx, expert_ids,
                          static_cast<T*>(y), ldy);
        });
    });
}

}  // extern "C"
