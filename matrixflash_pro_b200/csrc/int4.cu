// 4-bit weights: w = (q - z) * s with a scale s and zero point z per row and group of 32, 64 or 128
// columns. Quantising, reading back, and the product with a few rows (decoding).
#include "copy_ring.h"
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
// a / b; a 64-bit division only where a needs it (it takes four times as long as all else that a thread does).
__device__ __forceinline__ long long quotient(long long a, int b) {
    if (static_cast<unsigned long long>(a) >> 32) return a / b;
    return static_cast<unsigned>(a) / static_cast<unsigned>(b);
}

// The integer nearest to w / s, ties to even: the quotient of two FP32 numbers in double precision is never rounded
// onto or across a border between two integers below 2^24.
__device__ __noinline__ int exact_code(float w, float s) {
    return static_cast<int>(rint(fmin(fmax(static_cast<double>(w) / s, -64.0), 64.0)));
}

// clamp(nearest integer to w / s + z, 0, 15), from inv = 1 / s in FP32. The integer that w inv gives may be the wrong
// one next to a border between two; the remainder r = w - q s, exact in FP32, tells: q moves where r is above s / 2, or
// is s / 2 and q odd (16-bit weights and scales meet such ties often: one in a few hundred). below = the FP32 number
// under half = s / 2.
constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer, in the low bits
__device__ __forceinline__ int fast_code(float w, float s, float inv, float half, float below, int z) {
    const float m = fmaf(w, inv, kRound);
    const float r = fmaf(kRound - m, s, w);
    int q = __float_as_int(m);
    const float most = q & 1 ? below : half;
    if (r > most) ++q;
    if (r < -most) --q;
    return __viaddmin_s32_relu(q, z - 0x4b400000, 15);
}

// x / divisor (15 or 7) rounded to double and then to FP32, x = hi - lo. Where x is an FP32 number, so is rounding the
// quotient once: it is never within 2^-30 of the middle between two of them.
__device__ __forceinline__ double scale_of(float hi, float lo, float divisor) {
    const float x = hi - lo, back = x - hi;
    if ((hi - (x - back)) + (-lo - back) == 0.0f) return __fdiv_rn(x, divisor);
    return (static_cast<double>(hi) - lo) / divisor;
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

// Sixteen elements and eight bytes of codes per lane (the bytes of one lane's codes are a whole word or two), so two,
// four or eight lanes to a group, and one division in double precision for a warp's 16, 8 or 4 groups. Bound by
// instruction issue: 31 instructions an element (4096x11008 bf16: issue slots 82% busy, 48 us of which 17 would do for
// the memory); a warp per group, as a first version had it, spent most of its time on the division and on stores of
// single bytes.
// vec: rows of w that start on 16 bytes.
template <typename T, typename TS, int GROUP>
__global__ void __launch_bounds__(256) quantize_int4_kernel(const Int4Params p, const T* __restrict__ w, long long ldw,
                                                            long long stride_w, int cells, bool vec) {
    constexpr int kEach = 16, kLanes = GROUP / kEach;
    const long long unit = blockIdx.x * 256ll + threadIdx.x;  // a lane's 16 columns of a row; `cells` of them a row
    const long long row = quotient(unit, cells);
    const int j0 = static_cast<int>(unit - row * cells) * kEach;
    const bool live = row < p.rows;
    float v[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] = 0.0f;
    if (live) {
        const long long e = p.experts == 1 ? 0 : quotient(row, p.n);
        const T* src = w + e * stride_w + (row - e * p.n) * ldw + j0;
        if (vec && j0 + kEach <= p.k) {
            constexpr int kPer = 16 / sizeof(T);
#pragma unroll
            for (int i = 0; i < kEach / kPer; ++i) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(src) + i);
                const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
                for (int j = 0; j < kPer; ++j) v[i * kPer + j] = to_f32(t[j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (j0 + i < p.k) v[i] = to_f32(src[i]);
        }
    }
    float lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) lo = fminf(lo, v[i]), hi = fmaxf(hi, v[i]);
#pragma unroll
    for (int d = kLanes / 2; d; d /= 2) {
        lo = fminf(lo, __shfl_xor_sync(~0u, lo, d));
        hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, d));
    }
    const double range = p.zeros ? scale_of(hi, lo, 15.0f) : scale_of(fmaxf(-lo, hi), 0.0f, 7.0f);
    TS scale = saturated_scale<TS>(range);
    if (to_f32(scale) == 0.0f) scale = from_f32<TS>(1.0f);
    const float s = to_f32(scale), inv = 1.0f / s;
    // A saturated scale (quotients beyond the fast path's integers) or one without an FP32 reciprocal.
    const bool odd = range > 2.0 * s || s < 1e-37f;
    const float half = 0.5f * s, below = __int_as_float(__float_as_int(half) - 1);
    int z = 8;
    if (p.zeros) z = odd ? min(max(exact_code(-lo, s), 0), 15) : fast_code(-lo, s, inv, half, below, 0);
    if (!live) return;
    if (threadIdx.x % kLanes == 0 && j0 < p.groups * GROUP) {
        const long long at = row * p.groups + j0 / GROUP;
        static_cast<TS*>(p.scales)[at] = scale;
        if (p.zeros) p.zeros[at] = static_cast<unsigned char>(z);
    }
    if (j0 / 2 >= p.row_bytes) return;
    uint32_t codes[2] = {0, 0};
    if (!odd) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            codes[i / 8] |= static_cast<uint32_t>(fast_code(v[i], s, inv, half, below, z)) << (4 * (i % 8));
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            codes[i / 8] |= static_cast<uint32_t>(min(max(exact_code(v[i], s) + z, 0), 15)) << (4 * (i % 8));
    }
    *reinterpret_cast<uint2*>(p.packed + row * p.row_bytes + j0 / 2) = make_uint2(codes[0], codes[1]);
}

// Sixteen columns of a row per lane: one load of codes, one scale, stores of 16 bytes where the rows allow it (vec).
// 4096x11008 bf16: 15 instructions an element, issue slots 74% busy, 26.5 us of which 17 would do for the memory.
template <typename TS, typename T>
__global__ void __launch_bounds__(256) dequantize_int4_kernel(const Int4Params p, T* __restrict__ out, long long ldo,
                                                              long long stride_o, int cells, bool vec) {
    constexpr int kEach = 16;
    const long long unit = blockIdx.x * 256ll + threadIdx.x;
    const long long row = quotient(unit, cells);
    const int j0 = static_cast<int>(unit - row * cells) * kEach;
    if (row >= p.rows || j0 >= p.k) return;
    const uint2 codes = __ldg(reinterpret_cast<const uint2*>(p.packed + row * p.row_bytes + j0 / 2));
    const long long at = row * p.groups + j0 / p.group;
    const float s = to_f32(static_cast<const TS*>(p.scales)[at]);
    const float z = 8388608.0f + (p.zeros ? static_cast<float>(p.zeros[at]) : 8.0f);
    const long long e = p.experts == 1 ? 0 : quotient(row, p.n);
    T* dst = out + e * stride_o + (row - e * p.n) * ldo + j0;
    alignas(16) T v[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        v[i] = from_f32<T>((__uint_as_float((((i < 8 ? codes.x : codes.y) >> (4 * (i % 8))) & 15u) | 0x4b000000u) - z) * s);  // 2^23 + q
    if (vec && j0 + kEach <= p.k) {
#pragma unroll
        for (int i = 0; i < kEach * static_cast<int>(sizeof(T)) / 16; ++i)
            reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(v)[i];
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (j0 + i < p.k) dst[i] = v[i];
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
// the same accumulator, small ones first (below 2^-110 the third one falls under BF16's smallest number, and up to
// 2^-134 of the value is lost).
//
// Which columns meet in one MMA step is free as long as A and B agree, so a word of eight codes serves two steps as
// it lies: (word >> 4 i) & 0x000f000f holds codes i and i + 4. The four lanes of a row take four words of one group
// at a time, so that all columns of a step share one scale.
//
// One block of 16 warps per SM takes an even share of the 16-row tiles. Its warps split the columns (KW warps,
// every KW-th chunk each) and, where there are fewer chunks than warps, the tiles. A warp goes chunk by chunk
// through the tiles, two side by side (two independent MMA chains), so a chunk of x is loaded and laid out once for
// all of them. Codes come by TMA into a ring that belongs to the warp; the scales and zero points of a block's tiles
// by one bulk copy (loads of a few bytes per row into registers cost as much time as all else together: 108 us
// against 61 for 9 of 16 experts of 2048 x 16384). Sums wait in shared memory, a slot per tile, warp and lane, and
// are added up in a fixed order.

// Codes as 16-bit floats. The bits of a code in the low half of a 16-bit word are a subnormal number, q times the
// type's smallest one (in bits 4-7: 16 times that; BF16's exponent field is still 0 or 1 there), and one FMA by a
// power of two less z gives (q - z) * kUnit exactly. A word of eight codes costs one shift, four ANDs, four FMAs.
struct Int4MathF16 {
    static constexpr float kUnit = 0x1p-10f;
    static constexpr uint32_t kLow = 0x74007400u, kHigh = 0x64006400u, kMinusLow = 0xf400f400u;  // 2^14, 2^10, -2^14
    __device__ __forceinline__ static uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
        uint32_t d;
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
        return d;
    }
    __device__ __forceinline__ static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                               const float (&c)[4]) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    }
};
struct Int4MathBf16 {
    static constexpr float kUnit = 0x1p-6f;
    static constexpr uint32_t kLow = 0x7f007f00u, kHigh = 0x7d007d00u, kMinusLow = 0xff00ff00u;  // 2^127, 2^123, -2^127
    __device__ __forceinline__ static uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
        uint32_t d;
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
        return d;
    }
    __device__ __forceinline__ static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                               const float (&c)[4]) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    }
};
template <typename T>
struct Int4Math : Int4MathF16 {
    static constexpr int kTerms = 1;
};
template <>
struct Int4Math<__nv_bfloat16> : Int4MathBf16 {
    static constexpr int kTerms = 1;
};
template <>
struct Int4Math<float> : Int4MathBf16 {
    static constexpr int kTerms = 3;
};

// -z * kUnit in both halves, z being byte `group` of zeros.
template <typename Math>
__device__ __forceinline__ uint32_t int4_zero(uint32_t zeros, int group) {
    return Math::fma2(__byte_perm(zeros, 0, 0x4040 + 0x0101 * group), Math::kMinusLow, 0x80008000u);
}
// (q - z) * kUnit for codes i and i + 4 of a word, i = 0..3.
template <typename Math>
__device__ __forceinline__ void int4_weights(uint32_t word, uint32_t zero, uint32_t (&out)[4]) {
    out[0] = Math::fma2(word & 0x000f000fu, Math::kLow, zero);
    out[1] = Math::fma2(word & 0x00f000f0u, Math::kHigh, zero);
    word >>= 8;
    out[2] = Math::fma2(word & 0x000f000fu, Math::kLow, zero);
    out[3] = Math::fma2(word & 0x00f000f0u, Math::kHigh, zero);
}

// Eight consecutive values of a row of x from column j on, 0 behind column k.
template <typename T>
struct GemvX8 {
    uint32_t w[2 * sizeof(T)];

    __device__ __forceinline__ void load(const T* row, int j, int k, bool vec) {
        if (vec && j + 8 <= k) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + j) + i);
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
        } else if constexpr (sizeof(T) == 2) {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(row) + j;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = j + 2 * i < k ? __ldg(h + 2 * i) : 0, hi = j + 2 * i + 1 < k ? __ldg(h + 2 * i + 1) : 0;
                w[i] = lo | hi << 16;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = j + i < k ? __ldg(reinterpret_cast<const uint32_t*>(row) + j + i) : 0;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 2 * static_cast<int>(sizeof(T)); ++i) w[i] = 0;
    }
    // B registers of the two steps that a word of codes serves: values (0, 4), (1, 5) and (2, 6), (3, 7), per term.
    template <int TERMS>
    __device__ __forceinline__ void lay_out(uint32_t (&b)[TERMS][4]) const {
        uint32_t v[TERMS][4];
        if constexpr (TERMS == 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[0][i] = w[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float lo = __uint_as_float(w[2 * i]), hi = __uint_as_float(w[2 * i + 1]);
                asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(v[0][i]) : "f"(hi), "f"(lo));
#pragma unroll
                for (int t = 1; t < TERMS; ++t) {
                    lo -= __uint_as_float(v[t - 1][i] << 16);
                    hi -= __uint_as_float(v[t - 1][i] & 0xffff0000u);
                    // An infinity is its own first term, and the others are 0 (inf - inf is NaN). A NaN stays one.
                    if (t == 1 && __uint_as_float(w[2 * i] & 0x7fffffffu) == __int_as_float(0x7f800000)) lo = 0.0f;
                    if (t == 1 && __uint_as_float(w[2 * i + 1] & 0x7fffffffu) == __int_as_float(0x7f800000)) hi = 0.0f;
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v[t][i]) : "f"(hi), "f"(lo));
                }
            }
        }
#pragma unroll
        for (int u = 0; u < TERMS; ++u)
#pragma unroll
            for (int step = 0; step < 2; ++step) {
                b[u][2 * step] = __byte_perm(v[u][step], v[u][step + 2], 0x5410);
                b[u][2 * step + 1] = __byte_perm(v[u][step], v[u][step + 2], 0x7632);
            }
    }
};

// Scales (or zero points, a byte each) of one row and chunk.
template <typename TS, int GROUPS>
struct alignas(GROUPS * sizeof(TS)) GemvScales {
    TS v[GROUPS];
};

// Copies `bytes` from global to shared memory, both 16-byte aligned: the whole 16 bytes by TMA onto `bar`, whose
// expected bytes it returns, the last few by this thread.
__device__ __forceinline__ uint32_t copy_bulk(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
    const uint32_t whole = bytes & ~15u;
    for (uint32_t i = whole; i < bytes; ++i)
        static_cast<unsigned char*>(to)[i] = static_cast<const unsigned char*>(from)[i];
    if (whole)
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to)),
                     "l"(from), "r"(whole), "r"(smem_u32(bar))
                     : "memory");
    return whole;
}

// Lane t's word i of the 64 bytes that 128 columns take: words of one group are GROUP / 32 slots in a row per lane.
template <int GROUP>
__device__ __forceinline__ int slot_word(int t, int i) {
    constexpr int kSlots = GROUP / 32;
    return i / kSlots * 4 * kSlots + t * kSlots + i % kSlots;
}

// Row of a tile (0..7, and 8 more) that lanes 4 g .. 4 g + 3 take. Any order would do; this one lets the lanes that
// read shared memory together read different banks of the swizzled box.
template <int GROUP, int HALVES>
__device__ __forceinline__ int tile_row(int g) {
    if (HALVES == 1 || GROUP == 32) return g;
    return GROUP == 64 ? (g << 1 & 6) | g >> 2 : g >> 1 | (g & 1) << 2;
}
template <int GROUP, int HALVES>
__device__ __forceinline__ int tile_lane(int row) {
    if (HALVES == 1 || GROUP == 32) return row;
    return GROUP == 64 ? row >> 1 | (row & 1) << 2 : (row << 1 & 6) | row >> 2;
}

constexpr int kGemvWarps = 16;
constexpr int kGemvDepth = 4;  // KB of codes in flight per warp: 64 KB per SM
constexpr int kGemvRing = kGemvWarps * kGemvDepth * 1024;
constexpr int kGemvSmem = 224 * 1024;  // the ring, then sums and scales of as many tiles as fit

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
            if (blockIdx.x == 0) report_bad_index();
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

// x_vec: 16-byte aligned rows of x; s_bulk: scales and zero points of whole chunks that a bulk copy can take; kw_log:
// log2 of the warps along k; most: tiles whose sums and scales shared memory holds.
template <typename T, typename TS, int GROUP, int RT, int HALVES>
__global__ void __launch_bounds__(32 * kGemvWarps, 1)
    gemv_int4_kernel(const __grid_constant__ CUtensorMap codes, const Int4Params p, int rows, const T* __restrict__ x,
                     long long ldx, const int* __restrict__ ids, T* __restrict__ y, long long ldy, bool x_vec, bool s_bulk,
                     int kw_log, int most, uint64_t wait_limit_ns) {
    using Math = Int4Math<T>;
    constexpr int kTerms = Math::kTerms, kCols = 8 * RT, kChunk = 128 * HALVES, kGroups = kChunk / GROUP;
    constexpr int kSlots = GROUP / 32, kDepth = kGemvDepth / HALVES;
    extern __shared__ __align__(1024) uint4 ring[];                   // [warp][stage][16 rows][4 * HALVES pieces]
    float4* sums = reinterpret_cast<float4*>(ring + kGemvRing / 16);  // [tile][kw][RT][lane]
    __shared__ GemvSegments seg;
    __shared__ uint64_t bars[kGemvWarps][kDepth], scale_bar;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, t = lane % 4;
    const int my_row = tile_row<GROUP, HALVES>(lane / 4);  // and 8 more
    if (warp == 0) gemv_segments(p, ids, rows, lane, seg);
    if (lane < kDepth) {
        mbar_init(&bars[warp][lane], 1);
        if (threadIdx.x == 0) mbar_init(&scale_bar, 1);
        fence_barrier_init();
        fence_proxy_async_smem();
    }
    __syncthreads();

    const int kw_count = 1 << kw_log, kw = warp & (kw_count - 1), tw = warp >> kw_log, tw_count = kGemvWarps >> kw_log;
    const int chunks = (p.k + kChunk - 1) / kChunk, tiles = (p.n + 15) / 16;
    uint4* my_ring = ring + warp * kGemvDepth * 64;
    float4* my_sums = sums + ((tw << kw_log) + kw) * RT * 32 + lane;
    TS* scales = reinterpret_cast<TS*>(sums + (most << kw_log) * RT * 32);                     // [tile][16 rows][group]
    unsigned char* zeros = reinterpret_cast<unsigned char*>(scales + most * 16 * p.groups);
    const bool whole = p.groups % kGroups == 0;  // every chunk has all its groups, vectors are aligned
    CopyRing<kDepth> copies;
    uint32_t scale_parity = 0;
    bool ok = true;
    // An even share of all tiles: segment d, tiles m0 .. of it, left of them in all.
    const unsigned all = static_cast<unsigned>(seg.count) * tiles, share = all / gridDim.x, more = all % gridDim.x;
    const unsigned from = blockIdx.x * share + min(blockIdx.x, more);
    int left = static_cast<int>(share + (blockIdx.x < more ? 1 : 0));
    int d = static_cast<int>(from / tiles), m0 = static_cast<int>(from - d * static_cast<unsigned>(tiles));
    for (int count; ok && left > 0; left -= count, m0 += count) {
        if (m0 == tiles) m0 = 0, ++d;
        count = min(min(left, tiles - m0), most);
        const int mine = (count - tw + tw_count - 1) / tw_count;  // tiles of this warp: tw, tw + tw_count, ..
        const long long row0 = static_cast<long long>(seg.expert[d]) * p.n;
        const int x_first = seg.begin[d], x_count = seg.begin[d + 1] - x_first;
        const TS* s_matrix = static_cast<const TS*>(p.scales) + row0 * p.groups;
        const unsigned char* z_matrix = p.zeros + row0 * p.groups;
        if (s_bulk && threadIdx.x == 0) {
            const long long first = static_cast<long long>(m0) * 16 * p.groups;
            const uint32_t cells = static_cast<uint32_t>(min(count * 16, p.n - m0 * 16)) * p.groups;
            uint32_t bytes = copy_bulk(scales, s_matrix + first, cells * static_cast<uint32_t>(sizeof(TS)), &scale_bar);
            if (p.zeros) bytes += copy_bulk(zeros, z_matrix + first, cells, &scale_bar);
            mbar_arrive_expect_tx(&scale_bar, bytes);
        }
        bool scales_here = !s_bulk;
        for (int c0 = 0; c0 < x_count; c0 += kCols) {
            // Codes: this warp's tiles of chunk kw, then of chunk kw + kw_count, ..
            int load_chunk = mine > 0 ? kw : chunks, load_tile = 0;
            const int box_row = static_cast<int>(row0) + (m0 + tw) * 16;  // rows past the matrix: read, or 0, and not used
            auto load = [&]() {
                if (load_chunk >= chunks) return;
                if (lane == 0) {
                    const unsigned s = copies.next();
                    mbar_arrive_expect_tx(&bars[warp][s], 1024 * HALVES);
                    tma_load_2d(my_ring + s * 64 * HALVES, &codes, &bars[warp][s], load_chunk * 64 * HALVES,
                                box_row + load_tile * tw_count * 16);
                }
                ++copies.issued;
                if (++load_tile == mine) load_tile = 0, load_chunk += kw_count;
            };
#pragma unroll 1
            for (int i = 0; i < kDepth; ++i) load();

            const T* xr[RT];  // the row of x in this lane's column of B
            bool live[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int c = c0 + 8 * r + lane / 4;
                live[r] = c < x_count;
                xr[r] = x + (live[r] ? seg.order[x_first + c] : 0) * ldx;
            }
            // Scales and zero points (a byte per group) of row r of the tiles, groups of half b of a chunk.
            using Scales = GemvScales<TS, 128 / GROUP>;
            auto read_scales = [&](int r, int chunk, int b, Scales& s, uint32_t& z) {
                constexpr int kHalf = 128 / GROUP;
                const int g0 = chunk * kGroups + b * kHalf;
                z = 0x08080808u;
                if (s_bulk && whole) {
                    s = *reinterpret_cast<const Scales*>(scales + r * p.groups + g0);
                    if (p.zeros) {
                        const unsigned char* at = zeros + r * p.groups + g0;
                        if (kHalf == 4) z = *reinterpret_cast<const uint32_t*>(at);
                        else if (kHalf == 2) z = *reinterpret_cast<const uint16_t*>(at);
                        else z = *at;
                    }
                    return;
                }
                const long long at = static_cast<long long>(min(m0 * 16 + r, p.n - 1)) * p.groups;
                const TS* sp = s_bulk ? scales + r * p.groups : s_matrix + at;
                const unsigned char* zp = s_bulk ? zeros + r * p.groups : z_matrix + at;
                if (p.zeros) z = 0;
#pragma unroll
                for (int i = 0; i < kHalf; ++i) {
                    const bool in = g0 + i < p.groups;
                    s.v[i] = in ? sp[g0 + i] : from_f32<TS>(0.0f);
                    if (p.zeros && in) z |= static_cast<uint32_t>(zp[g0 + i]) << (8 * i);
                }
            };

            uint32_t xb[HALVES][RT][4][kTerms][4];
            // N tiles from tile j on: independent chains of MMAs side by side. A wait that gives up ends it for the whole
            // warp, before anything is read or another copy started.
            auto step_over = [&](auto n_, int j, int chunk) {
                constexpr int N = decltype(n_)::value;
                const uint32_t* box[N];
#pragma unroll
                for (int u = 0; u < N; ++u) {
                    ok = ok && mbar_wait_bounded(&bars[warp][copies.stage(u)], copies.parity(u), wait_limit_ns, nullptr);
                    box[u] = reinterpret_cast<const uint32_t*>(my_ring + copies.stage(u) * 64 * HALVES);
                }
                ok = __all_sync(~0u, ok);
                if (!ok) return;
                float acc[N][RT][4];
#pragma unroll
                for (int b = 0; b < HALVES; ++b) {
                    Scales s[N][2];
                    uint32_t z[N][2], w[N][2][4];
#pragma unroll
                    for (int u = 0; u < N; ++u)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int r = my_row + 8 * h;
                            read_scales((tw + (j + u) * tw_count) * 16 + r, chunk, b, s[u][h], z[u][h]);
                            // 16-byte pieces are swizzled by the row: all 8 pieces of 128 bytes, or 4 of 64
                            const int swizzle = HALVES == 2 ? (r & 7) * 4 : (r >> 1 & 3) * 4;
#pragma unroll
                            for (int i = 0; i < 4; i += kSlots) {
                                const uint32_t* from_w = box[u] + r * 16 * HALVES + ((b * 16 + slot_word<GROUP>(t, i)) ^ swizzle);
                                if constexpr (kSlots == 4) {
                                    const uint4 v = *reinterpret_cast<const uint4*>(from_w);
                                    w[u][h][0] = v.x, w[u][h][1] = v.y, w[u][h][2] = v.z, w[u][h][3] = v.w;
                                } else if constexpr (kSlots == 2) {
                                    const uint2 v = *reinterpret_cast<const uint2*>(from_w);
                                    w[u][h][i] = v.x, w[u][h][i + 1] = v.y;
                                } else {
                                    w[u][h][i] = *from_w;
                                }
                            }
                        }
                    if (b == HALVES - 1) {
                        __syncwarp();  // every lane has read the boxes
                        copies.consumed += N;
#pragma unroll
                        for (int u = 0; u < N; ++u) load();
                    }
                    float part[N][RT][4];
                    uint32_t zero[N][2];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int group = i / kSlots;
#pragma unroll
                        for (int u = 0; u < N; ++u) {
                            uint32_t a[2][4];  // rows my_row + 8 h, codes (i, i + 4)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                if (i % kSlots == 0) zero[u][h] = int4_zero<Math>(z[u][h], group);
                                int4_weights<Math>(w[u][h][i], zero[u][h], a[h]);
                            }
#pragma unroll
                            for (int step = 0; step < 2; ++step) {
                                const uint32_t av[4] = {a[0][2 * step], a[1][2 * step], a[0][2 * step + 1], a[1][2 * step + 1]};
#pragma unroll
                                for (int r = 0; r < RT; ++r)
#pragma unroll
                                    for (int e = kTerms - 1; e >= 0; --e) {
                                        const uint32_t(&xv)[4] = xb[b][r][i][e];
                                        const float none[4] = {};
                                        const bool first = i % kSlots == 0 && step == 0 && e == kTerms - 1;
                                        if (first) Math::mma(part[u][r], av, xv[2 * step], xv[2 * step + 1], none);
                                        else Math::mma(part[u][r], av, xv[2 * step], xv[2 * step + 1], part[u][r]);
                                    }
                            }
                            if (i % kSlots == kSlots - 1) {
                                const float s0 = to_f32(s[u][0].v[group]), s1 = to_f32(s[u][1].v[group]);
#pragma unroll
                                for (int r = 0; r < RT; ++r)
#pragma unroll
                                    for (int e = 0; e < 4; ++e)
                                        acc[u][r][e] = b == 0 && i == kSlots - 1
                                                           ? (e < 2 ? s0 : s1) * part[u][r][e]
                                                           : fmaf(e < 2 ? s0 : s1, part[u][r][e], acc[u][r][e]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < N; ++u)
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        // tile tw + (j + u) tw_count: kw_count slots a tile, kw_count tw_count = kGemvWarps
                        float4& slot = my_sums[((j + u) * kGemvWarps * RT + r) * 32];
                        float4 v = make_float4(acc[u][r][0], acc[u][r][1], acc[u][r][2], acc[u][r][3]);
                        if (chunk != kw) {
                            const float4 o = slot;
                            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
                        }
                        slot = v;
                    }
            };
            for (int chunk = mine > 0 ? kw : chunks; ok && chunk < chunks; chunk += kw_count) {
                GemvX8<T> xn[HALVES][RT][4];
#pragma unroll
                for (int b = 0; b < HALVES; ++b)
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            xn[b][r][i].clear();
                            if (live[r])
                                xn[b][r][i].load(xr[r], chunk * kChunk + b * 128 + slot_word<GROUP>(t, i) * 8, p.k, x_vec);
                        }
#pragma unroll
                for (int b = 0; b < HALVES; ++b)
#pragma unroll
                    for (int r = 0; r < RT; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i) xn[b][r][i].template lay_out<kTerms>(xb[b][r][i]);
                if (!scales_here) {
                    ok = __all_sync(~0u, mbar_wait_bounded(&scale_bar, scale_parity, wait_limit_ns, nullptr));
                    scales_here = true;
                }
                int j = 0;
                for (; ok && j + 2 <= mine; j += 2) step_over(std::integral_constant<int, 2>(), j, chunk);
                if (ok && j < mine) step_over(std::integral_constant<int, 1>(), j, chunk);
            }
            if (!ok && lane == 0) report_status(kStatusTimeoutProducer, nullptr);
            ok = __syncthreads_and(ok);
            if (!ok) break;
            const int split = min(kw_count, chunks);
            for (int at = threadIdx.x; at < count * 16 * kCols; at += 32 * kGemvWarps) {
                const int i = at & 15, rest = at >> 4;  // consecutive threads: consecutive outputs
                const int c = rest % kCols, m = rest / kCols;
                const int out = (m0 + m) * 16 + i;
                if (c0 + c >= x_count || out >= p.n) continue;
                const float* v = reinterpret_cast<const float*>(sums + ((m << kw_log) * RT + c / 8) * 32) +
                                 (tile_lane<GROUP, HALVES>(i & 7) * 4 + c % 8 / 2) * 4 + (i >> 3) * 2 + (c & 1);
                float sum = 0.0f;
                for (int s = 0; s < split; ++s) sum += v[s * RT * 128];
                y[seg.order[x_first + c0 + c] * ldy + out] = from_f32<T>(sum * (1.0f / Math::kUnit));
            }
            __syncthreads();
        }
        scale_parity ^= 1;  // one copy of scales per round of tiles
    }
    // A wait that gave up leaves copies in flight; they land (or the limit passes) before the block ends.
    if (!ok) {
        bool landed = copies.drain([&](unsigned s, unsigned parity) { return mbar_wait_drain(&bars[warp][s], parity, wait_limit_ns); });
        if (left > 0 && s_bulk && threadIdx.x == 0) landed = mbar_wait_drain(&scale_bar, scale_parity, wait_limit_ns) && landed;
        if (!landed) report_status(kStatusTimeoutDrain, nullptr);
    }
    if (seg.begin[seg.count] < rows)  // rows of no expert
        for (int r = 0; r < rows; ++r) {
            const int e = ids[r];
            if (e >= 0 && e < p.experts) continue;
            for (int i = blockIdx.x * 32 * kGemvWarps + threadIdx.x; i < p.n; i += gridDim.x * 32 * kGemvWarps)
                y[r * ldy + i] = from_f32<T>(0.0f);
        }
}

// Boxes of 16 rows x 64 bytes (or 128) of the codes.
mfb_status_t encode_codes(CUtensorMap* map, const void* base, long long rows, int row_bytes, int halves) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(MFB_ECUDA, "cuTensorMapEncodeTiled entry point unavailable");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
    const cuuint32_t box[2] = {64u * halves, 16}, step[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, step,
                          CU_TENSOR_MAP_INTERLEAVE_NONE,
                          halves == 2 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(MFB_ECUDA, "cuTensorMapEncodeTiled failed (code " + std::to_string(static_cast<int>(r)) + ")");
    return MFB_OK;
}

template <typename T, typename TS, int GROUP>
mfb_status_t gemv_int4_launch(const Int4Params& p, int device, cudaStream_t stream, int rows, const T* x, long long ldx,
                              const int* ids, T* y, long long ldy) {
    const bool x_vec = (reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(ldx * sizeof(T))) % 16 == 0;
    auto bulk = [&](const void* base, int size) {
        return aligned16(base) && (p.experts == 1 || static_cast<long long>(p.n) * p.groups * size % 16 == 0);
    };
    bool s_bulk = bulk(p.scales, sizeof(TS)) && (!p.zeros || bulk(p.zeros, 1));
    const long long tiles = static_cast<long long>(ids ? rows : 1) * ((p.n + 15) / 16);
    if (tiles > 0x7fffffffLL) return fail(MFB_EINVAL, "problem has too many output tiles");
    const unsigned grid = static_cast<unsigned>(std::min<long long>(tiles, sm_count(device)));
    auto go = [&](auto rt, auto halves) -> mfb_status_t {
        constexpr int RT = decltype(rt)::value, HALVES = decltype(halves)::value;
        const auto kernel = &gemv_int4_kernel<T, TS, GROUP, RT, HALVES>;
        const int chunks = (p.k + 128 * HALVES - 1) / (128 * HALVES);
        CUtensorMap map{};
        if (p.k > 0 && p.rows > 0) MFB_TRY(encode_codes(&map, p.packed, p.rows, p.row_bytes, HALVES));
        static std::atomic<unsigned long long> raised{0};  // devices whose shared-memory limit is raised
        const unsigned long long bit = 1ull << (device & 63);
        if (!(raised.load(std::memory_order_acquire) & bit)) {
            MFB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemvSmem),
                         "cudaFuncSetAttribute(gemv_int4)");
            raised.fetch_or(bit, std::memory_order_release);
        }
        // Warps along k: the split with the fewest steps per warp; of equal ones the widest whose sums fit at once,
        // since every further round of tiles starts its loads anew.
        const long long each = (tiles + grid - 1) / grid;
        const long long scale_bytes = 16ll * p.groups * (sizeof(TS) + (p.zeros ? 1 : 0));
        if (scale_bytes > 32768) s_bulk = false;  // rows of millions of columns
        auto room = [&](int log) {
            return static_cast<int>((kGemvSmem - kGemvRing) / ((512ll * RT << log) + (s_bulk ? scale_bytes : 0)));
        };
        long long best = 0;
        int kw_log = -1;
        for (int log = 4; log >= 0; --log) {
            const long long steps = ((each << log) + kGemvWarps - 1) / kGemvWarps * ((chunks + (1 << log) - 1) >> log);
            if (kw_log < 0 || steps < best || (steps == best && room(kw_log) < each)) best = steps, kw_log = log;
        }
        const int most = room(kw_log);
        kernel<<<grid, 32 * kGemvWarps, kGemvSmem, stream>>>(map, p, rows, x, ldx, ids, y, ldy, x_vec, s_bulk, kw_log, most,
                                                             wait_limit_ns());
        MFB_CUDA_TRY(cudaGetLastError(), "gemv_int4 launch");
        return MFB_OK;
    };
    // Two column tiles of x keep 16 rows in one pass over the codes; FP32 rows have no registers for that, and neither
    // they nor two tiles for 256 columns of x at a time.
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    if constexpr (sizeof(T) == 2) {
        if (rows > 8 && !ids) return go(Two(), One());
        return go(One(), Two());
    } else {
        return go(One(), One());
    }
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
    if (p->rows > INT32_MAX - 65536 || m->k > INT32_MAX - 65536)
        return fail(MFB_EINVAL, "4-bit matrix dimension exceeds the 32-bit limit");
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

bool overlap(const void* a, long long a_bytes, const void* b, long long b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + static_cast<uintptr_t>(b_bytes) && y < x + static_cast<uintptr_t>(a_bytes);
}

// Whether [at, at + bytes) reaches into the codes, scales or zero points.
bool overlaps_matrix(const Int4Params& p, int scale_dtype, const void* at, long long bytes) {
    const long long scales = p.rows * p.groups;
    return overlap(at, bytes, p.packed, p.rows * p.row_bytes) ||
           overlap(at, bytes, p.scales, scales * dtype_bytes(scale_dtype)) || overlap(at, bytes, p.zeros, scales);
}

// Bytes from the first to behind the last element of `m`'s rows in a caller's matrix.
long long rows_extent(const Int4Params& p, int dtype, long long ld, long long stride) {
    return ((p.n - 1ll) * ld + (p.experts - 1ll) * stride + p.k) * dtype_bytes(dtype);
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
    if (overlaps_matrix(p, out->scale_dtype, w, rows_extent(p, dtype, ldw, stride_w)))
        return fail(MFB_EINVAL, "a 4-bit matrix cannot alias the weights that it is made from");
    DeviceGuard guard;
    MFB_TRY(select_device(device));
    const int cells = p.groups * (p.group / 16);  // whole groups, so that a group's lanes are in one warp
    const long long blocks = (p.rows * cells + 255) / 256;
    if (blocks > 0x7fffffffLL) return fail(MFB_EINVAL, "4-bit matrix has too many groups");
    const long long size = dtype_bytes(dtype);
    const bool vec = aligned16(w) && (p.n <= 1 || ldw * size % 16 == 0) && (p.experts == 1 || stride_w * size % 16 == 0);
    return with_dtype(dtype, [&](auto t) {
        return with_dtype(out->scale_dtype, [&](auto ts) {
            using T = decltype(t);
            using TS = decltype(ts);
            const auto kernel = out->group == 32   ? &quantize_int4_kernel<T, TS, 32>
                                : out->group == 64 ? &quantize_int4_kernel<T, TS, 64>
                                                   : &quantize_int4_kernel<T, TS, 128>;
            kernel<<<static_cast<unsigned>(blocks), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                p, static_cast<const T*>(w), ldw, stride_w, cells, vec);
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
    if (overlaps_matrix(p, m->scale_dtype, out, rows_extent(p, dtype, ldo, stride_o)))
        return fail(MFB_EINVAL, "the weights of a 4-bit matrix cannot alias its parts");
    DeviceGuard guard;
    MFB_TRY(select_device(device));
    const int cells = p.row_bytes / 8;
    const long long blocks = (p.rows * cells + 255) / 256;
    if (blocks > 0x7fffffffLL) return fail(MFB_EINVAL, "4-bit matrix is too large");
    const long long size = dtype_bytes(dtype);
    const bool vec = aligned16(out) && (p.n <= 1 || ldo * size % 16 == 0) && (p.experts == 1 || stride_o * size % 16 == 0);
    return with_dtype(m->scale_dtype, [&](auto ts) {
        return with_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            dequantize_int4_kernel<decltype(ts), T><<<static_cast<unsigned>(blocks), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
                p, static_cast<T*>(out), ldo, stride_o, cells, vec);
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
    if (reinterpret_cast<uintptr_t>(expert_ids) % 4) return fail(MFB_EINVAL, "expert ids must be aligned to 4 bytes");
    const long long y_bytes = ((rows - 1) * ldy + p.n) * dtype_bytes(dtype);
    if (p.k > 0 && overlap(y, y_bytes, x, ((rows - 1) * ldx + p.k) * dtype_bytes(dtype)))
        return fail(MFB_EINVAL, "GEMV output cannot alias x");
    if (overlaps_matrix(p, m->scale_dtype, y, y_bytes) || overlap(y, y_bytes, expert_ids, 4ll * rows))
        return fail(MFB_EINVAL, "GEMV output cannot alias the matrix or the expert ids");
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
