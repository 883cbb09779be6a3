// The tcgen05 kernel of the products grouped by expert.
//
// One accumulator tile D (M x N) has output columns on its M side and output rows on its N side:
//   forward:  D[f, t] = sum_k  op(B_e)[k, f] A[t, k]   N side: rows t of one group
//   gradient: D[j, i] = sum_t  B[t, j]       A[t, i]   contraction over the rows t of one group
// so a TMEM lane is an output column and an accumulator column an output row. Weights always fill the M
// side, whatever a group's size; the N side of an MMA may be any multiple of 16 (32 on SM pairs), so a
// group of 3 rows costs an MMA of 16 or 32 columns and not a tile of 128 rows.
//
// Group sizes are device data. Every CTA scans the offsets once into shared memory (tiles before each
// group), and its roles walk the same tile sequence, dealt out round-robin to the persistent workers.
//
// 16-bit operands whose rows TMA can address come by TMA, 64 of the contraction deep, 128-byte swizzle
// (K-major tiles a box of rows, MN-major tiles boxes of 64 columns). All others (FP32, odd
// strides) come by loader warps that read global memory into registers and write the same layout:
// 16-bit values as they are, FP32 as PLANES BF16 terms x = h + m + l (h cut, m and l rounded). Three are exact down
// to 2^-110; below, l falls under BF16's smallest number and up to 2^-134 of x is lost. An infinity has no terms
// (inf - inf) and gives NaN. Products hh, hm, mh, mm, hl, lh are kept (six MMAs per step, 1/6 of the BF16 rate); what
// is left out is below 2^-21 of |a b|. Two terms (TF32 precision) keep hh, hm, mh.
//
// The tensor core adds with truncation, so the accumulator restarts every 64 of the contraction (strict FP32) or 512
// (all others) and the epilogue warps add the chunks, rounding to nearest: the error does not grow with the
// contraction. (FP32 every 128 instead would save 5% of the time and take the error at k = 4096 from 1.9e-7 to 6e-7.)
// 16-bit operands, k = 4096, 8 experts of 1024 rows, graph replay, by the chunk: 256 662 us, error of the sums 2.4e-7
// (all products positive 3.8e-7); 512 589 us, 4.8e-7 (9e-7); 1024 573 us, 1e-6 (2.2e-6); never restarted 552 us, 4.4e-6
// (1.4e-5, and 8e-5 at k = 16384). 512 is the longest that keeps sums of both signs below 1e-6 for both types (BF16 as
// given, FP16 6.5e-7; 2.8e-6 where all products are positive). What it costs is the hand-over: the next chunk's MMAs
// wait for a buffer whose reader needs 3600 cycles, signals across the pair included, and a chunk's MMAs take 4096.
//
// Bounds, and what it reaches on a B200: 8192 rows over 8 experts, 4096x11008 bf16, single calls 570 us, 1296 TFLOP/s,
// the hand-over of chunks and a last wave (1376 tiles for 74 pairs); call after call 687 us, 1075 TFLOP/s, at 1.3 GHz
// under the power limit (cuBLAS sustains 1387). 32 rows over 32 experts, 2048x1024 bf16, 26.4 us by graph replay, 3.3
// TB/s (160 tiles for 148 SMs). FP32, 3000 rows over 16 experts, 1024x2048, 114 to 171 us by GPU, about 100 TFLOP/s
// of the 279 that six MMAs allow, the work on the terms and a last wave (tensor pipe 38% busy, issue slots 44%).
#pragma once

#include "mfb_device.cuh"
#include "mfb_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace mfb {

constexpr int kGroupedMaxGroups = 1024;
constexpr int kGroupedDepth = 64;  // contraction per stage: one 128-byte row of 16-bit values

struct GroupedParams {
    const int* offsets;
    int groups, rows;       // rows of A
    int n, k;               // C is .. x n; k: contraction (forward) or rows of each C_e (gradient)
    long long ldc, stride_c;
    void* c;
    int out_f32, bf16, zero_rest;
    int m_tiles;            // tiles along the M side (n)
    uint64_t wait_limit_ns;
    // Operands for the loader warps: M side (B) and N side (A). align: bytes that every row start is a multiple of.
    const char* m_base;
    const char* n_base;
    long long m_ld, m_stride, n_ld;  // bytes
    int m_align, n_align;
    int m_shared;  // all groups share one matrix: the tensor map has one
    int m_wide, n_wide;  // MN-major operands whose rows are whole 64-column boxes: one copy brings all boxes of a slab
};

// KS = 64-deep slabs per stage. A stage has a fixed cost of a few hundred cycles (barrier wait, commit) beside its
// MMAs, so four of them (one slab of 16-bit values) are too few.
template <int NT_, int CG_, int PLANES_, bool RIGHT_, bool M_MN_, bool TMA_, int KS_, int STAGES_>
struct GroupedConfig {
    static constexpr int NT = NT_, CG = CG_, PLANES = PLANES_, KS = KS_, STAGES = STAGES_;
    static constexpr bool RIGHT = RIGHT_, TMA = TMA_;
    static constexpr bool M_MN = RIGHT_ || M_MN_;  // M side stored MN-major
    static constexpr bool N_MN = RIGHT_;           // N side stored MN-major
    static constexpr int ES = PLANES == 1 ? 2 : 4;  // bytes of an operand element in memory
    static constexpr int BM = 128 * CG;
    static constexpr int NTC = NT / CG;  // N-side rows of a CTA
    static constexpr int kMPlane = 128 * 128, kNPlane = NTC * 128;
    static constexpr int kMBytes = PLANES * kMPlane, kNBytes = PLANES * kNPlane;
    static constexpr int kSlab = kMBytes + kNBytes;
    static constexpr int kStage = KS * kSlab;
    static constexpr int kSumStages = PLANES == 3 ? 1 : 512 / (kGroupedDepth * KS);  // stages per accumulator chunk
    static constexpr int kBarriers = STAGES * kStage;
    static constexpr int kTables = kBarriers + 8 * (4 * STAGES + 5) + 8;
    static constexpr int kSmem = kTables + 8 * (kGroupedMaxGroups + 1) + 1024;
    // Warps. TMA: one producer per operand. Else 16 loader warps, since turning FP32 into three terms (or reading odd
    // strides) takes many instructions; roles are whole warpgroups then and share out the registers anew: to the
    // epilogue's FP32 sums and 24 MMAs a slab, or to the loaders of 16-bit values, which keep two slabs (in all no more
    // than the launch has: 896 threads of 72).
    static constexpr int kLoaders = TMA ? 2 : 16;
    static constexpr int kMmaWarp = kLoaders, kFixWarp = kLoaders + 1;
    static constexpr int kEpiWarp0 = !TMA ? kLoaders + 4 : RIGHT ? kLoaders + 2 : kLoaders + 1;
    static constexpr int kLaunchRegs = 72;
    static constexpr int kLoaderRegs = PLANES == 1 ? 88 : 56, kMmaRegs = PLANES == 1 ? 40 : 72, kEpiRegs = PLANES == 1 ? 56 : 104;
    static_assert(512 * kLoaderRegs + 128 * kMmaRegs + 256 * kEpiRegs <= 896 * kLaunchRegs, "register shares");
    static constexpr int kEpiWarps = 8;
    static constexpr int kThreads = 32 * (kEpiWarp0 + kEpiWarps);
    // The chunks' sums stay in registers, or, where the loaders need those, in TMEM beside as many accumulators as fit.
    static constexpr bool kTmemSums = !TMA && PLANES == 1;
    static constexpr int kBuffers = kTmemSums && NT == 256 ? 1 : 2;  // accumulators
    static constexpr int kTmemCols = (kBuffers + (kTmemSums ? 1 : 0)) * NT <= 2 * NT ? 2 * NT : 4 * NT;
    // N of an MMA is a multiple of this: whole 64-column boxes per CTA where the N side is MN-major.
    static constexpr int kGranule = (RIGHT ? 64 : 16) * CG;
    // Arrivals that complete a filled stage, besides the bytes of TMA copies: the loader warps', and in the leader of
    // a pair one from the peer. (An arrival across the pair is slow, so the peer's idle MMA warp makes it.)
    __device__ static int full_count(bool leader) { return TMA ? 1 : kLoaders + (CG == 2 && leader ? 1 : 0); }
    static_assert(kSmem <= 227 * 1024, "shared memory");
    static_assert((kTmemCols & (kTmemCols - 1)) == 0 && kTmemCols <= 512 && kTmemCols >= 32, "TMEM allocation");
    static_assert(KS == 1 || (TMA && PLANES == 1), "only TMA stages hold several slabs");
    static_assert(!N_MN || NTC % 64 == 0, "MN-major boxes are 64 columns");
};

struct GroupedTile {
    int e;
    int f0;          // first output column of the tile
    int r0, r1;      // output rows [r0, r1)
    int cols;        // N of the MMAs
    int t0, t1;      // gradient: rows contracted over
    int steps, slabs, kb;  // 16-deep MMA steps and 64-deep slabs of the contraction, and stages
};

template <class Cfg>
struct GroupedTiles {
    const GroupedParams& p;
    const int* offset;      // [groups + 1], clamped
    const int* first_tile;  // [groups + 1]
    int tile, step, e;

    __device__ GroupedTiles(const GroupedParams& p_, const int* o, const int* f, int worker, int workers)
        : p(p_), offset(o), first_tile(f), tile(worker - workers), step(workers), e(0) {}

    __device__ bool next(GroupedTile& t) {
        tile += step;
        if (tile >= first_tile[p.groups]) return false;
        while (tile >= first_tile[e + 1]) ++e;
        const int i = tile - first_tile[e];
        t.e = e;
        t.t0 = offset[e];
        t.t1 = offset[e + 1];
        // Tiles that share M-side data follow each other. The output rows are dealt out evenly: 300 rows are
        // 160 + 140, not 256 + 44 (every tile is left some, since (tiles - 1) NT < rows and each <= NT).
        const int rows = Cfg::RIGHT ? p.k : t.t1 - t.t0;
        const int tiles = (rows + Cfg::NT - 1) / Cfg::NT;
        const int each = ((rows + tiles - 1) / tiles + Cfg::kGranule - 1) / Cfg::kGranule * Cfg::kGranule;
        const int ri = i % tiles * each;
        const int left = min(each, rows - ri);
        t.f0 = i / tiles * Cfg::BM;
        t.r0 = (Cfg::RIGHT ? 0 : t.t0) + ri;
        t.r1 = t.r0 + left;
        t.cols = (left + Cfg::kGranule - 1) / Cfg::kGranule * Cfg::kGranule;
        t.steps = ((Cfg::RIGHT ? t.t1 - t.t0 : p.k) + 15) / 16;
        t.slabs = (t.steps + kGroupedDepth / 16 - 1) / (kGroupedDepth / 16);
        t.kb = (t.slabs + Cfg::KS - 1) / Cfg::KS;
        return true;
    }
};

template <typename T>
__device__ __forceinline__ T grouped_round(float v);
template <>
__device__ __forceinline__ float grouped_round<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half grouped_round<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 grouped_round<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// Rows [first, first + 16) of a column, as far as there are `rows`; `at` is row 0's place.
template <typename T>
__device__ __forceinline__ void grouped_store16(const GroupedParams& p, long long at, int first, int rows, const float (&v)[16]) {
    T* to = static_cast<T*>(p.c) + at + first * p.ldc;
    if (first + 16 <= rows) {
#pragma unroll
        for (int j = 0; j < 16; ++j, to += p.ldc) *to = grouped_round<T>(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j, to += p.ldc)
            if (first + j < rows) *to = grouped_round<T>(v[j]);
    }
}

// This warpgroup's share of the registers from here on.
template <int REGS, int LAUNCH>
__device__ __forceinline__ void set_max_registers() {
    if constexpr (REGS < LAUNCH) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
    if constexpr (REGS > LAUNCH) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}

// Loads of operands on their way through registers. Whole pieces of 16 bytes and more are not kept in L1, which is small
// beside these tiles and holds what the roles spill; of odd rows, two loads share most lines.
__device__ __forceinline__ uint32_t load_once(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load_once(const uint16_t* p) {
    uint16_t v;
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}

__device__ __forceinline__ void store_shared16(uint32_t to, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Eight consecutive FP32 elements of a row in global memory.
struct GroupedChunk {
    uint32_t w[8];

    // All eight are there; `align`: bytes that the address is a multiple of.
    __device__ __forceinline__ void load(const char* src, int align) {
        if (align >= 32) {
            asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                         : "l"(src));
        } else if (align >= 16) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                             : "l"(src + 16 * i));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = load_once(reinterpret_cast<const uint32_t*>(src) + i);
        }
    }

    // Those in [.., rows) x [.., cols), zeros for the others.
    __device__ __forceinline__ void load_some(const char* base, long long ld, int align, int row, int rows, int col,
                                              int cols) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0;
        if (row >= rows || col >= cols) return;
        const char* src = base + row * ld + static_cast<long long>(col) * 4;
        if (col + 8 <= cols) {
            load(src, align);
            return;
        }
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < cols - col) w[i] = load_once(reinterpret_cast<const uint32_t*>(src) + i);
    }

    // Their BF16 terms, into 16 bytes of each plane at shared address `to`.
    template <int PLANES>
    __device__ __forceinline__ void store(uint32_t to, int plane_bytes) const {
        uint32_t t[PLANES][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo = __uint_as_float(w[2 * i]), hi = __uint_as_float(w[2 * i + 1]);
            t[0][i] = __byte_perm(w[2 * i], w[2 * i + 1], 0x7632);  // cut to the upper halves
#pragma unroll
            for (int pl = 1; pl < PLANES; ++pl) {
                lo -= __uint_as_float(t[pl - 1][i] << 16);
                hi -= __uint_as_float(t[pl - 1][i] & 0xffff0000u);
                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(t[pl][i]) : "f"(hi), "f"(lo));
            }
        }
#pragma unroll
        for (int pl = 0; pl < PLANES; ++pl) store_shared16(to + pl * plane_bytes, t[pl][0], t[pl][1], t[pl][2], t[pl][3]);
    }
};

// A tile's place in an operand: rows (columns, where it is MN-major) [first, first + width), which the operand has up
// to last. Put together where it is used, from the kernel's parameters and the tile, to leave the registers to the data.
template <int WIDTH, bool MN>
struct GroupedPlace {
    const char* base;
    long long ld;
    int align, first, width, last;

    __device__ __forceinline__ bool inside() const { return MN ? first + WIDTH <= last : first < last; }
};

// One FP32 operand's 64-deep slabs on the way from global memory through registers into shared memory: WIDTH rows of the
// tile (columns, where the operand is MN-major). K-major rows have 8 chunks of eight elements, MN-major ones WIDTH / 8.
template <class Cfg, int WIDTH, bool MN>
struct GroupedSide {
    static constexpr int ES = 4, kThreads = 32 * Cfg::kLoaders;
    using Place = GroupedPlace<WIDTH, MN>;
    static constexpr int kPerRow = MN ? WIDTH / 8 : 8;
    static constexpr int kChunks = (WIDTH * 8 + kThreads - 1) / kThreads;
    static constexpr int kApart = kThreads / kPerRow;  // rows between a thread's chunks
    static constexpr int kPlane = WIDTH * 128, kPrefetch = 4;
    GroupedChunk c[kChunks];
    const char* at[MN ? 1 : kChunks];  // this thread's chunks of the next slab

    // The contraction starts at d0.
    __device__ __forceinline__ void start(const Place& o, int d0, int id) {
        if (MN) {
            at[0] = o.base + (d0 + id / kPerRow) * o.ld + static_cast<long long>(o.first + id % kPerRow * 8) * ES;
        } else {
#pragma unroll
            for (int i = 0; i < (MN ? 1 : kChunks); ++i)  // rows past the end repeat the last: their results go nowhere
                at[i] = o.base + min(o.first + i * kApart + id / 8, o.last - 1) * o.ld +
                        static_cast<long long>(d0 + id % 8 * 8) * ES;
        }
    }

    __device__ __forceinline__ static bool has(int i, int id) {  // whether chunk i is one of the tile's
        return (WIDTH * 8) % kThreads == 0 || i * kThreads + id < WIDTH * 8;
    }

    // The slab from d0 on of a contraction that ends at d1.
    __device__ __forceinline__ void load(const Place& o, int d0, int d1, int id, int /* slabs to the next load */) {
        if (o.inside() && d0 + kGroupedDepth <= d1) {
            // The lines of a later slab on their way into L2: one slab in registers covers its latency, not HBM's.
            if (id % 4 == 0 && d0 + (kPrefetch + 1) * kGroupedDepth <= d1) {
#pragma unroll
                for (int i = 0; i < kChunks; ++i) {
                    if (!has(i, id) || (!MN && i * kApart >= o.width)) continue;
                    const char* later = MN ? at[0] + (i * kApart + kPrefetch * kGroupedDepth) * o.ld
                                           : at[MN ? 0 : i] + kPrefetch * kGroupedDepth * ES;
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(later));
                }
            }
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                if (!has(i, id)) continue;
                if (MN) {
                    c[i].load(at[0] + i * kApart * o.ld, o.align);
                } else if (i * kApart < o.width) {
                    c[i].load(at[i], o.align);
                    at[i] += kGroupedDepth * ES;
                }
            }
            if (MN) at[0] += kGroupedDepth * o.ld;
        } else {
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                if (!has(i, id)) continue;
                const int row = i * kApart + id / kPerRow, col = id % kPerRow * 8;
                if (MN) c[i].load_some(o.base, o.ld, o.align, d0 + row, d1, o.first + col, o.last);
                else c[i].load_some(o.base, o.ld, o.align, o.first + row, o.last, d0 + col, d1);
            }
        }
    }

    __device__ __forceinline__ void store(uint32_t tile, int width, int id) const {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            if (!has(i, id) || (!MN && i * kApart >= width)) continue;
            const int row = i * kApart + id / kPerRow, col = id % kPerRow, box = MN ? col / 8 : 0;
            c[i].template store<Cfg::PLANES>(tile + box * 8192 + row * 128 + (((col % 8) ^ (row & 7)) << 4), kPlane);
        }
    }
};

// The same for 16-bit operands that TMA cannot address, whose rows start at any even address: a warp takes 64 elements
// of a row at a time, a word per lane, so that a load touches one or two lines however the row lies. A warp's segments
// are a multiple of eight rows apart, so they all start on a word or all between words; then lanes pass halves on to
// their neighbours, and the first half of each segment comes by one load for all of them.
template <class Cfg, int WIDTH, bool MN>
struct GroupedSide16 {
    static constexpr int kWarps = Cfg::TMA ? 16 : Cfg::kLoaders;  // (TMA kernels do not use it)
    static constexpr int kSegments = WIDTH / kWarps;              // of 64 elements, per warp
    static constexpr int kBoxes = MN ? WIDTH / 64 : 1;
    static constexpr int kApart = kWarps / kBoxes;  // rows between a warp's segments
    static_assert(WIDTH % kWarps == 0 && kSegments <= 32 && kApart % 8 == 0, "segments");
    using Place = GroupedPlace<WIDTH, MN>;
    uint32_t w[kSegments];
    uint32_t edge;   // lane i: element 0 of segment i
    const char* at;  // segment 0 of the next slab
    bool shifted;    // what is in w starts between words

    __device__ __forceinline__ void start(const Place& o, int d0, int id) {
        const int warp = id / 32;
        const int row = MN ? d0 + warp / kBoxes : o.first + warp, col = MN ? o.first + warp % kBoxes * 64 : d0;
        at = o.base + row * o.ld + static_cast<long long>(col) * 2;
    }

    __device__ __forceinline__ void load(const Place& o, int d0, int d1, int id, int ahead) {
        const int lane = id % 32, warp = id / 32;
        const long long step = kApart * o.ld;
        // One element more than the segments have: a lane's word may end behind them.
        if (MN ? o.first + WIDTH < o.last && d0 + kGroupedDepth <= d1 : d0 + kGroupedDepth < d1) {
            const uint32_t between = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at)) & 2u;
            shifted = between != 0;
            if (lane < kSegments && (MN || o.first + warp + lane * kApart < o.last))
                edge = load_once(reinterpret_cast<const uint16_t*>(at + lane * step));
            const char* src = at + between + lane * 4;
#pragma unroll
            for (int i = 0; i < kSegments; ++i, src += step)
                if (MN || o.first + warp + i * kApart < o.last) w[i] = load_once(reinterpret_cast<const uint32_t*>(src));
        } else {
            shifted = false;
            const int col = (MN ? o.first + warp % kBoxes * 64 : d0) + 2 * lane, cols = MN ? o.last : d1;
            const uint16_t* src = reinterpret_cast<const uint16_t*>(at) + 2 * lane;
            int row = MN ? d0 + warp / kBoxes : o.first + warp;
            const int rows = MN ? d1 : o.last;
#pragma unroll
            for (int i = 0; i < kSegments; ++i, row += kApart, src += step / 2) {
                w[i] = 0;
                if (row < rows && col < cols) w[i] = load_once(src);
                if (row < rows && col + 1 < cols) w[i] |= load_once(src + 1) << 16;
            }
        }
        at += ahead * (MN ? kGroupedDepth * o.ld : kGroupedDepth * 2);
    }

    // Rows past the operand's end hold what they held: their results go nowhere.
    __device__ __forceinline__ void store(uint32_t tile, int width, int id) const {
        const int lane = id % 32, warp = id / 32, row = warp / kBoxes;
        const uint32_t to = tile + warp % kBoxes * 8192 + row * 128 + (((lane / 4) ^ (row & 7)) << 4) + lane % 4 * 4;
#pragma unroll
        for (int i = 0; i < kSegments; ++i) {
            if (!MN && warp + i * kApart >= width) continue;
            uint32_t v = w[i];
            if (shifted) {
                const uint32_t before = __shfl_up_sync(~0u, v, 1), first = __shfl_sync(~0u, edge, i);
                v = (lane ? before >> 16 : first) | v << 16;
            }
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + i * kApart * 128), "r"(v) : "memory");
        }
    }
};

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads, 1)
    grouped_tc_kernel(const __grid_constant__ CUtensorMap map_m, const __grid_constant__ CUtensorMap map_n,
                      const __grid_constant__ CUtensorMap map_n32, const __grid_constant__ CUtensorMap map_n16,
                      const GroupedParams p) {
    constexpr int NT = Cfg::NT, CG = Cfg::CG, PLANES = Cfg::PLANES, STAGES = Cfg::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Cfg::kBarriers);  // of the leader: both CTAs' stage is filled
    uint64_t* empty_bar = full_bar + STAGES;
    uint64_t* tail_bar = empty_bar + STAGES;  // a stage whose last rows are still to be cleared
    // In the leader: the peer's tail in this stage is cleared. One per stage, like tail_bar, so that no arrival is lost:
    // the peer's next tail there is loaded only after the MMA has consumed the stage, which it does after the leader
    // has waited for this one. (With one barrier for all stages the peer could clear two tails in different stages
    // before the leader waits for the first, whose phase would be over unseen.)
    uint64_t* peer_tail_bar = tail_bar + STAGES;
    uint64_t* acc_full_bar = peer_tail_bar + STAGES;
    uint64_t* acc_empty_bar = acc_full_bar + 2;  // used in the leader
    uint64_t* drain_bar = acc_empty_bar + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* offset = reinterpret_cast<int*>(smem + Cfg::kTables);
    int* first_tile = offset + kGroupedMaxGroups + 1;

    const int warp = threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    const int rank = CG == 2 ? static_cast<int>(cluster_ctarank()) : 0;
    const bool leader = rank == 0;
    const int worker = blockIdx.x / CG, workers = gridDim.x / CG;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full_bar[s], Cfg::full_count(leader));
            mbar_init(&empty_bar[s], 1);
            mbar_init(&tail_bar[s], 1);
            mbar_init(&peer_tail_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full_bar[b], 1);
            mbar_init(&acc_empty_bar[b], CG * Cfg::kEpiWarps);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async_smem();
    }
    if (warp == Cfg::kMmaWarp) {
        if (CG == 2) {
            tmem_alloc_pair(tmem_slot, Cfg::kTmemCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(tmem_slot, Cfg::kTmemCols);
            tmem_relinquish();
        }
    }
    if (warp == Cfg::kEpiWarp0) {
        // Clamped offsets (running maximum) and the tiles in front of each group, 32 groups at a time.
        int floor = 0, before = 0;
        for (int base = 0; base <= p.groups; base += 32) {
            const int i = base + lane;
            const int raw = i <= p.groups ? p.offsets[i] : 0;
            int v = min(max(raw, 0), p.rows);
            if (i > p.groups) v = 0;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int o = __shfl_up_sync(~0u, v, d);
                if (lane >= d) v = max(v, o);
            }
            v = max(v, floor);
            if (i <= p.groups) {
                offset[i] = v;
                if (v != raw && worker == 0 && leader) report_bad_index();
            }
            int prev = __shfl_up_sync(~0u, v, 1);
            if (lane == 0) prev = floor;
            floor = __shfl_sync(~0u, v, 31);
            // tiles of group i - 1, which ends here
            const int rows = Cfg::RIGHT ? p.k : v - prev;
            int tiles = i >= 1 && i <= p.groups ? (rows + NT - 1) / NT * p.m_tiles : 0;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int o = __shfl_up_sync(~0u, tiles, d);
                if (lane >= d) tiles += o;
            }
            tiles += before;
            if (i <= p.groups) first_tile[i] = tiles;
            before = __shfl_sync(~0u, tiles, 31);
        }
    }
    if (Cfg::TMA && warp == 0 && lane == 0) {
        tma_prefetch_desc(&map_m);
        tma_prefetch_desc(&map_n);
    }
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint64_t limit = p.wait_limit_ns;
    GroupedTiles<Cfg> work(p, offset, first_tile, worker, workers);
    GroupedTile t;

    auto give_up = [&](uint32_t bits) {
        report_status(bits, abort_flag);
        if (CG == 2) st_cluster_u32(map_to_cta(smem_u32(const_cast<int*>(abort_flag)), rank ^ 1), 1);
    };
    auto leader_bar = [&](uint64_t* bar) { return map_to_cta(smem_u32(bar), 0); };
    auto arrive_leader = [&](uint64_t* bar) {
        if (CG == 2) mbar_arrive_cluster(leader_bar(bar));
        else mbar_arrive(bar);
    };

    if (Cfg::TMA && warp < 2) {
        // ------------------------------------------------------------ TMA producers: M side, N side
        // Issuing copies is what a producer spends its time on, so each operand has its own; the M side's posts the
        // bytes of both.
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            while (ok && work.next(t)) {
                const int half = t.cols / CG;  // N-side rows of this CTA
                // A copy costs the issuing thread more than a few rows too many cost the memory: one box, larger than
                // needed, instead of several.
                const int n_rows = Cfg::N_MN ? (p.n_wide ? Cfg::NTC : half)
                                             : half > 32 ? Cfg::NTC : half > 16 ? 32 : 16;
                const uint32_t bytes = Cfg::kMPlane + n_rows * 128;
                const int f = t.f0 + 128 * rank, r = t.r0 + half * rank;
                for (int kb = 0; kb < t.kb; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (!mbar_wait_bounded(&empty_bar[s], ((it / STAGES) & 1) ^ 1, limit, abort_flag)) {
                        give_up(kStatusTimeoutProducer);
                        ok = false;
                        break;
                    }
                    const int slabs = min(Cfg::KS, t.slabs - kb * Cfg::KS);
                    const bool tail = Cfg::RIGHT && kb == t.kb - 1 && (t.t1 - t.t0) % 16 != 0;
                    uint64_t* bar = tail ? &tail_bar[s] : &full_bar[s];
                    if (warp == 0) {
                        if (tail) mbar_arrive_expect_tx(bar, slabs * bytes);
                        else if (leader) mbar_arrive_expect_tx(bar, CG * slabs * bytes);
                    }
                    const uint32_t to = map_to_cta(smem_u32(bar), tail ? rank : 0);
                    auto load = [&](uint8_t* dst, const CUtensorMap* map, int x, int y, int z) {
                        if (CG == 2) tma_load_3d_pair(dst, map, to, x, y, z);
                        else tma_load_3d(dst, map, bar, x, y, z);
                    };
                    auto load_wide = [&](uint8_t* dst, const CUtensorMap* map, int column, int y, int z) {
                        if (CG == 2) tma_load_4d_pair(dst, map, to, 0, y, column / 64, z);
                        else tma_load_4d(dst, map, bar, 0, y, column / 64, z);
                    };
                    const int z = Cfg::RIGHT || p.m_shared ? 0 : t.e;
                    for (int j = 0; j < slabs; ++j) {
                        uint8_t* m_tile = smem + s * Cfg::kStage + j * Cfg::kSlab;
                        uint8_t* n_tile = m_tile + Cfg::kMBytes;
                        const int d0 = (Cfg::RIGHT ? t.t0 : 0) + (kb * Cfg::KS + j) * kGroupedDepth;
                        if (warp == 0) {
                            if (!Cfg::M_MN) {
                                load(m_tile, &map_m, d0, f, z);
                            } else if (p.m_wide) {
                                load_wide(m_tile, &map_m, f, d0, z);
                            } else {
                                load(m_tile, &map_m, f, d0, z);
                                load(m_tile + 8192, &map_m, f + 64, d0, z);
                            }
                        } else if (!Cfg::N_MN) {
                            load(n_tile, half > 32 ? &map_n : half > 16 ? &map_n32 : &map_n16, d0, r, 0);
                        } else if (p.n_wide) {
                            load_wide(n_tile, &map_n, r, d0, 0);
                        } else {
                            for (int b = 0; b < n_rows / 64; ++b) load(n_tile + b * 8192, &map_n, r + 64 * b, d0, 0);
                        }
                    }
                }
            }
            // Drain: the copies in flight land (their stages are consumed) before this CTA ends.
            for (int j = it - STAGES < 0 ? 0 : it - STAGES; j < it; ++j) {
                if (!mbar_wait_drain(&empty_bar[j % STAGES], (j / STAGES) & 1, limit)) {
                    report_status(kStatusTimeoutDrain, nullptr);
                    break;
                }
            }
        }
    } else if (!Cfg::TMA && warp < Cfg::kLoaders) {
        // ------------------------------------------------------------ loader warps
        // A slab's chunks are dealt out to the threads; each keeps the next slabs' in registers while it writes this
        // one's. Where a slab lies inside the operand (all but edges) a chunk costs a pointer step and
        // its loads.
        set_max_registers<Cfg::kLoaderRegs, Cfg::kLaunchRegs>();
        using M = std::conditional_t<Cfg::ES == 2, GroupedSide16<Cfg, 128, Cfg::M_MN>, GroupedSide<Cfg, 128, Cfg::M_MN>>;
        using N = std::conditional_t<Cfg::ES == 2, GroupedSide16<Cfg, Cfg::NTC, Cfg::N_MN>, GroupedSide<Cfg, Cfg::NTC, Cfg::N_MN>>;
        // Slabs ahead in registers: two of 16-bit values, since one does not cover a load's latency; FP32's are too wide.
        constexpr int kAhead = PLANES == 1 ? 2 : 1;
        M m[kAhead];
        N n[kAhead];
        const int id = threadIdx.x;
        int it = 0;
        bool ok = true;
        while (ok && work.next(t)) {
            const int half = t.cols / CG;
            const int d0 = Cfg::RIGHT ? t.t0 : 0, d1 = Cfg::RIGHT ? t.t1 : p.k;
            auto m_place = [&] {
                return typename M::Place{p.m_base + (Cfg::RIGHT ? 0 : t.e * p.m_stride), p.m_ld, p.m_align, t.f0 + 128 * rank,
                                         128, p.n};
            };
            auto n_place = [&] {
                return typename N::Place{p.n_base, p.n_ld, p.n_align, t.r0 + half * rank, half, Cfg::RIGHT ? p.k : t.t1};
            };
            auto load = [&](M& mk, N& nk, int kb) {
                if (kb >= t.kb) return;
                mk.load(m_place(), d0 + kb * kGroupedDepth, d1, id, kAhead);
                nk.load(n_place(), d0 + kb * kGroupedDepth, d1, id, kAhead);
            };
            auto step_over = [&](M& mk, N& nk, int kb) {
                const int s = it % STAGES;
                ok = mbar_wait_bounded(&empty_bar[s], ((it / STAGES) & 1) ^ 1, limit, abort_flag);
                ok = __all_sync(~0u, ok);
                if (!ok) {
                    if (lane == 0) give_up(kStatusTimeoutProducer);
                    return;
                }
                const uint32_t m_tile = smem_u32(smem + s * Cfg::kStage);
                mk.store(m_tile, 128, id);
                nk.store(m_tile + Cfg::kMBytes, half, id);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full_bar[s]);
                load(mk, nk, kb + kAhead);
                ++it;
            };
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                m[i].start(m_place(), d0 + i * kGroupedDepth, id);
                n[i].start(n_place(), d0 + i * kGroupedDepth, id);
                load(m[i], n[i], i);
            }
            for (int kb = 0; ok && kb < t.kb; kb += kAhead) {
                step_over(m[0], n[0], kb);
                if (kAhead == 2 && ok && kb + 1 < t.kb) step_over(m[kAhead - 1], n[kAhead - 1], kb + 1);
            }
        }
    } else if (warp < Cfg::kEpiWarp0) {
        // By all warps of the MMA's warpgroup, the idle ones too: a warpgroup changes its share with one instruction.
        if (!Cfg::TMA) set_max_registers<Cfg::kMmaRegs, Cfg::kLaunchRegs>();
        if (!Cfg::TMA && CG == 2 && warp == Cfg::kMmaWarp && !leader) {
            // ------------------------------------------------------------ tells the leader of the peer's filled stages
            if (lane == 0) {
                int it = 0;
                bool ok = true;
                while (ok && work.next(t)) {
                    for (int kb = 0; kb < t.kb; ++kb, ++it) {
                        const int s = it % STAGES;
                        if (!mbar_wait_bounded(&full_bar[s], (it / STAGES) & 1, limit, abort_flag)) {
                            give_up(kStatusTimeoutProducer);
                            ok = false;
                            break;
                        }
                        mbar_arrive_cluster(leader_bar(&full_bar[s]));
                    }
                }
            }
        } else if (warp == Cfg::kMmaWarp) {
            // ------------------------------------------------------------ MMA issuer (leader)
            if (lane == 0 && leader) {
                int it = 0, buf = 0;
                bool ok = true;
                while (ok && work.next(t)) {
                    const uint32_t idesc =
                        umma_idesc_f16(Cfg::BM, t.cols, Cfg::M_MN, Cfg::N_MN, PLANES > 1 ? 1 : p.bf16);
                    uint32_t d_tmem = 0, acc = 0;
                    for (int kb = 0; kb < t.kb; ++kb, ++it) {
                        if (kb % Cfg::kSumStages == 0) {
                            const int b = buf % Cfg::kBuffers;
                            if (!mbar_wait_bounded<CG == 2>(&acc_empty_bar[b], (buf / Cfg::kBuffers & 1) ^ 1, limit, abort_flag)) {
                                give_up(kStatusTimeoutMma);
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                            d_tmem = tmem_base + b * NT;
                            acc = 0;
                        }
                        const int s = it % STAGES;
                        // (of loader warps and cleared tails: the peer's stores too, so acquired from the pair)
                        if (!mbar_wait_bounded<CG == 2>(&full_bar[s], (it / STAGES) & 1, limit, abort_flag)) {
                            give_up(kStatusTimeoutMma);
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const int slabs = Cfg::KS == 1 ? 1 : min(Cfg::KS, t.slabs - kb * Cfg::KS);
                        for (int j = 0; j < slabs; ++j) {
                            // 16-deep steps of this slab that the contraction still has
                            const int steps = min(kGroupedDepth / 16, t.steps - (kb * Cfg::KS + j) * (kGroupedDepth / 16));
                            const uint32_t m_addr = smem_u32(smem + s * Cfg::kStage + j * Cfg::kSlab);
                            const uint64_t m_desc = umma_smem_desc(m_addr, Cfg::M_MN ? 8192 : 16, 1024, kLayoutSwizzle128B);
                            const uint64_t n_desc =
                                umma_smem_desc(m_addr + Cfg::kMBytes, Cfg::N_MN ? 8192 : 16, 1024, kLayoutSwizzle128B);
                            const uint32_t m_lo = static_cast<uint32_t>(m_desc), m_hi = static_cast<uint32_t>(m_desc >> 32);
                            const uint32_t n_lo = static_cast<uint32_t>(n_desc), n_hi = static_cast<uint32_t>(n_desc >> 32);
                            auto mma = [&](int mp, int np, int ks) {  // descriptors count 16-byte units
                                umma_f16<CG>(d_tmem, m_lo + (mp * Cfg::kMPlane + ks * (Cfg::M_MN ? 2048 : 32)) / 16, m_hi,
                                             n_lo + (np * Cfg::kNPlane + ks * (Cfg::N_MN ? 2048 : 32)) / 16, n_hi, idesc, acc);
                                acc = 1;
                            };
                            // The small products of all steps first: every addition truncates relative to what the
                            // accumulator holds, so only the last four cut at the sum's own size.
                            constexpr int kTerms = PLANES == 3 ? 6 : PLANES == 2 ? 3 : 1;
                            constexpr int kMTerm[6] = {2, 0, 1, 1, 0, 0}, kNTerm[6] = {0, 2, 1, 0, 1, 0};
                            if (steps == kGroupedDepth / 16) {
    #pragma unroll
                                for (int i = 6 - kTerms; i < 6; ++i)
    #pragma unroll
                                    for (int ks = 0; ks < kGroupedDepth / 16; ++ks) mma(kMTerm[i], kNTerm[i], ks);
                            } else {
    #pragma unroll
                                for (int i = 6 - kTerms; i < 6; ++i)
                                    for (int ks = 0; ks < steps; ++ks) mma(kMTerm[i], kNTerm[i], ks);
                            }
                        }
                        if (CG == 2) umma_commit_pair(&empty_bar[s], 0x3);
                        else umma_commit(&empty_bar[s]);
                        if (kb % Cfg::kSumStages == Cfg::kSumStages - 1 || kb == t.kb - 1) {
                            if (CG == 2) umma_commit_pair(&acc_full_bar[buf % Cfg::kBuffers], 0x3);
                            else umma_commit(&acc_full_bar[buf % Cfg::kBuffers]);
                            ++buf;
                        }
                    }
                }
                if (CG == 2) umma_commit_pair(drain_bar, 0x1);
                else umma_commit(drain_bar);
                if (!mbar_wait_drain(drain_bar, 0, limit)) report_status(kStatusTimeoutDrain, nullptr);
            }
        } else if (Cfg::TMA && Cfg::RIGHT && warp == Cfg::kFixWarp) {
            // ------------------------------------------------------------ clears the rows behind a group
            // The last MMA step of a contraction over a group's rows may hold rows of the next group (or NaN of a
            // buffer's spare rows): both operands' become 0 before the MMA may read them.
            int it = 0;
            uint32_t phases = 0;  // parities of each stage's tail barriers
            bool ok = true;
            while (ok && work.next(t)) {
                const int rows = t.t1 - t.t0, valid = rows % kGroupedDepth, end = (valid + 15) / 16 * 16;
                it += t.kb;
                if (rows % 16 == 0) continue;
                const int s = (it - 1) % STAGES;
                const uint32_t phase = (phases >> s) & 1;
                ok = mbar_wait_bounded(&tail_bar[s], phase, limit, abort_flag);
                ok = __all_sync(~0u, ok);
                if (!ok) {
                    if (lane == 0) give_up(kStatusTimeoutProducer);
                    break;
                }
                phases ^= 1u << s;
                const uint32_t m_tile = smem_u32(smem + s * Cfg::kStage + (t.slabs - 1) % Cfg::KS * Cfg::kSlab);
                const int boxes = t.cols / CG / 64;
                for (int b = 0; b < 2 + boxes; ++b) {
                    const uint32_t box = m_tile + (b < 2 ? b * 8192 : Cfg::kMBytes + (b - 2) * 8192);
                    for (int at = valid * 128 + lane * 16; at < end * 128; at += 512) store_shared16(box + at, 0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
                // One arrival completes the stage: the leader's, after the peer's tail is cleared too.
                if (CG == 2 && !leader) {
                    if (lane == 0) mbar_arrive_cluster(leader_bar(&peer_tail_bar[s]));
                    continue;
                }
                if (CG == 2) {
                    ok = __all_sync(~0u, mbar_wait_bounded<true>(&peer_tail_bar[s], phase, limit, abort_flag));
                    if (!ok) {
                        if (lane == 0) give_up(kStatusTimeoutProducer);
                        break;
                    }
                }
                if (lane == 0) mbar_arrive(&full_bar[s]);
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue
        if (!Cfg::TMA) set_max_registers<Cfg::kEpiRegs, Cfg::kLaunchRegs>();
        const int quarter = warp & 3;                    // TMEM lanes of this warp
        const int part = (warp - Cfg::kEpiWarp0) >> 2;   // which of every two 16-column pieces
        const uint32_t acc_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        int buf = 0;
        bool ok = true;
        while (ok && work.next(t)) {
            const int f = t.f0 + 128 * rank + quarter * 32 + lane;
            const long long at = (Cfg::RIGHT ? t.e * p.stride_c : 0) + t.r0 * p.ldc + f;
            const int rows = f < p.n ? t.r1 - t.r0 : 0;  // this lane's column of each row
            auto store = [&](int q, const float (&v)[16]) {
                if (p.out_f32) grouped_store16<float>(p, at, q * 16, rows, v);
                else if (p.bf16) grouped_store16<__nv_bfloat16>(p, at, q * 16, rows, v);
                else grouped_store16<__half>(p, at, q * 16, rows, v);
            };
            if (t.kb == 0) {
                const float zero[16] = {};
                for (int q = part; q * 16 < t.cols; q += 2) store(q, zero);
                continue;
            }
            constexpr int kPieces = NT / 32;
            float sum[Cfg::kTmemSums ? 1 : kPieces][16];
            if constexpr (!Cfg::kTmemSums) {
#pragma unroll
                for (int i = 0; i < kPieces; ++i)
#pragma unroll
                    for (int j = 0; j < 16; ++j) sum[i][j] = 0.0f;
            }
            const uint32_t sums = acc_base + Cfg::kBuffers * NT;
            for (int kb = 0; kb < t.kb; kb += Cfg::kSumStages, ++buf) {
                const int b = buf % Cfg::kBuffers;
                ok = mbar_wait_bounded(&acc_full_bar[b], buf / Cfg::kBuffers & 1, limit, abort_flag);
                ok = __all_sync(~0u, ok);
                if (!ok) break;
                tc_fence_after();
                if constexpr (Cfg::kTmemSums) {
                    for (int q = part; q * 16 < t.cols; q += 2) {
                        uint32_t v[16], o[16];
                        tmem_ld_32x32b_x16(acc_base + b * NT + q * 16, v);
                        if (kb) tmem_ld_32x32b_x16(sums + q * 16, o);
                        tmem_ld_wait();
                        tmem_regs_ready(v);
                        if (kb) {
                            tmem_regs_ready(o);
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(o[j]) + __uint_as_float(v[j]));
                        }
                        tmem_st_32x32b_x16(sums + q * 16, v);
                    }
                    tmem_st_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) {
                        const int q = 2 * i + part;
                        if (q * 16 < t.cols) {
                            uint32_t v[16];
                            tmem_ld_32x32b_x16(acc_base + b * NT + q * 16, v);
                            tmem_ld_wait();
                            tmem_regs_ready(v);
#pragma unroll
                            for (int j = 0; j < 16; ++j) sum[i][j] += __uint_as_float(v[j]);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_leader(&acc_empty_bar[b]);
            }
            if (ok) {
                if constexpr (Cfg::kTmemSums) {
                    for (int q = part; q * 16 < t.cols; q += 2) {
                        uint32_t v[16];
                        tmem_ld_32x32b_x16(sums + q * 16, v);
                        tmem_ld_wait();
                        tmem_regs_ready(v);
#pragma unroll
                        for (int j = 0; j < 16; ++j) sum[0][j] = __uint_as_float(v[j]);
                        store(q, sum[0]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kPieces; ++i)
                        if ((2 * i + part) * 16 < t.cols) store(2 * i + part, sum[i]);
                }
            }
            if (!ok && lane == 0) give_up(kStatusTimeoutEpilogue);
        }
        if (!Cfg::RIGHT && p.zero_rest) {
            // Rows of no group: in front of the first and behind the last one.
            const int first = offset[0], last = offset[p.groups], rest = first + p.rows - last;
            const int id = (blockIdx.x * Cfg::kEpiWarps + warp - Cfg::kEpiWarp0), ids = gridDim.x * Cfg::kEpiWarps;
            for (int i = id; i < rest; i += ids) {
                const long long row = i < first ? i : last + (i - first);
                for (int j = lane; j < p.n; j += 32) {
                    if (p.out_f32) static_cast<float*>(p.c)[row * p.ldc + j] = 0.0f;
                    else static_cast<uint16_t*>(p.c)[row * p.ldc + j] = 0;
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync_all();  // both CTAs are done with each other's barriers and TMEM
    if (warp == Cfg::kMmaWarp) {
        tc_fence_after();
        if (CG == 2) tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
        else tmem_dealloc(tmem_base, Cfg::kTmemCols);
    }
}

}  // namespace mfb
