// gemm_i8.hip -- matrix product in 8-bit integers on gfx950's int8 MFMAs:
// y[m, n] = (sum_k x[m, k] w[n, k]) sx[m] sw[n] + bias[n], both operands with k contiguous, sums in
// 32-bit integers (exact: K < 2^17), scales and bias in fp32 behind them, one rounding to y's type.
//
// The weights are the MFMA's A operand and the rows of x its B, so that a lane holds one row of x and runs of four
// neighbouring n: scales of n come as 16-byte loads and results leave as 8 or 16 bytes.
// MFMA layout (32x32x32), lane l: A[l % 32][16 g .. 16 g + 15], g = l / 32; B likewise; D as the other 32x32
// shapes'.  The reduction runs in any order that both operands share.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "quant_rows.h"

namespace inf {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

namespace {

constexpr uint32_t kNowhere = 0x80000000u;  // past the end of every buffer resource
constexpr int kI8Step = 128;  // a step's k in any kernel; K ranges are whole ones

__device__ __forceinline__ i32x16 mfma32x32x32i8(i32x4 a, i32x4 b, i32x16 c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}
// The first n of 16 bytes, zeros behind them.
__device__ __forceinline__ i32x4 first_bytes(i32x4 v, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = n - 4 * i;
        v[i] = k >= 4 ? v[i] : k <= 0 ? 0 : v[i] & (int)((1u << (8 * k)) - 1);
    }
    return v;
}

// Four neighbouring columns from n on: their scales and bias.
template <typename E>
struct Columns {
    f32x4 sw, bias;
    bool whole;  // all four there, on 16 bytes
    __device__ __forceinline__ Columns(const GemmI8Params& p, int n) : whole(p.wide && n + 4 <= p.N) {
        const typename E::T* b = (const typename E::T*)p.bias;
        sw = bias = f32x4{0.f, 0.f, 0.f, 0.f};
        if (whole) {
            sw = ld4(p.sw + n);
            if (b) bias = ld4(b + n);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < p.N) {
                    sw[i] = p.sw[n + i];
                    if (b) bias[i] = E::ld(b + n + i);
                }
        }
    }
    // Their results in row m.  NT: past the caches, where whole lines are written.
    template <bool NT>
    __device__ __forceinline__ void store(const GemmI8Params& p, int m, int n, i32x4 sum, float sx) const {
        typename E::T* y = (typename E::T*)p.y + (int64_t)m * p.ldy + n;
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = fmaf((float)sum[i] * sx, sw[i], bias[i]);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < p.N) E::st(y + i, v[i]);
        } else if constexpr (!NT) {
            st4(y, v);
        } else if constexpr (sizeof(typename E::T) == 4) {
            __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(y));
        } else {
            __builtin_nontemporal_store(u16x4{f32_to_bf16(v[0]), f32_to_bf16(v[1]), f32_to_bf16(v[2]), f32_to_bf16(v[3])},
                                        reinterpret_cast<u16x4*>(y));
        }
    }
};

}  // namespace

// ============================================================================
// Tiles.  A workgroup of WN x WM waves forms BN x BM results, each wave 32 x 32 blocks of them in its registers, with
// k in steps of 128 bytes through a ring of S buffers in LDS, filled by direct-to-LDS loads S - 1 steps ahead.
// A step's 16-byte pieces of a row lie in an order that varies with the row, so that any eight rows' pieces of
// one k lie in different banks.  A direct-to-LDS load fills 16 bytes a lane in the lanes' order, so the
// lanes fetch the pieces in that order: eight lanes still take one run of a row.
//
// One barrier a step, before its last 32 k: by then every wave has read all of the step's operands (the last 32 k's are
// in registers), so its buffer takes the loads of S steps on, while the products of these 32 k hide the first reads of
// the next step's.
//
// What bounds it, and what it measured (bf16 results):
//   tiles of 256 (two waves a SIMD, 128 KB of LDS): 16384 x 8192 x 8192 in 884-916 us, 2.4-2.5 POP/s, matrix cores busy
//     67 % at 1.76 GHz: the power limit sets that clock.  Four waves of 128 x 128 took 1050, steps of 64 with S = 4 more too;
//   tiles of 128 (two workgroups a CU, one's results leave while the other's products run): 8192 x 2304 x 768 in fp32
//     30-35 us, of which 75 MB of results are 15 and every step of k 1.7: both in part in the open.  Tiles of 128 x
//     192, 128 x 256 and 64 x 128 took 35-37, steps of 64 37;
//   tiles of 64: weights, 32 x 16384 x 4096 in 12.7 us, 5.3 TB/s; or L2's latency and rate, 333 x 4096 x 4096 in 15.
// ============================================================================
template <typename E, int BN, int BM, int WN, int WM, int S, bool SPLIT>
__global__ __launch_bounds__(64 * WN * WM, WN * WM * ((BN + BM) * kI8Step * S > 81920 ? 1 : 2) / 4) void gemm_i8_kernel(
    GemmI8Params p) {
    constexpr int NW = WN * WM, BK = kI8Step;
    constexpr int FN = BN / WN / 32, FM = BM / WM / 32;
    constexpr int P = BK / 16, RI = 64 / P;                     // pieces a row; rows a load instruction
    constexpr int IN = BN / RI / NW, IM = BM / RI / NW;         // instructions a wave and step
    constexpr int KS = BK / 32;
    static_assert(BN % (RI * NW) == 0 && BM % (RI * NW) == 0, "whole instructions");
    static_assert(S == 2 || S == 4, "steps named at compile time");
    // arrays of their own, so that the compiler can tell the loads into one from the reads of the others
    __shared__ __attribute__((aligned(16))) char w0[BN * BK], x0[BM * BK], w1[BN * BK], x1[BM * BK];
    __shared__ __attribute__((aligned(16))) char w2[S > 2 ? BN * BK : 16], x2[S > 2 ? BM * BK : 16],
        w3[S > 2 ? BN * BK : 16], x3[S > 2 ? BM * BK : 16];

    const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave % WN, wm = wave / WN;

    // Neighbouring workgroups go to different XCDs: each XCD takes a run of the tiles, in bands of 8 row tiles.
    const int per = (p.items + 7) / 8;
    int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || t >= p.items) return;
    int split = 0;
    if constexpr (SPLIT) {
        split = t / (p.tiles_m * p.tiles_n);
        t -= split * p.tiles_m * p.tiles_n;
    }
    const int band = t / (8 * p.tiles_n), m_first = 8 * band, bm = min(8, p.tiles_m - m_first);
    t -= band * 8 * p.tiles_n;
    const int m0 = (m_first + t % bm) * BM, n0 = t / bm * BN;
    const int k_first = SPLIT ? split * p.kchunk : 0;
    const int k_end = SPLIT ? min(p.K, k_first + p.kchunk) : p.K;
    const int k16 = (k_end + 15) & ~15;  // rows are read in whole pieces

    const int8_t* W = p.w + (int64_t)n0 * p.ldw;
    const int8_t* X = p.x + (int64_t)m0 * p.ldx;
    const int rows_n = min(p.N - n0, BN), rows_m = min(p.M - m0, BM);
    auto order = [](int row) { return row & 7; };
    const int piece = 16 * ((lane % P) ^ order(lane / P));  // this lane's of a step's row
    uint32_t vw[IN], vx[IM];
#pragma unroll
    for (int i = 0; i < IN; ++i) {
        const int r = RI * (wave + NW * i) + lane / P;
        vw[i] = r < rows_n ? (uint32_t)((int64_t)r * p.ldw + piece) : kNowhere;
    }
#pragma unroll
    for (int i = 0; i < IM; ++i) {
        const int r = RI * (wave + NW * i) + lane / P;
        vx[i] = r < rows_m ? (uint32_t)((int64_t)r * p.ldx + piece) : kNowhere;
    }
    auto load = [&](char* wd, char* xd, int k0) {  // a step behind the end reads nothing: zeros
        const bool in = piece < k16 - k0;
        const auto rw = buffer_rsrc(W + k0, k0 < k16 ? (uint32_t)((int64_t)(rows_n - 1) * p.ldw + k16 - k0) : 0u);
        const auto rx = buffer_rsrc(X + k0, k0 < k16 ? (uint32_t)((int64_t)(rows_m - 1) * p.ldx + k16 - k0) : 0u);
#pragma unroll
        for (int i = 0; i < IN; ++i) buffer_ld16_lds(rw, wd + 1024 * (wave + NW * i), in ? vw[i] : kNowhere);
#pragma unroll
        for (int i = 0; i < IM; ++i) buffer_ld16_lds(rx, xd + 1024 * (wave + NW * i), in ? vx[i] : kNowhere);
    };
    // All waves' LDS reads are done, and their loads but those of the newest `steps` steps.  (__syncthreads() would
    // wait for all loads into LDS.)
    auto meet = [](auto steps) {
        constexpr int n = decltype(steps)::value * (IN + IM);
        static_assert(n < 64, "the counter's range");
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((n & 15) | (n >> 4) << 14 | 7 << 4);  // vmcnt(n) lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    i32x16 acc[FN][FM];
#pragma unroll
    for (int a = 0; a < FN; ++a)
#pragma unroll
        for (int b = 0; b < FM; ++b) acc[a][b] = i32x16{};

    const int row_n = wn * (BN / WN) + l32, row_m = wm * (BM / WM) + l32;
    struct Frags {
        i32x4 a[FN], b[FM];
    };
    auto read = [&](Frags& f, const char* wc, const char* xc, int s) {
        const int at = 16 * ((2 * s + g) ^ order(l32));
#pragma unroll
        for (int i = 0; i < FN; ++i) f.a[i] = *reinterpret_cast<const i32x4*>(wc + (row_n + 32 * i) * BK + at);
#pragma unroll
        for (int i = 0; i < FM; ++i) f.b[i] = *reinterpret_cast<const i32x4*>(xc + (row_m + 32 * i) * BK + at);
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j) acc[i][j] = mfma32x32x32i8(f.a[i], f.b[j], acc[i][j]);
    };
    // the reads of the next 32 k between the products of these
    auto interleave = [] {
        constexpr int R = FN + FM, M = FN * FM;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // a read
            __builtin_amdgcn_sched_group_barrier(0x008, M >= 2 * R ? 2 : 1, 0);  // products
        }
        if constexpr (M < 2 * R && M > R) __builtin_amdgcn_sched_group_barrier(0x008, M - R, 0);
    };
    using std::integral_constant;
    Frags f[2];
    // the step of k0 in its buffer; the next one's buffer.  LAST: k may end in this step.
    auto step = [&](auto last, int k0, char* wc, char* xc, const char* wnext, const char* xnext) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (s + 1 < KS) {
                read(f[(s + 1) & 1], wc, xc, s + 1);
            } else {
                meet(integral_constant<int, S - 2>{});
                load(wc, xc, k0 + S * BK);
                read(f[(s + 1) & 1], wnext, xnext, 0);
            }
            if constexpr (decltype(last)::value) {
                if (k_end % 16) {  // the last piece's bytes behind the end
#pragma unroll
                    for (int i = 0; i < FM; ++i)
                        f[s & 1].b[i] = first_bytes(f[s & 1].b[i], k_end - (k0 + 32 * s + 16 * g));
                }
            }
            multiply(f[s & 1]);
            interleave();
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    load(w0, x0, k_first);
    load(w1, x1, k_first + BK);
    if constexpr (S > 2) {
        load(w2, x2, k_first + 2 * BK);
        load(w3, x3, k_first + 3 * BK);
    }
    meet(integral_constant<int, S - 1>{});
    read(f[0], w0, x0, 0);
    int k0 = k_first;
    const std::false_type whole;
    const std::true_type last;
    if constexpr (S > 2) {
        for (; k0 + 4 * BK <= k_end; k0 += 4 * BK) {
            step(whole, k0, w0, x0, w1, x1);
            step(whole, k0 + BK, w1, x1, w2, x2);
            step(whole, k0 + 2 * BK, w2, x2, w3, x3);
            step(whole, k0 + 3 * BK, w3, x3, w0, x0);
        }
        if (k0 < k_end) step(last, k0, w0, x0, w1, x1);
        if (k0 + BK < k_end) step(last, k0 + BK, w1, x1, w2, x2);
        if (k0 + 2 * BK < k_end) step(last, k0 + 2 * BK, w2, x2, w3, x3);
        if (k0 + 3 * BK < k_end) step(last, k0 + 3 * BK, w3, x3, w0, x0);
    } else {
        for (; k0 + 2 * BK <= k_end; k0 += 2 * BK) {
            step(whole, k0, w0, x0, w1, x1);
            step(whole, k0 + BK, w1, x1, w0, x0);
        }
        if (k0 < k_end) step(last, k0, w0, x0, w1, x1);
        if (k0 + BK < k_end) step(last, k0 + BK, w1, x1, w0, x0);
    }

    // Results leave in whole lines: each wave turns 32 rows of its block at a time in LDS (a lane holds runs of four
    // columns of one row), pieces of 16 bytes at places that vary with the row, as above.  (From the registers, 16 bytes of
    // 64 rows a store: 8192 x 2304 x 768 in fp32 48 us instead of 31.)
    __syncthreads();
    constexpr int U = BN / WN / 4;                       // pieces of four results in a wave's row
    constexpr int HOLD = (BN < BM ? BN : BM) * BK / (32 * U * 16);  // waves' blocks in an array of the ring
    static_assert(HOLD * 4 >= NW, "a block in LDS for every wave");
    const int which = wave / HOLD;
    i32x4* turn = reinterpret_cast<i32x4*>(which == 0 ? w0 : which == 1 ? x0 : which == 2 ? w1 : x1) + wave % HOLD * 32 * U;
    // a lane's columns stay the same: what scales them is loaded once, and its rows' scales ahead of the stores
    static_assert(64 % U == 0, "one piece of the columns to a lane");
    const int m_wave = m0 + wm * (BM / WM) + lane / U, n = n0 + wn * (BN / WN) + 4 * (lane % U);
    float sx[FM][U / 2];
    if constexpr (!SPLIT) {
#pragma unroll
        for (int h = 0; h < FM; ++h)
#pragma unroll
            for (int i = 0; i < U / 2; ++i) sx[h][i] = p.sx[min(m_wave + 32 * h + 64 / U * i, p.M - 1)];
    }
    const Columns<E> columns(p, SPLIT ? p.N : n);
#pragma unroll
    for (int h = 0; h < FM; ++h) {
#pragma unroll
        for (int f = 0; f < FN; ++f)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                turn[l32 * U + ((8 * f + 2 * j + g) ^ (l32 & 7))] =
                    i32x4{acc[f][h][4 * j], acc[f][h][4 * j + 1], acc[f][h][4 * j + 2], acc[f][h][4 * j + 3]};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < U / 2; ++i) {
            const int r = lane / U + 64 / U * i, m = m_wave + 32 * h + 64 / U * i;
            const i32x4 v = turn[r * U + (lane % U ^ (r & 7))];
            if (m >= p.M || n >= p.N) continue;
            if constexpr (SPLIT)
                *reinterpret_cast<i32x4*>(p.part + ((int64_t)split * p.M + m) * p.ldp + n) = v;
            else
                columns.template store<true>(p, m, n, v, sx[h][i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Adds the K ranges' sums (rows of ldp, whole fours).
template <typename E>
__global__ __launch_bounds__(256) void gemm_i8_join_kernel(GemmI8Params p) {
    const int per_row = p.ldp / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)p.M * per_row) return;
    const int m = (int)(i / per_row), n = (int)(i % per_row) * 4;
    const int32_t* src = p.part + (int64_t)m * p.ldp + n;
    i32x4 sum = *reinterpret_cast<const i32x4*>(src);
    for (int s = 1; s < p.ksplit; ++s)
        sum += *reinterpret_cast<const i32x4*>(src + (int64_t)s * p.M * p.ldp);
    Columns<E>(p, n).template store<false>(p, m, n, sum, p.sx[m]);
}

// ============================================================================
// Few rows: a workgroup takes 32 outputs and all rows of x, and its four waves every fourth step of 128 k each, in a
// ring of S buffers of its own: no barriers, and the whole device's loads are under way at once.  Weights pass
// through LDS in whole lines (loaded straight into registers, 16 rows x 64 bytes at a time, with x out of the caches for
// every 16 outputs, 32 x 16384 x 4096 took 16 us, 13 so).  The waves' sums meet in LDS.
//
// FUSED: x comes as it is, and the workgroup quantises all of it while its first weights are on their way.
// Every workgroup does, so that pays where x is small: 1 x 2304 x 768 fp32 4.9 us, of which 2 are a launch.
// ============================================================================
constexpr int kRowsWaves = 4;

template <typename E, int FM, int S, bool FUSED>
__global__ __launch_bounds__(64 * kRowsWaves) void gemm_i8_rows_kernel(GemmI8Params p) {
    constexpr int BK = kI8Step, BN = 32, NW = kRowsWaves;
    constexpr int XB = FUSED ? 0 : 32 * FM;                  // rows of x in the ring
    constexpr int L = (BN + XB) / 8;                         // load instructions a step
    constexpr int STEP = (BN + XB) * BK;
    static_assert(S == 3 || S == 4, "steps named at compile time");
    __shared__ __attribute__((aligned(16))) char r0[NW * STEP], r1[NW * STEP], r2[NW * STEP],
        r3[S > 3 ? NW * STEP : 16];
    extern __shared__ __attribute__((aligned(16))) char xq[];  // FUSED: [M][x_stride]
    __shared__ float scales[8];
    __shared__ uint32_t tops[NW];

    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = blockIdx.x * BN, k16 = (p.K + 15) & ~15;
    const int8_t* W = p.w + (int64_t)n0 * p.ldw;
    const int rows_n = min(p.N - n0, BN);
    const int piece = 16 * ((lane & 7) ^ (lane >> 3));
    uint32_t vw[BN / 8], vx[XB ? XB / 8 : 1];
#pragma unroll
    for (int i = 0; i < BN / 8; ++i) {
        const int r = 8 * i + (lane >> 3);
        vw[i] = r < rows_n ? (uint32_t)((int64_t)r * p.ldw + piece) : kNowhere;
    }
#pragma unroll
    for (int i = 0; i < XB / 8; ++i) {
        const int r = 8 * i + (lane >> 3);
        vx[i] = r < p.M ? (uint32_t)((int64_t)r * p.ldx + piece) : kNowhere;
    }
    auto load = [&](char* ring, int k0) {  // a step behind the end reads nothing: zeros
        char* to = ring + wave * STEP;
        const bool in = piece < k16 - k0;
        const auto rw = buffer_rsrc(W + k0, k0 < k16 ? (uint32_t)((int64_t)(rows_n - 1) * p.ldw + k16 - k0) : 0u);
#pragma unroll
        for (int i = 0; i < BN / 8; ++i) buffer_ld16_lds(rw, to + 1024 * i, in ? vw[i] : kNowhere);
        if constexpr (XB > 0) {
            const auto rx = buffer_rsrc(p.x + k0, k0 < k16 ? (uint32_t)((int64_t)(p.M - 1) * p.ldx + k16 - k0) : 0u);
#pragma unroll
            for (int i = 0; i < XB / 8; ++i) buffer_ld16_lds(rx, to + BN * BK + 1024 * i, in ? vx[i] : kNowhere);
        }
    };
    // This wave's step i.  Workgroups start at different places of the whole rounds of the waves: rows are often powers
    // of two apart, and steps of one k then lie in few of the memory's channels (8 x 8192 x 8192: 20.2 us, 13.5 so).
    constexpr int NEXT = BK * NW;
    const int rounds = p.K / NEXT, turn = rounds ? blockIdx.x % rounds : 0;
    auto k_of = [&](int i) {
        const int j = i < rounds ? (i + turn < rounds ? i + turn : i + turn - rounds) : i;
        return j * NEXT + BK * wave;
    };
    load(r0, k_of(0));
    load(r1, k_of(1));
    load(r2, k_of(2));
    if constexpr (S > 3) load(r3, k_of(3));

    const int x_stride = ((p.K + BK - 1) & ~(BK - 1)) + 16;
    if constexpr (FUSED) {
        // one row to all waves, or rows to waves
        const bool one = p.M == 1;
        const int T = one ? 64 * NW : 64, t = one ? tid : lane;
        for (int m = one ? 0 : wave; m < p.M; m += NW) {
            const typename E::T* x = (const typename E::T*)p.xf + (int64_t)m * p.ldxf;
            constexpr int C = kChunk<E>;
            uint32_t top = 0;
            auto most = [&](auto vec) {
#pragma unroll 2
                for (int c = C * t; c < p.K; c += C * T) {
                    float v[C];
                    load_chunk<E, decltype(vec)::value, false>(x, c, p.K, v);
#pragma unroll
                    for (int i = 0; i < C; ++i) top = max(top, magnitude(v[i]));
                }
            };
            if (p.wide_x) most(std::true_type{});
            else most(std::false_type{});
            top = wave_all(top, [](uint32_t a, uint32_t b) { return max(a, b); });
            if (one) {
                if (lane == 0) tops[wave] = top;
                __syncthreads();
                top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
            }
            const RowScale s(top);
            auto write = [&](auto vec) {
#pragma unroll 2
                for (int c = C * t; c < x_stride - 16; c += C * T) {
                    float v[C];
                    int q[C];
                    load_chunk<E, decltype(vec)::value, false>(x, c, p.K, v);
                    round_all(v, s, q);
                    store_chunk(xq + m * x_stride + c, q);
                }
            };
            if (p.wide_x) write(std::true_type{});
            else write(std::false_type{});
            if (t == 0) scales[m] = s.scale;
        }
        __syncthreads();
    }

    i32x16 acc[FM];
#pragma unroll
    for (int h = 0; h < FM; ++h) acc[h] = i32x16{};
    const char* xrow = xq + min(l32, p.M - 1) * x_stride;  // a column past the rows is not written
    auto step = [&](auto last, char* ring, int i) {  // last: k may end in this step
        const int k0 = k_of(i);
        const char* from = ring + wave * STEP;
        asm volatile("" ::: "memory");
        constexpr int n = (S - 1) * L;
        static_assert(n < 64, "the counter's range");
        __builtin_amdgcn_s_waitcnt((n & 15) | (n >> 4) << 14 | 7 << 4 | 15 << 8);  // this step's loads have landed
        asm volatile("" ::: "memory");
        i32x4 a[4], b[4][FM];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int at = 16 * ((2 * s + g) ^ (l32 & 7));
            a[s] = *reinterpret_cast<const i32x4*>(from + l32 * BK + at);
#pragma unroll
            for (int h = 0; h < FM; ++h)
                b[s][h] = FUSED ? *reinterpret_cast<const i32x4*>(xrow + min(k0, x_stride - 16 - BK) + 32 * s + 16 * g)
                                : *reinterpret_cast<const i32x4*>(from + (BN + 32 * h + l32) * BK + at);
        }
        if (!FUSED && decltype(last)::value && k0 + BK > p.K) {  // the last piece's bytes behind the end
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int h = 0; h < FM; ++h) b[s][h] = first_bytes(b[s][h], p.K - (k0 + 32 * s + 16 * g));
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);  // read: the buffer is free
        asm volatile("" ::: "memory");
        load(ring, k_of(i + S));
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int h = 0; h < FM; ++h) acc[h] = mfma32x32x32i8(a[s], b[s][h], acc[h]);
    };
    const std::false_type whole;
    const std::true_type last;
    const int steps = (p.K - BK * wave + NEXT - 1) / NEXT;  // 0 or less: none
    int i = 0;
    for (; i + S <= rounds; i += S) {
        step(whole, r0, i);
        step(whole, r1, i + 1);
        step(whole, r2, i + 2);
        if constexpr (S > 3) step(whole, r3, i + 3);
    }
    if (i < steps) step(last, r0, i);
    if (i + 1 < steps) step(last, r1, i + 1);
    if (i + 2 < steps) step(last, r2, i + 2);
    if constexpr (S > 3)
        if (i + 3 < steps) step(last, r3, i + 3);

    __syncthreads();
    int* sums = reinterpret_cast<int*>(r0);  // [NW][16 FM][64]
    static_assert(STEP >= 16 * FM * 64 * 4, "the sums fit in a buffer");
#pragma unroll
    for (int h = 0; h < FM; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) sums[((wave * FM + h) * 16 + r) * 64 + lane] = acc[h][r];
    __syncthreads();
    for (int i = wave; i < 4 * FM; i += NW) {
        const int h = i >> 2, j = i & 3;
        i32x4 v = {};
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += sums[((w * FM + h) * 16 + 4 * j + r) * 64 + lane];
        const int m = 32 * h + l32, n = n0 + 8 * j + 4 * g;
        if (m < p.M && n < p.N) Columns<E>(p, n).template store<false>(p, m, n, v, FUSED ? scales[m] : p.sx[m]);
    }
}

// Tiles of 64 by ranges, at most.
constexpr int kI8Ranges = 384;

int64_t gemm_i8_split_rows(int64_t N) { return 64 * (kI8Ranges / 2 / ((N + 63) / 64)); }

GemmI8Plan gemm_i8_plan(int64_t M, int64_t N, int64_t K, bool quantised) {
    GemmI8Plan plan;
    plan.kchunk = (int)((K + kI8Step - 1) / kI8Step * kI8Step);
    auto tiles = [&](int64_t t) { return ((M + t - 1) / t) * ((N + t - 1) / t); };
    const int64_t steps = (K + kI8Step - 1) / kI8Step;
    // Few rows: where their kernel is at most one workgroup a CU and no row too long for one (us, its and tiles of 64):
    // 32 x 4096 x 4096 6.9 and 9.6, 8 x 8192 x 8192 13.5 and 14.0; but 32 x 16384 x 4096 19 and 12.9,
    // 32 x 4096 x 16384 21 and 15.2.  One row goes the same way past this border, where its x is quantised by a launch of its
    // own (whole calls, weights from memory): 1 x 8192 x 8192, inside, 17.5; 1 x 16384 x 4096 20.8, 1 x 4096 x 14336 26.5.
    if (M <= 64 && (N + 31) / 32 <= 256 && steps <= 64) {
        plan.kind = GemmI8Plan::kRows;
        // x quantised by every workgroup, where that takes no longer than a launch of its own (us, so and with one): 1 x 2304
        // x 768 4.1 and 6.0, 1 x 4096 x 4096 6.9 and 7.8, 4 x 2304 x 768 4.8 and 6.2, 8 x 768 x 768 6.1 and 6.2; but 4 x 4096
        // x 4096 13.1 and 8.2, 32 x 2304 x 64 9.1 and 5.9.
        plan.fused = !quantised && (M == 1 || (M <= 8 && (M + 3) / 4 * K <= 1024));
        return plan;
    }
    // Tiles of 256, one workgroup a CU (us, theirs and tiles of 128, bf16 results): 4096 x 4096 x 4096 67 and 88, x 512 18.1 and
    // 20.3; with 69 % of a round's CUs busy, 2816 x 4096 x 4096, 56 and 65, but 53 %, 4352 x 4096 x 4096, 108 and 94.  A short
    // K leaves the results' writing in the open, which two workgroups a CU hide: 75 %, 16384 x 2304 x 768 in
    // fp32, 70 and 55.  The rule counts tiles, full or not: few rows of a vocabulary's width take them for their weights
    // (whole calls): 1 x 50257 x 4096 62 us, 32 62, 64 68; of 128, 1 x 50257 x 768 15.4, 1 x 28672 x 8192 52.
    const int64_t t256 = tiles(256), rounds = (t256 + 255) / 256;
    if (steps >= 4 && t256 * 10 >= rounds * 256 * (steps >= 16 ? 7 : 9)) {
        plan.kind = GemmI8Plan::k256;
    } else if (tiles(128) >= (steps >= 24 ? 192 : 208)) {
        // Of 128, three steps ahead where one a CU has nothing else to hide the memory (that fills its LDS): 2048 x 2048 x 4096
        // 24.9, one step ahead 31.5, of 64 28.7; 768 x 4096 x 4096, 192 of them, 21.1, 25.3 and 22.8; but 1408 x 2048 x 4096, 176
        // of them, 22.9 and of 64 21.1.  A shorter K, one step ahead and of 64: 2048 x 2048 x 2048 15.6 (three ahead 16.4) and
        // 16.1, 1792 x 2048 x 1024 10.2 and 10.2; 208 of them, 1664 x 2048 x 4096 25.5 and 29.5.
        plan.kind = GemmI8Plan::k128;
        plan.deep = tiles(128) <= 256 && steps >= 24;
    } else {
        plan.kind = GemmI8Plan::k64;
        // Where there is one tile a CU, or two, nothing but their own loads hides the memory: three steps ahead and one
        // (weights from memory) 128 x 8192 x 8192 24 and 47, 333 x 4096 x 4096 18.7 and 24.9; but with three tiles a CU, 768 x
        // 4096 x 4096, 28.8 and 22.8.
        plan.deep = tiles(64) <= 512 && steps >= 16;
        // K ranges, for a join of about 5 us, where they take 24 steps off the longest: 128 x 1024 x 8192 9.9 in eight,
        // 15.7 in one; 200 x 2048 x 4096 (three) 11.9 and 9.9.
        const int64_t ks = std::min<int64_t>(kI8Ranges / tiles(64), steps / 8);
        if (ks > 1 && steps * (ks - 1) > 24 * ks) {
            plan.kchunk = (int)((steps + ks - 1) / ks * kI8Step);
            plan.ksplit = (int)((K + plan.kchunk - 1) / plan.kchunk);
        }
    }
    return plan;
}

template <typename E, int BN, int BM, int WN, int WM, int S, bool SPLIT>
static void launch_tiles(GemmI8Params& p, hipStream_t s) {
    p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = (p.N + BN - 1) / BN;
    p.items = p.tiles_m * p.tiles_n * p.ksplit;
    hipLaunchKernelGGL((gemm_i8_kernel<E, BN, BM, WN, WM, S, SPLIT>), dim3((unsigned)((p.items + 7) / 8 * 8)),
                       dim3(64 * WN * WM), 0, s, p);
}

template <typename E>
static int launch_t(GemmI8Params p, const GemmI8Plan& plan, hipStream_t s) {
    p.ksplit = plan.ksplit;
    p.kchunk = plan.kchunk;
    if (plan.kind == GemmI8Plan::kRows) {
        const dim3 grid((unsigned)((p.N + 31) / 32)), block(64 * kRowsWaves);
        if (plan.fused) {
            const size_t lds = (size_t)p.M * (((p.K + 127) & ~127) + 16);
            hipLaunchKernelGGL((gemm_i8_rows_kernel<E, 1, 4, true>), grid, block, lds, s, p);
        } else if (p.M <= 32) {
            hipLaunchKernelGGL((gemm_i8_rows_kernel<E, 1, 4, false>), grid, block, 0, s, p);
        } else {
            hipLaunchKernelGGL((gemm_i8_rows_kernel<E, 2, 3, false>), grid, block, 0, s, p);
        }
    } else if (plan.kind == GemmI8Plan::k256) {
        launch_tiles<E, 256, 256, 2, 4, 2, false>(p, s);
    } else if (plan.kind == GemmI8Plan::k128) {
        if (plan.deep) launch_tiles<E, 128, 128, 2, 2, 4, false>(p, s);
        else launch_tiles<E, 128, 128, 2, 2, 2, false>(p, s);
    } else if (p.ksplit > 1) {
        launch_tiles<E, 64, 64, 2, 2, 4, true>(p, s);
        hipLaunchKernelGGL((gemm_i8_join_kernel<E>), dim3((unsigned)(((int64_t)p.M * (p.ldp / 4) + 255) / 256)),
                           dim3(256), 0, s, p);
    } else if (plan.deep) {
        launch_tiles<E, 64, 64, 2, 2, 4, false>(p, s);
    } else {
        launch_tiles<E, 64, 64, 2, 2, 2, false>(p, s);
    }
    return (int)hipGetLastError();
}

int launch_gemm_i8(const GemmI8Params& p, const GemmI8Plan& plan, int bf16, hipStream_t s) {
    return bf16 ? launch_t<BF16>(p, plan, s) : launch_t<F32>(p, plan, s);
}

}  // namespace inf
