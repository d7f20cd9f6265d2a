// gemm_i8.hip -- matrix product in 8-bit integers on gfx950's int8 MFMAs:
// y[m, n] = (sum_k x[m, k] w[n, k]) sx[m] sw[n] + bias[n], both operands with k contiguous, sums in
// 32-bit integers (exact: K < 2^17), scales and bias in fp32 behind them, one rounding to y's type.
//
// The weights are the MFMA's A operand and the rows of x its B, so that a lane holds one row of x and runs of four
// neighbouring n: scales of n come as 16-byte loads and results leave as 8 or 16 bytes.
// MFMA layouts, lane l: A[l % 32][16 g .. 16 g + 15], g = l / 32 (32x32x32), A[l % 16][16 g ..], g = l / 16
// (16x16x64); B likewise; D as the other 32x32 and 16x16 shapes'.  The reduction runs in any order that
// both operands share.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"

namespace inf {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

namespace {

constexpr int kBK = 128;             // k of a tile: 128 bytes of a row
constexpr uint32_t kNowhere = 0x80000000u;  // past the end of every buffer resource

__device__ __forceinline__ i32x16 mfma32x32x32i8(i32x4 a, i32x4 b, i32x16 c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ i32x4 mfma16x16x64i8(i32x4 a, i32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
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

// Four neighbouring results of row m from column n on.
template <typename E>
__device__ __forceinline__ void finish4(const GemmI8Params& p, int m, int n, i32x4 sum, float sx) {
    typename E::T* y = (typename E::T*)p.y + (int64_t)m * p.ldy + n;
    const typename E::T* bias = (const typename E::T*)p.bias;
    // the same roundings however the columns are aligned
    auto one = [&](int i, float sw, float b) { return fmaf((float)sum[i] * sx, sw, b); };
    if (p.wide && n + 4 <= p.N) {
        const f32x4 sw = ld4(p.sw + n), b = bias ? ld4(bias + n) : f32x4{0.f, 0.f, 0.f, 0.f};
        st4(y, f32x4{one(0, sw[0], b[0]), one(1, sw[1], b[1]), one(2, sw[2], b[2]), one(3, sw[3], b[3])});
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < p.N) E::st(y + i, one(i, p.sw[n + i], bias ? E::ld(bias + n + i) : 0.f));
    }
}

}  // namespace

// ============================================================================
// Tiles.  A workgroup of WN x WM waves forms BN x BM results, each wave 32 x 32 blocks of them in its registers, with
// k in steps of 128 bytes through double-buffered LDS, filled by direct-to-LDS loads one step ahead.
// LDS rows are 128 bytes, their eight 16-byte pieces at places c ^ (row % 8): any eight rows' pieces of one
// c lie in different banks.  A direct-to-LDS load fills 16 bytes a lane in the lanes' order, so the lanes
// fetch the pieces in that order: eight lanes still take one whole line of a row.
// ============================================================================
template <typename E, int BN, int BM, int WN, int WM, bool SPLIT>
__global__ __launch_bounds__(64 * WN * WM, 2) void gemm_i8_kernel(GemmI8Params p) {
    constexpr int NW = WN * WM;
    constexpr int FN = BN / WN / 32, FM = BM / WM / 32;
    constexpr int IN = BN / 8 / NW, IM = BM / 8 / NW;  // load instructions a wave and step
    static_assert(BN % (8 * NW) == 0 && BM % (8 * NW) == 0, "whole instructions");
    __shared__ __attribute__((aligned(16))) char ws0[BN * kBK], ws1[BN * kBK], xs0[BM * kBK], xs1[BM * kBK];

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
    const int piece = 16 * ((lane & 7) ^ (lane >> 3));  // this lane's of a step's row
    uint32_t vw[IN], vx[IM];
#pragma unroll
    for (int i = 0; i < IN; ++i) {
        const int r = 8 * (wave + NW * i) + (lane >> 3);
        vw[i] = r < rows_n ? (uint32_t)((int64_t)r * p.ldw + piece) : kNowhere;
    }
#pragma unroll
    for (int i = 0; i < IM; ++i) {
        const int r = 8 * (wave + NW * i) + (lane >> 3);
        vx[i] = r < rows_m ? (uint32_t)((int64_t)r * p.ldx + piece) : kNowhere;
    }
    auto load = [&](char* wd, char* xd, int k0) {
        const bool in = piece < k16 - k0;
        const auto rw = buffer_rsrc(W + k0, k0 < k16 ? (uint32_t)((int64_t)(rows_n - 1) * p.ldw + k16 - k0) : 0u);
        const auto rx = buffer_rsrc(X + k0, k0 < k16 ? (uint32_t)((int64_t)(rows_m - 1) * p.ldx + k16 - k0) : 0u);
#pragma unroll
        for (int i = 0; i < IN; ++i) buffer_ld16_lds(rw, wd + 1024 * (wave + NW * i), in ? vw[i] : kNowhere);
#pragma unroll
        for (int i = 0; i < IM; ++i) buffer_ld16_lds(rx, xd + 1024 * (wave + NW * i), in ? vx[i] : kNowhere);
    };

    i32x16 acc[FN][FM];
#pragma unroll
    for (int a = 0; a < FN; ++a)
#pragma unroll
        for (int b = 0; b < FM; ++b) acc[a][b] = i32x16{};

    load(ws0, xs0, k_first);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    const int row_n = wn * (BN / WN) + l32, row_m = wm * (BM / WM) + l32;
    auto step = [&](int k0, const char* wc, const char* xc, char* wd, char* xd) {
        load(wd, xd, k0 + kBK);
        const bool ragged = k0 + kBK > k_end && k_end % 16;
#pragma unroll
        for (int s = 0; s < kBK / 32; ++s) {
            const int at = 16 * ((2 * s + g) ^ (l32 & 7));
            i32x4 a[FN], b[FM];
#pragma unroll
            for (int f = 0; f < FN; ++f)
                a[f] = *reinterpret_cast<const i32x4*>(wc + (row_n + 32 * f) * kBK + at);
#pragma unroll
            for (int f = 0; f < FM; ++f)
                b[f] = *reinterpret_cast<const i32x4*>(xc + (row_m + 32 * f) * kBK + at);
            if (ragged) {
#pragma unroll
                for (int f = 0; f < FM; ++f) b[f] = first_bytes(b[f], k_end - (k0 + 32 * s + 16 * g));
            }
#pragma unroll
            for (int f = 0; f < FN; ++f)
#pragma unroll
                for (int h = 0; h < FM; ++h) acc[f][h] = mfma32x32x32i8(a[f], b[h], acc[f][h]);
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
    };
    for (int k0 = k_first; k0 < k_end; k0 += 2 * kBK) {
        step(k0, ws0, xs0, ws1, xs1);
        if (k0 + kBK < k_end) step(k0 + kBK, ws1, xs1, ws0, xs0);
    }

#pragma unroll
    for (int h = 0; h < FM; ++h) {
        const int m = m0 + row_m + 32 * h;
        if (m >= p.M) continue;
        const float sx = SPLIT ? 0.f : p.sx[m];
#pragma unroll
        for (int f = 0; f < FN; ++f)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = n0 + wn * (BN / WN) + 32 * f + 8 * j + 4 * g;
                const i32x4 v = {acc[f][h][4 * j], acc[f][h][4 * j + 1], acc[f][h][4 * j + 2], acc[f][h][4 * j + 3]};
                if constexpr (SPLIT) {
                    if (n < p.N)
                        *reinterpret_cast<i32x4*>(p.part + ((int64_t)split * p.M + m) * p.ldp + n) = v;
                } else if (n < p.N) {
                    finish4<E>(p, m, n, v, sx);
                }
            }
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
    finish4<E>(p, m, n, sum, p.sx[m]);
}

// ============================================================================
// Few rows: the weights go from memory straight into registers, each byte once.  A workgroup takes R x 16 outputs, its
// NW waves a K range each, all of a step's loads ahead of its products; x comes out of the caches.
// ============================================================================
template <typename E, int MT, int R, int NW>
__global__ __launch_bounds__(64 * NW) void gemm_i8_rows_kernel(GemmI8Params p) {
    constexpr int U = MT * R >= 4 ? 2 : 4;  // steps of 64 k whose loads are under way together
    __shared__ i32x4 sums[NW][R * MT][64];
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * (16 * R);
    const int8_t* w[R];
    const int8_t* x[MT];
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = p.w + (int64_t)min(n0 + 16 * r + l16, p.N - 1) * p.ldw + 16 * g;
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = p.x + (int64_t)min(16 * t + l16, p.M - 1) * p.ldx + 16 * g;
    i32x4 acc[R][MT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[r][t] = i32x4{};
    const int steps = (p.K + 63) / 64, per = (steps + NW - 1) / NW;
    const int s1 = min(steps, per * (wave + 1));
    const i32x4 zero = {};
    for (int s = per * wave; s < s1; s += U) {
        i32x4 a[U][R], b[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // a piece behind the end is read where the row's last one is, and counts as zeros
            const int k = min(64 * (s + u), p.last_piece - 16 * g);
#pragma unroll
            for (int r = 0; r < R; ++r) a[u][r] = *reinterpret_cast<const i32x4*>(w[r] + k);
#pragma unroll
            for (int t = 0; t < MT; ++t) b[u][t] = *reinterpret_cast<const i32x4*>(x[t] + k);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u >= s1) break;
            const int left = p.K - (64 * (s + u) + 16 * g);
            if (64 * (s + u) + 64 > p.K) {
#pragma unroll
                for (int t = 0; t < MT; ++t) b[u][t] = left >= 16 ? b[u][t] : left <= 0 ? zero : first_bytes(b[u][t], left);
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[r][t] = mfma16x16x64i8(a[u][r], b[u][t], acc[r][t]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) sums[wave][r * MT + t][lane] = acc[r][t];
    __syncthreads();
    for (int i = threadIdx.x; i < R * MT * 64; i += 64 * NW) {
        const int rt = i >> 6, r = rt / MT, t = rt % MT, m = 16 * t + (i & 15), n = n0 + 16 * r + 4 * ((i >> 4) & 3);
        i32x4 v = sums[0][rt][i & 63];
#pragma unroll
        for (int k = 1; k < NW; ++k) v += sums[k][rt][i & 63];
        if (m < p.M && n < p.N) finish4<E>(p, m, n, v, p.sx[m]);
    }
}

GemmI8Plan gemm_i8_plan(int64_t M, int64_t N, int64_t K) {
    GemmI8Plan plan;
    if (M <= kI8FewRows) {
        plan.kind = GemmI8Plan::kRows;
        return plan;
    }
    plan.kind = M * N >= (int64_t)256 * 256 * 192 ? GemmI8Plan::kLarge : GemmI8Plan::kMedium;
    const int64_t tile = plan.kind == GemmI8Plan::kLarge ? 256 : 128;
    const int64_t tiles = ((M + tile - 1) / tile) * ((N + tile - 1) / tile);
    const int64_t steps = (K + kBK - 1) / kBK;
    if (plan.kind == GemmI8Plan::kMedium) {
        const int64_t want = std::min<int64_t>(512 / std::max<int64_t>(tiles, 1), steps / 4);
        plan.ksplit = (int)std::max<int64_t>(1, std::min<int64_t>(want, 8));
    }
    plan.kchunk = (int)((steps + plan.ksplit - 1) / plan.ksplit * kBK);
    plan.ksplit = (int)((K + plan.kchunk - 1) / plan.kchunk);
    return plan;
}

template <typename E, int BN, int BM, int WN, int WM, bool SPLIT>
static void launch_tiles(GemmI8Params& p, hipStream_t s) {
    p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = (p.N + BN - 1) / BN;
    p.items = p.tiles_m * p.tiles_n * p.ksplit;
    hipLaunchKernelGGL((gemm_i8_kernel<E, BN, BM, WN, WM, SPLIT>), dim3((unsigned)((p.items + 7) / 8 * 8)),
                       dim3(64 * WN * WM), 0, s, p);
}

template <typename E>
static int launch_t(GemmI8Params p, const GemmI8Plan& plan, hipStream_t s) {
    p.ksplit = plan.ksplit;
    p.kchunk = plan.kchunk;
    p.last_piece = (p.K - 1) / 16 * 16;
    if (plan.kind == GemmI8Plan::kRows) {
        const dim3 grid((unsigned)((p.N + 15) / 16));
        auto go = [&](auto mt) {
            hipLaunchKernelGGL((gemm_i8_rows_kernel<E, decltype(mt)::value, 1, 4>), grid, dim3(256), 0, s, p);
        };
        if (p.M <= 16) go(std::integral_constant<int, 1>{});
        else if (p.M <= 32) go(std::integral_constant<int, 2>{});
        else go(std::integral_constant<int, 4>{});
    } else if (plan.kind == GemmI8Plan::kLarge) {
        launch_tiles<E, 256, 256, 2, 4, false>(p, s);
    } else if (p.ksplit > 1) {
        launch_tiles<E, 128, 128, 2, 2, true>(p, s);
        hipLaunchKernelGGL((gemm_i8_join_kernel<E>), dim3((unsigned)(((int64_t)p.M * (p.ldp / 4) + 255) / 256)),
                           dim3(256), 0, s, p);
    } else {
        launch_tiles<E, 128, 128, 2, 2, false>(p, s);
    }
    return (int)hipGetLastError();
}

int launch_gemm_i8(const GemmI8Params& p, const GemmI8Plan& plan, int bf16, hipStream_t s) {
    return bf16 ? launch_t<BF16>(p, plan, s) : launch_t<F32>(p, plan, s);
}

}  // namespace inf
