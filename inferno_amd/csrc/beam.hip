// beam.hip -- beam search's selection: of a group's beams x vocabulary candidates the best
// `beams` by score + logit - lse.
//
// The logits are read once.  A workgroup holds up to 8192 columns of one beam in registers, forms
// their maximum and sum of exponentials and finds their best `beams`; a second launch joins a
// beam's parts to its lse and ranks what is left of a group, some hundreds of candidates, by the
// whole score in 64 bits.  Within a beam the score's order is the logits', so the first step needs
// no lse and is exact; between beams scores can lie close together, and there the sums of
// exponentials are held in 64 bits as well.  Equal scores go to the lower beam, then the lower
// token.
//
// The best few of many: with each lane's largest value known, the beams-th largest of a wave's 64 is
// at most the beams-th largest of all its values, so only values from it up can matter: about as
// many as there are beams.  They are picked into LDS, and each counts those that are better.
#include "common.h"
#include "kernels.h"

namespace inf {

namespace {

constexpr int kBeamCols = 8192;  // columns of a workgroup at most: 32 per thread, in registers
constexpr int kBeamList = 1024;  // candidates in LDS; more of them (equal ones) are picked one by one

// Order of the floats as unsigned numbers, -0 as 0, NaN below -inf; 0 stands for no value.
__device__ __forceinline__ uint32_t ordered_logit(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 1u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t ordered_score(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    if ((b & 0x7fffffffffffffffull) > 0x7ff0000000000000ull) return 1ull;
    return b >> 63 ? ~b : b | (1ull << 63);
}

// A lower bound, exact down to bit LOW, of the n-th largest of the wave's values.
template <int LOW>
__device__ __forceinline__ uint32_t wave_nth(uint32_t v, int n) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= LOW; --bit) {
        const uint32_t up = t | (1u << bit);
        if (__popcll(__ballot(v >= up)) >= n) t = up;
    }
    return t;
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
    const uint32_t lo = __shfl_xor((uint32_t)v, m, 64), hi = __shfl_xor((uint32_t)(v >> 32), m, 64);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ double shfl_xor_d(double v, int m) {
    return __longlong_as_double((long long)shfl_xor64((uint64_t)__double_as_longlong(v), m));
}

// Whether a beam reads its logits: not if it is finished, or its score is not finite (then all
// its candidates have that score).
__device__ __forceinline__ bool beam_lives(const BeamSelectParams& p, int64_t row) {
    return !(p.finished && p.finished[row]) && isfinite(p.scores[row]);
}

}  // namespace

// N: columns per thread, 256 N per workgroup.
template <typename E, int N>
__global__ __launch_bounds__(256, N == 32 ? 7 : 1) void beam_part_kernel(BeamSelectParams p) {
    using T = typename E::T;
    constexpr int GE = 16 / sizeof(T), NV = N / GE;  // columns of a 16-byte load, loads per thread
    __shared__ uint64_t list[kBeamList];
    __shared__ int count;
    __shared__ float wmax[4];
    __shared__ double wsum[4];
    __shared__ uint64_t wbest[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t row = blockIdx.x / p.nsplit;
    const int split = blockIdx.x % p.nsplit;
    if (!beam_lives(p, row)) return;
    // Columns counted from the 16-byte boundary at or before the row's start; this workgroup's, from
    // its first one on, are those in [lo, hi).
    const T* x = (const T*)p.logits + row * p.ld;
    const int mis = (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) % GE);
    const int64_t c0 = (int64_t)split * (256 * N);
    const int lo = split == 0 ? mis : 0, hi = (int)min((int64_t)(256 * N), p.vocab + mis - c0);
    x += c0 - mis;
    float v[N];  // columns outside are -inf
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int c = (u * 256 + tid) * GE;
        if (c >= lo && c + GE <= hi) {
            const u32x4 raw = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x + c));
#pragma unroll
            for (int e = 0; e < GE; ++e) {
                if constexpr (sizeof(T) == 4)
                    v[u * GE + e] = __uint_as_float(raw[e]);
                else
                    v[u * GE + e] = __uint_as_float(e & 1 ? raw[e >> 1] & 0xffff0000u : raw[e >> 1] << 16);
            }
        } else {
#pragma unroll
            for (int e = 0; e < GE; ++e) v[u * GE + e] = c + e >= lo && c + e < hi ? E::ld(x + c + e) : -INFINITY;
        }
    }
    auto column = [&](int i) { return (i / GE * 256 + tid) * GE + i % GE; };
    auto key = [&](int i) {
        return (uint64_t)ordered_logit(v[i]) << 32 | (uint32_t)~(uint32_t)(c0 - mis + column(i));
    };
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) mx = fmaxf(mx, v[i]);
    const uint32_t lane_best = ordered_logit(mx);
    mx = wave_all(mx, [](float a, float b) { return fmaxf(a, b); });
    const float ref = mx == -INFINITY ? 0.f : mx;
    // four terms in 32 bits, which are off by 2^-23 of them at most, all further in 64
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        float t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = fast_exp2((v[i + e] - ref) * kLog2e);
        sum += (double)((t[0] + t[1]) + (t[2] + t[3]));
    }
    sum = wave_all(sum, [](double a, double b) { return a + b; });
    if (lane == 0) {
        wmax[wave] = mx;
        wsum[wave] = sum;
    }
    if (tid == 0) count = 0;
    const float least = logit_of(max(wave_nth<16>(lane_best, p.beams), ordered_logit(-INFINITY)));
    __syncthreads();
    if (tid == 0) {
        const float M = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
        double S = 0.0;
        for (int i = 0; i < 4; ++i) S += wmax[i] == -INFINITY ? wsum[i] : wsum[i] * exp((double)wmax[i] - (double)M);
        p.maxs[blockIdx.x] = M;
        p.sums[blockIdx.x] = S;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (v[i] >= least && column(i) >= lo && column(i) < hi) {
            const int at = atomicAdd(&count, 1);
            if (at < kBeamList) list[at] = key(i);
        }
    __syncthreads();
    const int n = count;
    uint64_t* out = p.cand + (int64_t)blockIdx.x * p.beams;
    if (n <= kBeamList) {
        if (tid < p.beams && tid >= n) out[tid] = 0;  // fewer columns than beams
        // four lanes count for one value
        for (int i0 = 0; i0 < n; i0 += 64) {
            const int i = i0 + (tid >> 2);
            const uint64_t mine = list[min(i, n - 1)];
            int better = 0;
#pragma unroll 4
            for (int j = tid & 3; j < n; j += 4) better += list[j] > mine;
            better += (int)dpp_u32<0xB1>((uint32_t)better);
            better += (int)dpp_u32<0x4E>((uint32_t)better);
            if (i < n && (tid & 3) == 0 && better < p.beams) out[better] = mine;
        }
        return;
    }
    uint64_t before = ~0ull;
    for (int k = 0; k < p.beams; ++k) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint64_t y = v[i] >= least && column(i) >= lo && column(i) < hi ? key(i) : 0;
            if (y < before && y > best) best = y;
        }
        best = wave_all(best, [](uint64_t a, uint64_t b) { return max(a, b); });
        if (lane == 0) wbest[wave] = best;
        __syncthreads();
        before = max(max(wbest[0], wbest[1]), max(wbest[2], wbest[3]));
        if (tid == 0) out[k] = before;
        __syncthreads();
    }
}

__global__ __launch_bounds__(256) void beam_join_kernel(BeamSelectParams p) {
    enum { kLives, kFinished, kFlat };  // a flat beam's candidates are the first tokens, all with its score
    __shared__ double base[kMaxBeams];  // score - lse; the score of a beam that is finished or flat
    __shared__ int kind[kMaxBeams];
    __shared__ uint64_t ls[kBeamList], lt[kBeamList];
    __shared__ int count;
    __shared__ uint64_t ws[4], wt[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t row0 = (int64_t)blockIdx.x * p.beams;
    const int per = p.nsplit * p.beams, total = p.beams * per;
    // The candidates' logits and columns do not wait for the lse; up to 256 U of them stay in registers.
    // Each part's are in order, so that a lane's step to step is no multiple of the beams: lanes that held
    // only best ones, and lanes that held only last ones, would bound the best few badly.
    constexpr int U = 8;
    uint64_t cand[U];
    auto index = [&](int i0, int u) { return i0 + 256 * u + ((tid + 41 * u) & 255); };
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            cand[u] = i0 + 256 * u < total && index(i0, u) < total ? p.cand[row0 * per + index(i0, u)] : 0;
    };
    load(0);
    static_assert(kMaxBeams * 8 <= 256, "eight lanes per beam");
    if (const int b = tid >> 3; b < p.beams) {
        const int64_t row = row0 + b;
        const float score = p.scores[row];
        const bool finished = p.finished && p.finished[row];
        // up to 32 parts: four a lane, loaded together
        constexpr int P = 4;
        float m[P], M = -INFINITY;
        double s[P], S = 0.0;
        for (int i0 = 0; i0 < p.nsplit; i0 += 8 * P) {
            float top = M;
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const int i = i0 + 8 * k + (tid & 7);
                m[k] = i < p.nsplit ? p.maxs[row * p.nsplit + i] : -INFINITY;
                s[k] = i < p.nsplit ? p.sums[row * p.nsplit + i] : 0.0;
                top = fmaxf(top, m[k]);
            }
            top = fmaxf(top, __uint_as_float(dpp_u32<0xB1>(__float_as_uint(top))));
            top = fmaxf(top, __uint_as_float(dpp_u32<0x4E>(__float_as_uint(top))));
            top = fmaxf(top, __uint_as_float(dpp_u32<0x141>(__float_as_uint(top))));
            if (M != -INFINITY) S *= exp((double)M - (double)top);
#pragma unroll
            for (int k = 0; k < P; ++k)
                if (i0 + 8 * k < p.nsplit) S += m[k] == -INFINITY ? s[k] : s[k] * exp((double)m[k] - (double)top);
            M = top;
        }
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) S += shfl_xor_d(S, d);
        if ((tid & 7) == 0) {
            // a NaN or +inf among the logits, or nothing above -inf: the sum is NaN, infinite or 0
            const double lse = (double)M + log(S);
            const bool lives = !finished && isfinite(score), fine = isfinite(lse);
            base[b] = !lives ? (double)score : fine ? (double)score - lse : __longlong_as_double(0x7ff8000000000000ll);
            kind[b] = finished ? kFinished : lives && fine ? kLives : kFlat;
        }
    }
    if (tid == 0) count = 0;
    __syncthreads();
    // Candidate i of the group: its score as an ordered number (0: there is none) and its place.
    auto candidate = [&](int i, uint64_t c, uint64_t& at) -> uint64_t {
        const int b = i / per, j = i - b * per;
        uint32_t token = (uint32_t)j;
        double score = base[b];
        if (kind[b] == kLives) {
            if (!c) return 0;
            token = ~(uint32_t)c;
            score += (double)logit_of((uint32_t)(c >> 32));
        } else if (kind[b] == kFinished) {
            if (j) return 0;
            token = (uint32_t)p.eos;
        } else if (j >= p.beams || j >= p.vocab) {
            return 0;
        }
        at = (uint64_t)b << 32 | token;
        return ordered_score(score);
    };
    auto emit = [&](int k, uint64_t s, uint64_t at) {
        const int b = (int)(at >> 32), token = (int)(uint32_t)at;
        const int64_t o = row0 + k;
        p.tokens[o] = token;
        p.parents[o] = b;
        p.scores_out[o] = (float)__longlong_as_double((long long)(s == 1 ? 0x7ff8000000000000ull
                                                                  : s >> 63 ? s & ~(1ull << 63) : ~s));
        if (p.finished_out) p.finished_out[o] = kind[b] == kFinished || token == p.eos;
    };
    uint32_t best = 0;
    uint64_t at = 0;
    auto pick = [&](uint64_t s, uint32_t least) {
        if (s && (uint32_t)(s >> 32) >= least) {
            const int k = atomicAdd(&count, 1);
            if (k < kBeamList) {
                ls[k] = s;
                lt[k] = at;
            }
        }
    };
    for (int i0 = 0; i0 < total; i0 += 256 * U) {
        if (i0) load(i0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + 256 * u < total && index(i0, u) < total)
                best = max(best, (uint32_t)(candidate(index(i0, u), cand[u], at) >> 32));
    }
    const uint32_t least = wave_nth<4>(best, p.beams);
    for (int i0 = 0; i0 < total; i0 += 256 * U) {
        if (total > 256 * U) load(i0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + 256 * u < total && index(i0, u) < total)
                pick(candidate(index(i0, u), cand[u], at), least);
    }
    __syncthreads();
    const int n = count;
    if (n <= kBeamList) {
        for (int i0 = 0; i0 < n; i0 += 64) {
            const int i = i0 + (tid >> 2);
            const uint64_t s = ls[min(i, n - 1)], t = lt[min(i, n - 1)];
            int better = 0;
#pragma unroll 4
            for (int j = tid & 3; j < n; j += 4) better += ls[j] > s || (ls[j] == s && lt[j] < t);
            better += (int)dpp_u32<0xB1>((uint32_t)better);
            better += (int)dpp_u32<0x4E>((uint32_t)better);
            if (i < n && (tid & 3) == 0 && better < p.beams) emit(better, s, t);
        }
        return;
    }
    uint64_t s0 = ~0ull, t0 = 0;  // the one picked last
    for (int k = 0; k < p.beams; ++k) {
        uint64_t s1 = 0, t1 = ~0ull;
        for (int i = tid; i < total; i += 256) {
            const uint64_t s = candidate(i, p.cand[row0 * per + i], at);
            if (s && (s < s0 || (s == s0 && at > t0)) && (s > s1 || (s == s1 && at < t1))) {
                s1 = s;
                t1 = at;
            }
        }
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) {
            const uint64_t s = shfl_xor64(s1, m), t = shfl_xor64(t1, m);
            if (s > s1 || (s == s1 && t < t1)) {
                s1 = s;
                t1 = t;
            }
        }
        if (lane == 0) {
            ws[wave] = s1;
            wt[wave] = t1;
        }
        __syncthreads();
        s0 = ws[0];
        t0 = wt[0];
        for (int w = 1; w < 4; ++w)
            if (ws[w] > s0 || (ws[w] == s0 && wt[w] < t0)) {
                s0 = ws[w];
                t0 = wt[w];
            }
        if (tid == 0) emit(k, s0, t0);
        __syncthreads();
    }
}

// Columns per workgroup: 8192, fewer (half the time of a workgroup, twice the parts to join) where the
// device would not be filled.
void beam_select_plan(int64_t groups, int beams, int64_t vocab, int* nsplit, int64_t* chunk) {
    int64_t ch = kBeamCols;
    while (ch > 2048 && groups * beams * ((vocab + ch - 1) / ch) < 256) ch /= 2;
    *chunk = ch;
    *nsplit = (int)((vocab + 7 + ch - 1) / ch);  // a row starts up to 7 columns behind a 16-byte boundary
}

template <typename E>
static int launch_select_t(const BeamSelectParams& p, hipStream_t s) {
    const dim3 grid((unsigned)(p.groups * p.beams * p.nsplit));
    switch (p.chunk) {
        case 2048: hipLaunchKernelGGL((beam_part_kernel<E, 8>), grid, dim3(256), 0, s, p); break;
        case 4096: hipLaunchKernelGGL((beam_part_kernel<E, 16>), grid, dim3(256), 0, s, p); break;
        default: hipLaunchKernelGGL((beam_part_kernel<E, 32>), grid, dim3(256), 0, s, p); break;
    }
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)p.groups), dim3(256), 0, s, p);
    return (int)hipGetLastError();
}

int launch_beam_select(const BeamSelectParams& p, int bf16, hipStream_t s) {
    return bf16 ? launch_select_t<BF16>(p, s) : launch_select_t<F32>(p, s);
}

}  // namespace inf
