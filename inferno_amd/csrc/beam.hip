// beam.hip -- beam search's selection: of a group's beams x vocabulary candidates the best
// `beams` by score + logit - lse.
//
// The logits are read once.  A workgroup holds up to 8192 columns of one beam in registers, forms
// their maximum and sum of exponentials and finds their best `beams`; a second launch joins a
// beam's parts to its lse and ranks what is left of a group, some hundreds of candidates, by the
// whole score in 64 bits.  Within a beam the score's order is the logits', so the first step needs
// no lse and is exact; between beams scores can lie close together, and there the sums of
// exponentials are held in 64 bits as well (the exponentials themselves are 32-bit).  Equal scores go to
// the lower beam, then the lower token.
//
// The best few of many: with each lane's largest value known, the beams-th largest of a wave's 64 is
// at most the beams-th largest of all its values, so only values from the best wave's up can matter:
// two or three times as many as there are beams.  They are picked into LDS, and each counts those
// that are better.
//
// 32 groups of 8 beams, 50257 bf16 columns, 26 MB: 16.1 us, 10.8 the first launch (4.3 would be the
// reads alone at HBM's rate, 2 a launch; all its workgroups run at once, so that what follows the reads
// is not hidden by others' reads) and 5.3 the second.  One group of 4 beams, 8192 fp32 columns: 8.9 us,
// two launches of 4 us each that are latency throughout.  Much of that is the fetching of code that
// runs once: loops stay rolled where values are few.
#include "common.h"
#include "kernels.h"

namespace inf {

namespace {

constexpr int kBeamCols = 8192;  // columns of a workgroup at most: 32 per thread, in registers
constexpr int kBeamList = 1024;  // candidates in LDS; more of them (equal ones) are picked one by one

// 16 bytes from any address of an element.
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
__device__ __forceinline__ u32x4 ld16_any(const float* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4_a4*>(p));
}
__device__ __forceinline__ u32x4 ld16_any(const uint16_t* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2*>(p));
}

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

// A group's candidate, its score an ordered number; `at` is the beam and, inverted, the logit: logits may differ
// by less than the last bit of their scores.
struct Ranked {
    uint64_t score, at;
    uint32_t token;
    __device__ __forceinline__ bool before(const Ranked& o) const {
        return score > o.score || (score == o.score && (at < o.at || (at == o.at && token < o.token)));
    }
};

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
    __shared__ uint32_t wnth[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t row = blockIdx.x / p.nsplit;
    const int split = blockIdx.x % p.nsplit;
    if (!beam_lives(p, row)) return;
    // This workgroup's columns are [0, hi) from its first one on.  They are counted from the row's start, so that equal
    // rows are summed alike wherever they lie: 16 bytes are loaded from any address that a column has.
    const int64_t c0 = (int64_t)split * (256 * N);
    const T* x = (const T*)p.logits + row * p.ld + c0;
    const int hi = (int)min((int64_t)(256 * N), p.vocab - c0);
    // The whole 16-byte pieces are this thread's N columns, and the few columns behind them one more.  Every load stands
    // alone, at a place inside the row: under a condition the compiler would wait for each before the next.
    const int last = hi / GE * GE - GE, edge = last + GE + tid;
    const bool tail = edge < hi;
    float v[N + 1];  // columns outside are -inf
    v[N] = -INFINITY;
    u32x4 raw[NV];
    if (last >= 0) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
            raw[u] = ld16_any(x + min((u * 256 + tid) * GE, last));
    }
    if (tail) v[N] = E::ld(x + edge);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int c = (u * 256 + tid) * GE;
        const bool in = c <= last;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t two = in ? raw[u][e] : sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
            if constexpr (sizeof(T) == 4) {
                v[u * GE + e] = __uint_as_float(two);
            } else {
                v[u * GE + 2 * e] = __uint_as_float(two << 16);
                v[u * GE + 2 * e + 1] = __uint_as_float(two & 0xffff0000u);
            }
        }
    }
    auto key = [&](float y, int c) {
        return (uint64_t)ordered_logit(y) << 32 | (uint32_t)~(uint32_t)(c0 + c);
    };
    float mx = v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) mx = fmaxf(mx, v[i]);
    const uint32_t lane_best = ordered_logit(mx);
    mx = wave_all(mx, [](float a, float b) { return fmaxf(a, b); });
    const float ref = mx == -INFINITY ? 0.f : mx;
    // Terms in 32 bits: one at d below the maximum is off by (2.25 |d| + 2) 2^-24 of itself (difference, product,
    // log2 e and v_exp_f32), and sums of four by 2^-23 more.  All further sums in 64.  |d| has a mean of at most 18 under the
    // terms' shares (2^31 columns), so the lse is off by 2^-18 at most.
    double sum = fast_exp2((v[N] - ref) * kLog2e);
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
    const uint32_t nth = wave_nth<16>(lane_best, p.beams);
    if (lane == 0) wnth[wave] = nth;
    __syncthreads();
    // Columns of -inf, those outside among them, are not picked.
    constexpr float kLowest = -3.402823466e38f;
    const float least = logit_of(max(max(max(wnth[0], wnth[1]), max(wnth[2], wnth[3])), ordered_logit(kLowest)));
    if (tid == 0) {
        const float M = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
        double S = 0.0;
        for (int i = 0; i < 4; ++i) S += wmax[i] == -INFINITY ? wsum[i] : wsum[i] * exp((double)wmax[i] - (double)M);
        p.maxs[blockIdx.x] = M;
        p.sums[blockIdx.x] = S;
    }
    auto pick = [&](float y, int c) {
        const int at = atomicAdd(&count, 1);
        if (at < kBeamList) list[at] = key(y, c);
    };
    if (v[N] >= least) pick(v[N], edge);
    uint32_t hits = 0;  // few, and read again: a copy of the code for each column would take longer to fetch
#pragma unroll
    for (int i = 0; i < N; ++i) hits |= (v[i] >= least) << i;
#pragma unroll 1
    for (; hits; hits &= hits - 1) {
        const int i = __builtin_ctz(hits), c = (i / GE * 256 + tid) * GE + i % GE;
        pick(E::ld(x + c), c);
    }
    __syncthreads();
    const int n = count;
    uint64_t* out = p.cand + (int64_t)blockIdx.x * p.beams;
    if (n <= kBeamList) {
        if (n < p.beams && wave == 0) {
            // fewer above -inf than beams: the lowest columns of the others (where there is a NaN, nobody asks)
            int at = n;
            for (int c = 0; c < hi && at < p.beams; c += 64) {
                const bool rest = c + lane < hi && !(E::ld(x + c + lane) >= kLowest);
                const uint64_t m = __ballot(rest);
                const int i =
                    __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, at));
                if (rest && i < p.beams) out[i] = key(-INFINITY, c + lane);
                at += __popcll(m);
            }
            if (lane < p.beams && lane >= at) out[lane] = 0;  // fewer columns than beams
        }
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
#pragma unroll 4
        for (int c = tid; c < hi; c += 256) {
            const uint64_t y = key(E::ld(x + c), c);
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

// One workgroup of 16 waves a group (4 waves: 17.1 us instead of 16.8 with 32 groups of 8 beams and 50257 bf16
// columns, 24.0 instead of 20.7 with 16 groups of 16 beams).
__global__ __launch_bounds__(1024) void beam_join_kernel(BeamSelectParams p) {
    constexpr int W = 16, kThreads = 64 * W;
    enum { kLives, kFinished, kFlat };  // a flat beam's candidates are the first tokens, all with its score
    __shared__ double base[kMaxBeams];  // score - log(sum); the score of a beam that is finished or flat
    // The logits' maximum.  It is taken from the logits first: where they are far from 0 (all at the type's lowest value,
    // a row without tokens), a sum with the lse would lose the score.
    __shared__ float maximum[kMaxBeams];
    __shared__ int kind[kMaxBeams];
    __shared__ uint64_t ls[kBeamList], lt[kBeamList];
    __shared__ uint32_t lk[kBeamList];
    __shared__ int count;
    __shared__ Ranked wr[W];
    __shared__ uint32_t wall[W];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int64_t row0 = (int64_t)blockIdx.x * p.beams;
    const int per = p.nsplit * p.beams;  // candidates of a beam
    // A wave takes whole beams, wave, wave + W, ..., 64 of a beam's candidates at a time, so that a beam's state is the
    // same for all lanes.  Up to U such rounds stay in registers, loaded before the lse is known.  Each part's
    // candidates are in order, so the lanes are turned from round to round: lanes that held only best ones, and
    // lanes that held only last ones, would bound the best few badly.
    constexpr int U = 2;  // more only cost time: 17.2 us with 4, 17.5 with 8, of 16.8
    const int rounds = (per + 63) / 64, all = (p.beams - wave + W - 1) / W * rounds;  // 0 or less: no beam
    struct At {
        int b, i, turn;
    };
    auto start = [&] { return At{wave, 0, 0}; };
    auto next = [&](At& a) {
        a.turn += 41;
        if (++a.i == rounds) {
            a.i = 0;
            a.b += W;
        }
    };
    auto place = [&](const At& a) { return 64 * a.i + ((lane + a.turn) & 63); };
    uint64_t cand[U];
    auto load = [&](At& a) {
#pragma unroll
        for (int u = 0; u < U; ++u) {  // one load after the other, under no condition
            cand[u] = p.cand[(row0 + min(a.b, p.beams - 1)) * per + min(place(a), per - 1)];
            next(a);
        }
    };
    At loaded = start();
    load(loaded);
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
                const int64_t i = row * p.nsplit + min(i0 + 8 * k + (tid & 7), p.nsplit - 1);
                m[k] = p.maxs[i];
                s[k] = p.sums[i];
            }
#pragma unroll
            for (int k = 0; k < P; ++k) {
                if (i0 + 8 * k + (tid & 7) >= p.nsplit) {
                    m[k] = -INFINITY;
                    s[k] = 0.0;
                }
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
            const double ls = log(S);
            const bool lives = !finished && isfinite(score), fine = isfinite(M) && isfinite(ls);
            base[b] = !lives ? (double)score : fine ? (double)score - ls : __longlong_as_double(0x7ff8000000000000ll);
            maximum[b] = M;
            kind[b] = finished ? kFinished : lives && fine ? kLives : kFlat;
        }
    }
    if (tid == 0) count = 0;
    __syncthreads();
    // Beam b's candidate c, the j-th (a score of 0: there is none).
    auto candidate = [&](int b, int j, uint64_t c) -> Ranked {
        Ranked r{0, (uint64_t)b << 32, (uint32_t)j};
        double score = base[b];
        if (kind[b] == kLives) {
            if (!c) return r;
            r.token = ~(uint32_t)c;
            r.at |= ~(uint32_t)(c >> 32);
            score += (double)logit_of((uint32_t)(c >> 32)) - (double)maximum[b];
        } else if (kind[b] == kFinished) {
            if (j) return r;
            r.token = (uint32_t)p.eos;
        } else if (j >= p.beams || j >= p.vocab) {
            return r;
        }
        r.score = ordered_score(score);
        return r;
    };
    auto scan = [&](auto f) {  // f(candidate) for this lane's candidates
        At a = start();
        if (all > U) loaded = a;
        for (int r = 0; r < all; r += U) {
            if (all > U) load(loaded);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r + u < all) {
                    const int j = place(a);
                    if (j < per)
                        if (const Ranked r = candidate(a.b, j, cand[u]); r.score) f(r);
                }
                next(a);
            }
        }
    };
    auto emit = [&](int k, const Ranked& r) {
        const int b = (int)(r.at >> 32), token = (int)r.token;
        const uint64_t s = r.score;
        const int64_t o = row0 + k;
        p.tokens[o] = token;
        p.parents[o] = b;
        p.scores_out[o] = (float)__longlong_as_double((long long)(s == 1 ? 0x7ff8000000000000ull
                                                                  : s >> 63 ? s & ~(1ull << 63) : ~s));
        if (p.finished_out) p.finished_out[o] = kind[b] == kFinished || token == p.eos;
    };
    uint32_t best = 0;
    scan([&](const Ranked& r) { best = max(best, (uint32_t)(r.score >> 32)); });
    // The group's `beams`-th is no less than any wave's.
    const uint32_t nth = wave_nth<4>(best, p.beams);
    if (lane == 0) wall[wave] = nth;
    __syncthreads();
    uint32_t least = 0;
    for (int w = 0; w < W; ++w) least = max(least, wall[w]);
    scan([&](const Ranked& r) {
        if ((uint32_t)(r.score >> 32) >= least) {
            const int k = atomicAdd(&count, 1);
            if (k < kBeamList) {
                ls[k] = r.score;
                lt[k] = r.at;
                lk[k] = r.token;
            }
        }
    });
    __syncthreads();
    const int n = count;
    if (n <= kBeamList) {
        for (int i0 = 0; i0 < n; i0 += kThreads / 4) {
            const int i = i0 + (tid >> 2);
            const int own = min(i, n - 1);
            const Ranked r{ls[own], lt[own], lk[own]};
            int better = 0;
#pragma unroll 4
            for (int j = tid & 3; j < n; j += 4) better += Ranked{ls[j], lt[j], lk[j]}.before(r);
            better += (int)dpp_u32<0xB1>((uint32_t)better);
            better += (int)dpp_u32<0x4E>((uint32_t)better);
            if (i < n && (tid & 3) == 0 && better < p.beams) emit(better, r);
        }
        return;
    }
    Ranked last{~0ull, 0, 0};  // the one picked last
    for (int k = 0; k < p.beams; ++k) {
        Ranked top{0, ~0ull, ~0u};
        scan([&](const Ranked& r) {
            if (last.before(r) && r.before(top)) top = r;
        });
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) {
            const Ranked r{shfl_xor64(top.score, m), shfl_xor64(top.at, m), (uint32_t)__shfl_xor(top.token, m, 64)};
            if (r.before(top)) top = r;
        }
        if (lane == 0) wr[wave] = top;
        __syncthreads();
        last = wr[0];
        for (int w = 1; w < W; ++w)
            if (wr[w].before(last)) last = wr[w];
        if (tid == 0) emit(k, last);
        __syncthreads();
    }
}

// Columns per workgroup: 8192, fewer (half the time of a workgroup, twice the parts to join) where the
// device would not be filled (beams of 50257 bf16 columns, us, 8192 and 4096: 64 beams 11.6 and 12.5, 256 16.0
// and 18.1; 32 beams, 4096 and 2048: 11.3 and 13.4).
void beam_select_plan(int64_t groups, int beams, int64_t vocab, int* nsplit, int64_t* chunk) {
    int64_t ch = kBeamCols;
    while (ch > 2048 && groups * beams * ((vocab + ch - 1) / ch) < 256) ch /= 2;
    *chunk = ch;
    *nsplit = (int)((vocab + ch - 1) / ch);
}

template <typename E>
static int launch_select_t(const BeamSelectParams& p, hipStream_t s) {
    const dim3 grid((unsigned)(p.groups * p.beams * p.nsplit));
    switch (p.chunk) {
        case 2048: hipLaunchKernelGGL((beam_part_kernel<E, 8>), grid, dim3(256), 0, s, p); break;
        case 4096: hipLaunchKernelGGL((beam_part_kernel<E, 16>), grid, dim3(256), 0, s, p); break;
        default: hipLaunchKernelGGL((beam_part_kernel<E, 32>), grid, dim3(256), 0, s, p); break;
    }
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)p.groups), dim3(1024), 0, s, p);
    return (int)hipGetLastError();
}

int launch_beam_select(const BeamSelectParams& p, int bf16, hipStream_t s) {
    return bf16 ? launch_select_t<BF16>(p, s) : launch_select_t<F32>(p, s);
}

}  // namespace inf
