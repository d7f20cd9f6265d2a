// paged4.hip -- a key-value cache in 4 bits and pages: writing new tokens to it, reading positions back, and
// attention of one new token per row over it.
//
// Blocks of 32 channels of a token's key or value share a power of two 2^(byte - 127); each channel is one of
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it (two bits of exponent, one of mantissa, as the MX formats' FP4), with a sign.
// Channel 2 i lies in the low half of byte i.  The format is the one that gfx950 converts to and from in
// hardware, scale included, two values an instruction, and every value is exact in bf16 and fp32: attention
// over the cache is attention over those values.  (A scale of 32 bits per row and even steps of 4 bits have the
// same error on normal channels, but cost a multiplication and an addition for each value.)
//
// The power is that of the block's largest magnitude, two lower, so that this one lies in [4, 8); 6 to 8 go to 6.
// It is at least 2^-125: no value that is held is subnormal.  A block with an infinity or a NaN has byte 255, and
// all of it reads as NaN.
//
// Key j of a row lies in slot j % P of page table[row][j / P], as in the cache of full precision; P is at least
// 16, so that a tile of 16 keys lies in one page.  The scales of a block of neighbouring slots lie next to each other.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "paged_shares.h"

namespace inf {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

namespace {

__device__ __forceinline__ f32x4 mfma16x16x32bf16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ int page_of(const Paged4View& c, const int32_t* table, int j) {
    const int p = table[j >> c.page_shift];
    return (unsigned)p < (unsigned)c.n_pages ? p : -1;
}

// 2^(byte - 127), NaN for 255.
__device__ __forceinline__ float block_scale(uint32_t byte) {
    return __uint_as_float(byte == 255 ? 0x7fc00000u : byte << 23);
}

// Eight channels of a block: four bytes.
__device__ __forceinline__ bf16x8 to_bf16(uint32_t codes, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0),
                 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2),
                 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <typename E>
__device__ __forceinline__ void store1(E* dst, float v) {
    if constexpr (sizeof(E) == 4)
        *dst = v;
    else
        *dst = f32_to_bf16(v);
}

}  // namespace

// ============================================================================
// Append and read: a thread takes eight channels of a token's key and of its value, four neighbouring threads a
// block; channels fastest, then heads, then tokens, as a projection's output lies.  Bound by HBM.
// ============================================================================
namespace {

struct Encoded {
    uint32_t codes, byte;
};
template <typename E>
__device__ __forceinline__ Encoded encode8(const E* src) {
    const f32x4 a = ld4(src), b = ld4(src + 4);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        top = max(top, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
    top = max(top, dpp_u32<0xB1>(top));  // the block's four threads: quad_perm [1,0,3,2], [2,3,0,1]
    top = max(top, dpp_u32<0x4E>(top));
    const uint32_t e = top >> 23;
    const uint32_t byte = e == 255 ? 255u : max(e, 4u) - 2;
    const float s = __uint_as_float((e == 255 ? 127u : byte) << 23);
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, a[0], a[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, a[2], a[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, b[0], b[1], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, b[2], b[3], s, 3);
    return {q, byte};
}

template <typename E>
__device__ __forceinline__ void store8(E* dst, uint32_t codes, float scale) {
    f32x4 v[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x2 x = i == 0 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)
                       : i == 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)
                       : i == 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)
                                : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
        v[i >> 1][2 * (i & 1)] = (float)x[0];
        v[i >> 1][2 * (i & 1) + 1] = (float)x[1];
    }
    st4(dst, v[0]);
    st4(dst + 4, v[1]);
}

}  // namespace

template <int D, typename E>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4AppendParams p) {
    constexpr int P = D / 8;
    const int row = blockIdx.y;
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int th = i / P, c = i % P;
    const int t = th / p.c.heads, h = th - t * p.c.heads;
    const int count = p.counts ? min(p.counts[row], p.Tn) : p.Tn;
    if (t >= count) return;  // a block's threads stay together
    const int64_t slot = (int64_t)p.c.lens[row] - count + t;
    if (slot < 0 || slot >= p.c.cap()) return;
    const int page = page_of(p.c, p.c.table + row * p.c.table_stride, (int)slot);
    if (page < 0) return;
    const int at = (int)slot & ((1 << p.c.page_shift) - 1);
    const Encoded k = encode8((const E*)p.k + row * p.sk.b + h * p.sk.h + t * p.sk.t + 8 * c);
    const Encoded v = encode8((const E*)p.v + row * p.sv.b + h * p.sv.h + t * p.sv.t + 8 * c);
    *reinterpret_cast<uint32_t*>(p.c.k + page * p.c.sk.b + h * p.c.sk.h + at * p.c.sk.t + 4 * c) = k.codes;
    *reinterpret_cast<uint32_t*>(p.c.v + page * p.c.sv.b + h * p.c.sv.h + at * p.c.sv.t + 4 * c) = v.codes;
    if (c % 4 == 0) {
        p.c.ks[page * p.c.sks.b + h * p.c.sks.h + c / 4 * p.c.sks.t + at] = (uint8_t)k.byte;
        p.c.vs[page * p.c.svs.b + h * p.c.svs.h + c / 4 * p.c.svs.t + at] = (uint8_t)v.byte;
    }
}

// Positions first[row] + t as dense rows; zeros outside the row, NaN where its table names no page of the pool's.
template <int D, typename E>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4ReadParams p) {
    constexpr int P = D / 8;
    const int row = blockIdx.y;
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int ht = i / P, c = i % P;
    const int h = ht / p.Tn, t = ht - h * p.Tn;
    if (h >= p.c.heads) return;
    const int64_t slot = (p.first ? (int64_t)p.first[row] : 0) + t;
    uint32_t k = 0, v = 0;
    float ks = 1.f, vs = 1.f;
    if (slot >= 0 && slot < p.c.lens[row] && slot < p.c.cap()) {
        const int page = page_of(p.c, p.c.table + row * p.c.table_stride, (int)slot);
        if (page < 0) {
            ks = vs = __builtin_nanf("");
        } else {
            const int at = (int)slot & ((1 << p.c.page_shift) - 1);
            k = *reinterpret_cast<const uint32_t*>(p.c.k + page * p.c.sk.b + h * p.c.sk.h + at * p.c.sk.t + 4 * c);
            v = *reinterpret_cast<const uint32_t*>(p.c.v + page * p.c.sv.b + h * p.c.sv.h + at * p.c.sv.t + 4 * c);
            ks = block_scale(p.c.ks[page * p.c.sks.b + h * p.c.sks.h + c / 4 * p.c.sks.t + at]);
            vs = block_scale(p.c.vs[page * p.c.svs.b + h * p.c.svs.h + c / 4 * p.c.svs.t + at]);
        }
    }
    store8((E*)p.k + row * p.sk.b + h * p.sk.h + t * p.sk.t + 8 * c, k, ks);
    store8((E*)p.v + row * p.sv.b + h * p.sv.h + t * p.sv.t + 8 * c, v, vs);
}

namespace {

template <typename F>
int by_type(int D, int bf16, F f) {
    using std::integral_constant;
    auto go = [&](auto d) { bf16 ? f(d, uint16_t{}) : f(d, float{}); };
    switch (D) {
        case 32: go(integral_constant<int, 32>{}); break;
        case 64: go(integral_constant<int, 64>{}); break;
        case 128: go(integral_constant<int, 128>{}); break;
        default: return (int)hipErrorInvalidValue;
    }
    return (int)hipGetLastError();
}

}  // namespace

int launch_kv4_append(const Kv4AppendParams& p, int bf16, hipStream_t s) {
    const int64_t n = (int64_t)p.Tn * p.c.heads * (p.c.D / 8);
    const dim3 grid((unsigned)((n + 255) / 256), (unsigned)p.c.rows);
    return by_type(p.c.D, bf16, [&](auto d, auto e) {
        hipLaunchKernelGGL((kv4_append_kernel<decltype(d)::value, decltype(e)>), grid, dim3(256), 0, s, p);
    });
}

int launch_kv4_read(const Kv4ReadParams& p, int bf16, hipStream_t s) {
    const int64_t n = (int64_t)p.Tn * p.c.heads * (p.c.D / 8);
    const dim3 grid((unsigned)((n + 255) / 256), (unsigned)p.c.rows);
    return by_type(p.c.D, bf16, [&](auto d, auto e) {
        hipLaunchKernelGGL((kv4_read_kernel<decltype(d)::value, decltype(e)>), grid, dim3(256), 0, s, p);
    });
}

// ============================================================================
// Attention of one query per row, as over the cache of full precision: steps of a row's keys shared out evenly to
// workgroups, one per key-value head in each share; four waves take T tiles of 16 keys of a step each; S^T = K Q^T
// (keys x heads), online softmax down the lane's column, O^T += V^T P^T; parts joined by a second launch.
//
// Keys and values become bf16 in registers, exactly.  fp32 queries and their probabilities are taken in three bf16
// parts (24 bits), bf16 ones' probabilities in two.
// ============================================================================
namespace {

constexpr int kKv4PerCu = 3;  // workgroups of a CU: what the registers allow

template <int D>
__device__ __forceinline__ int kv4_steps(int len, int max_len) {
    constexpr int step = kv4_step(D);
    return len > max_len ? 0 : (max(len, 0) + step - 1) / step;
}

}  // namespace

template <int D, typename E>
__global__ __launch_bounds__(256, kKv4PerCu) void kv4_split_kernel(Kv4DecodeParams p) {
    constexpr bool F = sizeof(E) == 4;
    constexpr int PARTS = F ? 3 : 1;      // of q
    constexpr int STEP = kv4_step(D);
    constexpr int T = STEP / 64;          // tiles of 16 keys per wave
    constexpr int NK = D / 32;            // words of a key row per lane: products of a tile
    constexpr int VD = D / 16;            // columns of a value row per lane
    constexpr int LD = D + 4;
    extern __shared__ __attribute__((aligned(16))) float lds[];  // o [4][heads][LD], then m, l [4][16]

    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int ht = p.head_tiles;
    int unit = blockIdx.x, tile = 0;
    if (ht > 1) {
        const int grp = blockIdx.x >> 3;
        tile = grp % ht;
        unit = grp / ht * 8 + (blockIdx.x & 7);
        if (unit >= p.c.heads * (p.groups ? p.groups : p.c.rows)) return;
    }
    const int h = unit % p.c.heads, group = unit / p.c.heads;
    const int g0 = tile * 16, gn = min(16, p.G - g0);  // query heads of this tile
    const int row0 = p.groups ? blockIdx.y * kPagedBlock : group;
    const int nrows = p.groups ? min(kPagedBlock, p.c.rows - row0) : 1;

    // Lane i: the first step of the block's row i.  This share's are [step, stop) of them; row r, the first
    // one, has [begin, end).
    const int mylen = lane < nrows ? p.c.lens[row0 + lane] : 0;
    int step = 0, r = 0, begin = 0, steps = kv4_steps<D>(mylen, p.max_len), starts = steps;
    if (nrows > 1) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int up = __shfl_up(starts, d, 64);
            if (lane >= d) starts += up;
        }
    }
    const int all = __builtin_amdgcn_readlane(starts, nrows - 1);
    int stop = all, end = __builtin_amdgcn_readlane(starts, 0);
    starts -= steps;
    if (p.groups) {
        if (unit == 0 && tile == 0 && wave == 0) {
            if (lane < nrows) p.first[row0 + lane] = starts;
            if (lane == 0) p.first[p.c.rows + blockIdx.y] = all;
        }
        const Shares shares(all, p.groups);
        step = shares.start(group);
        stop = shares.start(group + 1);
    } else if (!all) {  // an empty row is 0, one longer than max_len NaN
        const int len = __builtin_amdgcn_readlane(mylen, 0);
        for (int i = tid; i < gn * D; i += 256)
            store1((E*)p.o + row0 * p.so.b + (h * p.G + g0 + i / D) * p.so.h + i % D,
                   len > p.max_len ? __builtin_nanf("") : 0.f);
    }
    if (step >= stop) return;
    if (nrows > 1) {
        // the last row that starts at or before `step`
        r = __popcll(__ballot(lane < nrows && starts <= step)) - 1;
        begin = __builtin_amdgcn_readlane(starts, r);
        end = r + 1 < nrows ? __builtin_amdgcn_readlane(starts, r + 1) : all;
    }
    const int mask = (1 << p.c.page_shift) - 1, last_page = p.c.max_pages - 1;
    // this lane's places in a tile: key col, channels D / 4 * g on; values of keys 4 g + r, channels VD * col on
    const uint8_t* K = p.c.k + h * p.c.sk.h;
    const uint8_t* V = p.c.v + h * p.c.sv.h;
    const uint8_t* KS = p.c.ks + h * p.c.sks.h;
    const uint8_t* VS = p.c.vs + h * p.c.svs.h;
    const int k_at = col * (int)p.c.sk.t + g * (D / 8), ks_at = g * D / 128 * (int)p.c.sks.t + col;
    const int v_at = 4 * g * (int)p.c.sv.t + col * (VD / 2), vs_at = col * D / 512 * (int)p.c.svs.t + 4 * g;
    uint32_t kr[T][NK], ksr[T], vr[T][4], vsr[T];

    for (;;) {  // the rows of the share
        const int row = row0 + r, s0 = step - begin, s1 = min(stop, end) - begin;
        const int32_t* table = p.c.table + row * p.c.table_stride;
        const int base0 = s0 * STEP + 16 * T * wave;
        const int len = __builtin_amdgcn_readlane(mylen, r);
        int next[T] = {};
        auto read_pages = [&](int base) {
#pragma unroll
            for (int t = 0; t < T; ++t)
                next[t] = table[min(__builtin_amdgcn_readfirstlane(base + 16 * t) >> p.c.page_shift, last_page)];
        };
        read_pages(base0);
        const int j1 = min(len, s1 * STEP);

        // Q^T: column = head, the channels that a key's words have
        bf16x8 qf[NK][PARTS];
        {
            const E* q = (const E*)p.q + row * p.sq.b + (int64_t)(h * p.G + g0 + min(col, gn - 1)) * p.sq.h + g * (D / 4);
#pragma unroll
            for (int s = 0; s < NK; ++s) {
                const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                const f32x4 a = col < gn ? ld4(q + 8 * s) : zero, b = col < gn ? ld4(q + 8 * s + 4) : zero;
                if constexpr (F) {
                    const Bf3x8 x = split3(a, b);
                    qf[s][0] = x.h;
                    qf[s][1] = x.m;
                    qf[s][2] = x.l;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        qf[s][0][i] = (__bf16)a[i];
                        qf[s][0][4 + i] = (__bf16)b[i];
                    }
                }
            }
        }

        f32x4 acc[VD];
#pragma unroll
        for (int j = 0; j < VD; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        bool bad = false;
        for (int base = base0; base < j1; base += STEP) {
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const bool in = (unsigned)next[t] < (unsigned)p.c.n_pages;
                bad |= !in && base + 16 * t < j1;
                const int64_t page = in ? next[t] : 0;
                const int at = __builtin_amdgcn_readfirstlane(base + 16 * t) & mask;
                const uint8_t* kp = K + page * p.c.sk.b + at * p.c.sk.t + k_at;
                if constexpr (NK == 4) {
                    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp));
#pragma unroll
                    for (int s = 0; s < 4; ++s) kr[t][s] = x[s];
                } else if constexpr (NK == 2) {
                    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(kp));
                    kr[t][0] = x[0];
                    kr[t][1] = x[1];
                } else {
                    kr[t][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(kp));
                }
                ksr[t] = KS[page * p.c.sks.b + at + ks_at];
                const uint8_t* vp = V + page * p.c.sv.b + at * p.c.sv.t + v_at;
#pragma unroll
                for (int r = 0; r < 4; ++r, vp += p.c.sv.t) {
                    if constexpr (VD == 8)
                        vr[t][r] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(vp));
                    else if constexpr (VD == 4)
                        vr[t][r] = __builtin_nontemporal_load(reinterpret_cast<const uint16_t*>(vp));
                    else
                        vr[t][r] = __builtin_nontemporal_load(vp);
                }
                vsr[t] = *reinterpret_cast<const uint32_t*>(VS + page * p.c.svs.b + at + vs_at);
            }
            if (base + STEP < j1) read_pages(base + STEP);
            __builtin_amdgcn_sched_barrier(0);  // all of the step's loads before its first product
            float x[4 * T];
#pragma unroll
            for (int t = 0; t < T; ++t) {
                f32x4 st = {0.f, 0.f, 0.f, 0.f};
                const float ks = block_scale(ksr[t]);
#pragma unroll
                for (int s = 0; s < NK; ++s) {
                    const bf16x8 k = to_bf16(kr[t][s], ks);
#pragma unroll
                    for (int i = PARTS - 1; i >= 0; --i) st = mfma16x16x32bf16(k, qf[s][i], st);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) x[4 * t + r] = st[r] * p.cs;
            }
            if (base + 16 * T > j1) {  // keys behind the end: nothing of what their slots hold counts
#pragma unroll
                for (int i = 0; i < 4 * T; ++i)
                    if (base + 16 * (i >> 2) + 4 * g + (i & 3) >= j1) {
                        x[i] = -INFINITY;
                        vr[i >> 2][i & 3] = 0;
                        vsr[i >> 2] = (vsr[i >> 2] & ~(255u << (8 * (i & 3)))) | 127u << (8 * (i & 3));
                    }
            }
            float mx = m;
#pragma unroll
            for (int i = 0; i < 4 * T; ++i) mx = fmaxf(mx, x[i]);
            mx = max_xor32(max_xor16(mx));
            const float ref = mx == -INFINITY ? 0.f : mx;  // no key above -inf yet: keep everything at 0
            const float alpha = fast_exp2(m - ref);
            m = mx;
            l *= alpha;
#pragma unroll
            for (int j = 0; j < VD; ++j) acc[j] *= alpha;
#pragma unroll
            for (int i = 0; i < 4 * T; ++i) {
                x[i] = fast_exp2(x[i] - ref);
                l += x[i];
            }
#pragma unroll
            for (int t = 0; t < T; t += 2) {  // 32 keys a product
                bf16x8 ph, pm, pl;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    ph[i] = (__bf16)x[4 * t + i];
                    const float rest = x[4 * t + i] - (float)ph[i];
                    pm[i] = (__bf16)rest;
                    if constexpr (F) pl[i] = (__bf16)(rest - (float)pm[i]);
                }
                uint32_t vb[8][VD / 2];  // eight keys' pairs of columns
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t w = vr[t + (i >> 2)][i & 3];
                    const float vs = block_scale(vsr[t + (i >> 2)] >> (8 * (i & 3)) & 255);
                    vb[i][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vs, 0));
                    if constexpr (VD >= 4)
                        vb[i][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vs, 1));
                    if constexpr (VD >= 8) {
                        vb[i][2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vs, 2));
                        vb[i][3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vs, 3));
                    }
                }
#pragma unroll
                for (int j = 0; j < VD; ++j) {
                    const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;  // high or low halves of two words
                    u32x4 a;
#pragma unroll
                    for (int i = 0; i < 4; ++i) a[i] = __builtin_amdgcn_perm(vb[2 * i + 1][j >> 1], vb[2 * i][j >> 1], sel);
                    const bf16x8 v = __builtin_bit_cast(bf16x8, a);
                    if constexpr (F) acc[j] = mfma16x16x32bf16(v, pl, acc[j]);
                    acc[j] = mfma16x16x32bf16(v, pm, acc[j]);
                    acc[j] = mfma16x16x32bf16(v, ph, acc[j]);
                }
            }
        }

        // Join the waves: lane (col, g) holds head col's o[VD (4 g + r) + j] in acc[j][r].
        l += shfl_xor(l, 16);
        l += shfl_xor(l, 32);
        if (__any(bad)) l = __builtin_nanf("");
        float* ms = lds + 4 * gn * LD;
        float* ls = ms + 64;
        if (col < gn) {
            float* dst = lds + (wave * gn + col) * LD + 4 * VD * g;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < VD; ++j) dst[VD * r + j] = acc[j][r];
        }
        if (g == 0) {
            ms[wave * 16 + col] = m;
            ls[wave * 16 + col] = l;
        }
        __syncthreads();
        for (int i = tid; i < gn * D; i += 256) {
            const int head = i / D, d = i % D;
            const float M = fmaxf(fmaxf(ms[head], ms[16 + head]), fmaxf(ms[32 + head], ms[48 + head]));
            const float ref = M == -INFINITY ? 0.f : M;
            float L = 0.f, o = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float wt = fast_exp2(ms[w * 16 + head] - ref);
                L += ls[w * 16 + head] * wt;
                o += lds[(w * gn + head) * LD + d] * wt;
            }
            const int hq = h * p.G + g0 + head;
            if (!p.groups) {
                store1((E*)p.o + row * p.so.b + hq * p.so.h + d, o / L);
            } else {
                // rows and shares meet in one order: row + share is a number of their own
                const int64_t at = ((int64_t)row + blockIdx.y * p.groups + group) * p.Hq + hq;
                p.part[at * D + d] = o;
                if (d == 0) *reinterpret_cast<f32x2*>(p.stats + 2 * at) = f32x2{M, L};
            }
        }
        step += s1 - s0;
        if (step >= stop) return;
        begin = step;
        do {  // past empty rows
            ++r;
            end = r + 1 < nrows ? __builtin_amdgcn_readlane(starts, r + 1) : all;
        } while (end <= step);
        __syncthreads();  // the join's LDS is read
    }
}

// Joins a row's parts: a workgroup for each row and query head.
template <int D, typename E>
__global__ __launch_bounds__(256) void kv4_join_kernel(Kv4DecodeParams p) {
    __shared__ float wsh[kPagedMaxGroups];
    __shared__ f32x4 osh[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x / p.Hq, hq = blockIdx.x % p.Hq;
    const int len = p.c.lens[row], steps = kv4_steps<D>(len, p.max_len);
    E* out = (E*)p.o + row * p.so.b + hq * p.so.h;
    if (!steps) {
        if (tid < D) store1(out + tid, len > p.max_len ? __builtin_nanf("") : 0.f);
        return;
    }
    const int block = row / kPagedBlock, start = p.first[row];
    const Shares shares(p.first[p.c.rows + block], p.groups);
    const int part0 = shares.of(start);
    const RowParts parts = {shares.of(start + steps - 1) - part0 + 1, (int64_t)row + block * p.groups + part0};
    const int64_t at = parts.at * p.Hq + hq;  // part i: Hq further on each
    const f32x2* stats = reinterpret_cast<const f32x2*>(p.stats) + at;
    float M = -INFINITY, L = 0.f;
    for (int i = lane; i < parts.n; i += 64) {
        const f32x2 x = stats[(int64_t)i * p.Hq];
        join_part(M, L, x[0], x[1]);
        if (wave == 0) wsh[i] = x[0];
    }
    const float last = M;
    M = wave_all(M, [](float x, float y) { return fmaxf(x, y); });
    const float ref = M == -INFINITY ? 0.f : M;
    L = wave_all(L * fast_exp2(last - ref), [](float x, float y) { return x + y; });
    __syncthreads();
    constexpr int W = D / 4, NG = 256 / W;  // lanes to a part, parts at a time
    const int d = 4 * (tid % W), grp = tid / W;
    const float* part = p.part + at * D + d;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = grp; i < parts.n; i += NG)
        o += *reinterpret_cast<const f32x4*>(part + (int64_t)i * p.Hq * D) * fast_exp2(wsh[i] - ref);
    osh[tid] = o;
    __syncthreads();
    if (tid < D) {
        float r = 0.f;
        for (int i = 0; i < min(NG, parts.n); ++i) r += osh[i * W + tid / 4][tid % 4];
        store1(out + tid, r / L);
    }
}

// Whole rows to the workgroups, with no parts to join, where there are as many (row, head) pairs for each slot of
// the device as the longest row has steps.
int kv4_groups(int rows, int heads, int G, int max_len, int D) {
    const int step = kv4_step(D);
    const int64_t slots = 256 * kKv4PerCu, pairs = (int64_t)heads * ((G + 15) / 16);
    const int64_t steps = ((int64_t)max_len + step - 1) / step;
    if (steps == 1 || rows * pairs >= slots * steps) return 0;
    const int64_t most = std::min(rows, kPagedBlock) * steps;
    return (int)std::max<int64_t>(1, std::min({slots / pairs, most, (int64_t)kPagedMaxGroups}));
}

int launch_attn_decode_kv4(const Kv4DecodeParams& p, int bf16, hipStream_t s) {
    const dim3 grid((unsigned)paged_units(p.c.rows, p.c.heads, p.head_tiles, p.groups),
                    p.groups ? (unsigned)paged_blocks(p.c.rows) : 1u);
    const size_t lds = (size_t)(4 * std::min(p.G, 16) * (p.c.D + 4) + 128) * sizeof(float);
    return by_type(p.c.D, bf16, [&](auto d, auto e) {
        constexpr int D = decltype(d)::value;
        using E = decltype(e);
        hipLaunchKernelGGL((kv4_split_kernel<D, E>), grid, dim3(256), lds, s, p);
        if (p.groups)
            hipLaunchKernelGGL((kv4_join_kernel<D, E>), dim3((unsigned)((int64_t)p.c.rows * p.Hq)), dim3(256), 0, s, p);
    });
}

}  // namespace inf
