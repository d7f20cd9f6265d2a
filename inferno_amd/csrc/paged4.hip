// paged4.hip -- a key-value cache in 4 bits and pages: writing new tokens to it, reading positions back, and
// attention of one new token per row over it.
//
// Blocks of 32 channels of a token's key or value share a power of two 2^(byte - 127); each channel is one of
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it (two bits of exponent, one of mantissa, as the MX formats' FP4), with a sign.
// Channel 2 i lies in the low half of byte i.  The format is the one that gfx950 converts to and from in
// hardware, scale included, two values an instruction, and every value is exact in bf16 and fp32: attention
// over the cache is attention over those values.  (Even steps of 4 bits with a scale of 32 bits a row cost a
// multiplication for each value, with an offset an addition too.  RMS errors, relative, as FP4, in even steps and with an
// offset: normal channels at D 32 0.115, 0.097, 0.078, at D 128 0.115, 0.117, 0.100; of the other channels where one in
// twenty is eight times as large, D 128, 0.23, 0.53, 0.39.)
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

// Byte i of a word as the conversions' scale, 2^(byte - 127), NaN for 255: they read its exponent alone, so that the
// word's other bits may stay.
template <int I = 0>
__device__ __forceinline__ float block_scale(uint32_t word) {
    return __uint_as_float(I < 3 ? word << (23 - 8 * I) : word >> 1);
}

// Loads of a tile's rows: scalar bases and the lanes' 32-bit offsets, past the caches.  (Through pointers, the compiler
// takes every address as a sum of vectors.)
constexpr int kNt = 2;
template <int BYTES>
__device__ __forceinline__ auto load_nt(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    if constexpr (BYTES == 16)
        return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, kNt));
    else if constexpr (BYTES == 8)
        return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)at, 0, kNt));
    else if constexpr (BYTES == 4)
        return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)at, 0, kNt);
    else if constexpr (BYTES == 2)
        return (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)at, 0, kNt);
    else
        return (uint32_t)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, (int)at, 0, kNt);
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
// Append: a thread takes eight channels of a token's key and of its value, four neighbouring threads a block; channels
// fastest, then heads, then tokens, as a projection's output lies.  The values are loaded while the token's page is looked up.
// 8 prompts of up to 1024 tokens, half of that on average, 12 heads of 64, fp32: 28 MB in 8.3 us, 3.4 TB/s; 16 of 512, 8 heads
// of 128, bf16, 42.5 MB in 12.5, the same: a wave writes runs of D / 2 bytes to several heads, and scales as single
// bytes.  64 single tokens 3.1, a launch and three dependent reads.
// ============================================================================
namespace {

struct Raw8 {
    f32x4 a, b;
};
template <typename E>
__device__ __forceinline__ Raw8 raw8(const E* src) {
    return {ld4(src), ld4(src + 4)};
}
struct Encoded {
    uint32_t codes, byte;
};
__device__ __forceinline__ Encoded encode8(const Raw8& x) {
    const f32x4 a = x.a, b = x.b;
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
    const Raw8 kx = raw8((const E*)p.k + row * p.sk.b + h * p.sk.h + t * p.sk.t + 8 * c);
    const Raw8 vx = raw8((const E*)p.v + row * p.sv.b + h * p.sv.h + t * p.sv.t + 8 * c);
    const int64_t slot = (int64_t)p.c.lens[row] - count + t;
    if (slot < 0 || slot >= p.c.cap()) return;
    const int page = page_of(p.c, p.c.table + row * p.c.table_stride, (int)slot);
    if (page < 0) return;
    const int at = (int)slot & ((1 << p.c.page_shift) - 1);
    const Encoded k = encode8(kx), v = encode8(vx);
    *reinterpret_cast<uint32_t*>(p.c.k + page * p.c.sk.b + h * p.c.sk.h + at * p.c.sk.t + 4 * c) = k.codes;
    *reinterpret_cast<uint32_t*>(p.c.v + page * p.c.sv.b + h * p.c.sv.h + at * p.c.sv.t + 4 * c) = v.codes;
    if (c % 4 == 0) {
        p.c.ks[page * p.c.sks.b + h * p.c.sks.h + c / 4 * p.c.sks.t + at] = (uint8_t)k.byte;
        p.c.vs[page * p.c.svs.b + h * p.c.svs.h + c / 4 * p.c.svs.t + at] = (uint8_t)v.byte;
    }
}

// ============================================================================
// Read: positions first[row] + t as dense rows; zeros outside the row, NaN where its table names no page of the pool's.  A
// thread takes CH channels of a key and of its value, one store of 16 bytes each (8 where bf16 rows are aligned to that
// only), past the caches and in the results' order.  Bound by what it writes: 16 rows of 4512 positions, 8 heads of 128, bf16, in
// 82 us, 4.6 TB/s read and written.  Stores that fill no whole line cost twice that past the caches (40 -> 97 us at 100 MB).
// ============================================================================
namespace {

template <int CH>
__device__ __forceinline__ uint32_t codes_of(const uint8_t* row, int c) {
    if constexpr (CH == 8)
        return *reinterpret_cast<const uint32_t*>(row + 4 * c);
    else
        return *reinterpret_cast<const uint16_t*>(row + 2 * c);
}

template <int CH, typename E>
__device__ __forceinline__ void store_ch(E* dst, uint32_t codes, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0),
                 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
    if constexpr (sizeof(E) == 4) {
        __builtin_nontemporal_store(f32x4{(float)a[0], (float)a[1], (float)b[0], (float)b[1]},
                                    reinterpret_cast<f32x4*>(dst));
    } else if constexpr (CH == 8) {
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4, to_bf16(codes, scale)), reinterpret_cast<u32x4*>(dst));
    } else {
        __builtin_nontemporal_store(u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)},
                                    reinterpret_cast<u32x2*>(dst));
    }
}

}  // namespace

constexpr int kReadPer = 4;  // positions of a thread, all of whose loads are under way together

template <int D, typename E, int CH>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4ReadParams p, int blocks) {
    constexpr int P = D / CH, N = 256 / P;
    const int row = blockIdx.y, h = blockIdx.x / blocks;
    const int c = threadIdx.x % P, block = c * CH / 32;
    const int t0 = (blockIdx.x - h * blocks) * (N * kReadPer) + threadIdx.x / P;
    const int64_t first = p.first ? (int64_t)p.first[row] : 0, len = min((int64_t)p.c.lens[row], p.c.cap());
    const int32_t* table = p.c.table + row * p.c.table_stride;
    int page[kReadPer];
#pragma unroll
    for (int u = 0; u < kReadPer; ++u) {
        const int64_t slot = first + t0 + N * u;
        const bool in = t0 + N * u < p.Tn && slot >= 0 && slot < len;
        page[u] = in ? page_of(p.c, table, (int)slot) : -2;  // -1: no page of the pool's, -2: outside the row
    }
    uint32_t k[kReadPer], v[kReadPer];
    float ks[kReadPer], vs[kReadPer];
#pragma unroll
    for (int u = 0; u < kReadPer; ++u) {
        const int at = (int)(first + t0 + N * u) & ((1 << p.c.page_shift) - 1);
        k[u] = v[u] = 0;
        ks[u] = vs[u] = page[u] == -1 ? __builtin_nanf("") : 1.f;
        if (page[u] >= 0) {
            k[u] = codes_of<CH>(p.c.k + page[u] * p.c.sk.b + h * p.c.sk.h + at * p.c.sk.t, c);
            v[u] = codes_of<CH>(p.c.v + page[u] * p.c.sv.b + h * p.c.sv.h + at * p.c.sv.t, c);
            ks[u] = block_scale(p.c.ks[page[u] * p.c.sks.b + h * p.c.sks.h + block * p.c.sks.t + at]);
            vs[u] = block_scale(p.c.vs[page[u] * p.c.svs.b + h * p.c.svs.h + block * p.c.svs.t + at]);
        }
    }
#pragma unroll
    for (int u = 0; u < kReadPer; ++u) {
        const int t = t0 + N * u;
        if (t >= p.Tn) return;
        store_ch<CH>((E*)p.k + row * p.sk.b + h * p.sk.h + t * p.sk.t + CH * c, k[u], ks[u]);
        store_ch<CH>((E*)p.v + row * p.sv.b + h * p.sv.h + t * p.sv.t + CH * c, v[u], vs[u]);
    }
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
    const int ch = bf16 && p.wide ? 8 : 4, per = 256 / (p.c.D / ch) * kReadPer;
    const int blocks = (p.Tn + per - 1) / per;
    const dim3 grid((unsigned)(blocks * p.c.heads), (unsigned)p.c.rows);
    return by_type(p.c.D, bf16, [&](auto d, auto e) {
        constexpr int D = decltype(d)::value;
        using E = decltype(e);
        if (ch == 8)
            hipLaunchKernelGGL((kv4_read_kernel<D, E, sizeof(E) == 2 ? 8 : 4>), grid, dim3(256), 0, s, p, blocks);
        else
            hipLaunchKernelGGL((kv4_read_kernel<D, E, 4>), grid, dim3(256), 0, s, p, blocks);
    });
}

// ============================================================================
// Attention of one query per row, as over the cache of full precision: steps of a row's keys shared out evenly to
// workgroups, one per key-value head in each share; four waves take T tiles of 16 keys of a step each; S^T = K Q^T
// (keys x heads), online softmax down the lane's column, O^T += V^T P^T; parts joined by a second launch.
//
// Keys and values become bf16 in registers, exactly.  fp32 queries and their probabilities are taken in three bf16
// parts (24 bits), bf16 ones' probabilities in two (2^-17, below the result's own rounding).
//
// Bound by memory, and near it by what the CUs do with it: 64 rows of up to 8191 keys, 8 heads of 128 with four query heads
// each, bf16: 286 MB in 54-59 us, 4.9-5.3 TB/s (from the caches 39-45: the load path is busy for 68 % of the time, the vector
// units for 40); 4 rows of 131071, two heads, eight query heads each: 143 MB in 31.3; 32 rows of 2048, 12 heads of 64, fp32:
// 54 MB in 17, half of it waits.  The join's launch is another 4-5.  A step's loads ahead of the last one's products (two
// register sets) gave nothing, nor did two or four workgroups a CU at D = 128; two tiles' values in one load of twice the width,
// exchanged between neighbouring lanes, took 61, 34.5 and 18.3.
// ============================================================================
namespace {

constexpr int kv4_per_cu(int D) { return D == 128 ? 3 : 4; }  // workgroups of a CU: what the registers allow

// What a wave keeps in LDS where its scores pass through it.
constexpr int kv4_wave_floats(bool f32, int HB) {
    const int keys = kKv4Step / 4;
    return HB == 16 ? 0 : (f32 ? 3 : 1) * HB * keys + (f32 ? 3 : 2) * HB * keys / 2 + 16;
}

__device__ __forceinline__ int kv4_steps(int len, int max_len) {
    return len > max_len ? 0 : (max(len, 0) + kKv4Step - 1) / kKv4Step;
}

}  // namespace

// HB: 16, or 1, 2 or 4, at least as many as there are query heads.  A product's result has heads along the
// lanes, so that with few of them most lanes' softmax would be for nothing: below 16, the wave's scores pass through LDS to
// all lanes, 64 / HB of them a head, and the probabilities back.  And the columns that are left take the other bf16
// parts of queries and probabilities, part k of head i in column k HB + i: one product instead of two or three.
// (With the join, us, so and with 16: 32 rows of 2048 keys, 12 heads of 64, fp32, one query head each 19.1 and 24.2, two 20.7
// and 24.0, four 23.1 and 24.8; 32 of 4096, 8 heads of 128, bf16, four 35.4 and 37.0; but eight in bf16, with a fourth kind,
// 38.9 and 39.0.)
template <int D, typename E, int HB>
__global__ __launch_bounds__(256, kv4_per_cu(D)) void kv4_split_kernel(Kv4DecodeParams p) {
    constexpr bool F = sizeof(E) == 4;
    constexpr int PARTS = F ? 3 : 1;      // of q
    constexpr int STEP = kKv4Step;
    constexpr int T = STEP / 64;          // tiles of 16 keys per wave
    constexpr int NK = D / 32;            // words of a key row per lane: products of a tile
    constexpr int VD = D / 16;            // columns of a value row per lane
    constexpr int LD = D + 4;
    constexpr int KEYS = 16 * T;          // of a wave's step
    constexpr int LPH = 64 / HB, NV = KEYS / LPH;  // HB < 16: lanes of a head, keys of a lane
    constexpr int PP = F ? 3 : 2;         // bf16 parts of a probability
    static_assert(HB == 16 || PP * HB <= 16, "a column for every part");
    // o [4][heads][LD], then m, l [4][16]; before that, HB < 16: every wave's scores [PARTS][HB][KEYS], parts of
    // probabilities [PP][HB][KEYS] and factors [HB].  From q_at on, fp32: parts of q [3][heads, or HB][D].
    extern __shared__ __attribute__((aligned(16))) float lds[];

    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
    int step = 0, r = 0, begin = 0, steps = kv4_steps(mylen, p.max_len), starts = steps;
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
    const uint32_t k_at = col * (uint32_t)p.c.sk.t + g * (D / 8);
    uint32_t v_at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v_at[i] = (4 * g + i) * (uint32_t)p.c.sv.t + col * (VD / 2);
    // A step's scales come in one load: tile t's of keys 4 q .. and block b to lane t + T q + 4 T b, and from there to
    // the lanes that need them.  (With two loads for each tile's scales, 4 rows of 131071 keys took 32.4 us,
    // 31.3 so.)
    static_assert(4 * T * NK <= 64, "a lane for every four scales");
    const int scale_block = min(lane / (4 * T), NK - 1), scale_key = lane / T % 4 * 4;
    const uint8_t* KS = p.c.ks + h * p.c.sks.h + scale_block * p.c.sks.t + scale_key;
    const uint8_t* VS = p.c.vs + h * p.c.svs.h + scale_block * p.c.svs.t + scale_key;
    const int ks_lane = 4 * (T * (col / 4) + 4 * T * (g * D / 128)), ks_bit = 8 * (col % 4);
    const int vs_lane = 4 * (T * g + 4 * T * (col * D / 512));
    uint32_t kr[T][NK], ksr[T], vr[T][4], vsr[T];
    const int qn = HB == 16 ? gn : HB;
    float* mine = lds + wave * kv4_wave_floats(F, HB);

    for (;;) {  // the rows of the share
        const int row = row0 + r, s0 = step - begin, s1 = min(stop, end) - begin;
        const int32_t* table = p.c.table + row * p.c.table_stride;
        const int base0 = s0 * STEP + 16 * T * wave;
        const int len = __builtin_amdgcn_readlane(mylen, r);
        // Lane t: the page of the step's tile t, read a step ahead (behind the end, where the table may hold anything, it
        // is not used), and then the places of the tile's rows and scales, which go to scalar registers from there.
        const int tile_key = 16 * (lane & (T - 1));
        auto read_pages = [&](int base) { return table[min((base + tile_key) >> p.c.page_shift, last_page)]; };
        int next = read_pages(base0);
        const int j1 = min(len, s1 * STEP);

        // Q^T: column = head, the channels that a key's words have.  fp32: its parts lie in LDS, [3][heads][D] for all waves
        // (in registers they would be 48 at D = 128: spills).
        bf16x8 qf[F ? 1 : NK];
        if constexpr (F) {
            __bf16* dst = reinterpret_cast<__bf16*>(lds + p.q_at);
            for (int i = tid; i < gn * (D / 8); i += 256) {
                const int head = i / (D / 8), d = i % (D / 8) * 8;
                const E* q = (const E*)p.q + row * p.sq.b + (int64_t)(h * p.G + g0 + head) * p.sq.h + d;
                const Bf3x8 x = split3(ld4(q), ld4(q + 4));
                *reinterpret_cast<bf16x8*>(dst + head * D + d) = x.h;
                *reinterpret_cast<bf16x8*>(dst + (qn + head) * D + d) = x.m;
                *reinterpret_cast<bf16x8*>(dst + (2 * qn + head) * D + d) = x.l;
            }
            __syncthreads();
        } else {
            const E* q = (const E*)p.q + row * p.sq.b + (int64_t)(h * p.G + g0 + min(col, gn - 1)) * p.sq.h + g * (D / 4);
#pragma unroll
            for (int s = 0; s < NK; ++s) {
                const u32x2* src = reinterpret_cast<const u32x2*>(q + 8 * s);
                const u32x2 a = src[0], b = src[1];
                qf[s] = __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]});
            }
        }

        f32x4 acc[VD];
#pragma unroll
        for (int j = 0; j < VD; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        bool bad = false;
        for (int base = base0; base < j1; base += STEP) {
            uint64_t places[2];
            uint32_t ks_words, vs_words;
            {
                const bool in = (unsigned)next < (unsigned)p.c.n_pages;
                bad |= !in && base + tile_key < j1;
                const uint32_t page = in ? next : 0, at = (base + tile_key) & mask;
                places[0] = (uint64_t)K + page * (uint64_t)p.c.sk.b + (uint64_t)at * (uint32_t)p.c.sk.t;
                places[1] = (uint64_t)V + page * (uint64_t)p.c.sv.b + (uint64_t)at * (uint32_t)p.c.sv.t;
                ks_words = *reinterpret_cast<const uint32_t*>(KS + page * (uint64_t)p.c.sks.b + at);
                vs_words = *reinterpret_cast<const uint32_t*>(VS + page * (uint64_t)p.c.svs.b + at);
            }
            if (base + STEP < j1) next = read_pages(base + STEP);
#pragma unroll
            for (int t = 0; t < T; ++t) {
                auto rows = [&](int i, uint32_t bytes) {
                    const uint64_t a = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(places[i] >> 32), t) << 32 |
                                       (uint32_t)__builtin_amdgcn_readlane((int)places[i], t);
                    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(a), (short)0, (int)bytes, 0x00020000);
                };
                const auto kp = rows(0, 15 * (uint32_t)p.c.sk.t + D / 2);
                const auto k = load_nt<4 * NK>(kp, k_at);
                if constexpr (NK == 1) {
                    kr[t][0] = k;
                } else {
#pragma unroll
                    for (int s = 0; s < NK; ++s) kr[t][s] = k[s];
                }
                const auto vp = rows(1, 15 * (uint32_t)p.c.sv.t + D / 2);
#pragma unroll
                for (int r = 0; r < 4; ++r) vr[t][r] = load_nt<VD / 2>(vp, v_at[r]);
            }
            __builtin_amdgcn_sched_barrier(0);  // all of the step's loads before its first product
#pragma unroll
            for (int t = 0; t < T; ++t) {
                ksr[t] = (uint32_t)__builtin_amdgcn_ds_bpermute(ks_lane + 4 * t, (int)ks_words) >> ks_bit;
                vsr[t] = (uint32_t)__builtin_amdgcn_ds_bpermute(vs_lane + 4 * t, (int)vs_words);
            }
            f32x4 st[T] = {};
            const __bf16* qs = reinterpret_cast<const __bf16*>(lds + p.q_at) +
                               (HB == 16 ? min(col, gn - 1) : min(col, 3 * HB - 1)) * D + g * (D / 4);
            constexpr int QP = HB == 16 ? PARTS : 1;  // products a word
#pragma unroll
            for (int s = 0; s < NK; ++s) {
                bf16x8 q[QP];
                if constexpr (F) {
#pragma unroll
                    for (int i = 0; i < QP; ++i) q[i] = *reinterpret_cast<const bf16x8*>(qs + i * gn * D + 8 * s);
                } else {
                    q[0] = qf[s];
                }
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const bf16x8 k = to_bf16(kr[t][s], block_scale(ksr[t]));
#pragma unroll
                    for (int i = QP - 1; i >= 0; --i) st[t] = mfma16x16x32bf16(k, q[i], st[t]);
                }
            }
            const bool ends = base + KEYS > j1;  // keys behind the end: nothing of what their slots hold counts
            if (ends) {
#pragma unroll
                for (int i = 0; i < 4 * T; ++i)
                    if (base + 16 * (i >> 2) + 4 * g + (i & 3) >= j1) {
                        st[i >> 2][i & 3] = -INFINITY;
                        vr[i >> 2][i & 3] = 0;
                        vsr[i >> 2] = (vsr[i >> 2] & ~(255u << (8 * (i & 3)))) | 127u << (8 * (i & 3));
                    }
            }
            // x: this lane's scores, then their probabilities: its head's, in the order of the products (HB = 16), or
            // NV neighbouring keys of head lane / LPH
            constexpr int NX = HB == 16 ? 4 * T : NV;
            float x[NX];
            if constexpr (HB == 16) {
#pragma unroll
                for (int i = 0; i < NX; ++i) x[i] = st[i >> 2][i & 3];
            } else {
                if (col < PARTS * HB) {
#pragma unroll
                    for (int t = 0; t < T; ++t) *reinterpret_cast<f32x4*>(mine + col * KEYS + 16 * t + 4 * g) = st[t];
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                const float* src = mine + min(lane / LPH, gn - 1) * KEYS + lane % LPH * NV;
#pragma unroll
                for (int i = 0; i < NX; ++i) {
                    x[i] = src[i];
                    if constexpr (F) x[i] += src[HB * KEYS + i] + src[2 * HB * KEYS + i];
                }
            }
            float mx = m;
#pragma unroll
            for (int i = 0; i < NX; ++i) mx = fmaxf(mx, x[i]);
            if constexpr (HB == 16) {
                mx = max_xor32(max_xor16(mx));
            } else {
                if constexpr (LPH >= 2) mx = fmaxf(mx, dpp_mov<0xB1>(mx));
                if constexpr (LPH >= 4) mx = fmaxf(mx, dpp_mov<0x4E>(mx));
                if constexpr (LPH >= 8) mx = fmaxf(mx, dpp_mov<0x141>(mx));
                if constexpr (LPH >= 16) mx = fmaxf(mx, dpp_mov<0x140>(mx));
                if constexpr (LPH >= 32) mx = max_xor16(mx);
                if constexpr (LPH >= 64) mx = max_xor32(mx);
            }
            const float ref = mx == -INFINITY ? 0.f : mx;  // no key above -inf yet: keep everything at 0
            // differences before the scale: the largest one's is 0 at any magnitude, where a product less a rounded product may
            // be anything
            const float alpha = fast_exp2((m - ref) * p.cs);
            const bool moved = __any(mx != m);
            m = mx;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NX; ++i) {
                x[i] = fast_exp2((x[i] - ref) * p.cs);
                l += x[i];
            }
            float scale_acc = alpha;
            __bf16* parts = reinterpret_cast<__bf16*>(mine + PARTS * HB * KEYS);
            if constexpr (HB < 16) {
                __bf16* dst = parts + lane / LPH * KEYS + lane % LPH * NV;
                if constexpr (NV == 1) {
                    float a = x[0];
#pragma unroll
                    for (int k = 0; k < PP; ++k) {
                        const __bf16 h = (__bf16)a;
                        dst[k * HB * KEYS] = h;
                        a -= (float)h;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < NX - 1; i += 2) {  // words of two neighbouring keys
                        float a = x[i], b = x[i + 1];
#pragma unroll
                        for (int k = 0; k < PP; ++k) {
                            const bf16x2 h = {(__bf16)a, (__bf16)b};
                            *reinterpret_cast<bf16x2*>(dst + k * HB * KEYS + i) = h;
                            a -= (float)h[0];
                            b -= (float)h[1];
                        }
                    }
                }
                float* factors = mine + PARTS * HB * KEYS + PP * HB * KEYS / 2;
                if (moved && lane % LPH == 0) factors[lane / LPH] = alpha;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                if (moved) scale_acc = factors[col % HB];
            }
            if (moved) {
#pragma unroll
                for (int j = 0; j < VD; ++j) acc[j] *= scale_acc;
            }
#pragma unroll
            for (int t = 0; t < T; t += 2) {  // 32 keys a product
                bf16x8 ph, pm, pl;
                if constexpr (HB == 16) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        ph[i] = (__bf16)x[4 * t + i];
                        const float rest = x[4 * t + i] - (float)ph[i];
                        pm[i] = (__bf16)rest;
                        if constexpr (F) pl[i] = (__bf16)(rest - (float)pm[i]);
                    }
                } else {
                    // keys 4 g .. of the two tiles; a column past the parts is not used
                    const __bf16* src = parts + min(col, PP * HB - 1) * KEYS + 16 * t + 4 * g;
                    const bf16x4 lo = *reinterpret_cast<const bf16x4*>(src), hi = *reinterpret_cast<const bf16x4*>(src + 16);
                    ph = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                }
                uint32_t vb[8][VD / 2];  // eight keys' pairs of columns
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t w = vr[t + (i >> 2)][i & 3];
                    const uint32_t sw = vsr[t + (i >> 2)];
                    const float vs = (i & 3) == 0 ? block_scale<0>(sw) : (i & 3) == 1 ? block_scale<1>(sw)
                                   : (i & 3) == 2 ? block_scale<2>(sw) : block_scale<3>(sw);
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
                    if constexpr (HB == 16) {
                        if constexpr (F) acc[j] = mfma16x16x32bf16(v, pl, acc[j]);
                        acc[j] = mfma16x16x32bf16(v, pm, acc[j]);
                    }
                    acc[j] = mfma16x16x32bf16(v, ph, acc[j]);
                }
            }
        }

        // Join the waves: lane (col, g) holds head col's o[VD (4 g + r) + j] in acc[j][r].
        if constexpr (HB == 16) {
            l += shfl_xor(l, 16);
            l += shfl_xor(l, 32);
        } else {
            l = group_sum<(LPH < 32 ? LPH : 32)>(l);
            if constexpr (LPH == 64) l += shfl_xor(l, 32);
            // the parts' columns (row_shl: lane i <- i + n), the small ones first
#pragma unroll
            for (int j = 0; j < VD; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float low = dpp_mov<0x100 + HB>(acc[j][r]);
                    if constexpr (F) low += dpp_mov<0x100 + 2 * HB>(acc[j][r]);
                    acc[j][r] += low;
                }
            __syncthreads();  // the waves' scores are read
        }
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
        if (HB == 16 ? g == 0 : lane % LPH == 0) {
            ms[wave * 16 + (HB == 16 ? col : lane / LPH)] = m * p.cs;
            ls[wave * 16 + (HB == 16 ? col : lane / LPH)] = l;
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
    const int len = p.c.lens[row], steps = kv4_steps(len, p.max_len);
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

// Whole rows to the workgroups, with no parts to join, where they are short (a step takes about 1 us, the join and its launch 3;
// graph replays, whole and shared out, us: one row, 12 heads fp32, 500 keys 5.4 and 7.8, 1000 7.4 and 7.7; 32 rows
// 7.5 and 10.6, 11.3 and 13.6), and where there are as many (row, head) pairs for each slot of the device as the
// longest row has steps.
int kv4_groups(int rows, int heads, int G, int max_len, int D, bool most) {
    const int64_t slots = 256 * kv4_per_cu(D), pairs = (int64_t)heads * ((G + 15) / 16);
    const int64_t steps = ((int64_t)max_len + kKv4Step - 1) / kKv4Step;
    if (steps <= 4 || rows * pairs >= slots * steps) return 0;
    const int64_t all = std::min(rows, kPagedBlock) * steps;
    const int64_t groups = std::max<int64_t>(1, std::min({slots / pairs, all, (int64_t)kPagedMaxGroups}));
    if (most) return (int)groups;
    const int64_t share = (all + groups - 1) / groups;  // of the longest rows; no more shares than come out even
    return (int)((all + share - 1) / share);
}

int launch_attn_decode_kv4(const Kv4DecodeParams& p, int bf16, hipStream_t s) {
    const dim3 grid((unsigned)paged_units(p.c.rows, p.c.heads, p.head_tiles, p.groups),
                    p.groups ? (unsigned)paged_blocks(p.c.rows) : 1u);
    const int heads = std::min(p.G, 16);
    return by_type(p.c.D, bf16, [&](auto d, auto e) {
        constexpr int D = decltype(d)::value;
        using E = decltype(e);
        auto go = [&](auto hb) {
            constexpr int HB = decltype(hb)::value;
            constexpr bool F = sizeof(E) == 4;
            Kv4DecodeParams a = p;
            a.q_at = std::max(4 * heads * (D + 4) + 128, 4 * kv4_wave_floats(F, HB));
            const size_t lds = (size_t)(a.q_at + (F ? 3 * (HB == 16 ? heads : HB) * D / 2 : 0)) * sizeof(float);
            hipLaunchKernelGGL((kv4_split_kernel<D, E, HB>), grid, dim3(256), lds, s, a);
        };
        using std::integral_constant;
        if (heads == 1) go(integral_constant<int, 1>{});
        else if (heads == 2) go(integral_constant<int, 2>{});
        else if (heads <= 4) go(integral_constant<int, 4>{});
        else go(integral_constant<int, 16>{});
        if (p.groups)
            hipLaunchKernelGGL((kv4_join_kernel<D, E>), dim3((unsigned)((int64_t)p.c.rows * p.Hq)), dim3(256), 0, s, p);
    });
}

}  // namespace inf
