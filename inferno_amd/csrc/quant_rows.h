// quant_rows.h -- rows in 8 bits, shared by the kernels that quantise them.
//
// A row's scale is its largest magnitude times 1/127, its values whole multiples of it, q = rint(x / scale).
// The quotient is rounded as if it were exact, ties to even: x times the scale's reciprocal may
// come out on the wrong side of the middle between two whole numbers, so the remainder x - q scale, which one
// fused multiply-add gives exactly (it is a multiple of the last places of x and scale, and
// below scale), is compared with half the scale.  The same x then has the same q on any machine.
//
// A row with an infinity or a NaN has scale NaN and zeros; one whose scale would be subnormal has scale 0 and
// zeros.  Magnitudes are compared as whole numbers, where NaN is above infinity and both above the others.
#pragma once

#include "common.h"

namespace inf {

constexpr float kInv127 = 1.0f / 127.0f;

// The scale of a row whose largest magnitude has these bits, and its reciprocal (0 where all are zeros).
struct RowScale {
    float scale, inv;
    __device__ __forceinline__ explicit RowScale(uint32_t top) {
        const float s = __uint_as_float(top) * kInv127;
        const bool bad = top >= 0x7f800000u, tiny = s < 1.17549435e-38f;
        scale = bad ? __builtin_nanf("") : tiny ? 0.f : s;
        inv = bad || tiny ? 0.f : 1.f / s;
    }
};

// rint(x / scale) for N values.
template <int N>
__device__ __forceinline__ void round_all(const float (&x)[N], const RowScale& s, int (&q)[N]) {
    const float half = 0.5f * s.scale;
    float r[N], e[N], worst = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        r[i] = s.inv == 0.f ? 0.f : rintf(x[i] * s.inv);
        e[i] = s.inv == 0.f ? 0.f : fmaf(-r[i], s.scale, x[i]);
        worst = fmaxf(worst, fabsf(e[i]));
    }
    if (__any(worst >= half)) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool odd = (int)r[i] & 1;
            if (e[i] > half || (e[i] == half && odd)) r[i] += 1.f;
            if (e[i] < -half || (e[i] == -half && odd)) r[i] -= 1.f;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = (int)fminf(fmaxf(r[i], -127.f), 127.f);
}

template <int N>
__device__ __forceinline__ uint32_t pack4(const int (&q)[N], int at) {
    return (uint32_t)(q[at] & 255) | (uint32_t)(q[at + 1] & 255) << 8 | (uint32_t)(q[at + 2] & 255) << 16 |
           (uint32_t)(q[at + 3] & 255) << 24;
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The columns that a thread takes at a time: 16 bytes.
template <typename E>
constexpr int kChunk = 16 / (int)sizeof(typename E::T);

// Chunk of columns from c on, zeros behind the last.  VEC: rows on 16 bytes; NT: past the caches.
template <typename E, bool VEC, bool NT>
__device__ __forceinline__ void load_chunk(const typename E::T* row, int c, int cols, float (&x)[kChunk<E>]) {
    constexpr int N = kChunk<E>;
    if (VEC && c + N <= cols) {
        const u32x4* src = reinterpret_cast<const u32x4*>(row + c);
        const u32x4 v = NT ? __builtin_nontemporal_load(src) : *src;
#pragma unroll
        for (int i = 0; i < N; ++i)
            x[i] = __uint_as_float(N == 4 ? v[i & 3] : i & 1 ? v[(i >> 1) & 3] & 0xffff0000u : v[(i >> 1) & 3] << 16);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = c + i < cols ? E::ld(row + c + i) : 0.f;
    }
}

// The chunk's whole numbers, a byte each.
template <int N>
__device__ __forceinline__ void store_chunk(void* q, const int (&r)[N]) {
    if constexpr (N == 8)
        *reinterpret_cast<uint2*>(q) = make_uint2(pack4(r, 0), pack4(r, 4));
    else
        *reinterpret_cast<uint32_t*>(q) = pack4(r, 0);
}

}  // namespace inf
