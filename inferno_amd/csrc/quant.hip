// quant.hip -- rows (or columns) of a matrix in 8 bits (quant_rows.h): for each its scale, and its values as whole
// multiples of it.
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "quant_rows.h"

namespace inf {

// W waves a row, 16 bytes of it a thread at a time, U times that held between the two passes over the row; a longer
// row (32 KB on) is read twice.  q's rows are written up to whole 16 bytes, with zeros.
// Bound by memory: 16384 x 8192 bf16 in 66 us, 6.0 TB/s of rows read and values written (89 in 8-byte pieces through the
// caches; 75 with a quarter of a row held and the rest read again); 8192 x 768 fp32 7.3; few rows are a launch and two
// waits, 32 x 4096 bf16 3.7.
template <typename E, int W, int U, bool VEC>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeParams p) {
    constexpr int T = 64 * W, C = kChunk<E>;
    __shared__ uint32_t tops[4];
    const int tid = threadIdx.x % T, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * (4 / W) + threadIdx.x / T;
    const bool there = row < p.rows;
    const typename E::T* x = (const typename E::T*)p.x + (there ? row : 0) * p.ldx;
    const int cols = (int)p.cols;
    float v[U][C];
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) load_chunk<E, VEC, true>(x, C * (tid + T * u), cols, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < C; ++i) top = max(top, magnitude(v[u][i]));
    for (int c = C * (tid + T * U); c < cols; c += C * T) {
        float y[C];
        load_chunk<E, VEC, false>(x, c, cols, y);
#pragma unroll
        for (int i = 0; i < C; ++i) top = max(top, magnitude(y[i]));
    }
    top = wave_all(top, [](uint32_t a, uint32_t b) { return max(a, b); });
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) tops[wave] = top;
        __syncthreads();
        top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    }
    if (!there) return;
    const RowScale s(top);
    int8_t* q = p.q + row * p.ldq;
    const int end = (cols + 15) & ~15;
    auto write = [&](int c, const float (&y)[C]) {
        int r[C];
        round_all(y, s, r);
        if (c < end) store_chunk(q + c, r);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) write(C * (tid + T * u), v[u]);
    for (int c = C * (tid + T * U); c < end; c += C * T) {
        float y[C];
        load_chunk<E, VEC, false>(x, c, cols, y);
        write(c, y);
    }
    if (tid == 0) p.scale[row] = s.scale;
}

// Columns of x as rows of q (weights [in, out], one scale for each output): a workgroup takes 32 columns, reads
// them for their largest magnitudes and again, 16 rows a thread, for their values, which it so writes
// transposed without passing through LDS.  8192 x 8192 fp32 111 us: once for a model's weights, not taken further.
template <typename E>
__global__ __launch_bounds__(1024) void quantize_columns_kernel(QuantizeParams p) {
    __shared__ uint32_t tops[32][33];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + c;
    const bool there = col < p.cols;
    const typename E::T* x = (const typename E::T*)p.x + (there ? col : 0);
    uint32_t top = 0;
#pragma unroll 8
    for (int64_t r = g; r < p.rows; r += 32) top = max(top, magnitude(E::ld(x + r * p.ldx)));
    tops[g][c] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 32; ++i) top = max(top, tops[i][c]);
    const RowScale s(top);
    const int64_t end = (p.rows + 15) & ~(int64_t)15;
    for (int64_t r0 = 16 * g; r0 < end; r0 += 512) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = r0 + i < p.rows ? E::ld(x + (r0 + i) * p.ldx) : 0.f;
        int q[16];
        round_all(v, s, q);
        if (there)
            *reinterpret_cast<uint4*>(p.q + col * p.ldq + r0) =
                make_uint4(pack4(q, 0), pack4(q, 4), pack4(q, 8), pack4(q, 12));
    }
    if (there && g == 0) p.scale[col] = s.scale;
}

template <typename E, bool VEC>
static void launch_rows(const QuantizeParams& p, hipStream_t s) {
    auto go = [&](auto w, auto u) {
        constexpr int W = decltype(w)::value, U = decltype(u)::value;
        hipLaunchKernelGGL((quantize_rows_kernel<E, W, U, VEC>), dim3((unsigned)((p.rows + 4 / W - 1) / (4 / W))),
                           dim3(256), 0, s, p);
    };
    using std::integral_constant;
    using C1 = integral_constant<int, 1>;
    using C2 = integral_constant<int, 2>;
    using C4 = integral_constant<int, 4>;
    using C8 = integral_constant<int, 8>;
    const int64_t chunks = (p.cols + kChunk<E> - 1) / kChunk<E>;
    if (quantize_by_wave(p.rows, p.cols, (int)sizeof(typename E::T))) {
        if (chunks <= 64) go(C1{}, C1{});
        else if (chunks <= 128) go(C1{}, C2{});
        else go(C1{}, C4{});
    } else if (chunks <= 256) {
        go(C4{}, C1{});
    } else if (chunks <= 512) {
        go(C4{}, C2{});
    } else if (chunks <= 1024) {
        go(C4{}, C4{});
    } else {
        go(C4{}, C8{});
    }
}

int launch_quantize(const QuantizeParams& p, int transpose, int bf16, hipStream_t s) {
    if (transpose) {
        const dim3 grid((unsigned)((p.cols + 31) / 32));
        if (bf16)
            hipLaunchKernelGGL((quantize_columns_kernel<BF16>), grid, dim3(1024), 0, s, p);
        else
            hipLaunchKernelGGL((quantize_columns_kernel<F32>), grid, dim3(1024), 0, s, p);
    } else if (bf16) {
        p.wide ? launch_rows<BF16, true>(p, s) : launch_rows<BF16, false>(p, s);
    } else {
        p.wide ? launch_rows<F32, true>(p, s) : launch_rows<F32, false>(p, s);
    }
    return (int)hipGetLastError();
}

}  // namespace inf
