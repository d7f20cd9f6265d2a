// capi_quant.cpp -- the extern "C" entry points of matrices in 8 bits (include/inferno_hip.h): argument
// validation on the host, workspace sizing, launches.  Nothing here allocates.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "inferno_hip.h"
#include "kernels.h"
#include "overlap.h"

namespace {

constexpr size_t kAlign = 256;
constexpr int64_t kMaxLd = int64_t(1) << 22;   // rows of a tile are addressed with 32-bit offsets
constexpr int64_t kMaxK = (int64_t(1) << 17) - 1;  // 2^7 2^7 K stays inside 32 bits
constexpr int64_t kMaxMN = int64_t(1) << 30;
constexpr int64_t kMaxThreads = (int64_t(1) << 32) - 1;  // of a launch

bool dtype_ok(int dt) { return dt == INF_F32 || dt == INF_BF16; }
int esz(inf_dtype dt) { return dt == INF_F32 ? 4 : 2; }
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
int hip_status(int e) { return e == 0 ? INF_OK : INF_ERR_HIP; }
size_t round_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }
int64_t whole16(int64_t n) { return (n + 15) / 16 * 16; }

// A matrix in 8 bits: rows on 16 bytes.
int check_i8(const void* q, int64_t ld, int64_t cols) {
    if (!q) return INF_ERR_NULL_POINTER;
    if (ld < whole16(cols) || ld > kMaxLd) return INF_ERR_BAD_STRIDE;
    return aligned(q, 16) && ld % 16 == 0 ? INF_OK : INF_ERR_ALIGNMENT;
}

int check_product(int64_t M, int64_t N, int64_t K) {
    if (M < 1 || N < 1 || K < 1 || M > kMaxMN || N > kMaxMN) return INF_ERR_BAD_SHAPE;
    if (K > kMaxK) {
        inf::set_error_detail("product in 8 bits: K of at most " + std::to_string(kMaxK) + ", got " + std::to_string(K));
        return INF_ERR_UNSUPPORTED;
    }
    // tiles, and the join's threads, in one grid
    return ((M + 127) / 128 + 1) * ((N + 127) / 128 + 1) * 8 * 512 > kMaxThreads || M * ((N + 3) / 4) > kMaxThreads - 256
               ? INF_ERR_BAD_SHAPE
               : INF_OK;
}

// What a product needs behind its operands, and a linear layer for its rows in 8 bits.
size_t part_bytes(const inf::GemmI8Plan& plan, int64_t M, int64_t N) {
    return plan.ksplit > 1 ? round_up((size_t)plan.ksplit * M * ((N + 3) / 4 * 4) * 4) : 0;
}
size_t q_bytes(int64_t M, int64_t K) { return round_up((size_t)M * whole16(K)); }
size_t scale_bytes(int64_t M) { return round_up((size_t)M * 4); }
size_t linear_bytes(const inf::GemmI8Plan& plan, int64_t M, int64_t N, int64_t K) {
    return plan.fused ? 0 : q_bytes(M, K) + scale_bytes(M) + part_bytes(plan, M, N);
}

// Bytes of up to M rows: fewer rows may have more K ranges, and so need more.
template <typename F>
size_t most_bytes(int64_t M, int64_t N, int64_t K, bool quantised, F bytes) {
    size_t n = bytes(inf::gemm_i8_plan(M, N, K, quantised), M);
    const int64_t split = inf::gemm_i8_split_rows(N);
    for (int64_t m = 64; m < M && m <= split; m += 64)
        n = std::max(n, bytes(inf::gemm_i8_plan(m, N, K, quantised), m));
    return n;
}

// A matrix of elements of this type.
inf::Memory elements(const void* x, int64_t ld, int64_t rows, int64_t cols, inf_dtype dt) {
    return {x, rows, inf::Memory::bytes(ld, esz(dt)), cols * esz(dt)};
}

// The arguments that both forms of the product share.
int check_rest(const int8_t* w, int64_t ldw, const float* sw, const void* bias, const void* y, int64_t ldy, int64_t M,
               int64_t N, int64_t K, inf_dtype dt, const void* workspace, size_t ws_bytes, size_t need) {
    if (!sw || !y) return INF_ERR_NULL_POINTER;
    if (ldy < N) return INF_ERR_BAD_STRIDE;
    const size_t es = (size_t)esz(dt);
    if (!aligned(sw, 4) || !aligned(y, es) || !aligned(bias, es)) return INF_ERR_ALIGNMENT;
    // other workgroups read these while one writes its results
    const inf::Memory my = elements(y, ldy, M, N, dt), mw(workspace, (int64_t)need);
    auto read = [&](const inf::Memory& m) {
        return m.over({w, N, ldw, K}) || m.over({sw, 4 * N}) || m.over({bias, (int64_t)es * N});
    };
    if (read(my) || my.over(mw)) return INF_ERR_BAD_STRIDE;
    if (need && (!workspace || ws_bytes < need)) return INF_ERR_WORKSPACE;
    if (need && !aligned(workspace, kAlign)) return INF_ERR_ALIGNMENT;
    return read(mw) ? INF_ERR_BAD_STRIDE : INF_OK;
}

// Rows of elements that can be read four at a time.
bool by_four(const void* x, int64_t ldx, inf_dtype dt) { return ldx % 4 == 0 && aligned(x, 4 * (size_t)esz(dt)); }

// Rows that can be read 16 bytes at a time.
bool on_16(const void* x, int64_t ldx, inf_dtype dt) { return ldx * esz(dt) % 16 == 0 && aligned(x, 16); }

// What both forms of the product have in common.
inf::GemmI8Params product(const int8_t* w, int64_t ldw, const float* sw, const void* bias, void* y, int64_t ldy,
                          int64_t M, int64_t N, int64_t K, inf_dtype dt) {
    inf::GemmI8Params p{};
    p.w = w;
    p.sw = sw;
    p.bias = bias;
    p.y = y;
    p.ldw = ldw; p.ldy = ldy;
    p.M = (int)M; p.N = (int)N; p.K = (int)K;
    p.wide = by_four(y, ldy, dt) && aligned(bias, 4 * (size_t)esz(dt)) && aligned(sw, 16);
    p.ldp = (int)((N + 3) / 4 * 4);
    return p;
}

int quantize(const void* x, int64_t ldx, int64_t rows, int64_t cols, int transpose, int8_t* q, int64_t ldq,
             float* scale, inf_dtype dt, hipStream_t stream) {
    inf::QuantizeParams p{};
    p.x = x;
    p.q = q;
    p.scale = scale;
    p.rows = rows; p.cols = cols;
    p.ldx = ldx; p.ldq = ldq;
    p.wide = on_16(x, ldx, dt);
    return hip_status(inf::launch_quantize(p, transpose, dt == INF_BF16, stream));
}

int check_x(const void* x, int64_t ldx, int64_t cols, inf_dtype dt) {
    if (!x) return INF_ERR_NULL_POINTER;
    if (ldx < cols) return INF_ERR_BAD_STRIDE;
    return aligned(x, (size_t)esz(dt)) ? INF_OK : INF_ERR_ALIGNMENT;
}

}  // namespace

extern "C" {

int inf_quantize_i8(const void* x, int64_t ldx, int64_t rows, int64_t cols, int transpose, int8_t* q, int64_t ldq,
                    float* scale, inf_dtype dt, void* stream) {
    if (!dtype_ok(dt)) return INF_ERR_BAD_DTYPE;
    if (rows < 0 || cols < 1 || rows > kMaxMN || cols > kMaxMN) return INF_ERR_BAD_SHAPE;
    if (transpose && rows < 1) return INF_ERR_BAD_SHAPE;
    if (rows == 0) return INF_OK;
    if (inf::quantize_threads(rows, cols, transpose, esz(dt)) > kMaxThreads) return INF_ERR_BAD_SHAPE;
    int st = check_x(x, ldx, cols, dt);
    if (st != INF_OK) return st;
    if (!scale) return INF_ERR_NULL_POINTER;
    if (!aligned(scale, 4)) return INF_ERR_ALIGNMENT;
    if ((st = check_i8(q, ldq, transpose ? rows : cols))) return st;
    // other workgroups still read x
    const int64_t n = transpose ? cols : rows, k = whole16(transpose ? rows : cols);
    const inf::Memory mx = elements(x, ldx, rows, cols, dt), mq(q, n, ldq, k), ms(scale, 4 * n);
    if (mx.over(mq) || mx.over(ms) || mq.over(ms)) return INF_ERR_BAD_STRIDE;
    return quantize(x, ldx, rows, cols, transpose, q, ldq, scale, dt, (hipStream_t)stream);
}

int inf_gemm_i8_workspace(int64_t M, int64_t N, int64_t K, size_t* out_bytes) {
    if (!out_bytes) return INF_ERR_NULL_POINTER;
    *out_bytes = 0;
    const int st = check_product(M, N, K);
    if (st == INF_OK)
        *out_bytes = most_bytes(M, N, K, true, [&](const auto& plan, int64_t m) { return part_bytes(plan, m, N); });
    return st;
}

int inf_gemm_i8(int64_t M, int64_t N, int64_t K, const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w,
                int64_t ldw, const float* w_scale, const void* bias, void* y, int64_t ldy, inf_dtype dt,
                void* workspace, size_t ws_bytes, void* stream) {
    if (!dtype_ok(dt)) return INF_ERR_BAD_DTYPE;
    int st = check_product(M, N, K);
    if (st != INF_OK || (st = check_i8(x, ldx, K)) || (st = check_i8(w, ldw, K))) return st;
    if (!x_scale) return INF_ERR_NULL_POINTER;
    if (!aligned(x_scale, 4)) return INF_ERR_ALIGNMENT;
    const inf::GemmI8Plan plan = inf::gemm_i8_plan(M, N, K, true);
    if ((st = check_rest(w, ldw, w_scale, bias, y, ldy, M, N, K, dt, workspace, ws_bytes, part_bytes(plan, M, N))))
        return st;
    const inf::Memory mx(x, M, ldx, K), ms(x_scale, 4 * M);
    for (const inf::Memory& m : {elements(y, ldy, M, N, dt), inf::Memory(workspace, (int64_t)part_bytes(plan, M, N))})
        if (m.over(mx) || m.over(ms)) return INF_ERR_BAD_STRIDE;
    inf::GemmI8Params p = product(w, ldw, w_scale, bias, y, ldy, M, N, K, dt);
    p.x = x;
    p.ldx = ldx;
    p.sx = x_scale;
    p.part = static_cast<int32_t*>(workspace);
    return hip_status(inf::launch_gemm_i8(p, plan, dt == INF_BF16, (hipStream_t)stream));
}

int inf_linear_i8_workspace(int64_t M, int64_t N, int64_t K, size_t* out_bytes) {
    if (!out_bytes) return INF_ERR_NULL_POINTER;
    *out_bytes = 0;
    const int st = check_product(M, N, K);
    if (st == INF_OK)
        *out_bytes = most_bytes(M, N, K, false, [&](const auto& plan, int64_t m) { return linear_bytes(plan, m, N, K); });
    return st;
}

int inf_linear_i8(int64_t M, int64_t N, int64_t K, const void* x, int64_t ldx, const int8_t* w, int64_t ldw,
                  const float* w_scale, const void* bias, void* y, int64_t ldy, inf_dtype dt, void* workspace,
                  size_t ws_bytes, void* stream) {
    if (!dtype_ok(dt)) return INF_ERR_BAD_DTYPE;
    int st = check_product(M, N, K);
    if (st != INF_OK || (st = check_x(x, ldx, K, dt)) || (st = check_i8(w, ldw, K))) return st;
    if (inf::quantize_threads(M, K, 0, esz(dt)) > kMaxThreads) return INF_ERR_BAD_SHAPE;
    const inf::GemmI8Plan plan = inf::gemm_i8_plan(M, N, K, false);
    if ((st = check_rest(w, ldw, w_scale, bias, y, ldy, M, N, K, dt, workspace, ws_bytes, linear_bytes(plan, M, N, K))))
        return st;
    const inf::Memory mx = elements(x, ldx, M, K, dt);
    if (mx.over(elements(y, ldy, M, N, dt)) || mx.over({workspace, (int64_t)linear_bytes(plan, M, N, K)}))
        return INF_ERR_BAD_STRIDE;
    inf::GemmI8Params p = product(w, ldw, w_scale, bias, y, ldy, M, N, K, dt);
    if (plan.fused) {
        p.xf = x;
        p.ldxf = ldx;
        p.wide_x = on_16(x, ldx, dt);
    } else {
        char* ws = static_cast<char*>(workspace);
        int8_t* q = reinterpret_cast<int8_t*>(ws);
        float* scale = reinterpret_cast<float*>(ws + q_bytes(M, K));
        p.x = q;
        p.ldx = whole16(K);
        p.sx = scale;
        p.part = reinterpret_cast<int32_t*>(ws + q_bytes(M, K) + scale_bytes(M));
        if ((st = quantize(x, ldx, M, K, 0, q, p.ldx, scale, dt, (hipStream_t)stream))) return st;
    }
    return hip_status(inf::launch_gemm_i8(p, plan, dt == INF_BF16, (hipStream_t)stream));
}

}  // extern "C"
