// paged.hip -- a key-value cache in pages: writing new tokens to it, attention of one new
// token per row over it, eviction from it, and its reordering under beam search.
//
// Key j of a row lies in slot j % P of page table[row][j / P] (P a power of two), the same
// page for every key-value head and for keys and values.  Page numbers come from device
// memory, so each is checked against the pool's size before it is used: one out of range
// is never followed (a store is dropped; attention makes the row NaN).
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "paged_shares.h"

namespace inf {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

namespace {

__device__ __forceinline__ f32x4 mfma16x16x32bf16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16x16x4(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ u32x4 ld16_nt(const char* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}

// The page that holds position j of a row, -1 where the table names none of the pool's.
__device__ __forceinline__ int page_of(const PagedView& c, const int32_t* table, int j) {
    const int p = table[j >> c.page_shift];
    return (unsigned)p < (unsigned)c.n_pages ? p : -1;
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
// Append.  One thread per 16-byte piece (8-byte where bf16 rows are aligned to that only)
// of a token's key and of its value, pieces of a row fastest, then heads, then tokens: the
// source, a projection's output, is read in the order that it has, and each row of D
// elements is one contiguous run on both sides.  A copy, bound by HBM: 32 prompts of up to 1024
// tokens, 12 heads of D 64, fp32, 200 MB in 33 us, 6.2 TB/s (stores through the caches: 42), 8 of
// them 50 MB in 10 to 12 us, 4.3 to 4.9 TB/s; one token in each of 64 rows is a launch, 3.2 us.
// ============================================================================
template <int BYTES>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendParams p, int pieces, int esz) {
    using V = typename std::conditional<BYTES == 16, u32x4, u32x2>::type;
    const int row = blockIdx.y;
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int th = i / pieces, c = i - th * pieces;
    const int t = th / p.c.heads, h = th - t * p.c.heads;
    const int count = p.counts ? min(p.counts[row], p.Tn) : p.Tn;
    if (t >= count) return;
    const int len = p.c.lens[row];
    const int64_t slot = (int64_t)len - count + t;
    if (slot < 0 || slot >= p.c.cap()) return;
    const int page = page_of(p.c, p.c.table + row * p.c.table_stride, (int)slot);
    if (page < 0) return;
    const int in_page = (int)slot & ((1 << p.c.page_shift) - 1);
    const char* ks = (const char*)p.k + (row * p.sk.b + h * p.sk.h + t * p.sk.t) * esz + c * BYTES;
    const char* vs = (const char*)p.v + (row * p.sv.b + h * p.sv.h + t * p.sv.t) * esz + c * BYTES;
    char* kd = (char*)p.c.k + (page * p.c.sk.b + h * p.c.sk.h + in_page * p.c.sk.t) * esz + c * BYTES;
    char* vd = (char*)p.c.v + (page * p.c.sv.b + h * p.c.sv.h + in_page * p.c.sv.t) * esz + c * BYTES;
    const V kx = *reinterpret_cast<const V*>(ks);
    const V vx = *reinterpret_cast<const V*>(vs);
    __builtin_nontemporal_store(kx, reinterpret_cast<V*>(kd));
    __builtin_nontemporal_store(vx, reinterpret_cast<V*>(vd));
    if (c == 0) {
        const int64_t m = ((int64_t)row * p.c.heads + h) * p.c.cap() + slot;
        if (p.weights) p.weights[m] = 0.f;
        if (p.positions) p.positions[m] = p.seen ? p.seen[row] - count + t : (int)slot;
    }
}

int launch_kv_append(const KvAppendParams& p, int bf16, hipStream_t s) {
    const int esz = bf16 ? 2 : 4, bytes = p.wide ? 16 : 8;
    const int pieces = p.c.D * esz / bytes;
    const int64_t n = (int64_t)p.Tn * p.c.heads * pieces;
    const dim3 grid((unsigned)((n + 255) / 256), (unsigned)p.c.rows);
    if (p.wide)
        hipLaunchKernelGGL((kv_append_kernel<16>), grid, dim3(256), 0, s, p, pieces, esz);
    else
        hipLaunchKernelGGL((kv_append_kernel<8>), grid, dim3(256), 0, s, p, pieces, esz);
    return (int)hipGetLastError();
}

// ============================================================================
// Attention of one query per row: s_j = q k_j scale, p = softmax(s), o = sum_j p_j v_j, for
// the G query heads of a key-value head at once.
//
// The work is cut in steps of 64 to 512 keys of a row, 64 KB.  All steps of up to 64 rows, one after the other, are
// shared out evenly to `groups` of workgroups, one workgroup per key-value head in each, as many as the
// device holds at once: rows of any lengths keep it busy to the end.  (Chunks of a fixed size left a last
// round of workgroups that was partly empty: 64 rows of 1 to 8191 positions, bf16, 8 heads of D 128 with 4
// query heads each, took 203 us, 173 now: 957 MB at 5.5 TB/s.)
// The heads of a group read the same pages at the same time, which lie next to each other: with the heads'
// workgroups apart that case took 319 us instead of 225.  Where a share ends in the middle of a row, the
// row's parts are joined by a second launch.
//
// Each of a workgroup's four waves takes 16 KB of a step, T tiles of 16 keys, all of whose loads are under way
// before its first product: 192 KB a CU, which is what keeps HBM busy.  (The next step's loads ahead of this
// one's products as well: 2 waves a SIMD instead of 3, 12% slower.)  The products run on the matrix cores with up
// to 16 query heads as the columns: S^T = K Q^T (keys x heads), then O^T += V^T P^T (D x heads).  A head's
// scores, maximum, sum and output then lie in one lane column, so that the softmax needs two exchanges per step,
// and each lane's probabilities are the second product's operand as they are: its sum over keys may run in any
// order, so the value rows are loaded in the order that the first product's result has.  A lane holds D / 16
// neighbouring columns of four value rows a tile; one column of them is (half of) one operand (bf16: eight 16-bit
// halves of two tiles picked together; fp32: a register each).  Neither operand passes through LDS, and a row of K
// or V is read from HBM once for all heads, past the caches (16% of the fp32 case's time).  bf16 probabilities are
// taken in two parts (16 bits), whose products cost no time here.
//
// Keys behind the end are read as the last one and their scores are -inf, their values zero, so whatever
// their slots hold does not count.
//
// Bound by HBM where rows are long: 64 rows of 8191, 8 heads of D 128, 4 query heads each, bf16, 339 us, 6.3 TB/s,
// the rate of a plain streaming read; 32 rows of 2048, 12 heads of D 64, fp32, 64 us, 6.3 TB/s.  One row of 1000 takes
// 6 us and its join 3.6: two launches, and a chain of five reads that depend on each other.
// ============================================================================
namespace {

constexpr int kPagedPerCu = 3;           // workgroups of a CU: what the registers allow
constexpr int kPagedHold = 12 << 10;     // bytes of LDS in which a wave holds scores: 144 KB a CU

template <int D, typename E>
__device__ __forceinline__ int paged_steps(int len, int max_len) {
    constexpr int step = paged_step(D, sizeof(E) == 2);
    return len > max_len ? 0 : (max(len, 0) + step - 1) / step;
}

}  // namespace

// SMALL: pages of fewer than 16 keys.  WEIGH: scores are written for the weights (in all variants: 8% slower where
// the registers are few, D 128 in fp32).
template <int D, typename E, bool SMALL, bool WEIGH>
__global__ __launch_bounds__(256, kPagedPerCu) void paged_split_kernel(PagedDecodeParams p) {
    constexpr int ES = sizeof(E);
    constexpr int STEP = paged_step(D, ES == 2);
    constexpr int T = STEP / 64;          // tiles of 16 keys per wave
    constexpr int NK = D * ES / 64;       // 16-byte pieces of a key row per lane
    constexpr int VD = D / 16;            // columns of a value row per lane
    constexpr int VW = VD * ES / 4;       // ... in 32-bit words
    constexpr int LD = D + 4;
    // o [4][heads][LD], then m, l [4][16]; before that, the scores held
    extern __shared__ __attribute__((aligned(16))) float lds[];

    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 15, g = lane >> 4;
    // the tiles of more than 16 query heads read the same keys: neighbours on one XCD
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
    int step = 0, r = 0, begin = 0, steps = paged_steps<D, E>(mylen, p.max_len), starts = steps;
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
    const E* K = (const E*)p.c.k + h * p.c.sk.h;
    const E* V = (const E*)p.c.v + h * p.c.sv.h;
    u32x4 kr[T][NK];
    uint32_t vr[T][4][VW];

    for (;;) {  // the rows of the share
        const int row = row0 + r, s0 = step - begin, s1 = min(stop, end) - begin;
        const int32_t* table = p.c.table + row * p.c.table_stride;
        const int base0 = s0 * STEP + 16 * T * wave;
        // Pages of 16 keys or more: one page for each tile of 16 keys, the same for all lanes, read a step
        // ahead (behind the end, where the table may hold anything, they are not used).
        const int len = __builtin_amdgcn_readlane(mylen, r);
        int next[T] = {};
        auto read_pages = [&](int base) {
#pragma unroll
            for (int t = 0; t < T; ++t)
                next[t] = table[min(__builtin_amdgcn_readfirstlane(base + 16 * t) >> p.c.page_shift, last_page)];
        };
        if constexpr (!SMALL) read_pages(base0);
        const int j1 = min(len, s1 * STEP);

        // Q^T: column = head, rows 16 bytes of d as the key rows are read
        u32x4 qf[NK];
        {
            const E* q = (const E*)p.q + row * p.sq.b + (int64_t)(h * p.G + g0 + min(col, gn - 1)) * p.sq.h;
#pragma unroll
            for (int s = 0; s < NK; ++s) {
                const u32x2* src = reinterpret_cast<const u32x2*>((const char*)q + 64 * s + 16 * g);
                const u32x2 a = src[0], b = src[1];
                qf[s] = col < gn ? u32x4{a[0], a[1], b[0], b[1]} : u32x4{0, 0, 0, 0};
            }
        }

        f32x4 acc[VD];
#pragma unroll
        for (int j = 0; j < VD; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        bool bad = false;
        // Scores are held in LDS and written many steps at a time: a few writes among the reads take HBM from the
        // 6.3 TB/s of reads alone to the 4.9 of a copy (two rows of 131071, 2 heads of D 128, 8 query heads each,
        // bf16: 67.4 us with a write per step, 63.4 so; the rows of 1 to 8191 above 232 and 213).
        float* sc = WEIGH ? p.scores + ((int64_t)row * p.Hq + h * p.G + g0) * p.score_ld : nullptr;
        float* hold = lds + wave * (kPagedHold / 4);
        const int most = kPagedHold / (64 * T * gn);
        int held = 0;
        auto flush = [&](int base) {  // the steps before `base`; the wave's other lanes wrote some of them
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (int i = lane; i < held * gn * 4 * T; i += 64) {
                const int key = 4 * (i % (4 * T)), sh = i / (4 * T), s = sh / gn, head = sh - s * gn;
                *reinterpret_cast<f32x4*>(sc + head * p.score_ld + base - (held - s) * STEP + key) =
                    *reinterpret_cast<const f32x4*>(hold + 4 * i);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            held = 0;
        };
        int base = base0;
        for (; base < j1; base += STEP) {
            // rows behind the end are read as the last key's
            int page[T] = {};
            if constexpr (!SMALL) {
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const bool in = (unsigned)next[t] < (unsigned)p.c.n_pages;
                    bad |= !in && base + 16 * t < j1;
                    page[t] = in ? next[t] : 0;
                }
                if (base + STEP < j1) read_pages(base + STEP);
            }
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const int key = min(base + 16 * t + col, j1 - 1);
                int pg = page[t];
                if constexpr (SMALL) {
                    pg = page_of(p.c, table, key);
                    bad |= pg < 0;
                    pg = max(pg, 0);
                }
                const char* src = (const char*)(K + pg * p.c.sk.b + (key & mask) * p.c.sk.t) + 16 * g;
#pragma unroll
                for (int s = 0; s < NK; ++s)
                    kr[t][s] = ld16_nt(src + 64 * s);
            }
#pragma unroll
            for (int t = 0; t < T; ++t) {
                // pages of four keys or more: one page for the lane's four
                int pg = page[t];
                if constexpr (SMALL) pg = max(page_of(p.c, table, min(base + 16 * t + 4 * g, j1 - 1)), 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = min(base + 16 * t + 4 * g + r, j1 - 1);
                    if constexpr (SMALL)
                        if (r && p.c.page_shift < 2) pg = max(page_of(p.c, table, key), 0);
                    const char* src = (const char*)(V + pg * p.c.sv.b + (key & mask) * p.c.sv.t + VD * col);
                    if constexpr (VW == 1) {
                        vr[t][r][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(src));
                    } else if constexpr (VW == 2) {
                        const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(src));
                        vr[t][r][0] = x[0];
                        vr[t][r][1] = x[1];
                    } else {
#pragma unroll
                        for (int w = 0; w < VW; w += 4) {
                            const u32x4 x = ld16_nt(src + 4 * w);
#pragma unroll
                            for (int e = 0; e < 4; ++e) vr[t][r][w + e] = x[e];
                        }
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // all of the step's loads before its first product
            f32x4 st[T] = {};
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int s = 0; s < NK; ++s) {
                    if constexpr (ES == 2) {
                        st[t] = mfma16x16x32bf16(__builtin_bit_cast(bf16x8, kr[t][s]),
                                                 __builtin_bit_cast(bf16x8, qf[s]), st[t]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            st[t] = mfma16x16x4(__uint_as_float(kr[t][s][e]), __uint_as_float(qf[s][e]), st[t]);
                    }
                }
            float x[4 * T];
#pragma unroll
            for (int i = 0; i < 4 * T; ++i) x[i] = st[i >> 2][i & 3] * p.cs;
            if (base + 16 * T > j1) {
#pragma unroll
                for (int i = 0; i < 4 * T; ++i)
                    if (base + 16 * (i >> 2) + 4 * g + (i & 3) >= j1) {
                        x[i] = -INFINITY;
#pragma unroll
                        for (int w = 0; w < VW; ++w) vr[i >> 2][i & 3][w] = 0;
                    }
            }
            if constexpr (WEIGH) {
                if (held == most) flush(base);
                if (col < gn) {
#pragma unroll
                    for (int t = 0; t < T; ++t)
                        *reinterpret_cast<f32x4*>(hold + (held * gn + col) * 16 * T + 16 * t + 4 * g) =
                            f32x4{x[4 * t], x[4 * t + 1], x[4 * t + 2], x[4 * t + 3]};
                }
                ++held;
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
            if constexpr (ES == 2) {
#pragma unroll
                for (int t = 0; t < T; t += 2) {  // 32 keys a product
                    bf16x8 ph, pm;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        ph[i] = (__bf16)x[4 * t + i];
                        pm[i] = (__bf16)(x[4 * t + i] - (float)ph[i]);
                    }
#pragma unroll
                    for (int j = 0; j < VD; ++j) {
                        const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;  // high or low halves of two words
                        u32x4 a;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            a[i] = __builtin_amdgcn_perm(vr[t + (i >> 1)][2 * (i & 1) + 1][j >> 1],
                                                         vr[t + (i >> 1)][2 * (i & 1)][j >> 1], sel);
                        acc[j] = mfma16x16x32bf16(__builtin_bit_cast(bf16x8, a), ph, acc[j]);
                        acc[j] = mfma16x16x32bf16(__builtin_bit_cast(bf16x8, a), pm, acc[j]);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4 * T; ++i)
#pragma unroll
                    for (int j = 0; j < VD; ++j)
                        acc[j] = mfma16x16x4(__uint_as_float(vr[i >> 2][i & 3][j]), x[i], acc[j]);
            }
        }

        if constexpr (WEIGH) {
            flush(base);
            __syncthreads();
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

template <int D, typename E>
__device__ __forceinline__ RowParts row_parts(const PagedDecodeParams& p, int row, int len) {
    const int steps = paged_steps<D, E>(len, p.max_len);
    if (!steps) return {0, 0};
    const int block = row / kPagedBlock, start = p.first[row], all = p.first[p.c.rows + block];
    const Shares shares(all, p.groups);
    const int g0 = shares.of(start), g1 = shares.of(start + steps - 1);
    return {g1 - g0 + 1, (int64_t)row + block * p.groups + g0};
}

// Joins the parts: the first rows * Hq workgroups write o, the others (where weights are asked
// for) take 1024 positions of a (row, key-value head) each and add the heads' probabilities
// exp2(score - max) / sum to the weights, in the order of the heads.
template <int D, typename E>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedDecodeParams p, int wblocks, int wide) {
    __shared__ float wsh[kPagedMaxGroups];
    __shared__ f32x4 osh[256];
    __shared__ f32x2 heads[4][8], scale[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nout = p.c.rows * p.Hq;
    if ((int)blockIdx.x < nout) {
        const int row = blockIdx.x / p.Hq, hq = blockIdx.x % p.Hq;
        const int len = p.c.lens[row];
        E* out = (E*)p.o + row * p.so.b + hq * p.so.h;
        const RowParts parts = row_parts<D, E>(p, row, len);
        if (!parts.n) {
            if (tid < D) store1(out + tid, len > p.max_len ? __builtin_nanf("") : 0.f);
            return;
        }
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
        return;
    }
    const int b = blockIdx.x - nout;
    const int rh = b / wblocks, j0 = (b % wblocks) * 1024;
    const int row = rh / p.c.heads, h = rh % p.c.heads;
    const int len = p.c.lens[row];
    const int n = min(len, p.max_len);
    if (j0 >= n) return;
    const RowParts parts = row_parts<D, E>(p, row, len);
    const int64_t hq0 = (int64_t)row * p.Hq + h * p.G;
    const int j = j0 + 4 * tid;  // this thread's 4 positions; scores are padded to whole steps
    const int64_t wat = (int64_t)rh * p.c.cap() + j;
    const bool whole = j + 4 <= n && p.c.cap() % 4 == 0 && wide;
    f32x4 w = {0.f, 0.f, 0.f, 0.f};
    if (p.w_in) {
        if (whole) {
            w = *reinterpret_cast<const f32x4*>(p.w_in + wat);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j + e < n) w[e] = p.w_in[wat + e];
        }
    }
    constexpr int U = 8;  // heads whose scores are loaded together, under no condition, which each load would wait for
    const float* scores = p.scores + hq0 * p.score_ld + min(j, (n - 1) & ~3);
    for (int h0 = 0; h0 < p.G; h0 += U) {
        const int gn = min(U, p.G - h0);
        f32x4 sc[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
            sc[i] = *reinterpret_cast<const f32x4*>(scores + (int64_t)min(h0 + i, p.G - 1) * p.score_ld);
        // thread t: head t % 8, every 32nd part
        const int mine = tid & 7;
        float M = -INFINITY, L = 0.f;
        if (mine < gn) {
            const f32x2* stats = reinterpret_cast<const f32x2*>(p.stats) + parts.at * p.Hq + h * p.G + h0 + mine;
#pragma unroll 8
            for (int s = tid >> 3; s < parts.n; s += 32) {
                const f32x2 x = stats[(int64_t)s * p.Hq];
                join_part(M, L, x[0], x[1]);
            }
        }
#pragma unroll
        for (int d = 8; d < 64; d <<= 1) {
            const float m = shfl_xor(M, d), l = shfl_xor(L, d);
            join_part(M, L, m, l);
        }
        if (lane < 8) heads[wave][lane] = f32x2{M, L};
        __syncthreads();
        if (tid < 8) {
#pragma unroll
            for (int k = 1; k < 4; ++k) join_part(M, L, heads[k][tid][0], heads[k][tid][1]);
            scale[tid] = f32x2{M, !parts.n || M == -INFINITY ? __builtin_nanf("") : 1.f / L};
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (i < gn)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] += fast_exp2(sc[i][e] - scale[i][0]) * scale[i][1];
    }
    if (whole) {
        *reinterpret_cast<f32x4*>(p.w_out + wat) = w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (j + e < n) p.w_out[wat + e] = w[e];
    }
}

// Whole rows to the workgroups, with no parts to join, where there are many short ones: as many (row, head)
// pairs for each slot of the device as the longest row has steps.  fp32, 12 heads of D 64, rows of up to n
// positions, whole and in shares, us: 700 rows 117 and 142 (n = 300), 179 and 201 (500), 311 and 324 (900);
// 260 rows 48 and 57 (300), 74 and 79 (500), but 126 and 123 (900); 256 rows 203 and 187 (1500); 70 rows of
// 1500 75 and 60.
int paged_groups(int rows, int heads, int G, int max_len, int D, int bf16, bool weights) {
    const int step = paged_step(D, bf16);
    const int64_t slots = 256 * kPagedPerCu, pairs = (int64_t)heads * ((G + 15) / 16);
    const int64_t steps = ((int64_t)max_len + step - 1) / step;
    if (!weights && (steps == 1 || rows * pairs >= slots * steps)) return 0;
    const int64_t most = std::min(rows, kPagedBlock) * steps;
    return (int)std::max<int64_t>(1, std::min({slots / pairs, most, (int64_t)kPagedMaxGroups}));
}

template <int D, typename E>
static int launch_paged_t(const PagedDecodeParams& p, hipStream_t s) {
    const dim3 grid((unsigned)paged_units(p.c.rows, p.c.heads, p.head_tiles, p.groups),
                    p.groups ? (unsigned)paged_blocks(p.c.rows) : 1u);
    size_t lds = (size_t)(4 * (p.G < 16 ? p.G : 16) * (D + 4) + 128) * sizeof(float);
    if (p.scores) lds = std::max<size_t>(lds, 4 * kPagedHold);  // the same LDS first holds scores
    auto split = [&](auto small) {
        constexpr bool kSmall = decltype(small)::value;
        if (p.scores)
            hipLaunchKernelGGL((paged_split_kernel<D, E, kSmall, true>), grid, dim3(256), lds, s, p);
        else
            hipLaunchKernelGGL((paged_split_kernel<D, E, kSmall, false>), grid, dim3(256), lds, s, p);
    };
    if (p.c.page_shift < 4)
        split(std::true_type{});
    else
        split(std::false_type{});
    if (p.groups) {
        const int wblocks = p.scores ? (p.max_len + 1023) / 1024 : 0;
        const int wide = (reinterpret_cast<uintptr_t>(p.w_in) | reinterpret_cast<uintptr_t>(p.w_out)) % 16 == 0;
        const int64_t blocks = (int64_t)p.c.rows * p.Hq + (int64_t)p.c.rows * p.c.heads * wblocks;
        hipLaunchKernelGGL((paged_join_kernel<D, E>), dim3((unsigned)blocks), dim3(256), 0, s, p, wblocks, wide);
    }
    return (int)hipGetLastError();
}

int launch_attn_decode_paged(const PagedDecodeParams& p, int bf16, hipStream_t s) {
    switch (p.c.D) {
        case 32: return bf16 ? launch_paged_t<32, uint16_t>(p, s) : launch_paged_t<32, float>(p, s);
        case 64: return bf16 ? launch_paged_t<64, uint16_t>(p, s) : launch_paged_t<64, float>(p, s);
        case 128: return bf16 ? launch_paged_t<128, uint16_t>(p, s) : launch_paged_t<128, float>(p, s);
        default: return (int)hipErrorInvalidValue;
    }
}

// ============================================================================
// Eviction.  A (row, head) with more than `keep` positions keeps the `recent` newest and, of
// the others, those of the largest weights (equal ones: the lower slot).  One workgroup finds
// the weight of the last one kept, by a radix select over the weights as ordered integers, and
// lists the holes before the cut and the kept positions behind it; then every hole takes one
// of those.  Attention does not mind the order of the keys, so nothing else moves: a
// tenth of the cache evicted moves a tenth of it at most, where closing the gaps would move
// nearly all.  No position is both read and written, so moves run in any order.
//
// Half of 2048 positions, 32 rows of 12 heads of D 64, fp32: 62 us, 11 of them the selection;
// the moves are single rows of 256 bytes, 230 MB read and written at 4.5 TB/s.  64 of 32832
// positions, 2 rows of 8 heads: 32 us, of which 28 are the selection on 16 CUs, five walks over
// a row's keys.  (Other CUs copying the weights meanwhile: 1 us less, not worth their code.)
// ============================================================================
namespace {

// Order of the floats as unsigned numbers, -0 as 0; NaN, below all, is 0.  Infinity is 0xff800000.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x != x ? 0u : b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}

// Slots whose keys fit in LDS beside the rest (144 KB of the 160); longer rows read their weights
// again in every pass.
constexpr int kEvictLds = 36 << 10;

}  // namespace

// W waves, each with one stretch of the slots, 256 at a time, four to a lane, so that what comes before a
// slot is the waves before, the rounds before, the lanes before and the lane's own.
template <int W, bool LDS, bool VEC>
__global__ __launch_bounds__(64 * W) void kv_evict_select_kernel(KvEvictParams p) {
    constexpr int kThreads = 64 * W, kBins = 2048, PER = kBins / kThreads;
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t part[W], part2[W];
    __shared__ uint32_t found[2];
    extern __shared__ __attribute__((aligned(16))) uint32_t skeys[];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int rh = blockIdx.x, row = rh / p.c.heads;
    const int stored = p.c.lens[row], len = min(max(stored, 0), (int)p.c.cap());
    const float* w = p.w_in + (int64_t)rh * p.c.cap();
    const int32_t* pos = p.pos_in + (int64_t)rh * p.c.cap();
    float* wo = p.w_out + (int64_t)rh * p.c.cap();
    int32_t* po = p.pos_out + (int64_t)rh * p.c.cap();
    int32_t* list = p.list + (int64_t)rh * (2 * p.moves + 1);
    const int keep = p.keep;
    const bool copy = wo != w || po != pos;
    if (len <= keep || stored > p.max_len) {
        if (tid == 0) list[2 * p.moves] = 0;
        if (copy)
            for (int j = tid; j < len; j += kThreads) {
                wo[j] = w[j];
                po[j] = pos[j];
            }
        return;
    }
    const int rounds = (len + 4 * kThreads - 1) / (4 * kThreads);
    const int first = 256 * wave * rounds + 4 * lane;
    // Four slots from j on, one by one where rows are not aligned; behind the end, anything.  Loads never stand
    // under a condition: the compiler would wait for each before the next.
    auto load4 = [&](const uint32_t* src, int j) -> u32x4 {
        if constexpr (VEC) return *reinterpret_cast<const u32x4*>(src + min(j, (len - 1) & ~3));
        u32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = src[min(j + e, len - 1)];
        return x;
    };
    struct Meta {
        u32x4 w, pos;
    };
    // f(j, x) for this lane's groups of four slots in order, x = load(j); U of them are loaded together.  Every loop
    // runs a few rounds only, so the time is that of fetching its code: little of it (two rows of 32832 slots, 8
    // heads: 36 us with U = 4 for keys in LDS as well, 32 so).
    auto each = [&](auto load, auto f) {
        constexpr int U = 2;
#pragma unroll 1
        for (int i = 0; i < rounds; i += U) {
            decltype(load(0)) x[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                x[u] = load(first + 256 * (i + u));
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u < rounds) f(first + 256 * (i + u), x[u]);
        }
    };
    const uint32_t *wbits = reinterpret_cast<const uint32_t*>(w), *pbits = reinterpret_cast<const uint32_t*>(pos);
    // Positions past `safe` stay.
    int safe = INT32_MAX;
    bool all_safe = false;
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
    if (p.recent) {
        int top = INT32_MIN;
        each([&](int j) { return load4(pbits, j); }, [&](int j, u32x4 x) {
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, j + e < len ? (int)x[e] : INT32_MIN);
        });
        top = wave_all(top, [](int x, int y) { return max(x, y); });
        if (lane == 0) part[wave] = (uint32_t)top;
        __syncthreads();
        for (int i = 0; i < W; ++i) top = max(top, (int)part[i]);
        const int64_t s = (int64_t)top - p.recent;
        all_safe = s < INT32_MIN;
        safe = all_safe ? INT32_MIN : (int)s;
    } else {
        __syncthreads();
    }
    // Above every weight's key, and alone in its bin of every pass.  Slots behind the end have it too, and are
    // taken off the counts.
    constexpr uint32_t kSafe = 0xffffffffu;
    auto keys_of = [&](int j, Meta x) {
        u32x4 k;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            k[e] = (int)x.pos[e] > safe || all_safe ? kSafe : ordered(__uint_as_float(x.w[e]));
        if (j + 4 > len) {
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = j + e < len ? k[e] : kSafe;
        }
        return k;
    };
    auto meta = [&](int j) { return Meta{load4(wbits, j), p.recent ? load4(pbits, j) : u32x4{0u, 0u, 0u, 0u}}; };
    each(meta, [&](int j, Meta x) {
        const u32x4 k = keys_of(j, x);
        if (LDS && j < len) *reinterpret_cast<u32x4*>(&skeys[j]) = k;
        // often the whole wave has one bin (recent slots, equal weights)
        const uint32_t one = __builtin_amdgcn_readfirstlane(k[0] >> 21);
        if (__all((k[0] >> 21) == one && (k[1] >> 21) == one && (k[2] >> 21) == one && (k[3] >> 21) == one)) {
            if (lane == 0) atomicAdd(&hist[one], 256u);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) atomicAdd(&hist[k[e] >> 21], 1u);
        }
    });
    auto keys = [&](auto f) {  // f(j, four keys)
        if constexpr (LDS) {
#pragma unroll 1
            for (int i = 0; i < rounds; ++i) {
                const int j = first + 256 * i;
                const u32x4 k = *reinterpret_cast<const u32x4*>(&skeys[min(j, (len - 1) & ~3)]);
                f(j, j < len ? k : u32x4{kSafe, kSafe, kSafe, kSafe});
            }
        } else
            each(meta, [&](int j, Meta x) { f(j, keys_of(j, x)); });
    };
    __syncthreads();

    // The keep-th largest key, eleven bits at a time from the top; `need` of those that share the bits found
    // so far are kept.
    uint32_t last = kSafe, need = (uint32_t)keep;
    const uint32_t safes = hist[kBins - 1] - (uint32_t)(4 * kThreads * rounds - len);
    if (safes < need) {
        need -= safes;
        __syncthreads();
        if (tid == 0) hist[kBins - 1] = 0;
        __syncthreads();
        uint32_t prefix = 0;
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 10 : 11;
            const uint32_t bins = 1u << width;
            if (pass) {
                keys([&](int, u32x4 k) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if ((k[e] >> (shift + width)) == prefix)
                            atomicAdd(&hist[(k[e] >> shift) & (bins - 1)], 1u);
                });
                __syncthreads();
            }
            // thread t: PER bins from the top, behind those of the threads before
            uint32_t n[PER], mine = 0;
            uint32_t* mybins = hist + (kBins - PER * (tid + 1));
#pragma unroll
            for (int i = 0; i < PER; ++i) mine += n[i] = mybins[PER - 1 - i];
            uint32_t before = mine;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t up = __shfl_up(before, d, 64);
                if (lane >= d) before += up;
            }
            if (lane == 63) part[wave] = before;
            before -= mine;
            __syncthreads();
            for (int i = 0; i < wave; ++i) before += part[i];
            if (before < need && before + mine >= need) {
                uint32_t bin = 0;
                bool done = false;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    done |= before + n[i] >= need;
                    if (!done) {
                        before += n[i];
                        ++bin;
                    }
                }
                found[0] = prefix << width | (kBins - 1 - (PER * tid + bin));
                found[1] = need - before;
            }
#pragma unroll
            for (int i = 0; i < PER; ++i) mybins[i] = 0;
            __syncthreads();
            prefix = found[0];
            need = found[1];
        }
        last = prefix;
    }

    // Kept: the keys above `last`, and the first `need` slots of those equal to it.
    uint32_t gt = 0, eq = 0;
    keys([&](int, u32x4 k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            gt += k[e] > last;
            eq += k[e] == last;
        }
    });
    gt = wave_all(gt, [](uint32_t x, uint32_t y) { return x + y; });
    eq = wave_all(eq, [](uint32_t x, uint32_t y) { return x + y; });
    const int behind = 256 * rounds - min(max(len - 256 * wave * rounds, 0), 256 * rounds);  // the end
    (last == kSafe ? eq : gt) -= behind;
    __syncthreads();
    if (lane == 0) {
        part[wave] = gt;
        part2[wave] = eq;
    }
    __syncthreads();
    uint32_t eq_before = 0, kept_before = 0;
    for (int i = 0; i < wave; ++i) {
        const uint32_t e = part2[i];
        kept_before += part[i] + (eq_before < need ? min(e, need - eq_before) : 0u);
        eq_before += e;
    }
    auto below = [](uint64_t mask, uint32_t n) {  // n and its bits under this lane
        return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, n));
    };
    // Lists four slots; kept: which of them are.
    auto place = [&](int j, u32x4 k, bool (&kept)[4]) {
        bool same[4];
        uint64_t m[4];
        const int in = len - j;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            kept[e] = k[e] > last && e < in;
            same[e] = k[e] == last && e < in;
        }
        if (__any(same[0] || same[1] || same[2] || same[3])) {
            uint32_t rank = eq_before;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[e] = __ballot(same[e]);
                rank = below(m[e], rank);
                eq_before += __popcll(m[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                kept[e] |= same[e] && rank < need;
                rank += same[e];
            }
        }
        uint32_t before = kept_before;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            m[e] = __ballot(kept[e]);
            before = below(m[e], before);
            kept_before += __popcll(m[e]);
        }
        if (j < len) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool front = j + e < keep;
                if (front != kept[e] && e < in)  // a hole, or one to fill one (the last kept comes first)
                    list[front ? j + e - (int)before : p.moves + keep - 1 - (int)before] = j + e;
                if (j + e == keep) list[2 * p.moves] = keep - (int)before;  // holes before the cut
                before += kept[e];
            }
        }
    };
    if (copy)
        each([&](int j) { return Meta{load4(wbits, j), load4(pbits, j)}; }, [&](int j, Meta x) {
            u32x4 k;
            if constexpr (LDS)
                k = *reinterpret_cast<const u32x4*>(&skeys[min(j, (len - 1) & ~3)]);
            else
                k = keys_of(j, p.recent ? x : Meta{x.w, u32x4{0u, 0u, 0u, 0u}});
            bool kept[4];
            place(j, k, kept);
            // a hole gets its own from the moves that follow
            if (VEC && j + 4 <= keep) {
                *reinterpret_cast<u32x4*>(wo + j) = x.w;
                *reinterpret_cast<u32x4*>(po + j) = x.pos;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (kept[e] && j + e < keep) {
                        wo[j + e] = __uint_as_float(x.w[e]);
                        po[j + e] = (int)x.pos[e];
                    }
            }
        });
    else
        keys([&](int j, u32x4 k) {
            bool kept[4];
            place(j, k, kept);
        });
}

// Each move: a row of K, one of V, its weight and its position.  A thread takes its 16-byte
// piece of U of them, the loads of all U together.
template <int U>
__global__ __launch_bounds__(256) void kv_evict_move_kernel(KvEvictParams p, int pieces, int esz, int blocks) {
    const int rh = blockIdx.x / blocks, block = blockIdx.x % blocks, row = rh / p.c.heads, h = rh % p.c.heads;
    const int32_t* list = p.list + (int64_t)rh * (2 * p.moves + 1);
    const int n = list[2 * p.moves];
    const int per = 256 / pieces;  // moves of a workgroup at a time
    const int i0 = block * per * U + threadIdx.x / pieces, c = threadIdx.x % pieces;
    if (block == 0 && h == 0 && threadIdx.x == 0) {
        const int len = p.c.lens[row];
        p.lens_out[row] = len > p.keep && len <= p.max_len ? p.keep : len;
    }
    if (i0 >= n) return;
    const int32_t* table = p.c.table + row * p.c.table_stride;
    const int mask = (1 << p.c.page_shift) - 1;
    const int64_t at = (int64_t)rh * p.c.cap();
    int src[U], dst[U], ps[U], pd[U];
    u32x4 kx[U], vx[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = min(i0 + u * per, n - 1);  // the last one again where there are no more
        dst[u] = list[i];
        src[u] = list[p.moves + n - 1 - i];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        pd[u] = page_of(p.c, table, dst[u]);
        ps[u] = page_of(p.c, table, src[u]);
    }
    const int64_t ko = h * p.c.sk.h, vo = h * p.c.sv.h;
    const char *K = (const char*)p.c.k + 16 * c, *V = (const char*)p.c.v + 16 * c;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int pg = max(ps[u], 0), slot = src[u] & mask;
        kx[u] = ld16_nt(K + (pg * p.c.sk.b + ko + slot * p.c.sk.t) * esz);
        vx[u] = ld16_nt(V + (pg * p.c.sv.b + vo + slot * p.c.sv.t) * esz);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (i0 + u * per >= n) break;
        const int slot = dst[u] & mask;
        if (pd[u] >= 0 && ps[u] >= 0) {
            *reinterpret_cast<u32x4*>((char*)K + (pd[u] * p.c.sk.b + ko + slot * p.c.sk.t) * esz) = kx[u];
            *reinterpret_cast<u32x4*>((char*)V + (pd[u] * p.c.sv.b + vo + slot * p.c.sv.t) * esz) = vx[u];
        }
        if (c == 0) {
            p.w_out[at + dst[u]] = p.w_in[at + src[u]];
            p.pos_out[at + dst[u]] = p.pos_in[at + src[u]];
        }
    }
    // No page to copy from: NaN, so that attention sees it here as it did there.  Apart from the copies, whose stores
    // would take 2% longer with both.
    bool lost = false;
#pragma unroll
    for (int u = 0; u < U; ++u) lost |= ps[u] < 0;
    if (__any(lost)) {
        const uint32_t nan = esz == 2 ? 0x7fc07fc0u : 0x7fc00000u;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * per >= n || ps[u] >= 0 || pd[u] < 0) continue;
            const int slot = dst[u] & mask;
            *reinterpret_cast<u32x4*>((char*)K + (pd[u] * p.c.sk.b + ko + slot * p.c.sk.t) * esz) =
                *reinterpret_cast<u32x4*>((char*)V + (pd[u] * p.c.sv.b + vo + slot * p.c.sv.t) * esz) =
                    u32x4{nan, nan, nan, nan};
        }
    }
}

int launch_kv_evict(const KvEvictParams& p, int bf16, hipStream_t s) {
    const int esz = bf16 ? 2 : 4, pieces = p.c.D * esz / 16, blocks = p.move_blocks;
    const int64_t rh = (int64_t)p.c.rows * p.c.heads;
    const dim3 grid((unsigned)rh);
    const size_t lds = ((size_t)p.max_len + 3) / 4 * 16;
    const uintptr_t any = reinterpret_cast<uintptr_t>(p.w_in) | reinterpret_cast<uintptr_t>(p.w_out) |
                          reinterpret_cast<uintptr_t>(p.pos_in) | reinterpret_cast<uintptr_t>(p.pos_out);
    auto select = [&](auto v) {
        constexpr bool kVec = decltype(v)::value;
        if (evict_threads(p.max_len) == 256)
            hipLaunchKernelGGL((kv_evict_select_kernel<4, true, kVec>), grid, dim3(256), lds, s, p);
        else if (p.max_len <= kEvictLds)
            hipLaunchKernelGGL((kv_evict_select_kernel<16, true, kVec>), grid, dim3(1024), lds, s, p);
        else
            hipLaunchKernelGGL((kv_evict_select_kernel<16, false, kVec>), grid, dim3(1024), 0, s, p);
    };
    if (any % 16 == 0 && p.c.cap() % 4 == 0)
        select(std::true_type{});
    else
        select(std::false_type{});
    const dim3 g2((unsigned)(rh * blocks));
    if (p.move_unroll == 4)
        hipLaunchKernelGGL((kv_evict_move_kernel<4>), g2, dim3(256), 0, s, p, pieces, esz, blocks);
    else
        hipLaunchKernelGGL((kv_evict_move_kernel<1>), g2, dim3(256), 0, s, p, pieces, esz, blocks);
    return (int)hipGetLastError();
}

// ============================================================================
// Reordering under beam search.  Full pages are only read from here on, so a beam takes its
// parent's by number.  The last, partly filled page will be written by each beam on its own: a
// beam that is not its own parent copies it into its spare page, and the page that it had becomes
// its spare.  Nobody writes a page that another one reads, so one launch does it for all layers.
// A copy, bound by HBM: 32 x 8 beams, 12 layers of 12 heads of D 64, 28 positions of the last page of 32, bf16, 463 MB
// in 78 us, 5.9 TB/s (stores through the caches: 87 us).  One search of 4 beams is a launch, 3.7 us.
// ============================================================================
__global__ __launch_bounds__(256) void beam_reorder_kernel(BeamReorderParams p, int pieces, int esz) {
    const int row = blockIdx.x, layer = blockIdx.y;
    const int first = row / p.beams * p.beams;
    const int len = min(max(p.c.lens[first], 0), (int)p.c.cap());
    const int full = len >> p.c.page_shift, part = len & ((1 << p.c.page_shift) - 1);
    const int pb = p.parents[row];
    const bool ok = (unsigned)pb < (unsigned)p.beams;
    const int parent = first + (ok ? pb : 0);
    const int32_t* own = p.c.table + row * p.c.table_stride;
    const int32_t* from = p.c.table + parent * p.c.table_stride;
    const bool other = ok && parent != row && part;
    const int src = other ? from[full] : -1, dst = p.spare[row];
    const bool copy = (unsigned)src < (unsigned)p.c.n_pages;
    if (layer == 0 && blockIdx.z == 0) {
        int32_t* out = p.table_out + row * p.table_out_stride;
        for (int i = threadIdx.x; i < p.c.max_pages; i += 256) {
            int v = own[i];
            if (!ok && len) v = -1;  // no such parent: the row names no page, and reads as NaN
            else if (i < full) v = from[i];
            else if (i == full && other) v = copy ? dst : src;  // no page to copy: its number, which reads as NaN
            out[i] = v;
        }
        if (threadIdx.x == 0) p.spare_out[row] = copy ? own[full] : dst;
    }
    if (!copy || (unsigned)dst >= (unsigned)p.c.n_pages) return;
    const int n = p.c.heads * part * pieces;
    for (int i = blockIdx.z * 256 + threadIdx.x; i < n; i += 256 * gridDim.z) {
        const int hs = i / pieces, c = i - hs * pieces;
        const int h = hs / part, t = hs - h * part;
        const int64_t ko = layer * p.k_layer + h * p.c.sk.h + t * p.c.sk.t;
        const int64_t vo = layer * p.v_layer + h * p.c.sv.h + t * p.c.sv.t;
        const u32x4 kx = *reinterpret_cast<const u32x4*>((const char*)p.c.k + (ko + src * p.c.sk.b) * esz + 16 * c);
        const u32x4 vx = *reinterpret_cast<const u32x4*>((const char*)p.c.v + (vo + src * p.c.sv.b) * esz + 16 * c);
        __builtin_nontemporal_store(
            kx, reinterpret_cast<u32x4*>((char*)p.c.k + (ko + dst * p.c.sk.b) * esz + 16 * c));
        __builtin_nontemporal_store(
            vx, reinterpret_cast<u32x4*>((char*)p.c.v + (vo + dst * p.c.sv.b) * esz + 16 * c));
    }
}

int launch_beam_reorder(const BeamReorderParams& p, int bf16, hipStream_t s) {
    const int esz = bf16 ? 2 : 4, pieces = p.c.D * esz / 16;
    // pieces of a whole page; a workgroup takes up to two rounds of them
    const int64_t n = ((int64_t)p.c.heads * pieces << p.c.page_shift);
    int64_t z = (n + 511) / 512;
    if (z > 1024) z = 1024;
    const dim3 grid((unsigned)p.c.rows, (unsigned)p.layers, (unsigned)z);
    hipLaunchKernelGGL(beam_reorder_kernel, grid, dim3(256), 0, s, p, pieces, esz);
    return (int)hipGetLastError();
}

}  // namespace inf
