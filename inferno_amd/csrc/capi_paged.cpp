// capi_paged.cpp -- the extern "C" entry points of generation from a paged
// key-value cache (include/inferno_hip.h): argument validation on the host,
// workspace sizing, launches.  Nothing here allocates.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <string>
#include <utility>

#include "inferno_hip.h"
#include "kernels.h"

namespace {

constexpr size_t kAlign = 256;
constexpr int64_t kMaxRowStride = int64_t(1) << 22;  // as the other attention views'
constexpr int64_t kMaxBlocks = int64_t(1) << 30;
constexpr int64_t kMaxThreads = (int64_t(1) << 32) - 1;  // of a launch, along one axis of its grid

bool dtype_ok(int dt) { return dt == INF_F32 || dt == INF_BF16; }
int esz(inf_dtype dt) { return dt == INF_F32 ? 4 : 2; }
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
int hip_status(int e) { return e == 0 ? INF_OK : INF_ERR_HIP; }
size_t round_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }
inf::View4 view(const inf_strides& s) { return inf::View4{s.b, s.h, s.t}; }

// Strides of a [b, h, t, D] view whose rows allow accesses of `bytes` bytes.
int check_view(const void* p, const inf_strides& s, int es, int bytes) {
    if (!p) return INF_ERR_NULL_POINTER;
    if (s.d != 1 || s.b < 0 || s.h < 0 || s.t < 0 || s.t > kMaxRowStride) return INF_ERR_BAD_STRIDE;
    const int64_t n = bytes / es;
    if (!aligned(p, (size_t)bytes) || s.b % n || s.h % n || s.t % n) return INF_ERR_ALIGNMENT;
    return INF_OK;
}

// Every element of a written view has an address of its own: ordered by stride, each is at
// least the span of the dims inside it.
int check_apart(const inf_strides& s, int64_t B, int64_t H, int64_t T, int64_t D, int64_t layers = 1,
                int64_t layer_stride = 0) {
    struct Dim { int64_t n, stride; } d[4] = {{layers, layer_stride}, {B, s.b}, {H, s.h}, {T, s.t}};
    std::sort(d, d + 4, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    int64_t span = D;
    for (const Dim& x : d) {
        if (x.n <= 1) continue;
        if (x.stride < span) return INF_ERR_BAD_STRIDE;
        span = x.stride * (x.n - 1) + span;
    }
    return INF_OK;
}

int check_shape(const inf_paged_kv* c) {
    if (!c) return INF_ERR_NULL_POINTER;
    if (!dtype_ok(c->dt)) return INF_ERR_BAD_DTYPE;
    if (c->rows < 1 || c->heads < 1 || c->D < 1 || c->page_size < 1 || c->max_pages < 1 || c->n_pages < 1)
        return INF_ERR_BAD_SHAPE;
    if (c->D != 32 && c->D != 64 && c->D != 128) return INF_ERR_UNSUPPORTED;
    if (c->page_size & (c->page_size - 1)) {
        inf::set_error_detail("paged cache: page_size must be a power of two, got " + std::to_string(c->page_size));
        return INF_ERR_UNSUPPORTED;
    }
    if (c->rows > 65535 || (int64_t)c->rows * c->heads > (1 << 24) ||
        (int64_t)c->max_pages * c->page_size > (1 << 30))
        return INF_ERR_BAD_SHAPE;
    return INF_OK;
}

// The cache, for a call that reads it, or writes it too.
int check_cache(const inf_paged_kv* c, bool written, inf::PagedView* out) {
    int st = check_shape(c);
    if (st != INF_OK) return st;
    if ((st = check_view(c->k, c->sk, esz(c->dt), 16)) || (st = check_view(c->v, c->sv, esz(c->dt), 16))) return st;
    if (!c->table || !c->lens) return INF_ERR_NULL_POINTER;
    if (!aligned(c->table, 4) || !aligned(c->lens, 4)) return INF_ERR_ALIGNMENT;
    if (c->table_stride < c->max_pages) return INF_ERR_BAD_STRIDE;
    if (written && ((st = check_apart(c->sk, c->n_pages, c->heads, c->page_size, c->D)) ||
                    (st = check_apart(c->sv, c->n_pages, c->heads, c->page_size, c->D))))
        return st;
    int shift = 0;
    while ((1 << shift) < c->page_size) ++shift;
    *out = inf::PagedView{c->k, c->v, view(c->sk), view(c->sv), c->table, c->lens, c->table_stride,
                          c->rows, c->heads, c->n_pages, c->max_pages, shift, c->D};
    return INF_OK;
}

// Whether arrays of 4-byte elements overlap (either may be null: then not).
bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + 4 * (uintptr_t)nb && y < x + 4 * (uintptr_t)na;
}
// The same of arrays of one size, without being the same.
bool overlap_partly(const void* a, const void* b, int64_t n) { return a != b && overlap(a, n, b, n); }
// ... of [rows, heads, capacity] arrays.
bool overlap_partly(const inf_paged_kv* c, const void* a, const void* b) {
    return overlap_partly(a, b, (int64_t)c->rows * c->heads * c->max_pages * c->page_size);
}

int64_t capacity(const inf_paged_kv* c) { return (int64_t)c->max_pages * c->page_size; }

// The decode's workspace: the shares' results (one per row and share that meet, so at most rows +
// shares), the rows' first steps, the scores.
struct DecodeSizes {
    int groups;
    int64_t score_ld;
    size_t part, stats, first, scores;
    size_t total() const { return part + stats + first + scores; }
};
DecodeSizes decode_sizes(const inf_paged_kv* c, int q_heads, int max_len, bool weights) {
    DecodeSizes s{};
    const int bf16 = c->dt == INF_BF16, step = inf::paged_step(c->D, bf16), blocks = inf::paged_blocks(c->rows);
    s.groups = inf::paged_groups(c->rows, c->heads, q_heads / c->heads, max_len, c->D, bf16, weights);
    if (s.groups == 0) return s;
    const size_t parts = ((size_t)c->rows + (size_t)blocks * s.groups) * q_heads;
    s.part = round_up(parts * c->D * sizeof(float));
    s.stats = round_up(parts * 2 * sizeof(float));
    s.first = round_up(((size_t)c->rows + blocks) * sizeof(int32_t));
    s.score_ld = ((int64_t)max_len + step - 1) / step * step;
    if (weights) s.scores = round_up((size_t)c->rows * q_heads * s.score_ld * sizeof(float));
    return s;
}

int check_decode(const inf_paged_kv* c, int q_heads, int max_len) {
    const int st = check_shape(c);
    if (st != INF_OK) return st;
    if (q_heads < 1 || q_heads % c->heads || max_len < 1 || max_len > capacity(c)) return INF_ERR_BAD_SHAPE;
    if ((int64_t)c->rows * q_heads > (1 << 24)) return INF_ERR_BAD_SHAPE;
    // the steps of a block of rows are counted in 32 bits
    if ((int64_t)std::min(c->rows, inf::kPagedBlock) * (max_len / inf::paged_step(c->D, c->dt == INF_BF16) + 1) >
        (1 << 30))
        return INF_ERR_BAD_SHAPE;
    return INF_OK;
}

int check_evict(const inf_paged_kv* c, int keep, int max_len) {
    const int st = check_shape(c);
    if (st != INF_OK) return st;
    if (keep < 1 || max_len < 1 || max_len > capacity(c)) return INF_ERR_BAD_SHAPE;
    return INF_OK;
}

int evict_moves(int keep, int max_len) { return std::max(0, std::min(keep, max_len - keep)); }

int check_beams(int64_t groups, int beams, int64_t vocab) {
    if (groups < 1 || beams < 1 || vocab < 1 || vocab > INT32_MAX) return INF_ERR_BAD_SHAPE;
    if (beams > inf::kMaxBeams) {
        inf::set_error_detail("beam selection: at most " + std::to_string(inf::kMaxBeams) + " beams, got " +
                              std::to_string(beams));
        return INF_ERR_UNSUPPORTED;
    }
    if (groups > (1 << 24)) return INF_ERR_BAD_SHAPE;
    int ns = 0;
    int64_t ch = 0;
    inf::beam_select_plan(groups, beams, vocab, &ns, &ch);
    return groups * beams * ns * 256 > kMaxThreads || groups * 1024 > kMaxThreads ? INF_ERR_BAD_SHAPE : INF_OK;
}

}  // namespace

extern "C" {

int inf_kv_append(const inf_paged_kv* cache, const void* k, inf_strides sk, const void* v, inf_strides sv,
                  const int32_t* counts, int T, float* weights, int32_t* positions, const int32_t* seen,
                  void* stream) {
    inf::KvAppendParams p{};
    int st = check_cache(cache, true, &p.c);
    if (st != INF_OK) return st;
    if (T < 0) return INF_ERR_BAD_SHAPE;
    if (T == 0) return INF_OK;
    const int es = esz(cache->dt);
    if ((st = check_view(k, sk, es, 4 * es)) || (st = check_view(v, sv, es, 4 * es))) return st;
    if ((int64_t)T * cache->heads * cache->D > kMaxBlocks) return INF_ERR_BAD_SHAPE;
    p.k = k; p.v = v;
    p.sk = view(sk); p.sv = view(sv);
    p.counts = counts;
    p.Tn = T;
    p.wide = check_view(k, sk, es, 16) == INF_OK && check_view(v, sv, es, 16) == INF_OK;
    p.weights = weights;
    p.positions = positions;
    p.seen = seen;
    return hip_status(inf::launch_kv_append(p, cache->dt == INF_BF16, (hipStream_t)stream));
}

int inf_attn_decode_paged_workspace(const inf_paged_kv* cache, int q_heads, int max_len, int weights,
                                    size_t* out_bytes) {
    if (!out_bytes) return INF_ERR_NULL_POINTER;
    *out_bytes = 0;
    const int st = check_decode(cache, q_heads, max_len);
    if (st != INF_OK) return st;
    const DecodeSizes s = decode_sizes(cache, q_heads, max_len, weights != 0);
    *out_bytes = s.total();
    return INF_OK;
}

int inf_attn_decode_paged(const inf_paged_kv* cache, const void* q, inf_strides sq, void* o, inf_strides so,
                          int q_heads, int max_len, float scale, const float* weights_in, float* weights_out,
                          void* workspace, size_t ws_bytes, void* stream) {
    inf::PagedDecodeParams p{};
    int st = check_decode(cache, q_heads, max_len);
    if (st != INF_OK || (st = check_cache(cache, false, &p.c))) return st;
    if (!(scale > 0.f) || !std::isfinite(scale)) return INF_ERR_BAD_SCALE;
    const int es = esz(cache->dt);
    if ((st = check_view(q, sq, es, 4 * es)) || (st = check_view(o, so, es, 4 * es)) ||
        (st = check_apart(so, cache->rows, q_heads, 1, cache->D)))
        return st;
    if (weights_in && !weights_out) return INF_ERR_NULL_POINTER;
    if (overlap_partly(cache, weights_in, weights_out)) return INF_ERR_BAD_STRIDE;
    const DecodeSizes s = decode_sizes(cache, q_heads, max_len, weights_out != nullptr);
    const int64_t tiles = (q_heads / cache->heads + 15) / 16;
    const int64_t join = q_heads + (weights_out ? (int64_t)cache->heads * ((max_len + 1023) / 1024) : 0);
    if (inf::paged_units(cache->rows, cache->heads, (int)tiles, s.groups) * 256 > kMaxThreads ||
        (s.groups && cache->rows * join * 256 > kMaxThreads))
        return INF_ERR_BAD_SHAPE;
    if (s.total() && (!workspace || ws_bytes < s.total())) return INF_ERR_WORKSPACE;
    if (s.total() && !aligned(workspace, kAlign)) return INF_ERR_ALIGNMENT;
    p.q = q; p.o = o;
    p.sq = view(sq); p.so = view(so);
    p.Hq = q_heads;
    p.G = q_heads / cache->heads;
    p.head_tiles = (int)tiles;
    p.max_len = max_len;
    p.groups = s.groups;
    p.cs = scale * 1.4426950408889634f;
    char* ws = static_cast<char*>(workspace);
    p.part = reinterpret_cast<float*>(ws);
    p.stats = reinterpret_cast<float*>(ws + s.part);
    p.first = reinterpret_cast<int32_t*>(ws + s.part + s.stats);
    if (weights_out) p.scores = reinterpret_cast<float*>(ws + s.part + s.stats + s.first);
    p.score_ld = s.score_ld;
    p.w_in = weights_in;
    p.w_out = weights_out;
    return hip_status(inf::launch_attn_decode_paged(p, cache->dt == INF_BF16, (hipStream_t)stream));
}

int inf_kv_evict_workspace(const inf_paged_kv* cache, int keep, int max_len, size_t* out_bytes) {
    if (!out_bytes) return INF_ERR_NULL_POINTER;
    *out_bytes = 0;
    const int st = check_evict(cache, keep, max_len);
    if (st != INF_OK) return st;
    *out_bytes = round_up((size_t)cache->rows * cache->heads * (2 * (size_t)evict_moves(keep, max_len) + 1) * 4);
    return INF_OK;
}

int inf_kv_evict(const inf_paged_kv* cache, const float* weights_in, float* weights_out, const int32_t* positions_in,
                 int32_t* positions_out, int32_t* lens_out, int keep, int recent, int max_len, void* workspace,
                 size_t ws_bytes, void* stream) {
    inf::KvEvictParams p{};
    int st = check_evict(cache, keep, max_len);
    if (st != INF_OK || (st = check_cache(cache, true, &p.c))) return st;
    if (recent < 0 || recent > keep) return INF_ERR_BAD_SHAPE;
    if (!weights_in || !weights_out || !positions_in || !positions_out || !lens_out) return INF_ERR_NULL_POINTER;
    if (overlap_partly(cache, weights_in, weights_out) || overlap_partly(cache, positions_in, positions_out) ||
        overlap_partly(cache->lens, lens_out, cache->rows))
        return INF_ERR_BAD_STRIDE;
    size_t need = 0;
    inf_kv_evict_workspace(cache, keep, max_len, &need);
    if (!workspace || ws_bytes < need) return INF_ERR_WORKSPACE;
    if (!aligned(workspace, 4)) return INF_ERR_ALIGNMENT;
    p.w_in = weights_in; p.w_out = weights_out;
    p.pos_in = positions_in; p.pos_out = positions_out;
    p.lens_out = lens_out;
    p.keep = keep; p.recent = recent; p.max_len = max_len;
    p.moves = evict_moves(keep, max_len);
    p.list = static_cast<int32_t*>(workspace);
    const int64_t rh = (int64_t)cache->rows * cache->heads;
    p.move_unroll = inf::evict_unroll(rh, p.moves, cache->D, cache->dt == INF_BF16);
    const int64_t blocks = inf::evict_blocks(p.moves, p.move_unroll, cache->D, cache->dt == INF_BF16);
    if (rh * inf::evict_threads(max_len) > kMaxThreads || rh * blocks * 256 > kMaxThreads) return INF_ERR_BAD_SHAPE;
    p.move_blocks = (int)blocks;
    return hip_status(inf::launch_kv_evict(p, cache->dt == INF_BF16, (hipStream_t)stream));
}

int inf_beam_select_workspace(int64_t groups, int beams, int64_t vocab, size_t* out_bytes) {
    if (!out_bytes) return INF_ERR_NULL_POINTER;
    *out_bytes = 0;
    const int st = check_beams(groups, beams, vocab);
    if (st != INF_OK) return st;
    int ns = 0;
    int64_t ch = 0;
    inf::beam_select_plan(groups, beams, vocab, &ns, &ch);
    const size_t parts = (size_t)groups * beams * ns;
    *out_bytes = round_up(parts * 8) + round_up(parts * 8 * beams) + round_up(parts * 4);
    return INF_OK;
}

int inf_beam_select(const void* logits, int64_t ld, const float* scores, const int32_t* finished, int64_t groups,
                    int beams, int64_t vocab, int32_t eos, int32_t* tokens, int32_t* parents, float* scores_out,
                    int32_t* finished_out, inf_dtype dt, void* workspace, size_t ws_bytes, void* stream) {
    if (!dtype_ok(dt)) return INF_ERR_BAD_DTYPE;
    const int st = check_beams(groups, beams, vocab);
    if (st != INF_OK) return st;
    if (!logits || !scores || !tokens || !parents || !scores_out) return INF_ERR_NULL_POINTER;
    if (eos >= vocab || (finished && eos < 0)) return INF_ERR_BAD_SHAPE;
    if (ld < vocab) return INF_ERR_BAD_STRIDE;
    // a group's results must not lie over what another group still reads
    for (const void* out : std::initializer_list<const void*>{tokens, parents, scores_out, finished_out})
        if (overlap_partly(out, scores, groups * beams) || overlap_partly(out, finished, groups * beams))
            return INF_ERR_BAD_STRIDE;
    if (!aligned(logits, (size_t)esz(dt))) return INF_ERR_ALIGNMENT;
    size_t need = 0;
    inf_beam_select_workspace(groups, beams, vocab, &need);
    if (!workspace || ws_bytes < need) return INF_ERR_WORKSPACE;
    if (!aligned(workspace, kAlign)) return INF_ERR_ALIGNMENT;
    inf::BeamSelectParams p{};
    p.logits = logits; p.scores = scores; p.finished = finished;
    p.groups = groups; p.vocab = vocab; p.ld = ld;
    p.beams = beams;
    p.eos = eos < 0 ? -1 : eos;
    inf::beam_select_plan(groups, beams, vocab, &p.nsplit, &p.chunk);
    const size_t parts = (size_t)groups * beams * p.nsplit;
    char* ws = static_cast<char*>(workspace);
    p.sums = reinterpret_cast<double*>(ws);
    p.cand = reinterpret_cast<uint64_t*>(ws + round_up(parts * 8));
    p.maxs = reinterpret_cast<float*>(ws + round_up(parts * 8) + round_up(parts * 8 * beams));
    p.tokens = tokens; p.parents = parents; p.scores_out = scores_out; p.finished_out = finished_out;
    return hip_status(inf::launch_beam_select(p, dt == INF_BF16, (hipStream_t)stream));
}

int inf_beam_reorder(const inf_paged_kv* cache, int layers, int64_t k_layer_stride, int64_t v_layer_stride,
                     const int32_t* parents, int beams, int32_t* table_out, int64_t table_out_stride,
                     const int32_t* spare, int32_t* spare_out, void* stream) {
    inf::BeamReorderParams p{};
    int st = check_cache(cache, true, &p.c);
    if (st != INF_OK) return st;
    if (layers < 1 || layers > 65535 || beams < 1 || cache->rows % beams) return INF_ERR_BAD_SHAPE;
    if (!parents || !table_out || !spare || !spare_out) return INF_ERR_NULL_POINTER;
    if (layers > 1) {
        const int es = esz(cache->dt);
        if (k_layer_stride < 0 || v_layer_stride < 0) return INF_ERR_BAD_STRIDE;
        if (k_layer_stride * es % 16 || v_layer_stride * es % 16) return INF_ERR_ALIGNMENT;
        if ((st = check_apart(cache->sk, cache->n_pages, cache->heads, cache->page_size, cache->D, layers,
                              k_layer_stride)) ||
            (st = check_apart(cache->sv, cache->n_pages, cache->heads, cache->page_size, cache->D, layers,
                              v_layer_stride)))
            return st;
    }
    if (table_out_stride < cache->max_pages) return INF_ERR_BAD_STRIDE;
    // rows read the tables of other rows, and every layer its row's parent and spare page: the new ones lie elsewhere
    const int64_t rows = cache->rows, nt = (rows - 1) * cache->table_stride + cache->max_pages,
                  nu = (rows - 1) * table_out_stride + cache->max_pages;
    auto read = [&](const int32_t* out, int64_t n) {
        return overlap(out, n, cache->table, nt) || overlap(out, n, cache->lens, rows) ||
               overlap(out, n, parents, rows) || overlap(out, n, spare, rows);
    };
    if (read(table_out, nu) || read(spare_out, rows) || overlap(table_out, nu, spare_out, rows))
        return INF_ERR_BAD_STRIDE;
    if ((int64_t)cache->heads * cache->page_size * cache->D > kMaxBlocks) return INF_ERR_BAD_SHAPE;
    p.layers = layers;
    p.beams = beams;
    p.k_layer = k_layer_stride; p.v_layer = v_layer_stride;
    p.parents = parents;
    p.table_out = table_out;
    p.table_out_stride = table_out_stride;
    p.spare = spare; p.spare_out = spare_out;
    return hip_status(inf::launch_beam_reorder(p, cache->dt == INF_BF16, (hipStream_t)stream));
}

}  // extern "C"
