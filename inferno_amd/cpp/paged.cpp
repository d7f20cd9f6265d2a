// paged.cpp -- PagedKVCache (include/inferno/modules/pagedkvcache.h) and beam_select
// (include/inferno/functional/beam.h) over the C-ABI's paged entry points.
#include <algorithm>

#include "detail.h"
#include "inferno/functional/attention.h"
#include "inferno/functional/beam.h"
#include "inferno/gradengine/engine.h"
#include "inferno/modules/pagedkvcache.h"

namespace Inferno {

namespace {

inf_strides strides4(const Tensor& t) {
    const auto& s = t.strides();
    return inf_strides{(int64_t)s[0], (int64_t)s[1], (int64_t)s[2], (int64_t)s[3]};
}

int32_t* ints(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }
float* floats(const Tensor& t) { return static_cast<float*>(t.data_ptr()); }

void fill_int(const Tensor& t, size_t value) {
    detail::status_check(inf_fill(t.data_ptr(), (int64_t)t.numel(), 4, (uint32_t)value, detail::stream_of(t)), "inf_fill");
}

}  // namespace

// The C-ABI's view of one layer, for the step's rows.
struct PagedKVCache::Handle {
    inf_paged_kv kv;
    Handle(const PagedKVCache& c, size_t layer, bool prompt) {
        const auto& st = c.m_k.strides();
        const inf_strides s{(int64_t)st[1], (int64_t)st[2], (int64_t)st[3], 1};
        const size_t at = layer * st[0] * dtype_size(c.m_k.dtype()), per = c.m_table.shape()[1];
        const size_t beams = c.m_options.beams;
        // the prompt's rows are the first ones of the groups
        kv = inf_paged_kv{static_cast<char*>(c.m_k.data_ptr()) + at, static_cast<char*>(c.m_v.data_ptr()) + at, s, s,
                          ints(c.m_table), ints(c.m_lens), (int64_t)(prompt ? per * beams : per),
                          (int)(prompt ? c.m_groups : c.rows()), (int)c.m_heads, (int)c.m_dim,
                          (int)c.m_options.page_size, (int)per, (int)c.m_pages,
                          detail::inf_dt(c.m_k.dtype(), "PagedKVCache")};
    }
};

PagedKVCache::PagedKVCache(size_t layers, size_t groups, size_t heads, size_t capacity, size_t D, Device device,
                           DType dtype, Options options)
    : m_layers(layers), m_groups(groups), m_heads(heads), m_capacity(capacity), m_dim(D), m_options(options) {
    const size_t P = options.page_size;
    if (device.is_cpu()) throw Error("PagedKVCache: a HIP device expected");
    if (!layers || !groups || !heads || !capacity || !options.beams) throw Error("PagedKVCache: empty shape");
    if (D != 32 && D != 64 && D != 128) throw Error("PagedKVCache: head dim must be 32, 64 or 128");
    if (!P || (P & (P - 1))) throw Error("PagedKVCache: page_size must be a power of two");
    if (capacity > (size_t(1) << 28) || P > (size_t(1) << 16)) throw Error("PagedKVCache: capacity or page_size too large");
    if (options.beams > 32) throw Error("PagedKVCache: at most 32 beams");
    if (options.budget && options.beams > 1) throw Error("PagedKVCache: beams share pages, which a budget would rewrite");
    if (options.budget >= capacity || options.recent > options.budget)
        throw Error("PagedKVCache: need recent <= budget < capacity");
    detail::inf_dt(dtype, "PagedKVCache");
    const size_t per = (capacity + P - 1) / P, R = rows();
    m_pages = R * per + (options.beams > 1 ? R : 0);  // each row's own, and a spare one for reordering
    if (R > 65535 || m_pages > (size_t(1) << 30)) throw Error("PagedKVCache: too many rows or pages");
    m_k = Tensor(dtype, std::vector<size_t>{layers, m_pages, heads, P, D}, "paged_k", device, false);
    m_v = Tensor(dtype, std::vector<size_t>{layers, m_pages, heads, P, D}, "paged_v", device, false);
    std::vector<int32_t> own(R * per), spare(R);
    for (size_t i = 0; i < own.size(); ++i) own[i] = (int32_t)i;
    for (size_t i = 0; i < R; ++i) spare[i] = (int32_t)(R * per + i);
    m_table = Tensor(DType::Int32, own, std::vector<size_t>{R, per}, "paged_table", device);
    m_next_table = Tensor(DType::Int32, own, std::vector<size_t>{R, per}, "paged_table", device);
    m_spare = Tensor(DType::Int32, spare, std::vector<size_t>{R}, "paged_spare", device);
    m_next_spare = Tensor(DType::Int32, spare, std::vector<size_t>{R}, "paged_spare", device);
    m_lens = Tensor::zeros({R}, DType::Int32, device, "paged_lens");
    m_positions_seen = Tensor::zeros({R}, DType::Int32, device, "paged_seen");
    if (options.budget)
        for (size_t l = 0; l < layers; ++l) {
            m_weights.push_back(Tensor::zeros({R, heads, per * P}, DType::Float32, device, "paged_weights"));
            m_positions.push_back(Tensor::zeros({R, heads, per * P}, DType::Int32, device, "paged_positions"));
        }
}

// Grown on demand and reused: all calls are ordered on the device's library stream.
void* PagedKVCache::workspace(size_t bytes) {
    if (!bytes) return nullptr;
    if (!m_ws.defined() || m_ws.size() < bytes + 256)
        m_ws = Tensor(DType::Float32, std::vector<size_t>{bytes / 4 + 128}, "paged_ws", m_k.device(), false);
    const uintptr_t p = reinterpret_cast<uintptr_t>(m_ws.data_ptr());
    return reinterpret_cast<void*>((p + 255) & ~uintptr_t(255));
}

void PagedKVCache::begin(size_t t) {
    if (!t || (m_length && t != 1)) throw Error("PagedKVCache: after the prompt, one position per step");
    if (t > m_capacity) throw Error("PagedKVCache: the prompt is longer than the cache");
    if (m_length + t > m_capacity) {
        if (!m_options.budget) throw Error("PagedKVCache: the cache is full");
        evict();
    }
    detail::DeviceGuard g(m_k.device().index);
    m_step = t;
    fill_int(m_lens, m_length + t);
    if (m_options.budget) fill_int(m_positions_seen, m_seen + t);
}

Tensor PagedKVCache::attend(size_t layer, const Tensor& q, const Tensor& k, const Tensor& v) {
    if (!m_step) throw Error("PagedKVCache: attend() outside begin() and end()");
    if (layer >= m_layers) throw Error("PagedKVCache: no such layer");
    const bool prompt = m_length == 0;
    const std::vector<size_t> want{prompt ? m_groups : rows(), m_heads, m_step, m_dim};
    for (const Tensor* x : {&q, &k, &v}) {
        if (x->shape() != want) throw Error("PagedKVCache: q, k, v must be [rows, H, t, D] of this step");
        if (x->dtype() != m_k.dtype() || x->device() != m_k.device())
            throw Error("PagedKVCache: q, k, v must have the cache's dtype and device");
    }
    NoGradGuard ng;
    detail::DeviceGuard g(m_k.device().index);
    const Handle h(*this, layer, prompt);
    const bool budget = m_options.budget != 0;
    detail::status_check(inf_kv_append(&h.kv, k.data_ptr(), strides4(k), v.data_ptr(), strides4(v), nullptr, (int)m_step,
                                       budget ? floats(m_weights[layer]) : nullptr,
                                       budget ? ints(m_positions[layer]) : nullptr,
                                       budget ? ints(m_positions_seen) : nullptr, detail::stream_of(m_k)),
                         "inf_kv_append");
    if (m_step > 1) return scaled_dot_product_attention(q, k, v, true).contiguous();  // nothing cached before it
    Tensor out(m_k.dtype(), want, "paged_attention", m_k.device(), false);
    const int len = (int)(m_length + 1);
    size_t bytes = 0;
    detail::status_check(inf_attn_decode_paged_workspace(&h.kv, (int)m_heads, len, budget, &bytes),
                         "inf_attn_decode_paged_workspace");
    void* ws = workspace(bytes);
    float* w = budget ? floats(m_weights[layer]) : nullptr;
    detail::status_check(inf_attn_decode_paged(&h.kv, q.data_ptr(), strides4(q), out.data_ptr(), strides4(out),
                                               (int)m_heads, len, 1.0f / std::sqrt((float)m_dim), w, w, ws, bytes,
                                               detail::stream_of(m_k)),
                         "inf_attn_decode_paged");
    return out;
}

void PagedKVCache::end() {
    if (!m_step) throw Error("PagedKVCache: end() without begin()");
    const bool prompt = m_length == 0;
    m_length += m_step;
    m_seen += m_step;
    m_step = 0;
    if (prompt && m_options.beams > 1)
        reorder(Tensor::zeros({m_groups, m_options.beams}, DType::Int32, m_k.device(), "first_beam"));
}

void PagedKVCache::evict() {
    detail::DeviceGuard g(m_k.device().index);
    const int keep = (int)m_options.budget, len = (int)m_length;
    Tensor lens(DType::Int32, std::vector<size_t>{rows()}, "paged_lens", m_k.device(), false);
    fill_int(m_lens, m_length);
    for (size_t l = 0; l < m_layers; ++l) {
        const Handle h(*this, l, false);
        size_t bytes = 0;
        detail::status_check(inf_kv_evict_workspace(&h.kv, keep, len, &bytes), "inf_kv_evict_workspace");
        detail::status_check(inf_kv_evict(&h.kv, floats(m_weights[l]), floats(m_weights[l]), ints(m_positions[l]),
                                          ints(m_positions[l]), ints(lens), keep, (int)m_options.recent, len,
                                          workspace(bytes), bytes, detail::stream_of(m_k)),
                             "inf_kv_evict");
    }
    m_length = m_options.budget;
}

void PagedKVCache::reorder(const Tensor& parents) {
    if (m_step) throw Error("PagedKVCache: reorder() inside a step");
    if (m_options.beams < 2) throw Error("PagedKVCache: a cache without beams has nothing to reorder");
    if (parents.dtype() != DType::Int32 || parents.shape() != std::vector<size_t>{m_groups, m_options.beams} ||
        !parents.is_contiguous() || parents.device() != m_k.device())
        throw Error("PagedKVCache: parents must be dense Int32 [groups, beams] on the cache's device");
    detail::DeviceGuard g(m_k.device().index);
    fill_int(m_lens, m_length);
    const Handle h(*this, 0, false);
    const int64_t layer = (int64_t)m_k.strides()[0];
    detail::status_check(inf_beam_reorder(&h.kv, (int)m_layers, layer, layer, ints(parents), (int)m_options.beams,
                                          ints(m_next_table), (int64_t)m_table.shape()[1], ints(m_spare), ints(m_next_spare),
                                          detail::stream_of(m_k)),
                         "inf_beam_reorder");
    std::swap(m_table, m_next_table);
    std::swap(m_spare, m_next_spare);
}

BeamStep beam_select(const Tensor& logits, const Tensor& scores, const Tensor& finished, int eos) {
    if (logits.device().is_cpu()) throw Error("beam_select: tensors on a HIP device expected");
    if (scores.ndim() != 2 || scores.dtype() != DType::Float32 || !scores.is_contiguous())
        throw Error("beam_select: scores must be dense Float32 [groups, beams]");
    const size_t rows = scores.numel(), nd = logits.ndim();
    if ((nd != 2 && !(nd == 3 && logits.shape()[1] == 1)) || logits.shape()[0] != rows)
        throw Error("beam_select: logits must be [groups * beams, V]");
    const size_t V = logits.shape()[nd - 1];
    if (V > 1 && logits.strides()[nd - 1] != 1) throw Error("beam_select: the last dimension must be dense");
    if (finished.defined()) {
        if (finished.dtype() != DType::Int32 || finished.shape() != scores.shape() || !finished.is_contiguous())
            throw Error("beam_select: finished must be dense Int32 [groups, beams]");
        if (eos < 0) throw Error("beam_select: finished beams need eos");
        detail::same_device(logits, finished, "beam_select");
    }
    detail::same_device(logits, scores, "beam_select");
    const int64_t G = (int64_t)scores.shape()[0], K = (int64_t)scores.shape()[1];
    const Device dev = logits.device();
    BeamStep r;
    r.tokens = Tensor(DType::Int32, scores.shape(), "beam_tokens", dev, false);
    r.parents = Tensor(DType::Int32, scores.shape(), "beam_parents", dev, false);
    r.scores = Tensor(DType::Float32, scores.shape(), "beam_scores", dev, false);
    if (eos >= 0) r.finished = Tensor(DType::Int32, scores.shape(), "beam_finished", dev, false);
    detail::DeviceGuard g(dev.index);
    size_t bytes = 0;
    detail::status_check(inf_beam_select_workspace(G, (int)K, (int64_t)V, &bytes), "inf_beam_select_workspace");
    Tensor ws(DType::Float32, std::vector<size_t>{bytes / 4 + 64}, "beam_ws", dev, false);
    void* p = reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(ws.data_ptr()) + 255) & ~uintptr_t(255));
    const int64_t ld = rows > 1 ? (int64_t)logits.strides()[0] : (int64_t)V;
    detail::status_check(inf_beam_select(logits.data_ptr(), ld, floats(scores), finished.defined() ? ints(finished) : nullptr,
                                         G, (int)K, (int64_t)V, eos, ints(r.tokens), ints(r.parents), floats(r.scores),
                                         r.finished.defined() ? ints(r.finished) : nullptr,
                                         detail::inf_dt(logits.dtype(), "beam_select"), p, bytes,
                                         detail::stream_of(logits)),
                         "inf_beam_select");
    return r;
}

}  // namespace Inferno
