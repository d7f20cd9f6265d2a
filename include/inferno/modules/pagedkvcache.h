// pagedkvcache.h -- the keys and values of a model's attention layers for generation, in pages, on a HIP
// device: beam search that reorders page numbers instead of caches, and caches of a bounded size.
// No reference counterpart (the reference has no generation loop).
#pragma once

#include <vector>

#include "inferno/core/tensor.h"

namespace Inferno {

// The rows are `groups` x beams sequences of one length.  One model step of t positions is
//     cache.begin(t);  for every layer: y = cache.attend(layer, q, k, v);  cache.end();
// The first step is the prompt of each group, a row per group ([groups, H, t, D]); end() then gives
// every beam the prompt's cache (the full pages are shared).  All later steps have t = 1 and
// rows() rows.  A step that throws in between leaves the positions as begin() found them, or cut them, and the
// attention counted so far.
class PagedKVCache {
public:
    struct Options {
        size_t page_size = 16;  // a power of two
        size_t beams = 1;       // rows of a group
        // With a budget (1 .. capacity - 1), a full cache is cut to that many positions per head, the `recent`
        // newest and those that got the most attention in the single-position steps so far (a prompt of more than one
        // position adds none: a cache that is cut right after it keeps the first slots and the newest).
        // Without one a full cache throws.  Not together with beams, whose rows share pages.
        size_t budget = 0, recent = 0;
    };
    // D: 32, 64 or 128; Float32 or BFloat16.
    PagedKVCache(size_t layers, size_t groups, size_t heads, size_t capacity, size_t D, Device device, DType dtype,
                 Options options);

    size_t rows() const { return m_groups * m_options.beams; }
    size_t capacity() const { return m_capacity; }
    size_t length() const { return m_length; }  // positions held
    size_t seen() const { return m_seen; }      // positions there have been

    void begin(size_t t);
    // q, k, v [rows of the step, H, t, D] (rows' elements adjacent, 4-element aligned, as slices of a [B, t, 3C]
    // projection are): appends k and v to the layer's cache and returns the attention over it, dense.
    Tensor attend(size_t layer, const Tensor& q, const Tensor& k, const Tensor& v);
    void end();

    // Row i of every group becomes a copy of the group's row parents[i]; parents Int32 [groups, beams].
    void reorder(const Tensor& parents);

private:
    struct Handle;
    void* workspace(size_t bytes);
    void evict();
    size_t m_layers, m_groups, m_heads, m_capacity, m_dim, m_pages;
    Options m_options;
    Tensor m_k, m_v;                          // [layers, pages, H, page_size, D]
    Tensor m_table, m_next_table;             // Int32 [rows, pages of a row]
    Tensor m_spare, m_next_spare;             // Int32 [rows]
    Tensor m_lens, m_positions_seen;          // Int32 [rows]
    std::vector<Tensor> m_weights, m_positions;  // per layer [rows, H, capacity], with a budget
    Tensor m_ws;
    size_t m_length = 0, m_seen = 0, m_step = 0;
};

}  // namespace Inferno
