// overlap.h -- whether two strided views share memory, for the host's checks of results against what is read.
//
// A view is runs of bytes at up to three strides.  Where the larger strides of two views are alike, or one view fits
// between two neighbouring runs of the other, the answer is exact: keys and values that take turns in one buffer,
// columns of one matrix and parts of one page lie apart.  Else the views are taken as one piece each, from
// their first byte to their last.  An overlap is never missed.
#pragma once

#include <algorithm>
#include <cstdint>

namespace inf {

class Memory {
public:
    // A null pointer has no memory.
    Memory(const void* p, int64_t bytes) : Memory(p, 1, 0, 1, 0, 1, 0, bytes) {}
    Memory(const void* p, int64_t rows, int64_t pitch, int64_t run) : Memory(p, rows, pitch, 1, 0, 1, 0, run) {}
    // Strides in bytes, not negative.
    Memory(const void* p, int64_t B, int64_t sb, int64_t H, int64_t sh, int64_t T, int64_t st, int64_t run)
        : dim_{{B, sb}, {H, sh}, {T, st}}, run_(run) {
        if (!p || run <= 0) return;
        at_ = reinterpret_cast<uintptr_t>(p);
        const int64_t bytes = span(span(span(run, dim_[0]), dim_[1]), dim_[2]);
        end_ = at_ + std::min((uintptr_t)bytes, UINTPTR_MAX - at_);
    }

    // The bytes of so many elements, in 64 bits.
    static int64_t bytes(int64_t n, int es) { return std::min(n, kFar / es) * es; }

    bool over(const Memory& o) const {
        if (at_ >= o.end_ || o.at_ >= end_) return false;
        const Runs a(*this), b(o);
        return meet(a, 0, b, 0, (int64_t)(o.at_ - at_));
    }

private:
    struct Dim {
        int64_t n, stride;
    };
    static constexpr int64_t kFar = int64_t(1) << 61;
    // Bytes from the first to the last of `inner` ones at a stride.
    static int64_t span(int64_t inner, const Dim& d) {
        int64_t s = 0;
        return __builtin_mul_overflow(d.n - 1, d.stride, &s) || __builtin_add_overflow(s, inner, &s) ? kFar
                                                                                                     : std::min(s, kFar);
    }

    // A view's dims, the largest stride first.
    struct Runs {
        int n = 0;       // dims with more than one place
        Dim dim[3];
        int64_t span[4];  // of the dims from i on
        explicit Runs(const Memory& m) {
            for (const Dim& d : m.dim_) {
                if (d.n <= 1 || !d.stride) continue;  // what repeats itself is there once
                int i = n++;
                for (; i > 0 && dim[i - 1].stride < d.stride; --i) dim[i] = dim[i - 1];
                dim[i] = d;
            }
            span[n] = m.run_;
            for (int i = n - 1; i >= 0; --i) span[i] = Memory::span(span[i + 1], dim[i]);
        }
    };
    static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }

    // Whether a's dims from i on and b's from j on meet, b's first byte `off` behind a's.
    static bool meet(const Runs& a, int i, const Runs& b, int j, int64_t off) {
        if (off >= a.span[i] || -off >= b.span[j]) return false;
        if (i == a.n && j == b.n) return true;
        const int64_t sa = i < a.n ? a.dim[i].stride : 0, sb = j < b.n ? b.dim[j].stride : 0;
        const int64_t S = std::max(sa, sb);
        // the dims of the larger stride (both, if they are alike): b's index less a's is d, from there on off + d S
        const int ia = i + (sa == S), jb = j + (sb == S);
        const int64_t na = sa == S ? a.dim[i].n : 1, nb = sb == S ? b.dim[j].n : 1;
        if (a.span[ia] > S || b.span[jb] > S) return true;
        const int64_t first = std::max(1 - na, floor_div(-b.span[jb] - off, S) + 1);
        const int64_t last = std::min(nb - 1, floor_div(a.span[ia] - 1 - off, S));
        for (int64_t d = first; d <= last; ++d)  // two at most
            if (meet(a, ia, b, jb, off + d * S)) return true;
        return false;
    }

    uintptr_t at_ = 0, end_ = 0;
    Dim dim_[3];
    int64_t run_;
};

}  // namespace inf
