// overlap.h -- whether two strided views share memory, for the host's checks of results against what is read.
//
// A view is runs of bytes at up to three strides.  Where the larger strides of two views are alike, or one view fits
// between two neighbouring runs of the other, the answer is exact: keys and values that take turns in one buffer,
// columns of one matrix and parts of one page lie apart.  Else the views are taken as one piece each, from
// their first byte to their last.  An overlap is never missed.
#pragma once

#include <algorithm>
#include <cstdint>
#include <initializer_list>

namespace inf {

class Memory {
public:
    Memory() = default;
    Memory(const void* p, int64_t bytes) : Memory(p, 1, 0, 1, 0, 1, 0, bytes) {}
    Memory(const void* p, int64_t rows, int64_t pitch, int64_t run) : Memory(p, rows, pitch, 1, 0, 1, 0, run) {}
    // Strides in bytes, not negative.
    Memory(const void* p, int64_t B, int64_t sb, int64_t H, int64_t sh, int64_t T, int64_t st, int64_t run)
        : at_(reinterpret_cast<uintptr_t>(p)), run_(run) {
        for (const Dim& x : {Dim{B, sb}, Dim{H, sh}, Dim{T, st}})
            if (x.n > 1 && x.stride) dim_[n_++] = x;  // what repeats itself is there once
        std::sort(dim_, dim_ + n_, [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
        span_[n_] = run;
        for (int i = n_ - 1; i >= 0; --i) {
            int64_t s = 0;
            span_[i] = __builtin_mul_overflow(dim_[i].n - 1, dim_[i].stride, &s) ||
                               __builtin_add_overflow(s, span_[i + 1], &s) || s > kFar
                           ? kFar
                           : s;
        }
    }

    // The bytes of so many elements, in 64 bits.
    static int64_t bytes(int64_t n, int es) { return std::min(n, kFar / es) * es; }

    // A null pointer has no memory.
    bool over(const Memory& o) const {
        if (!at_ || !o.at_ || run_ <= 0 || o.run_ <= 0) return false;
        return at_ <= o.at_ ? meet(*this, 0, o, 0, distance(at_, o.at_)) : meet(o, 0, *this, 0, distance(o.at_, at_));
    }

private:
    struct Dim {
        int64_t n, stride;
    };
    static int64_t distance(uintptr_t a, uintptr_t b) { return b - a > (uintptr_t)kFar ? kFar : (int64_t)(b - a); }
    static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }

    // Whether a's dims from i on and b's from j on meet, b's first byte `off` behind a's.
    static bool meet(const Memory& a, int i, const Memory& b, int j, int64_t off) {
        if (off >= a.span_[i] || -off >= b.span_[j]) return false;
        if (i == a.n_ && j == b.n_) return true;
        const int64_t sa = i < a.n_ ? a.dim_[i].stride : 0, sb = j < b.n_ ? b.dim_[j].stride : 0;
        const int64_t S = std::max(sa, sb);
        // the dims of the larger stride (both, if they are alike): b's index less a's is d, from there on off + d S
        const int ia = i + (sa == S), jb = j + (sb == S);
        const int64_t na = sa == S ? a.dim_[i].n : 1, nb = sb == S ? b.dim_[j].n : 1;
        if (a.span_[ia] > S || b.span_[jb] > S) return true;
        const int64_t first = std::max(1 - na, floor_div(-b.span_[jb] - off, S) + 1);
        const int64_t last = std::min(nb - 1, floor_div(a.span_[ia] - 1 - off, S));
        for (int64_t d = first; d <= last; ++d)  // two at most
            if (meet(a, ia, b, jb, off + d * S)) return true;
        return false;
    }

    static constexpr int64_t kFar = int64_t(1) << 61;
    uintptr_t at_ = 0;
    int64_t run_ = 0;
    int n_ = 0;      // dims with more than one place
    Dim dim_[3];     // the largest stride first
    int64_t span_[4] = {};  // bytes from the first to the last of the dims from i on
};

}  // namespace inf
