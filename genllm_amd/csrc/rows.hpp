// rows.hpp -- which operands of a call share memory.  Host code.
//
// Operands are rows of bytes at up to three strides.  Views of one buffer meet in
// their address ranges without sharing a byte (q, k and v of a fused projection),
// so ranges alone do not answer it: two sets of rows, a at i0 s0 + i1 s1 + .., share
// memory where the difference of two rows' addresses lies between the rows' lengths.
#pragma once

#include <algorithm>
#include <cstdint>

namespace genllm {

struct Rows {
    const char* p = nullptr;  // null: no operand
    int64_t n[3] = {1, 1, 1}, stride[3] = {0, 0, 0};  // bytes
    int64_t bytes = 0;                                // of a row

    static Rows whole(const void* p, int64_t bytes) {
        Rows r;
        r.p = static_cast<const char*>(p), r.bytes = bytes;
        return r;
    }
    bool empty() const { return !p || bytes <= 0 || n[0] <= 0 || n[1] <= 0 || n[2] <= 0; }
    bool same_as(const Rows& o) const {
        return p == o.p && bytes == o.bytes && std::equal(n, n + 3, o.n) && std::equal(stride, stride + 3, o.stride);
    }
};

class RowSearch {
    using wide = __int128;
    struct Axis {
        wide s;      // > 0
        wide lo, hi; // of its factor
    };
    Axis axis_[6];
    int n_ = 0, nodes_ = 0;
    wide below_ = 0, above_ = 0;     // hits: -below < sum < above
    wide rest_lo_[7], rest_hi_[7];   // reach of the axes from i on
    bool skip_zero_ = false;

    void add(wide s, wide lo, wide hi) {
        if (s == 0 || lo == hi) return;  // no axis has a factor other than 0 alone
        if (s < 0) {
            s = -s;
            std::swap(lo, hi);
            lo = -lo, hi = -hi;
        }
        for (int i = 0; i < n_; ++i)
            if (axis_[i].s == s) {
                axis_[i].lo += lo, axis_[i].hi += hi;
                return;
            }
        axis_[n_++] = {s, lo, hi};
    }
    static wide floor_div(wide a, wide b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }

    bool visit(int i, wide sum, bool zero) {
        // strides without any order could make this long: then the answer is yes
        if (++nodes_ > 20000) return true;
        if (i == n_) return sum > -below_ && sum < above_ && !(zero && skip_zero_);
        const Axis& a = axis_[i];
        const wide first = std::max(a.lo, floor_div(-below_ - sum - rest_hi_[i + 1], a.s) + 1);
        const wide last = std::min(a.hi, -floor_div(-(above_ - sum - rest_lo_[i + 1]), a.s) - 1);
        for (wide c = first; c <= last; ++c)
            if (visit(i + 1, sum + c * a.s, zero && c == 0)) return true;
        return false;
    }
    bool run(wide start) {
        std::sort(axis_, axis_ + n_, [](const Axis& x, const Axis& y) { return x.s > y.s; });
        rest_lo_[n_] = rest_hi_[n_] = 0;
        for (int i = n_; i-- > 0;) {
            rest_lo_[i] = rest_lo_[i + 1] + axis_[i].lo * axis_[i].s;
            rest_hi_[i] = rest_hi_[i + 1] + axis_[i].hi * axis_[i].s;
        }
        if (start + rest_hi_[0] <= -below_ || start + rest_lo_[0] >= above_) return false;
        return visit(0, start, true);
    }

    // each stride clears all that the smaller ones reach: the usual tensors
    static bool nested(const Rows& a) {
        int d[3] = {0, 1, 2};
        const auto size = [&](int i) { return a.n[i] > 1 ? (a.stride[i] < 0 ? -wide(a.stride[i]) : wide(a.stride[i])) : 0; };
        if (size(d[0]) > size(d[1])) std::swap(d[0], d[1]);
        if (size(d[1]) > size(d[2])) std::swap(d[1], d[2]);
        if (size(d[0]) > size(d[1])) std::swap(d[0], d[1]);
        wide reach = a.bytes;
        for (int i : d) {
            if (a.n[i] < 2) continue;
            if (size(i) < reach) return false;
            reach += (a.n[i] - 1) * size(i);
        }
        return true;
    }

  public:
    // a row of a and a row of b have a byte in common
    bool shared(const Rows& a, const Rows& b) {
        if (a.empty() || b.empty()) return false;
        for (int d = 0; d < 3; ++d) add(a.stride[d], 0, a.n[d] - 1);
        for (int d = 0; d < 3; ++d) add(b.stride[d], -(b.n[d] - 1), 0);
        below_ = a.bytes, above_ = b.bytes;
        return run(wide(reinterpret_cast<uintptr_t>(a.p)) - wide(reinterpret_cast<uintptr_t>(b.p)));
    }
    // two different rows of a have
    bool shared_within(const Rows& a) {
        if (a.empty() || nested(a)) return false;
        for (int d = 0; d < 3; ++d) {
            if (a.n[d] > 1 && a.stride[d] == 0) return true;
            for (int e = 0; e < d; ++e)
                if (a.n[d] > 1 && a.n[e] > 1 && (a.stride[d] == a.stride[e] || a.stride[d] == -a.stride[e])) return true;
            add(a.stride[d], -(a.n[d] - 1), a.n[d] - 1);
        }
        below_ = above_ = a.bytes;
        skip_zero_ = true;
        return run(0);
    }
};

inline bool rows_shared(const Rows& a, const Rows& b) { return RowSearch().shared(a, b); }
inline bool rows_shared_within(const Rows& a) { return RowSearch().shared_within(a); }

struct NamedRows {
    const char* name;
    Rows rows;
    int64_t first = INT64_MAX, end = INT64_MIN;  // of the addresses; INT64_MAX, INT64_MIN: none, the reverse: any

    NamedRows(const char* name_, const Rows& r) : name(name_), rows(r) {
        if (r.empty()) return;
        const int64_t at = int64_t(reinterpret_cast<uintptr_t>(r.p));
        first = at;
        bool far = __builtin_add_overflow(at, r.bytes, &end);
        for (int d = 0; d < 3; ++d) {
            int64_t by;
            far |= __builtin_mul_overflow(r.n[d] - 1, r.stride[d], &by);
            far |= by < 0 ? __builtin_add_overflow(first, by, &first) : __builtin_add_overflow(end, by, &end);
        }
        if (far) first = INT64_MIN, end = INT64_MAX;
    }
    bool near(const NamedRows& o) const { return first < o.end && o.first < end; }
};

// The first pair of operands that share memory, `written` against all before them
// and against `read`, as "NAME overlaps NAME"; null where there is none.
// allowed(w, r): a pair that may.
template <int W, int R, typename F>
inline bool find_overlap(const NamedRows (&written)[W], const NamedRows (&read)[R], const F& allowed, const char*& a, const char*& b) {
    for (int i = 0; i < W; ++i) {
        a = written[i].name;
        for (int j = 0; j < i; ++j)
            if (b = written[j].name; written[i].near(written[j]) && rows_shared(written[i].rows, written[j].rows)) return true;
        for (int j = 0; j < R; ++j)
            if (b = read[j].name; written[i].near(read[j]) && !allowed(written[i].rows, read[j].rows) &&
                                  rows_shared(written[i].rows, read[j].rows))
                return true;
    }
    return false;
}

}  // namespace genllm
