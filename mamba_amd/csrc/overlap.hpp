// Whether tensors that a launch writes share elements.  Plain C++, so that the
// checks and a host program share the rule.
#pragma once
#include <algorithm>
#include <cstdint>
#include <utility>
#include <vector>

namespace ss {

// Whether blocks of `size` elements at i * s1 + j * s2 (i below n1, j below n2;
// strides not negative) overlap.
inline bool blocks_overlap(int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t size) {
    if (n1 < 1 || n2 < 1 || size < 1) return false;
    if ((n1 > 1 && s1 < size) || (n2 > 1 && s2 < size)) return true;
    if (n1 == 1 || n2 == 1) return false;
    if (n1 > n2) std::swap(n1, n2), std::swap(s1, s2);
    const auto inside = [&](int64_t n, int64_t s, int64_t of) { return __int128(n - 1) * s + size <= of; };
    if (inside(n1, s1, s2) || inside(n2, s2, s1)) return false;       // one dimension's blocks lie between the other's
    // two blocks lie i s1 - j s2 apart: for each i the j on both sides of zero
    for (int64_t i = 1; i < n1; ++i) {
        const __int128 d = __int128(i) * s1, j = d / s2;
        if (j >= 1 && j < n2 && d - j * s2 < size) return true;
        if (j + 1 < n2 && (j + 1) * s2 - d < size) return true;
    }
    return false;
}

struct Span { uintptr_t from, to; int64_t at; };      // bytes [from, to) of tensor `at`, not empty

// The first output (of `outs`, sorted here) that lies over another one, or over an
// input that is not its own in whole, by its `at`; -1: none.
inline int64_t outputs_clash(const std::vector<Span>& ins, std::vector<Span>& outs) {
    const auto before = [](const Span& a, const Span& b) { return a.from < b.from; };
    if (!std::is_sorted(outs.begin(), outs.end(), before)) std::sort(outs.begin(), outs.end(), before);
    for (size_t i = 1; i < outs.size(); ++i)
        if (outs[i].from < outs[i - 1].to) return outs[i].at;
    for (const Span& in : ins) {
        if (outs.empty() || in.to <= outs.front().from || in.from >= outs.back().to) continue;
        // outputs are apart, so the first that ends past the input's start is the one that may reach into it
        auto o = std::upper_bound(outs.begin(), outs.end(), in.from, [](uintptr_t v, const Span& s) { return v < s.to; });
        for (; o != outs.end() && o->from < in.to; ++o)
            if (o->at != in.at || o->from != in.from || o->to != in.to) return o->at;
    }
    return -1;
}

}  // namespace ss
