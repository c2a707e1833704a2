// g4q_overlap.h -- whether the strided tensors of a call share elements: host arithmetic on addresses and strides.
#pragma once

#include <algorithm>
#include <cstdint>

#include "g4q.h"

namespace g4q {

// Rows of d contiguous elements on up to three axes, the longest stride first (axes of one row are left out).
struct Lattice {
    using Wide = __int128;           // a caller's strides times counts may pass 64 bits
    int64_t stride[3], count[3], d;
    int axes = 0;

    void add(int64_t s, int64_t n) {
        if (n <= 1) return;
        int i = axes++;
        for (; i > 0 && stride[i - 1] < s; --i) stride[i] = stride[i - 1], count[i] = count[i - 1];
        stride[i] = s, count[i] = n;
    }

    // From the first row's first element to the last one's end, of the axes from `axis` on.
    Wide span(int axis = 0) const {
        Wide e = d;
        for (; axis < axes; ++axis) e += (Wide)stride[axis] * (count[axis] - 1);
        return e;
    }

    // No step of an axis is shorter than what lies inside of it, so no two rows share an element.
    bool nested() const {
        for (int i = 0; i < axes; ++i)
            if (stride[i] < span(i + 1)) return false;
        return true;
    }

    // Whether the same lattice, its first row `gap` elements on, shares an element with this one. Where the axes are nested
    // this is exact: the steps i between a row of each leave |gap - sum(i stride)| < d, and an axis has at most three
    // candidates for its i. Else lattices whose spans overlap are taken to share some.
    bool meets_shifted(Wide gap) const {
        if (gap >= span() || -gap >= span()) return false;
        return !nested() || differ_by(gap, 0);
    }

    // Whether d elements from `gap` elements behind the first row's first one on lie in some row too; exact likewise.
    bool meets_row(Wide gap) const {
        if (gap >= span() || -gap >= d) return false;
        return !nested() || holds(gap, 0);
    }

private:
    static Wide floor_div(Wide a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }

    bool differ_by(Wide gap, int axis) const {
        if (axis == axes) return gap < d && -gap < d;
        const int64_t s = stride[axis];
        const Wide reach = span(axis + 1), most = count[axis] - 1;   // |gap - i s| < reach
        Wide lo = -floor_div(reach - 1 - gap, s), hi = floor_div(gap + reach - 1, s);
        if (lo < -most) lo = -most;
        if (hi > most) hi = most;
        for (Wide i = lo; i <= hi; ++i)
            if (differ_by(gap - i * s, axis + 1)) return true;
        return false;
    }

    bool holds(Wide gap, int axis) const {
        if (axis == axes) return gap < d && -gap < d;
        const int64_t s = stride[axis];
        Wide lo = -floor_div(span(axis + 1) - 1 - gap, s), hi = floor_div(gap + d - 1, s);   // -d < gap - i s < the inner span
        if (lo < 0) lo = 0;
        if (hi > count[axis] - 1) hi = count[axis] - 1;
        for (Wide i = lo; i <= hi; ++i)
            if (holds(gap - i * s, axis + 1)) return true;
        return false;
    }
};

// M tokens of head rows.
inline Lattice rows_lattice(const G4qHeadRows& r, int64_t M, int64_t d) {
    Lattice l;
    l.d = d;
    l.add(r.token_stride, M);
    l.add(r.head_stride, r.n_heads);
    return l;
}

// Whether no two of the rows share an element. Tokens and heads that interleave without sharing one qualify: of the steps
// of the longer stride only those within the other axis' reach matter, which are no more than it has rows.
inline bool rows_apart(const G4qHeadRows& r, int64_t M, int64_t d) {
    const Lattice l = rows_lattice(r, M, d);
    if (l.nested()) return true;
    if (l.stride[l.axes - 1] < d) return false;
    const int64_t s = l.stride[1];                   // two axes, or the last would have been nested
    for (int64_t i = 1; i < l.count[0] && (Lattice::Wide)i * l.stride[0] < l.span(1); ++i) {
        const int64_t rest = (int64_t)((Lattice::Wide)i * l.stride[0] % s);
        const bool next = (Lattice::Wide)i * l.stride[0] - rest < (Lattice::Wide)s * (l.count[1] - 1);
        if (rest < d || (next && s - rest < d)) return false;
    }
    return true;
}

// Whether two tensors of M tokens of head rows may share elements, from the strides alone. Where these are alike (views of one
// buffer) the places of the rows tell, else tensors whose spans overlap may.
inline bool rows_may_meet(const G4qHeadRows& a, const G4qHeadRows& b, int64_t M, int64_t d) {
    struct Axes {
        int64_t outer, inner, span, inner_span;      // strides of the two axes, and extents in elements
    };
    auto axes = [&](const G4qHeadRows& t) {
        const int64_t ts = M > 1 ? t.token_stride : 0, hs = t.n_heads > 1 ? t.head_stride : 0;
        const bool tokens_out = ts >= hs;
        Axes x;
        x.outer = std::max(ts, hs), x.inner = std::min(ts, hs);
        x.inner_span = x.inner * ((tokens_out ? t.n_heads : M) - 1) + d;
        x.span = x.outer * ((tokens_out ? M : t.n_heads) - 1) + x.inner_span;
        return x;
    };
    const Axes x = axes(a), y = axes(b);
    const int64_t gap = b.data - a.data;             // both are 16-byte aligned
    if (gap >= x.span || -gap >= y.span) return false;
    if (x.outer != y.outer || x.outer < std::max(x.inner_span, y.inner_span)) return true;
    auto inner_meet = [&](int64_t g) {               // one row of each, b's g elements on
        if (g >= x.inner_span || -g >= y.inner_span) return false;
        if (x.inner != y.inner || x.inner < d) return true;
        const int64_t r = ((g % x.inner) + x.inner) % x.inner;
        return r < d || x.inner - r < d;
    };
    if (x.outer == 0) return inner_meet(gap);
    const int64_t r = ((gap % x.outer) + x.outer) % x.outer;
    return inner_meet(r) || inner_meet(r - x.outer);
}

// Whether they do: where they may, the rows are looked at one by one before a call is refused. Exact unless both tensors have
// rows that interleave.
inline bool rows_meet(const G4qHeadRows& a, const G4qHeadRows& b, int64_t M, int64_t d) {
    if (!rows_may_meet(a, b, M, d)) return false;
    const Lattice la = rows_lattice(a, M, d), lb = rows_lattice(b, M, d);
    if (!la.nested() && !lb.nested()) return true;
    const G4qHeadRows &walk = lb.nested() ? a : b, &at = lb.nested() ? b : a;
    const Lattice& l = lb.nested() ? lb : la;
    const int64_t tokens = walk.token_stride == 0 ? 1 : M;
    for (int64_t t = 0; t < tokens; ++t)
        for (int64_t h = 0; h < walk.n_heads; ++h)
            if (l.meets_row(walk.data - at.data + (Lattice::Wide)t * walk.token_stride + (Lattice::Wide)h * walk.head_stride)) return true;
    return false;
}

// The slots of a cache's k (or v), one row a head.
inline Lattice cache_lattice(const G4qPagedCache& c) {
    Lattice l;
    l.d = c.head_dim;
    l.add(c.page_stride, c.n_pages);
    l.add(c.head_stride, c.n_kv_heads);
    l.add(c.slot_stride, c.page_size);
    return l;
}

// What an append to the cache would write from several warps at once; null where every slot of k and v is its own.
inline const char* shared_slots(const G4qPagedCache& c) {
    const Lattice l = cache_lattice(c);
    if (!l.nested()) return "cache: pages, heads and slots must not overlap";
    if (l.meets_shifted(c.v - c.k)) return "cache: k and v share elements";
    return nullptr;
}

// Whether M tokens of head rows share elements with the cache's slots. Only rows between the ends of k or v are looked at one
// by one: those of a buffer that holds both.
inline bool meets_cache(const G4qHeadRows& r, int64_t M, const G4qPagedCache& c, const Lattice& l) {
    const Lattice::Wide last = (Lattice::Wide)r.token_stride * (M - 1) + (Lattice::Wide)r.head_stride * (r.n_heads - 1);
    for (const uint16_t* base : {c.k, c.v}) {
        const Lattice::Wide gap = r.data - base;
        if (gap >= l.span() || gap + last + l.d <= 0) continue;
        if (!l.nested()) return true;
        const int64_t tokens = r.token_stride == 0 ? 1 : M, heads = r.n_heads;
        for (int64_t t = 0; t < tokens; ++t)
            for (int64_t h = 0; h < heads; ++h)
                if (l.meets_row(gap + (Lattice::Wide)t * r.token_stride + (Lattice::Wide)h * r.head_stride)) return true;
    }
    return false;
}

}  // namespace g4q
