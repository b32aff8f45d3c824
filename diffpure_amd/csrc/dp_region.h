// What an argument covers in memory, and whether two arguments share a byte (host checks of the C entry points).
#pragma once
#include <stdint.h>

namespace dp {

// up to three axes of n places, s >= 0 bytes apart, of `row` bytes each; an axis of one place has no stride.  An argument that was not given: row 0.
struct Region {
    const char* name;
    intptr_t p;
    long long n[3], s[3], row;
    typedef __int128 Wide;              // (2^30 places 2^42 bytes apart)
    Wide end() const {
        Wide e = row;
        for (int i = 0; i < 3; ++i)
            if (n[i] > 1) e += (Wide)(n[i] - 1) * s[i];
        return e;
    }
    // all bytes lie within this many of the first, modulo m
    Wide within(long long m) const {
        Wide e = row;
        for (int i = 0; i < 3; ++i)
            if (n[i] > 1 && s[i] % m != 0) e += (Wide)(n[i] - 1) * s[i];
        return e;
    }
    // no two of its rows share a byte (for axes that nest, as those of any view of a dense tensor do)
    bool distinct() const {
        bool done[3] = {n[0] <= 1, n[1] <= 1, n[2] <= 1};
        Wide need = row;
        for (;;) {
            int at = -1;
            for (int i = 0; i < 3; ++i)
                if (!done[i] && (at < 0 || s[i] < s[at])) at = i;
            if (at < 0) return true;
            if (s[at] < need) return false;
            need += (Wide)(n[at] - 1) * s[at];
            done[at] = true;
        }
    }
};
inline Region flat(const char* name, const void* p, long long bytes) { return Region{name, (intptr_t)p, {1, 1, 1}, {0, 0, 0}, p ? bytes : 0}; }

// Whether a and b, b beginning `at` bytes behind a, may share a byte: by their largest stride first - of all pairs of places along it, the few whose remainders reach each other
// are looked at in turn (more than 8 are taken for a meeting: strides that do not nest).
inline bool meet(Region a, Region b, Region::Wide at) {
    if (at >= a.end() || -at >= b.end()) return false;
    long long m = 0;
    for (const Region* r : {&a, &b})
        for (int i = 0; i < 3; ++i)
            if (r->n[i] > 1 && r->s[i] > m) m = r->s[i];
    if (m == 0) return true;
    Region::Wide lo = 0, hi = 0;                          // b's place less a's
    for (int i = 0; i < 3; ++i) {
        if (a.n[i] > 1 && a.s[i] == m) { lo -= a.n[i] - 1; a.n[i] = 1; }
        if (b.n[i] > 1 && b.s[i] == m) { hi += b.n[i] - 1; b.n[i] = 1; }
    }
    const Region::Wide first = -(at + b.end()) / m - 1, last = (a.end() - at) / m + 1;
    if (first > lo) lo = first;
    if (last < hi) hi = last;
    int pairs = 0;
    for (Region::Wide k = lo; k <= hi; ++k) {
        const Region::Wide to = at + k * m;
        if (to >= a.end() || -to >= b.end()) continue;
        if (++pairs > 8 || meet(a, b, to)) return true;
    }
    return false;
}
// apart as wholes, or as different columns of rows at one pitch (views of one tensor: heads side by side, q | k | v of a head, a part of a wider row), or place by place
inline bool apart(const Region& a, const Region& b) {
    if (a.row == 0 || b.row == 0) return true;
    const Region::Wide at = (Region::Wide)b.p - a.p;
    if (at >= a.end() || -at >= b.end()) return true;
    for (const Region* r : {&a, &b})
        for (int i = 0; i < 3; ++i) {
            const long long m = r->s[i];
            if (r->n[i] <= 1 || m <= 0) continue;
            const Region::Wide col = (at % m + m) % m;
            if (col >= a.within(m) && col + b.within(m) <= m) return true;
        }
    return !meet(a, b, at);
}

// every written argument against the read ones and the other written ones: 0, or 1 with a message
inline int check_apart(const char* fn, const Region* w, int nw, const Region* r, int nr) {
    for (int i = 0; i < nw; ++i)
        for (int j = 0; j < nr; ++j)
            if (!apart(w[i], r[j])) {
                dp_set_error("%s: %s overlaps %s", fn, w[i].name, r[j].name);
                return 1;
            }
    for (int i = 0; i < nw; ++i) {
        if (w[i].row && !w[i].distinct()) {
            dp_set_error("%s: the rows of %s overlap", fn, w[i].name);
            return 1;
        }
        for (int j = 0; j < i; ++j)
            if (!apart(w[i], w[j])) {
                dp_set_error(w[i].p == w[j].p ? "%s: %s and %s begin at one address" : "%s: %s overlaps %s", fn, w[j].name, w[i].name);
                return 1;
            }
    }
    return 0;
}

}  // namespace dp
