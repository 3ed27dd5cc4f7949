// Whether tensors share memory: plain host arithmetic, so that it can be held against counting without a device.
#pragma once
#include <cstdint>

namespace trn {

// Whether two ranges of memory share nothing.
inline bool apart(const void* x, int64_t nx, const void* y, int64_t ny) {
    const uintptr_t p = (uintptr_t)x, q = (uintptr_t)y;
    return p + (uint64_t)nx <= q || q + (uint64_t)ny <= p;
}
// What a tensor of three strided axes and contiguous rows covers: strides and width in bytes, not negative, no axis empty.
struct Extent {
    const void* p; int64_t n[3], st[3], width;
    int64_t span() const { return (n[0] - 1) * st[0] + (n[1] - 1) * st[1] + (n[2] - 1) * st[2] + width; }
};
// Whether a byte of one lies at distance d from a byte of the other: n steps of the axes forward or m back, each axis wider than all below it.
inline bool reaches(int64_t d, int axes, const int64_t* st, const int64_t* n, const int64_t* m, int64_t w, int64_t v) {
    if (axes == 0) return -v < d && d < w;
    const int64_t s = st[axes - 1], q = d / s - (d % s < 0);
    for (int64_t k = q; k <= q + 1; ++k)
        if (-m[axes - 1] < k && k < n[axes - 1] && reaches(d - k * s, axes - 1, st, n, m, w, v)) return true;
    return false;
}
// Whether two tensors share memory.  Exactly where they have the same strides, each wider than all that lies between its steps (keys and values packed into
// one tensor by head, by token or by sequence); of others that lie within each other it is taken for granted.
inline bool meet(const Extent& x, const Extent& y) {
    if (apart(x.p, x.span(), y.p, y.span())) return false;
    int64_t st[3], n[3], m[3], all = x.width > y.width ? x.width : y.width;
    int axes = 0;
    for (int i = 0; i < 3; ++i) {
        if (x.n[i] == 1 && y.n[i] == 1) continue;
        const int64_t s = x.n[i] == 1 ? y.st[i] : x.st[i];
        if (y.n[i] != 1 && y.st[i] != s) return true;
        int j = axes++;
        for (; j > 0 && st[j - 1] > s; --j) { st[j] = st[j - 1]; n[j] = n[j - 1]; m[j] = m[j - 1]; }
        st[j] = s; n[j] = x.n[i]; m[j] = y.n[i];
    }
    for (int i = 0; i < axes; ++i) {
        if (st[i] < all) return true;
        all += ((n[i] > m[i] ? n[i] : m[i]) - 1) * st[i];
    }
    return reaches((int64_t)((uintptr_t)y.p - (uintptr_t)x.p), axes, st, n, m, x.width, y.width);
}

}  // namespace trn
