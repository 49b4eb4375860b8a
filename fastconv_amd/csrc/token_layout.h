// Whether what a call writes shares anything: rows along some axes, on the host.
#pragma once

struct fc_axis {
    long n, stride;      // entries, and elements from one to the next
};

// Rows of so many elements, n of them a stride apart, share none.
static inline bool fc_apart(long n, long stride, long row) { return n < 2 || stride >= row; }

// The same along up to three axes, in any order.  Where of those with more than one entry each lies at least as far apart as all nearer ones together reach, nothing
// is shared.  Rows that are woven into each other are gone through: two of them that share something differ by some entries of each axis, so that for every
// difference along the shorter axes the nearest one along the longest is looked at; layouts of more than 2^20 such differences are taken for ones that share.
template <int N>
static inline bool fc_apart(const fc_axis (&axes)[N], long row) {
    static_assert(N <= 3);
    fc_axis by[3] = {{1, 0}, {1, 0}, {1, 0}};
    int many = 0;
    for (const fc_axis &a : axes) {
        if (a.n < 2) continue;
        int at = many++;
        for (; at > 0 && by[at - 1].stride > a.stride; at--) by[at] = by[at - 1];
        by[at] = a;
    }
    __int128 reach = row;
    bool nested = true;
    for (int i = 0; i < many; i++) {
        if (by[i].stride < row) return false;
        nested = nested && by[i].stride >= reach;
        reach += (__int128)(by[i].n - 1) * by[i].stride;
    }
    if (nested) return true;
    int longest = 0;
    for (int i = 1; i < 3; i++)
        if (by[i].n > by[longest].n) longest = i;
    const fc_axis l = by[longest], a = by[longest == 0 ? 1 : 0], b = by[longest == 2 ? 1 : 2];
    if ((__int128)a.n * (2 * (__int128)b.n - 1) > (1 << 20)) return false;
    for (long i = 0; i < a.n; i++)
        for (long j = 1 - b.n; j < b.n; j++) {
            const __int128 off = (__int128)i * a.stride + (__int128)j * b.stride;
            const __int128 size = off < 0 ? -off : off, below = size / l.stride;      // entries of the longest axis that lead back, or one more
            for (__int128 k = below; k <= below + 1 && k < l.n; k++) {
                const __int128 left = size - k * l.stride;
                if ((i || j || k) && left < row && -left < row) return false;
            }
        }
    return true;
}
