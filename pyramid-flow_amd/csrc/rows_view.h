// Whether two pf_rows_view tensors share memory, on the host (no HIP in here).
#pragma once
#include <algorithm>
#include "pyflow_hip.h"

struct RowsDim { long long stride, n; };                     // elements; n > 1, stride > 0
// the elements at + sum_i k_i stride_i + [0, chunk), 0 <= k_i < n_i; strides fall
struct RowsSet {
    long long at, chunk;
    RowsDim dim[3];
    int dims;
    long long extent(int from) const {
        long long e = chunk;
        for (int i = from; i < dims; ++i) e += dim[i].stride * (dim[i].n - 1);
        return e;
    }
};

inline RowsSet rows_set(const pf_rows_view& v, int B, int L, int H, int D) {
    RowsSet s;
    s.at = (long long)((unsigned long long)v.p / 2);
    s.chunk = D;
    s.dims = 0;
    const RowsDim all[3] = {{v.batch, B}, {v.row, L}, {v.head, H}};
    for (const RowsDim& d : all)
        if (d.n > 1 && d.stride > 0) s.dim[s.dims++] = d;    // what is repeated (stride 0) is there once
    std::sort(s.dim, s.dim + s.dims, [](const RowsDim& x, const RowsDim& y) { return x.stride > y.stride; });
    return s;
}

// Takes the largest stride off (off both where it is the same: then only the difference of the two indices counts) and looks at the
// pairs whose extents meet: two or three for the layouts there are.  `steps` bounds what odd ones can cost; beyond it: shared.
inline bool rows_meet(const RowsSet& a, int da, long long at_a, const RowsSet& b, int db, long long at_b, int& steps) {
    const long long ea = a.extent(da), eb = b.extent(db);
    if (at_a + ea <= at_b || at_b + eb <= at_a) return false;
    if (da == a.dims && db == b.dims) return true;
    const long long sa = da < a.dims ? a.dim[da].stride : 0, sb = db < b.dims ? b.dim[db].stride : 0;
    if (sa < sb) return rows_meet(b, db, at_b, a, da, at_a, steps);
    const bool both = sa == sb;
    // a's inner set, shifted by k sa, against b (its inner set)
    const int ib = both ? db + 1 : db;
    const long long inner_a = a.extent(da + 1), inner_b = b.extent(ib);
    long long lo = both ? -(b.dim[db].n - 1) : 0, hi = a.dim[da].n - 1;
    // at_a + k sa + inner_a > at_b  and  at_a + k sa < at_b + inner_b
    const long long above = at_b - at_a - inner_a, below = at_b + inner_b - at_a;
    auto floor_div = [](long long x, long long y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
    lo = std::max(lo, floor_div(above, sa) + 1);
    hi = std::min(hi, floor_div(below - 1, sa));
    for (long long k = lo; k <= hi; ++k) {
        if (--steps < 0) return true;
        if (rows_meet(a, da + 1, at_a + k * sa, b, ib, at_b, steps)) return true;
    }
    return false;
}

inline bool rows_share(const pf_rows_view& x, int Bx, int Lx, int Hx, const pf_rows_view& y, int By, int Ly, int Hy, int D) {
    if (!Bx || !Lx || !Hx || !By || !Ly || !Hy) return false;
    const RowsSet a = rows_set(x, Bx, Lx, Hx, D), b = rows_set(y, By, Ly, Hy, D);
    int steps = 4096;
    return rows_meet(a, 0, a.at, b, 0, b.at, steps);
}

// the same elements under the same names
inline bool rows_same(const pf_rows_view& x, const pf_rows_view& y, int B, int L, int H) {
    return x.p == y.p && (B <= 1 || x.batch == y.batch) && (L <= 1 || x.row == y.row) && (H <= 1 || x.head == y.head);
}

// one element under several names: an output that is repeated or folded onto itself
inline bool rows_folded(const pf_rows_view& v, int B, int L, int H, int D) {
    if (!B || !L || !H) return false;
    if ((B > 1 && !v.batch) || (L > 1 && !v.row) || (H > 1 && !v.head)) return true;
    const RowsSet s = rows_set(v, B, L, H, D);
    for (int i = 0; i < s.dims; ++i)
        if (s.dim[i].stride < s.extent(i + 1)) return true;
    return false;
}
