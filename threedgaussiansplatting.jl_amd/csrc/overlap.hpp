// overlap.hpp — whether strided tensors share memory, on the host, before a call writes one while it reads another.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace tdgs {

// `rows` runs of `width` bytes, `step` bytes apart.
struct ByteRows {
    uint64_t at;
    int64_t rows, step, width;
    ByteRows(const void* p, int64_t rows_, int64_t step_, int64_t width_)
        : at((uint64_t)(uintptr_t)p), rows(rows_), step(step_), width(width_) {
        if (rows > 1 && step <= width) {   // one run, or all of them in one place
            width += (rows - 1) * step;
            rows = 1;
        }
        if (rows <= 1) step = width;
    }
    bool empty() const { return rows < 1 || width < 1; }
    uint64_t end() const { return at + (uint64_t)(rows - 1) * (uint64_t)step + (uint64_t)width; }
};

// The least x >= 0 with l <= a x mod m <= r, or -1 without one; 0 <= a < m, 0 <= l <= r < m. Where no multiple of a lies in
// l .. r itself, a x - m y does for some y > 0, that is m y mod a lies in -r .. -l mod a: the same question about smaller
// numbers, as in Euclid's algorithm.
inline __int128 first_in_range(__int128 a, __int128 m, __int128 l, __int128 r) {
    if (l == 0) return 0;
    if (a == 0) return -1;
    const __int128 x = (l + a - 1) / a;
    if (x * a <= r) return x;
    const __int128 y = first_in_range(m % a, a, a - r % a, a - l % a);
    return y < 0 ? -1 : (l + m * y + a - 1) / a;
}

// Whether two sets of rows share a byte; exact, for any strides.
inline bool rows_overlap(const ByteRows& a, const ByteRows& b) {
    if (a.empty() || b.empty() || a.end() <= b.at || b.end() <= a.at) return false;
    if (a.rows == 1 && b.rows == 1) return true;
    if (b.rows == 1) return rows_overlap(b, a);
    // a's rows i0 .. i1 reach into b's span; against rows of b's step without an end on either side, they meet the same rows
    const __int128 first = (__int128)b.at - (__int128)a.at - a.width + 1;       // a row that starts here ends on b's first byte
    const __int128 last = (__int128)b.end() - 1 - (__int128)a.at;
    const __int128 i0 = first <= 0 ? 0 : (first + a.step - 1) / a.step;
    const __int128 i1 = last / a.step < a.rows - 1 ? last / a.step : a.rows - 1;
    if (i0 > i1) return false;
    // row i starts at c + i s of a period of b, moved so that it meets a row where that is at most a.width + b.width - 2
    const __int128 m = b.step, w = (__int128)a.width + b.width - 2;
    if (w >= m) return true;
    __int128 c = ((__int128)a.at + i0 * a.step + a.width - 1 - (__int128)b.at) % m;
    if (c < 0) c += m;
    if (c <= w) return true;
    const __int128 x = first_in_range((__int128)a.step % m, m, m - c, m - c + w);
    return x >= 0 && x <= i1 - i0;
}

// Whether a tensor may be written over one whose elements are each read, for the same place, before that place is written: it
// is that tensor, or shares nothing with it.
inline bool same_or_apart(const ByteRows& w, const ByteRows& r) {
    return (w.at == r.at && w.rows == r.rows && w.step == r.step && w.width == r.width) || !rows_overlap(w, r);
}

// A tensor of up to three strided dimensions of contiguous runs of `width` bytes, strides in bytes: dimensions that go on where the
// one inside ends are taken together, from the smallest stride on.
struct ByteDims {
    uint64_t at;
    int64_t given[3], run;            // the strides as they came (0 of single ones), and the run's bytes
    int64_t count[3], step[3], width;
    int dims = 0;
    bool none = false, nested = true;   // nested: every step reaches past all that is inside, so that no run lies on another
    ByteDims(const void* p, const int64_t (&n)[3], const int64_t (&s)[3], int64_t width_) : at((uint64_t)(uintptr_t)p), run(width_), width(width_) {
        for (int i = 0; i < 3; ++i) {
            if (n[i] < 1) none = true;
            given[i] = n[i] > 1 ? s[i] : 0;
            if (n[i] <= 1) continue;
            int k = dims++;
            for (; k > 0 && step[k - 1] > s[i]; --k) {
                count[k] = count[k - 1];
                step[k] = step[k - 1];
            }
            count[k] = n[i];
            step[k] = s[i];
        }
        int64_t inside = width;
        int k = 0;
        for (int i = 0; i < dims; ++i) {
            if (step[i] < inside) nested = false;
            inside += (count[i] - 1) * step[i];
            if (k == 0 && step[i] <= width) {
                width += (count[i] - 1) * step[i];
            } else if (k > 0 && step[i] == step[k - 1] * count[k - 1]) {
                count[k - 1] *= count[i];
            } else {
                count[k] = count[i];
                step[k++] = step[i];
            }
        }
        dims = k;
    }
    // Of a tensor of the same shape: whether every element of both is in the same place.
    bool same(const ByteDims& o) const {
        return at == o.at && run == o.run && given[0] == o.given[0] && given[1] == o.given[1] && given[2] == o.given[2];
    }
    // Its last dimension's rows; what is inside counts as covered, which it is with one dimension or none.
    ByteRows rows() const {
        int64_t w = width;
        for (int i = 0; i + 1 < dims; ++i) w += (count[i] - 1) * step[i];
        return ByteRows((const void*)(uintptr_t)at, none ? 0 : dims ? count[dims - 1] : 1, dims ? step[dims - 1] : 0, w);
    }
};

// Whether they surely share a byte: told where each is rows of one step, or they start together.
inline bool dims_overlap(const ByteDims& a, const ByteDims& b) {
    if (a.none || b.none || !rows_overlap(a.rows(), b.rows())) return false;
    return (a.dims <= 1 && b.dims <= 1) || a.at == b.at;
}

}  // namespace tdgs
