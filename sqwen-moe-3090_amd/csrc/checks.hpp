// checks.hpp - what the entry points of the paged pool and of cached rows check their
// arguments with.
#pragma once
#include "common.hpp"

namespace sqa {

inline bool dense1(const sqa_tensor *t, int type, int64_t n, int64_t esize) {
    return t->type == type && t->ne[0] == n && t->ne[1] == 1 && t->ne[2] == 1 && t->ne[3] == 1 &&
           (n <= 1 || t->nb[0] == (uint64_t)esize) && (n == 0 || (t->data && (uintptr_t)t->data % esize == 0));
}

// n rows of `len` bytes, `step` bytes apart
struct Rows {
    uintptr_t at;
    uint64_t len, step;
    int64_t n;
    uintptr_t end() const { return at + (uint64_t)(n - 1) * step + len; }
};

inline Rows rows_of(const sqa_tensor *t) {  // ne[1] rows of ne[0] 4-byte values
    return Rows{(uintptr_t)t->data, 4 * (uint64_t)t->ne[0], t->nb[1], t->ne[1]};
}
inline Rows run_of(const sqa_tensor *t, uint64_t bytes) { return Rows{(uintptr_t)t->data, bytes, 0, bytes ? 1 : 0}; }

// Whether two sets of rows share a byte. Rows of one step, such as parts of a wider buffer's
// columns, may lie between each other; of different steps, all that lies between is taken as theirs.
inline bool meet(const Rows &a, const Rows &b) {
    if (a.n < 1 || b.n < 1 || a.end() <= b.at || b.end() <= a.at) return false;
    const uint64_t step = a.n == 1 ? b.step : a.step;
    if ((a.n > 1 && b.n > 1 && a.step != b.step) || (a.n == 1 && b.n == 1) || a.len > step || b.len > step) return true;
    const uint64_t r = b.at >= a.at ? (b.at - a.at) % step : (step - (a.at - b.at) % step) % step;  // b's start in a's row
    return r < a.len || step - r < b.len;
}

inline bool power_of_two(int64_t x) { return x > 0 && (x & (x - 1)) == 0; }

}  // namespace sqa
