// paged_merge.hpp - device code that the merges of split partials share: where a row's are.
#pragma once
#include "paged_attn.hpp"

namespace sqa {
namespace paged {

struct Row {
    const float *acc, *ml;  // of the row in its first slot
    int64_t step;           // floats of acc between its splits (ml: step / 128)
    int n;                  // 0: nothing to do
};

// Partials of head h of a token whose entry is w.
__device__ __forceinline__ Row partials(const Call &c, const int4 w, int h) {
    Row r{nullptr, nullptr, 0, 0};
    const int form = w.w & 3, step = w.w >> 2, kvh = group_of(c, h), row = w.z + h - kvh * c.G;
    const int rows = form == kFew ? c.rows_d : c.rows_c;
    const int64_t heads = form == kFew ? 1 : (int64_t)w.y * step, first = w.x + kvh * heads;
    // (arrays that are no plan's may leave here what the workspace held: any four numbers)
    if (form == kDone || form == kWhole || w.x < 0 || step < 1 || w.y < 1 || w.y > 256 || row < 0 || row >= rows ||
        first + (int64_t)(w.y - 1) * step >= (form == kFew ? c.slots_d : c.slots_c))
        return r;
    const int64_t at = first * rows + row;
    r.acc = (form == kFew ? c.acc_d : c.acc_c) + at * 256;
    r.ml = (form == kFew ? c.ml_d : c.ml_c) + at * 2;
    r.step = (int64_t)step * rows * 256;
    r.n = w.y;
    return r;
}

__device__ __forceinline__ const float *gate_row(const Call &c, int t, int h) {
    return reinterpret_cast<const float *>(c.gate + t * c.gate_nb2 + h * c.gate_nb1);
}

}  // namespace paged
}  // namespace sqa
