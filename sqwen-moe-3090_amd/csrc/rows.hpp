// rows.hpp - what the kernels over cached rows share with their entry points.
#pragma once
#include "common.hpp"

namespace sqa {

// Rows of a q4_0 cache read back: dst[i] = row idx[i] of src.
struct GetRows {
    const uint8_t *src;
    int64_t src_nb1, src_rows;
    const char *idx;
    int64_t idx_nb0;
    char *dst;
    int64_t dst_nb1;
    int64_t n;    // rows
    int blocks;   // q4_0 blocks of a row
};
int launch_get_rows_q4_0(const GetRows &p, bool half, hipStream_t s);

constexpr int kMostRot = 256;  // rotated dims of a head

// Rows moved: dst[to[i]] = src[from[i]], the first n_rot dims of every head rotated.
struct MoveRows {
    const uint8_t *src;
    uint8_t *dst;
    int64_t src_nb1, dst_nb1, src_rows, dst_rows;
    const char *from, *to;
    int64_t from_nb0, to_nb0;
    const int32_t *delta;  // [4 * n] or null (n_rot 0)
    int64_t n;
    int heads, head_dim;
    int n_rot;             // 0: rows are copied
    int sections[4], sect; // sect: the sections' sum
    double freq[kMostRot / 2];  // radians a position, of every rotation pair
};
int launch_move_rows_q4_0(const MoveRows &p, hipStream_t s);

}  // namespace sqa
