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
    // set by the launch: its first row, rows of a workgroup, reciprocal of a row's units
    int64_t first;
    int rows;
    float recip;
};
int launch_get_rows_q4_0(GetRows p, bool half, hipStream_t s);

constexpr int kMostRot = 256;  // rotated dims of a head
constexpr double kMostFreq = 1.25;  // radians a position: times 2^31 positions, below 3e9
constexpr int64_t kMostRowValues = 1 << 17;  // of a row: what the kernels' divisions by a reciprocal are exact for
constexpr int64_t kMostRowCount = (int64_t)1 << 40;

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
    // of every rotation pair: radians a position, which position (t, h, w, e) turns it
    double freq[kMostRot / 2];
    uint8_t component[kMostRot / 2];
    // set by the launch: its first row, rows of a workgroup, units that its threads rotate in one pass,
    // reciprocals of what they divide by
    int64_t first;
    int rows, pass;
    float recip_half, recip_turned, recip_lanes, recip_copy, recip_rest;
};
int launch_move_rows_q4_0(MoveRows p, hipStream_t s);

}  // namespace sqa
