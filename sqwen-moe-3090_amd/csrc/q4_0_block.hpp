// q4_0_block.hpp - ggml's quantize_row_q4_0_ref for one 32-value block held by
// 8 consecutive lanes (4 consecutive values each), bit for bit:
//   max  = value of largest |x| in the block, first occurrence on ties
//   d    = max / -8            (stored as fp16, round-to-nearest-even)
//   id   = d != 0 ? 1/d : 0    (correctly rounded fp32 division)
//   code = min(15, (int8_t)(x*id + 8.5f)) with the multiply and the add each
//          rounded on their own (contraction off: no fused multiply-add)
// An all-zero block therefore stores d = -0.0 (fp16 0x8000) and codes 8.
#pragma once
#include "common.hpp"

namespace sqa {

// x of another lane of the 8: quad permutes, row_half_mirror, row_shl:4.
template <int kCtrl, typename T>
__device__ __forceinline__ T dpp8(T x) {
    int i;
    __builtin_memcpy(&i, &x, 4);
    i = __builtin_amdgcn_update_dpp(i, i, kCtrl, 0xf, 0xf, false);
    __builtin_memcpy(&x, &i, 4);
    return x;
}

// v: this lane's 4 values (block elements 4t..4t+3, t = lane & 7); blk: the
// 18-byte block. All 8 lanes of the group must call it together.
__device__ __forceinline__ void quantize_q4_0_block8(const float v[4], int t, uint8_t *blk) {
    // x*id + 8.5f as two roundings: with contraction on (hipcc's default, and
    // inside HIP's __fmul_rn / __fadd_rn, which are plain * and +) it became one
    // fma (v_fmaak_f32), and a value whose x*id lies within half an ulp below a
    // half-integer then truncated to the code below ggml's
#pragma clang fp contract(off)
    // The largest |x| of the 8 lanes (a NaN counts as none), then the first element that has it and its
    // sign as one number, by DPP within 8 lanes: neighbours, neighbouring pairs, the mirrored half.
    float top = fmaxf(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fabsf(v[2])), fabsf(v[3]));
    top = fmaxf(top, 0.0f);
    top = fmaxf(top, dpp8<0xB1>(top));
    top = fmaxf(top, dpp8<0x4E>(top));
    top = fmaxf(top, dpp8<0x141>(top));
    uint32_t first = 64;
#pragma unroll
    for (int j = 3; j >= 0; --j)
        first = fabsf(v[j]) == top ? (uint32_t)(8 * t + 2 * j) | __float_as_uint(v[j]) >> 31 : first;
    first = min(first, dpp8<0xB1>(first));
    first = min(first, dpp8<0x4E>(first));
    first = min(first, dpp8<0x141>(first));
    const float mx = top == 0.0f ? 0.0f : first & 1 ? -top : top;

    const float d = mx / -8.0f;
    const float id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float y = v[j] * id + 8.5f;
        int c = (int)y;  // truncation toward zero, y in [0.5, 16.5] for finite input
        c = c < 15 ? c : 15;
        word |= (uint32_t)(c & 0xff) << (8 * j);
    }
    // qs[j] = code[j] | code[j+16] << 4: lanes 0..3 take the high nibbles from lanes 4..7.
    const uint32_t hi = dpp8<0x104>(word);
    if (t < 4) {
        const uint32_t qs = word | (hi << 4);
        uint16_t *p = reinterpret_cast<uint16_t *>(blk + 2 + 4 * t);
        p[0] = (uint16_t)(qs & 0xffff);
        p[1] = (uint16_t)(qs >> 16);
    } else if (t == 4) {
        const _Float16 dh = (_Float16)d;
        *reinterpret_cast<_Float16 *>(blk) = dh;
    }
}

}  // namespace sqa
