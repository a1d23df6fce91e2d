// rows_q4_0.hip - cached q4_0 rows read back (get_rows) and moved (move_rows), the
// counterparts of set_rows_q4_0.hip.
#include <math.h>

#include "q4_0_block.hpp"
#include "rows.hpp"

namespace sqa {
namespace {

constexpr int kThreads = 256;

// dst[i] = (code - 8) d of row idx[i]: 8 lanes a block, 4 values a lane.
template <bool kHalf>
__global__ __launch_bounds__(kThreads) void get_rows_q4_0_kernel(GetRows p) {
    const int64_t gid = (int64_t)blockIdx.x * kThreads + threadIdx.x, blk = gid >> 3;
    const int t = threadIdx.x & 7;
    if (blk >= p.n * p.blocks) return;
    const int64_t i = blk / p.blocks, b = blk - i * p.blocks;
    const int64_t r = *reinterpret_cast<const int64_t *>(p.idx + i * p.idx_nb0);
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (r >= 0 && r < p.src_rows) {
        const uint8_t *from = p.src + r * p.src_nb1 + b * SQA_Q4_0_BLOCK_BYTES;
        const float d = (float)*reinterpret_cast<const _Float16 *>(from);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)((from[2 + 4 * (t & 3) + j] >> (t < 4 ? 0 : 4) & 15) - 8) * d;
    }
    const int64_t at = b * SQA_QK4_0 + 4 * t;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (kHalf) reinterpret_cast<_Float16 *>(p.dst + i * p.dst_nb1)[at + j] = (_Float16)v[j];
        else reinterpret_cast<float *>(p.dst + i * p.dst_nb1)[at + j] = v[j];
    }
}

// One workgroup a token: the (cos, sin) of its rotation pairs, then the rotated blocks
// (8 lanes each, requantised), then the others' bytes.
__global__ __launch_bounds__(kThreads) void move_rows_q4_0_kernel(MoveRows p) {
#pragma clang fp contract(off)
    __shared__ float2 cs[128];
    const int tid = threadIdx.x;
    const int64_t i = blockIdx.x;
    const int64_t r = *reinterpret_cast<const int64_t *>(p.from + i * p.from_nb0);
    const int64_t w = *reinterpret_cast<const int64_t *>(p.to + i * p.to_nb0);
    if (r < 0 || r >= p.src_rows || w < 0 || w >= p.dst_rows) return;
    const int half = p.n_rot >> 1;
    if (tid < half) {
        const int sector = tid % p.sect;
        const int c = sector % 3 == 1 && sector < 3 * p.sections[1]   ? 1
                      : sector % 3 == 2 && sector < 3 * p.sections[2] ? 2
                      : sector % 3 == 0 && sector < 3 * p.sections[0] ? 0
                                                                      : 3;
        double sn, co;
        sincos((double)p.delta[i + c * p.n] * p.freq[tid], &sn, &co);
        cs[tid] = make_float2((float)co, (float)sn);
    }
    __syncthreads();
    const uint8_t *src = p.src + r * p.src_nb1;
    uint8_t *dst = p.dst + w * p.dst_nb1;
    const int turned = (p.n_rot + 31) / 32, blocks = p.head_dim / 32, lanes = 8 * turned;
    for (int l0 = 0; l0 < p.heads * lanes; l0 += kThreads) {
        const int l = l0 + tid, h = l / lanes, d0 = 4 * (l - h * lanes);
        const bool ok = h < p.heads;
        float out[4] = {};
        const uint8_t *head = src + (int64_t)(ok ? h : 0) * blocks * SQA_Q4_0_BLOCK_BYTES;
        auto value = [&](int d) {
            const uint8_t *b = head + (d >> 5) * SQA_Q4_0_BLOCK_BYTES;
            const int k = d & 31;
            return (float)((b[2 + (k & 15)] >> (k < 16 ? 0 : 4) & 15) - 8) * (float)*reinterpret_cast<const _Float16 *>(b);
        };
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = d0 + j;
            if (d >= p.n_rot) out[j] = value(d);
            else if (d < half) out[j] = value(d) * cs[d].x - value(d + half) * cs[d].y;
            else out[j] = value(d - half) * cs[d - half].y + value(d) * cs[d - half].x;
        }
        __syncthreads();  // dst may be src
        if (ok)
            quantize_q4_0_block8(out, tid & 7, dst + ((int64_t)h * blocks + (d0 >> 5)) * SQA_Q4_0_BLOCK_BYTES);
        __syncthreads();
    }
    const int rest = (blocks - turned) * (SQA_Q4_0_BLOCK_BYTES / 2);
    if (src != dst)
        for (int k = tid; k < p.heads * rest; k += kThreads) {
            const int64_t at = (int64_t)(k / rest) * blocks * (SQA_Q4_0_BLOCK_BYTES / 2) +
                               turned * (SQA_Q4_0_BLOCK_BYTES / 2) + k % rest;
            reinterpret_cast<uint16_t *>(dst)[at] = reinterpret_cast<const uint16_t *>(src)[at];
        }
}

}  // namespace

int launch_get_rows_q4_0(const GetRows &p, bool half, hipStream_t s) {
    if (p.n == 0) return SQA_OK;
    const int prof = profile_start("get_rows_q4_0", s);
    const dim3 grid((unsigned)((p.n * p.blocks * 8 + kThreads - 1) / kThreads));
    if (half) get_rows_q4_0_kernel<true><<<grid, dim3(kThreads), 0, s>>>(p);
    else get_rows_q4_0_kernel<false><<<grid, dim3(kThreads), 0, s>>>(p);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "get_rows_q4_0 launch");
}

int launch_move_rows_q4_0(const MoveRows &p, hipStream_t s) {
    if (p.n == 0) return SQA_OK;
    const int prof = profile_start("move_rows_q4_0", s);
    move_rows_q4_0_kernel<<<dim3((unsigned)p.n), dim3(kThreads), 0, s>>>(p);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "move_rows_q4_0 launch");
}

}  // namespace sqa
