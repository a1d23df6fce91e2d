// rows_q4_0.hip - cached q4_0 rows read back (get_rows) and moved (move_rows), the
// counterparts of set_rows_q4_0.hip.
//
// Both are one pass over the rows. get_rows is bound by the bytes it reads and writes: 131072
// rows of 512 values as F16 28 us, 6.2 TB/s, F32 45 us, 6.8 (a copy 4.8). move_rows of 100001 such
// rows with 64 rotated dims a head 24 us, in place 25: vector instructions (15 us without the rotated
// blocks, 14 of them with a table that costs nothing) and, below 20000 rows, four memory latencies in a
// row; without a rope 12, as a copy. A workgroup
// takes a run of rows; its threads go through the rows' units of a fixed size, whose row
// comes from a multiplication (the host provides the reciprocal).
#include <math.h>

#include "q4_0_block.hpp"
#include "rows.hpp"

namespace sqa {
namespace {

constexpr int kThreads = 256;

// 4 bytes at any even address (the hardware's loads and stores ask for no more)
typedef uint32_t uint32a __attribute__((aligned(2)));
typedef uint32_t uint32x2a __attribute__((ext_vector_type(2), aligned(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef uint32_t uint32x4 __attribute__((ext_vector_type(4)));

// u / n for 0 <= u <= 2^20 by the reciprocal of n: u + 1/2 is half of 1 / n or more from a whole
// quotient, and the float product off by 2^-22 of it (32-bit multiplications take four times as long).
__device__ __forceinline__ int div_by(int u, float recip) { return (int)(((float)u + 0.5f) * recip); }
__device__ __forceinline__ int mul(int a, int b) { return __mul24(a, b); }  // below 2^23 each

// get_rows: a unit is the 16 bytes that a lane stores, 8 values of F16 or 4 of F32: their codes
// (low or high nibbles of 8 or 4 bytes) and their block's scale. Rows whose starts are not 16 bytes
// apart, or at such addresses, go out value by value.
template <bool kHalf, bool kVec, bool kStream>
__global__ __launch_bounds__(kThreads) void get_rows_q4_0_kernel(GetRows p) {
    constexpr int kVals = kHalf ? 8 : 4, kPer = 32 / kVals;  // units of a block
    const int units = p.blocks * kPer;
    const int64_t i0 = p.first + (int64_t)blockIdx.x * p.rows;
    for (int u = threadIdx.x; u < (int)min((int64_t)p.rows, p.n - i0) * units; u += kThreads) {
        const int k = div_by(u, p.recip), c = u - mul(k, units), b = c / kPer, t = c % kPer;
        const int64_t i = i0 + k, r = *reinterpret_cast<const int64_t *>(p.idx + i * p.idx_nb0);
        float v[kVals] = {};
        if (r >= 0 && r < p.src_rows) {
            const uint8_t *from = p.src + r * p.src_nb1 + b * SQA_Q4_0_BLOCK_BYTES;
            const float d = (float)*reinterpret_cast<const _Float16 *>(from);
            from += 2 + kVals * (t % (kPer / 2));
            uint32_t q[kVals / 4];
            if constexpr (kHalf) {
                const uint32x2a x = *reinterpret_cast<const uint32x2a *>(from);
                q[0] = x[0], q[1] = x[1];
            } else {
                q[0] = *reinterpret_cast<const uint32a *>(from);
            }
            const int sh = t < kPer / 2 ? 0 : 4;
#pragma unroll
            for (int j = 0; j < kVals; ++j) v[j] = (float)((int)(q[j >> 2] >> (8 * (j & 3) + sh) & 15) - 8) * d;
        }
        char *row = p.dst + i * p.dst_nb1 + (int64_t)c * 16;
        if constexpr (kVec) {
            uint32x4 x;
            if constexpr (kHalf) {
                half8 h;
#pragma unroll
                for (int j = 0; j < kVals; ++j) h[j] = (_Float16)v[j];
                __builtin_memcpy(&x, &h, 16);
            } else {
                __builtin_memcpy(&x, v, 16);
            }
            if constexpr (kStream) __builtin_nontemporal_store(x, reinterpret_cast<uint32x4 *>(row));
            else *reinterpret_cast<uint32x4 *>(row) = x;
        } else {
#pragma unroll
            for (int j = 0; j < kVals; ++j) {
                if constexpr (kHalf) reinterpret_cast<_Float16 *>(row)[j] = (_Float16)v[j];
                else reinterpret_cast<float *>(row)[j] = v[j];
            }
        }
    }
}

// cos and sin of x radians, |x| < 2^31 pi / 2, good to some 2^-48 of 1 (for results rounded
// to fp32): x minus the nearest multiple of pi / 2, which two fmas take off as the double next
// to pi / 2 and what that leaves out, then the Taylor polynomials to x^16 and x^15 (the next
// terms are below 2^-53 up to pi / 4).
__device__ __forceinline__ float2 cos_sin(double x) {
    const double k = __builtin_rint(x * 0.63661977236758134308);  // 2 / pi
    double r = fma(-k, 1.57079632679489661923, x);
    r = fma(-k, 6.12323399573676603587e-17, r);
    const double y = r * r;
    double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
    s = fma(s, y, 1.0 / 6227020800.0), c = fma(c, y, -1.0 / 87178291200.0);
    s = fma(s, y, -1.0 / 39916800.0), c = fma(c, y, 1.0 / 479001600.0);
    s = fma(s, y, 1.0 / 362880.0), c = fma(c, y, -1.0 / 3628800.0);
    s = fma(s, y, -1.0 / 5040.0), c = fma(c, y, 1.0 / 40320.0);
    s = fma(s, y, 1.0 / 120.0), c = fma(c, y, -1.0 / 720.0);
    s = fma(s, y, -1.0 / 6.0), c = fma(c, y, 1.0 / 24.0);
    s = fma(s * y, r, r), c = fma(c, y, -0.5);
    c = fma(c, y, 1.0);
    const int q = (int)((int64_t)k & 3);
    const float sf = (float)s, cf = (float)c;
    const float co = q & 1 ? sf : cf, si = q & 1 ? cf : sf;
    return make_float2(q == 1 || q == 2 ? -co : co, q >= 2 ? -si : si);
}

// move_rows: the rows' places and the (cos, sin) of their rotation pairs go to LDS; a rotated
// block is 8 lanes of 4 values, which read their own codes and their partners' (half dims away,
// both 4 bytes at one place) and quantize again; the other blocks are copied. A thread has the loads
// of kTurns rotated units, or kCopies copied ones, in flight together. In place a head's partners must
// all be read before a block of it is stored: a pass of the threads then takes whole heads, and a
// barrier stands between its loads and its stores (a head's lanes may be in two wavefronts).
typedef uint32_t Bytes12 __attribute__((ext_vector_type(3), aligned(4)));
constexpr int kTurns = 2, kCopies = 4;

template <typename Copy, int kStep>
__global__ __launch_bounds__(kThreads) void move_rows_q4_0_kernel(MoveRows p) {
#pragma clang fp contract(off)
    const int64_t i0 = p.first + (int64_t)blockIdx.x * p.rows;
    const int rows = (int)min((int64_t)p.rows, p.n - i0);
    extern __shared__ __align__(16) uint8_t lds[];
    int64_t *places = reinterpret_cast<int64_t *>(lds);         // [rows] {offset in src or -1, in dst}
    float2 *cs = reinterpret_cast<float2 *>(lds + 16 * p.rows);  // [rows][half]
    const int tid = threadIdx.x, half = p.n_rot >> 1;
    if (tid < rows) {
        const int64_t r = *reinterpret_cast<const int64_t *>(p.from + (i0 + tid) * p.from_nb0);
        const int64_t w = *reinterpret_cast<const int64_t *>(p.to + (i0 + tid) * p.to_nb0);
        const bool ok = r >= 0 && r < p.src_rows && w >= 0 && w < p.dst_rows;
        places[2 * tid] = ok ? r * p.src_nb1 : -1;
        places[2 * tid + 1] = ok ? w * p.dst_nb1 : 0;
    }
    // rows that all move as far (a whole conversation, as a rule) share one row of the table: 100001
    // rows 36.6 -> 30.7 us (with the quantizer's exchanges still through LDS)
    bool same = true;
    if (half && tid < 4 * rows) same = p.delta[i0 + (tid >> 2) + (tid & 3) * p.n] == p.delta[i0 + (tid & 3) * p.n];
    same = __syncthreads_and(same);
    for (int u = tid; u < (same ? half : rows * half); u += kThreads) {
        const int k = div_by(u, p.recip_half), ic = u - mul(k, half);
        cs[u] = cos_sin((double)p.delta[i0 + k + p.component[ic] * p.n] * p.freq[ic]);
    }
    const int table = same ? 0 : half;
    const int turned = (p.n_rot + 31) >> 5, head_bytes = p.head_dim / SQA_QK4_0 * SQA_Q4_0_BLOCK_BYTES;
    const int lanes = 8 * turned, per_row = lanes * p.heads;
    __syncthreads();
    for (int u0 = 0; u0 < rows * per_row; u0 += p.pass) {
        float out[kTurns][4];
        uint8_t *to[kTurns];
#pragma unroll
        for (int n = 0; n < kTurns; ++n) {
            const int i = tid + n * kThreads, u = u0 + i;
            const int k = div_by(u, p.recip_turned), hl = u - mul(k, per_row), h = div_by(hl, p.recip_lanes);
            const int d0 = 4 * (hl - mul(h, lanes));
            const int64_t at = i < p.pass && k < rows ? places[2 * k] : -1;
            to[n] = nullptr;
            if (at < 0) continue;
            to[n] = p.dst + places[2 * k + 1] + mul(h, head_bytes) + (d0 >> 5) * SQA_Q4_0_BLOCK_BYTES;
            const uint8_t *head = p.src + at + mul(h, head_bytes);
            auto values = [&](int d, float (&x)[4]) {  // dims d .. d + 3 of the head
                const uint8_t *b = head + (d >> 5) * SQA_Q4_0_BLOCK_BYTES;
                const float s = (float)*reinterpret_cast<const _Float16 *>(b);
                const uint32_t q = *reinterpret_cast<const uint32a *>(b + 2 + (d & 15)) >> (d & 16 ? 4 : 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = (float)((int)(q >> (8 * j) & 15) - 8) * s;
            };
            float x[4], y[4];
            const bool low = d0 < half, turns = d0 < p.n_rot;
            const int ic = low ? d0 : turns ? d0 - half : 0;
            values(d0, x);
            values(!turns ? d0 : low ? d0 + half : ic, y);
            const float4 *t = reinterpret_cast<const float4 *>(cs + mul(k, table) + ic);
            const float4 t0 = t[0], t1 = t[1];
            const float c[4] = {t0.x, t0.z, t1.x, t1.z}, s[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // x0 c - x1 s, and x1 c + x0 s for the partner
                const float a = x[j] * c[j], b = y[j] * s[j];
                out[n][j] = turns ? a + (low ? -b : b) : x[j];
            }
        }
        if (p.src == p.dst) __syncthreads();
#pragma unroll
        for (int n = 0; n < kTurns; ++n)
            if (to[n]) quantize_q4_0_block8(out[n], tid & 7, to[n]);
    }
    // blocks without a rotated dim; in place they are there
    const int skip = turned * SQA_Q4_0_BLOCK_BYTES, step = kStep, rest = (head_bytes - skip) / step;
    const int per_copy = rest * p.heads;
    for (int u0 = tid; u0 < rows * per_copy; u0 += kCopies * kThreads) {
        Copy x[kCopies] = {};
        int64_t to[kCopies];
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
            const int u = u0 + j * kThreads, k = div_by(u, p.recip_copy), hc = u - mul(k, per_copy), h = div_by(hc, p.recip_rest);
            const int64_t at = k < rows ? places[2 * k] : -1;
            const int in_row = mul(h, head_bytes) + skip + step * (hc - mul(h, rest));
            to[j] = at < 0 ? -1 : places[2 * k + 1] + in_row;
            if (at >= 0) x[j] = *reinterpret_cast<const Copy *>(p.src + at + in_row);
        }
#pragma unroll
        for (int j = 0; j < kCopies; ++j)
            if (to[j] >= 0) *reinterpret_cast<Copy *>(p.dst + to[j]) = x[j];
    }
}

float recip(int64_t n) { return n > 0 ? 1.0f / (float)n : 0.0f; }

// Rows of a workgroup: from one pass of its threads over their units to `passes` of them, while four
// workgroups a CU are left (20000 rows moved 14.0 us with the least, 12.8 so).
int rows_of_workgroup(int64_t n, int64_t units, int passes, int most) {
    const int64_t many = passes * kThreads / units, one = kThreads / units, cus = device_cu_count();
    int64_t rows = n / (4 * cus);
    if (rows > many) rows = many;
    if (rows < one) rows = one;
    return (int)(rows < 1 ? 1 : rows > most ? most : rows);
}
// The launches of a call: one, but that none has 2^32 threads.
template <class P, class F>
void launch_all(P &p, const char *name, hipStream_t s, F launch) {
    const int prof = profile_start(name, s);
    const int64_t most = (int64_t)p.rows << 23;
    for (p.first = 0; p.first < p.n; p.first += most) {
        const int64_t n = p.n - p.first < most ? p.n - p.first : most;
        launch(dim3((unsigned)((n + p.rows - 1) / p.rows)));
    }
    profile_stop(prof, s);
}

}  // namespace

// Results of more than this go past the caches: 268 MB of F32 87 us with ordinary stores and 45 so,
// 134 MB of F16 50 and 28; with a kernel that reads them right after (in us, both together) 182
// and 172, 91 and 88; but 66 MB 45.5 and 47.3, 33 MB 23.3 and 25.5: those stay in the last cache.
constexpr int64_t kStreamBytes = 96 << 20;

int launch_get_rows_q4_0(GetRows p, bool half, hipStream_t s) {
    if (p.n == 0) return SQA_OK;
    const int64_t units = (half ? 4 : 8) * (int64_t)p.blocks, bytes = p.n * 16 * units;
    p.rows = rows_of_workgroup(p.n, units, 4, 16);
    p.recip = recip(units);
    const bool vec = (uintptr_t)p.dst % 16 == 0 && (p.dst_nb1 % 16 == 0 || p.n == 1);
    const bool stream = bytes > kStreamBytes;
    const auto kernel = half ? (!vec     ? get_rows_q4_0_kernel<true, false, false>
                                : stream ? get_rows_q4_0_kernel<true, true, true>
                                         : get_rows_q4_0_kernel<true, true, false>)
                             : (!vec     ? get_rows_q4_0_kernel<false, false, false>
                                : stream ? get_rows_q4_0_kernel<false, true, true>
                                         : get_rows_q4_0_kernel<false, true, false>);
    launch_all(p, "get_rows_q4_0", s, [&](dim3 grid) { kernel<<<grid, dim3(kThreads), 0, s>>>(p); });
    return hip_status(hipGetLastError(), "get_rows_q4_0 launch");
}

int launch_move_rows_q4_0(MoveRows p, hipStream_t s) {
    if (p.n == 0) return SQA_OK;
    const int64_t turned = (p.n_rot + 31) / 32, bytes = (p.head_dim / 32 - turned) * SQA_Q4_0_BLOCK_BYTES;
    // copies of 16 bytes where every run of whole heads or blocks allows them (144 a head of 256), of 12
    // where they are whole pairs of blocks, else of 2
    const uint64_t at = (uint64_t)(uintptr_t)p.src | (uint64_t)(uintptr_t)p.dst | (uint64_t)p.src_nb1 | (uint64_t)p.dst_nb1 |
                        (uint64_t)bytes | (uint64_t)(turned * SQA_Q4_0_BLOCK_BYTES) |
                        (uint64_t)(p.head_dim / 32 * SQA_Q4_0_BLOCK_BYTES);
    const int step = at % 16 == 0 ? 16 : at % 4 == 0 ? 12 : 2;
    const int64_t lanes = 8 * turned, rest = bytes / step;
    p.rows = rows_of_workgroup(p.n, (lanes + rest) * p.heads, 8, 32);
    p.recip_half = recip(p.n_rot / 2);
    p.recip_turned = recip(lanes * p.heads), p.recip_lanes = recip(lanes);
    // (between two caches a head may lie across two passes)
    p.pass = kTurns * kThreads;
    if (p.src == p.dst && lanes) p.pass -= p.pass % (int)lanes;
    p.recip_copy = recip(rest * p.heads), p.recip_rest = recip(rest);
    const size_t lds = (size_t)p.rows * (16 + (p.n_rot / 2) * sizeof(float2));
    const auto kernel = step == 16   ? move_rows_q4_0_kernel<uint32x4, 16>
                        : step == 12 ? move_rows_q4_0_kernel<Bytes12, 12>
                                     : move_rows_q4_0_kernel<uint16_t, 2>;
    launch_all(p, "move_rows_q4_0", s, [&](dim3 grid) { kernel<<<grid, dim3(kThreads), lds, s>>>(p); });
    return hip_status(hipGetLastError(), "move_rows_q4_0 launch");
}

}  // namespace sqa
