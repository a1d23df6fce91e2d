// lora.hip - low-rank adapters of many requests beside a shared projection:
// out = base + scale[id] B[id] (A[id] (x sigmoid(gate))), an id per token.
//
// Bound by memory: x, gate, base and out once each (64 to 100 KB a token group of 16 per
// 4096 + 2048 columns), the adapters in use out of L2; by latency for few tokens. Both
// kernels therefore do the two products in one launch, with A x in LDS between them.
//
// Few tokens (decode): a workgroup per token and part of the columns. Every byte that
// the token needs is asked for at the start (A rows, B rows, base beside x), so one
// memory latency stands before the sums; fp32 throughout.
//
// More: a workgroup takes 16 tokens. Its 8 wavefronts split K, each with all ranks:
// t^T = A x^T on v_mfma_f32_16x16x32_f16, A as it is, x as an fp16 pair: hi = fp16(x),
// lo = fp16((x - hi) 2^11), in sums of their own (the shift keeps lo clear of
// subnormals: 22 bits down to |x| = 2^-13, an absolute 2^-36 below). The eight partial
// t are added in LDS; then they split the columns, out^T = B t^T with t as a pair in
// the same way. The transposed forms leave a lane with 4 consecutive columns of one
// token: 16-byte accesses of base and out. Tokens of a tile with other adapters are
// served in further passes over the tile; a pass takes effect by a select per token,
// so no adapter's values reach another one's tokens, not even its NaN.
#include <mutex>

#include "paged.hpp"

namespace sqa {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float float4a __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxRank = 128;

struct Params {
    const char *base, *x, *gate;
    int64_t base_nb1, x_nb1, gate_nb1, dst_nb1;
    const _Float16 *a, *b;
    const int32_t *ids;
    const float *scale;
    char *dst;
    int K, N, r, n, M;
};

__device__ __forceinline__ floatx4 gated(floatx4 x, floatx4 g) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g[i]));
    return x;
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o);
    return x;
}

// ------------------------------------------------------------- few tokens

// Grid (tokens, parts of the columns). Wavefront w sums ranks w, w + 8, ...: a lane 8
// values of every 512.
__global__ __launch_bounds__(kThreads) void lora_token_kernel(Params p) {
    extern __shared__ float xs[];  // K values of x sigmoid(gate)
    __shared__ __align__(16) float t[kMaxRank];
    const int m = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int id = p.ids[m];
    const float *base = reinterpret_cast<const float *>(p.base + m * p.base_nb1);
    float *dst = reinterpret_cast<float *>(p.dst + m * p.dst_nb1);
    const int quads = p.N / 4, q0 = (int)((int64_t)quads * blockIdx.y / gridDim.y),
              q1 = (int)((int64_t)quads * (blockIdx.y + 1) / gridDim.y);
    if (id < 0 || id >= p.n) {
        for (int q = q0 + tid; q < q1; q += kThreads)
            reinterpret_cast<floatx4 *>(dst)[q] = reinterpret_cast<const floatx4 *>(base)[q];
        return;
    }
    const _Float16 *a = p.a + (int64_t)id * p.r * p.K, *b = p.b + (int64_t)id * p.N * p.r;
    const float sc = p.scale ? p.scale[id] : 1.0f;
    // the first rank's row and the first column's are on their way while x is gated
    constexpr int kAhead = 8;
    half8 an[kAhead];
    const bool first = wave < p.r;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        if (first && 512 * j + 8 * lane < p.K) an[j] = *reinterpret_cast<const half8 *>(a + (int64_t)wave * p.K + 512 * j + 8 * lane);
    const float *x = reinterpret_cast<const float *>(p.x + m * p.x_nb1);
    const float *g = p.gate ? reinterpret_cast<const float *>(p.gate + m * p.gate_nb1) : nullptr;
    for (int k = 4 * tid; k < p.K; k += 4 * kThreads) {
        floatx4 v = *reinterpret_cast<const float4a *>(x + k);
        if (g) v = gated(v, *reinterpret_cast<const float4a *>(g + k));
        *reinterpret_cast<floatx4 *>(xs + k) = v;
    }
    __syncthreads();
    for (int j = wave; j < p.r; j += kWaves) {
        float s0 = 0.0f, s1 = 0.0f;
        for (int k0 = 0; k0 < p.K; k0 += 512 * kAhead) {
            half8 av[kAhead];
#pragma unroll
            for (int q = 0; q < kAhead; ++q) av[q] = an[q];
            // the next stretch: of this rank, or the start of the next one
            const int kn = k0 + 512 * kAhead, jn = kn < p.K ? j : j + kWaves, k1 = kn < p.K ? kn : 0;
#pragma unroll
            for (int q = 0; q < kAhead; ++q)
                if (jn < p.r && k1 + 512 * q + 8 * lane < p.K)
                    an[q] = *reinterpret_cast<const half8 *>(a + (int64_t)jn * p.K + k1 + 512 * q + 8 * lane);
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const int k = k0 + 512 * q + 8 * lane;
                if (k < p.K) {
                    const floatx4 u = *reinterpret_cast<const floatx4 *>(xs + k), v = *reinterpret_cast<const floatx4 *>(xs + k + 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s0 = fmaf(u[i], (float)av[q][i], s0);
                        s1 = fmaf(v[i], (float)av[q][4 + i], s1);
                    }
                }
            }
        }
        const float s = wave_sum(s0 + s1);
        if (lane == 0) t[j] = s * sc;
    }
    __syncthreads();
    for (int c = 4 * q0 + tid; c < 4 * q1; c += kThreads) {
        const half8 *row = reinterpret_cast<const half8 *>(b + (int64_t)c * p.r);
        float s = base[c];
        for (int j = 0; j < p.r / 8; ++j) {
            const half8 bv = row[j];
            const floatx4 u = *reinterpret_cast<const floatx4 *>(t + 8 * j), v = *reinterpret_cast<const floatx4 *>(t + 8 * j + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s = fmaf(u[i], (float)bv[i], s);
                s = fmaf(v[i], (float)bv[4 + i], s);
            }
        }
        dst[c] = s;
    }
}

// ----------------------------------------------------------------- tiles

constexpr int kTile = 16;  // tokens of a workgroup

// hi = fp16(x) and lo = fp16((x - hi) 2^11) of 8 values
__device__ __forceinline__ void split(const float (&x)[8], half8 &hi, half8 &lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const _Float16 h = (_Float16)x[i];
        hi[i] = h;
        lo[i] = (_Float16)((x[i] - (float)h) * 2048.0f);
    }
}

// RT: tiles of 16 ranks, r <= 16 RT.
// MFMA operands (lane = 16 g + n): A[n][8g..8g+7], B[8g..8g+7][n], C[4g..4g+3][n].
template <int RT>
__global__ __launch_bounds__(kThreads, 2) void lora_tile_kernel(Params p) {
    extern __shared__ float part[];  // [8 waves][RT * 16 ranks][16 tokens], then t [16 tokens][RT * 16 + 4]
    constexpr int kR = 16 * RT, kTRow = kR + 4;
    float *t = part + kWaves * kR * kTile;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, n = lane & 15;
    const int m = (int)blockIdx.x * kTile + n;  // the lane's token
    const bool in = m < p.M;
    const int64_t row = in ? m : p.M - 1;
    int id = p.ids[row];
    id = in && id >= 0 && id < p.n ? id : -1;
    const float *x = reinterpret_cast<const float *>(p.x + row * p.x_nb1);
    const float *gt = p.gate ? reinterpret_cast<const float *>(p.gate + row * p.gate_nb1) : nullptr;
    const float *base = reinterpret_cast<const float *>(p.base + row * p.base_nb1);
    float *dst = reinterpret_cast<float *>(p.dst + row * p.dst_nb1);
    // K in steps of 32, N in tiles of 16: this wavefront's share
    const int k_steps = p.K / 32, k0 = k_steps * wave / kWaves, k1 = k_steps * (wave + 1) / kWaves;
    const int n_tiles = p.N / 16, c0 = n_tiles * wave / kWaves, c1 = n_tiles * (wave + 1) / kWaves;

    uint64_t todo = __ballot(id >= 0 && g == 0);
    bool done = false;  // whether dst holds base already (a later pass)
    if (!todo) {
        for (int c = c0; c < c1; ++c)
            if (in) *reinterpret_cast<floatx4 *>(dst + 16 * c + 4 * g) = *reinterpret_cast<const floatx4 *>(base + 16 * c + 4 * g);
        return;
    }
    while (todo) {
        const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
        const bool mine = id == cur;
        todo &= ~__ballot(mine && g == 0);
        const _Float16 *a = p.a + (int64_t)cur * p.r * p.K, *b = p.b + (int64_t)cur * p.N * p.r;
        const float sc = p.scale ? p.scale[cur] : 1.0f;
        floatx4 hi[RT], lo[RT];
#pragma unroll
        for (int q = 0; q < RT; ++q) hi[q] = lo[q] = floatx4{0.f, 0.f, 0.f, 0.f};
        // rows of A past r re-read its last one: their t is never used
        const _Float16 *ar[RT];
#pragma unroll
        for (int q = 0; q < RT; ++q) ar[q] = a + (int64_t)min(16 * q + n, p.r - 1) * p.K + 8 * g;
        constexpr int kU = 2;
        for (int s0 = k0; s0 < k1; s0 += kU) {
            floatx4 xv[kU][2], gv[kU][2];
            half8 av[kU][RT];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int k = 32 * min(s0 + u, k1 - 1) + 8 * g;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    xv[u][h] = *reinterpret_cast<const float4a *>(x + k + 4 * h);
                    if (gt) gv[u][h] = *reinterpret_cast<const float4a *>(gt + k + 4 * h);
                }
#pragma unroll
                for (int q = 0; q < RT; ++q) av[u][q] = *reinterpret_cast<const half8 *>(ar[q] + 32 * min(s0 + u, k1 - 1));
            }
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (s0 + u >= k1) break;
                float v[8];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const floatx4 w = gt ? gated(xv[u][h], gv[u][h]) : xv[u][h];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[4 * h + i] = w[i];
                }
                half8 xh, xl;
                split(v, xh, xl);
#pragma unroll
                for (int q = 0; q < RT; ++q) {
                    hi[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av[u][q], xh, hi[q], 0, 0, 0);
                    lo[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av[u][q], xl, lo[q], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int q = 0; q < RT; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                part[(wave * kR + 16 * q + 4 * g + i) * kTile + n] = fmaf(lo[q][i], 1.0f / 2048.0f, hi[q][i]);
        __syncthreads();
        for (int e = tid; e < kR * kTile; e += kThreads) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) s += part[w * kR * kTile + e];
            t[(e & 15) * kTRow + (e >> 4)] = e >> 4 < p.r ? s * sc : 0.0f;
        }
        __syncthreads();
        // t of the lane's token, ranks 32s + 8g ..
        constexpr int kS = (kR + 31) / 32;
        half8 th[kS], tl[kS];
#pragma unroll
        for (int s = 0; s < kS; ++s) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 32 * s + 8 * g < kR ? t[n * kTRow + 32 * s + 8 * g + i] : 0.0f;
            split(v, th[s], tl[s]);
        }
        // kC tiles of 16 columns at a time, all their loads before the first use
        constexpr int kC = RT == 8 ? 2 : 4;
        const float *from = done ? dst : base;
        for (int cc = c0; cc < c1; cc += kC) {
            floatx4 old[kC];
            half8 bv[kC][kS];
#pragma unroll
            for (int u = 0; u < kC; ++u) {
                const int c = min(cc + u, c1 - 1);
                old[u] = *reinterpret_cast<const floatx4 *>(from + 16 * c + 4 * g);
#pragma unroll
                for (int s = 0; s < kS; ++s) {
                    bv[u][s] = half8{};
                    if (32 * s + 8 * g < p.r) bv[u][s] = *reinterpret_cast<const half8 *>(b + (int64_t)(16 * c + n) * p.r + 32 * s + 8 * g);
                }
            }
#pragma unroll
            for (int u = 0; u < kC; ++u) {
                floatx4 h = {0.f, 0.f, 0.f, 0.f}, l = h;
#pragma unroll
                for (int s = 0; s < kS; ++s) {
                    h = __builtin_amdgcn_mfma_f32_16x16x32_f16(bv[u][s], th[s], h, 0, 0, 0);
                    l = __builtin_amdgcn_mfma_f32_16x16x32_f16(bv[u][s], tl[s], l, 0, 0, 0);
                }
                floatx4 o;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = mine ? old[u][i] + fmaf(l[i], 1.0f / 2048.0f, h[i]) : old[u][i];
                if (in && (mine || !done) && cc + u < c1) *reinterpret_cast<floatx4 *>(dst + 16 * (cc + u) + 4 * g) = o;
            }
        }
        done = true;
    }
}

}  // namespace

int launch_lora_add(const sqa_tensor &base, const sqa_tensor &x, const sqa_tensor *gate, const sqa_tensor &a,
                    const sqa_tensor &b, const sqa_tensor &ids, const sqa_tensor *scale, const sqa_tensor &dst,
                    hipStream_t s) {
    const Params p{(const char *)base.data, (const char *)x.data, gate ? (const char *)gate->data : nullptr,
                   (int64_t)base.nb[1], (int64_t)x.nb[1], gate ? (int64_t)gate->nb[1] : 0, (int64_t)dst.nb[1],
                   (const _Float16 *)a.data, (const _Float16 *)b.data, (const int32_t *)ids.data,
                   scale ? (const float *)scale->data : nullptr, (char *)dst.data, (int)x.ne[0], (int)base.ne[0],
                   (int)a.ne[1], (int)a.ne[2], (int)x.ne[1]};
    const int prof = profile_start("lora_add", s);
    // x of a token has to fit in LDS beside its ranks
    if (p.M <= 256 && p.K <= 15 * 1024) {
        const int parts = p.M <= 32 ? 4 : p.M <= 96 ? 2 : 1;
        lora_token_kernel<<<dim3((unsigned)p.M, (unsigned)parts), dim3(kThreads), (size_t)p.K * 4, s>>>(p);
    } else {
        const dim3 grid((unsigned)((p.M + kTile - 1) / kTile));
        auto lds = [](int rt) { return (size_t)(kWaves * 16 * rt * kTile + kTile * (16 * rt + 4)) * 4; };
        static std::once_flag once;  // the one form above the 64 KB that need no asking
        static hipError_t err = hipSuccess;
        std::call_once(once, [&] {
            err = hipFuncSetAttribute((const void *)lora_tile_kernel<8>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds(8));
        });
        if (err != hipSuccess) return hip_status(err, "lora_add LDS attribute");
        if (p.r <= 16) lora_tile_kernel<1><<<grid, dim3(kThreads), lds(1), s>>>(p);
        else if (p.r <= 32) lora_tile_kernel<2><<<grid, dim3(kThreads), lds(2), s>>>(p);
        else if (p.r <= 64) lora_tile_kernel<4><<<grid, dim3(kThreads), lds(4), s>>>(p);
        else lora_tile_kernel<8><<<grid, dim3(kThreads), lds(8), s>>>(p);
    }
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "lora_add launch");
}

}  // namespace sqa
