// lora.hip - low-rank adapters of many requests beside a shared projection:
// out = base + scale[id] B[id] (A[id] (x sigmoid(gate))), an id per token.
//
// One workgroup per token: its wavefronts take the ranks of A x in turn, then its
// threads the columns of the output.
#include "paged.hpp"

namespace sqa {
namespace {

constexpr int kThreads = 256;

struct Params {
    const char *base, *x, *gate;
    int64_t base_nb1, x_nb1, gate_nb1, dst_nb1;
    const _Float16 *a, *b;
    const int32_t *ids;
    const float *scale;
    char *dst;
    int K, N, r, n, M;
};

__global__ __launch_bounds__(kThreads) void lora_token_kernel(Params p) {
    __shared__ float t[128];
    const int m = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int id = p.ids[m];
    const float *base = reinterpret_cast<const float *>(p.base + m * p.base_nb1);
    float *dst = reinterpret_cast<float *>(p.dst + m * p.dst_nb1);
    const bool has = id >= 0 && id < p.n;
    if (has) {
        const float *x = reinterpret_cast<const float *>(p.x + m * p.x_nb1);
        const float *g = p.gate ? reinterpret_cast<const float *>(p.gate + m * p.gate_nb1) : nullptr;
        for (int j = wave; j < p.r; j += 4) {
            const _Float16 *a = p.a + ((int64_t)id * p.r + j) * p.K;
            float s = 0.0f;
            for (int k = lane; k < p.K; k += 64) {
                const float v = g ? x[k] * (1.0f / (1.0f + expf(-g[k]))) : x[k];
                s = fmaf(v, (float)a[k], s);
            }
            for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
            if (lane == 0) t[j] = s;
        }
    }
    __syncthreads();
    const float sc = has && p.scale ? p.scale[id] : 1.0f;
    for (int c = tid; c < p.N; c += kThreads) {
        float s = 0.0f;
        if (has) {
            const _Float16 *b = p.b + ((int64_t)id * p.N + c) * p.r;
            for (int j = 0; j < p.r; ++j) s = fmaf(t[j], (float)b[j], s);
        }
        dst[c] = has ? fmaf(sc, s, base[c]) : base[c];
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
    lora_token_kernel<<<dim3((unsigned)p.M), dim3(kThreads), 0, s>>>(p);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "lora_add launch");
}

}  // namespace sqa
