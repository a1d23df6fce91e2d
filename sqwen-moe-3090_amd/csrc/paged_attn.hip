// paged_attn.hip - attention of a batch of requests over a paged q4_0 pool.
//
// One workgroup per (token, query head): its 4 wavefronts walk the keys in turn, a
// lane holding 4 of the 256 dims, each with a softmax of its own that is kept
// online (running maximum and sum); the four are merged through LDS.
#include "paged.hpp"

namespace sqa {
namespace {

constexpr int kThreads = 256;

struct Params {
    const char *q;
    int64_t q_nb1, q_nb2;
    const uint8_t *k, *v;
    int64_t row_bytes, k_page, v_page;
    int32_t n_pages;
    int page, lp;
    const int32_t *table;
    int64_t table_stride;
    int W, B;
    const int32_t *q_start, *kv_len, *prefix;
    int n_tok, H, G;
    float scale, cap, bias;
    int nl2;
    const char *gate;
    int64_t gate_nb1, gate_nb2;
    float *dst;
};

__device__ __forceinline__ float h2f(uint16_t b) {
    _Float16 f;
    __builtin_memcpy(&f, &b, 2);
    return (float)f;
}

__global__ __launch_bounds__(kThreads) void paged_attn_kernel(Params p) {
    __shared__ int found;
    __shared__ float xo[4][256], xm[4], xl[4];
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    if (tid == 0) found = -1;
    __syncthreads();
    for (int b = tid; b < p.B; b += kThreads)
        if (p.q_start[b] <= t && t < p.q_start[b + 1]) found = b;
    __syncthreads();
    const int b = found;
    if (b < 0) return;
    const int kvh = h / p.G;
    const int64_t kv = min((int64_t)max(p.kv_len[b], 0), (int64_t)p.W << p.lp);
    const int64_t pos = (int64_t)p.kv_len[b] - p.q_start[b + 1] + t;
    int64_t see = pos + 1;
    if (p.prefix) see = max(see, (int64_t)p.prefix[b]);
    see = min(see, kv);
    // dims of the lane: elements 2i, 2i + 1, 16 + 2i, 17 + 2i of block blk
    const int blk = lane >> 3, i = lane & 7;
    const float *qr = reinterpret_cast<const float *>(p.q + t * p.q_nb1 + h * p.q_nb2) + 32 * blk + 2 * i;
    float q[4] = {qr[0], qr[1], qr[16], qr[17]};
    float amax = 0.0f;
    for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fabsf(q[j]));
    for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    const float id = amax != 0.0f ? 127.f / amax : 0.0f;
    const float qd = (float)(_Float16)(amax / 127.f) * p.scale;
    for (int j = 0; j < 4; ++j) q[j] = rintf(q[j] * id) * qd;
    const float slope = p.bias == 0.0f ? 0.0f
                        : h < p.nl2    ? exp2f(-p.bias * (float)(h + 1) / (float)p.nl2)
                                       : exp2f(-0.5f * p.bias * (float)(2 * (h - p.nl2) + 1) / (float)p.nl2);
    float m = -INFINITY, l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t j = wave; j < see; j += 4) {
        const int32_t id_p = p.table[b * p.table_stride + (j >> p.lp)];
        if (id_p < 0 || id_p >= p.n_pages) continue;
        const int64_t row = (j & (p.page - 1)) * p.row_bytes + kvh * kHeadRowBytes + 18 * blk;
        const uint16_t *kb = reinterpret_cast<const uint16_t *>(p.k + id_p * p.k_page + row);
        const uint16_t *vb = reinterpret_cast<const uint16_t *>(p.v + id_p * p.v_page + row);
        const uint32_t kc = kb[1 + i], vc = vb[1 + i];
        const float kd = h2f(kb[0]), vd = h2f(vb[0]);
        float s = kd * (q[0] * (float)((int)(kc & 15) - 8) + q[1] * (float)((int)(kc >> 8 & 15) - 8) +
                        q[2] * (float)((int)(kc >> 4 & 15) - 8) + q[3] * (float)((int)(kc >> 12) - 8));
        for (int x = 1; x < 64; x <<= 1) s += __shfl_xor(s, x);
        if (p.cap != 0.0f) s = p.cap * tanhf(s / p.cap);
        s -= slope * fabsf((float)(pos - j));
        const float mn = fmaxf(m, s), al = expf(m - mn), w = expf(s - mn);
        m = mn;
        l = l * al + w;
        const float wd = w * vd;
        o[0] = o[0] * al + wd * (float)((int)(vc & 15) - 8);
        o[1] = o[1] * al + wd * (float)((int)(vc >> 8 & 15) - 8);
        o[2] = o[2] * al + wd * (float)((int)(vc >> 4 & 15) - 8);
        o[3] = o[3] * al + wd * (float)((int)(vc >> 12) - 8);
    }
    const int d = 32 * blk + 2 * i;
    xo[wave][d] = o[0], xo[wave][d + 1] = o[1], xo[wave][d + 16] = o[2], xo[wave][d + 17] = o[3];
    if (lane == 0) xm[wave] = m, xl[wave] = l;
    __syncthreads();
    const float M = fmaxf(fmaxf(xm[0], xm[1]), fmaxf(xm[2], xm[3]));
    float r = 0.0f, L = 0.0f;
    if (M != -INFINITY)
        for (int w = 0; w < 4; ++w) {
            const float f = expf(xm[w] - M);
            r += f * xo[w][tid];
            L += f * xl[w];
        }
    r = L == 0.0f ? 0.0f : r / L;
    if (p.gate) {
        const float g = reinterpret_cast<const float *>(p.gate + t * p.gate_nb2 + h * p.gate_nb1)[tid];
        r *= 1.0f / (1.0f + expf(-g));
    }
    p.dst[((int64_t)t * p.H + h) * kHeadDim + tid] = r;
}

}  // namespace

size_t paged_attn_workspace(int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

int launch_paged_attn(const PagedArgs &a, hipStream_t s) {
    const sqa_tensor &q = *a.q, &k = *a.k;
    Params p{};
    p.q = (const char *)q.data, p.q_nb1 = (int64_t)q.nb[1], p.q_nb2 = (int64_t)q.nb[2];
    p.k = (const uint8_t *)k.data, p.v = (const uint8_t *)a.v->data;
    p.row_bytes = (int64_t)k.nb[2], p.k_page = (int64_t)k.nb[3], p.v_page = (int64_t)a.v->nb[3];
    p.n_pages = (int32_t)k.ne[3], p.page = (int)k.ne[2];
    while ((1 << p.lp) < p.page) ++p.lp;
    p.table = (const int32_t *)a.table->data, p.table_stride = (int64_t)a.table->nb[1] / 4;
    p.W = (int)a.table->ne[0], p.B = (int)a.table->ne[1];
    p.q_start = (const int32_t *)a.q_start->data, p.kv_len = (const int32_t *)a.kv_len->data;
    p.prefix = a.prefix ? (const int32_t *)a.prefix->data : nullptr;
    p.n_tok = (int)q.ne[1], p.H = (int)q.ne[2], p.G = (int)(q.ne[2] / k.ne[1]);
    p.scale = a.scale, p.cap = a.softcap, p.bias = a.max_bias;
    p.nl2 = 1;
    while (2 * p.nl2 <= p.H) p.nl2 *= 2;
    p.gate = a.gate ? (const char *)a.gate->data : nullptr;
    p.gate_nb1 = a.gate ? (int64_t)a.gate->nb[1] : 0, p.gate_nb2 = a.gate ? (int64_t)a.gate->nb[2] : 0;
    p.dst = (float *)a.dst->data;
    const int prof = profile_start("paged_attn", s);
    paged_attn_kernel<<<dim3((unsigned)p.n_tok, (unsigned)p.H), dim3(kThreads), 0, s>>>(p);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "paged_attn launch");
}

}  // namespace sqa
