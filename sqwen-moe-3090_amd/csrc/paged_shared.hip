// paged_shared.hip - attention of a batch whose groups of requests share long prefixes: a
// request's own pages and its group's pages under one softmax.
//
// The simple form: a wavefront takes one query row, 4 dims a lane, and goes through the
// keys of the shared prefix and then its own with a running maximum and sum.
#include "paged_attn.hpp"

namespace sqa {
namespace paged {
namespace {

struct Shared {
    Call c;                   // own part
    const int32_t *table;     // pages of the groups' prefixes
    int64_t table_stride, most_kv;
    const int32_t *len, *token_group;
    int groups;
};

struct Online {
    float m = -INFINITY, l = 0.0f, o[4] = {};
};

// Sum over the wavefront.
__device__ __forceinline__ float wsum(float x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o);
    return x;
}

// A lane's 4 dims of a head row: byte pair within its block.
__device__ __forceinline__ void row4(const uint8_t *row, int lane, float (&x)[4]) {
    const uint8_t *b = row + (lane >> 3) * SQA_Q4_0_BLOCK_BYTES;
    const int t = lane & 7;
    const float d = (float)*reinterpret_cast<const _Float16 *>(b);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (float)((b[2 + 4 * (t & 3) + j] >> (t < 4 ? 0 : 4) & 15) - 8) * d;
}

__device__ void keys(const Call &c, const int32_t *row, int n, int kvh, int lane, const float (&q)[4], float slope, int far,
                     Online &a) {
    for (int j = 0; j < n; ++j) {
        const int id = row[j >> c.lp];
        if ((uint32_t)id >= (uint32_t)c.n_pages) continue;
        const int64_t at = (int64_t)(j & (c.page - 1)) * c.row_bytes + kvh * kHeadRowBytes;
        float k[4];
        row4(c.k + id * c.k_page + at, lane, k);
        float s[1] = {wsum(fmaf(q[0], k[0], fmaf(q[1], k[1], fmaf(q[2], k[2], q[3] * k[3]))))};
        if (c.cap2 != 0.0f) cap_logits(s, c.cap2, c.cap_inv, 0.0f);
        if (c.bias != 0.0f) s[0] = fmaf(-slope, fabsf((float)(far - j)), s[0]);
        const float m = fmaxf(a.m, s[0]), al = a.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(a.m - m);
        const float p = s[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s[0] - m);
        row4(c.v + id * c.v_page + at, lane, k);
        a.m = m, a.l = fmaf(a.l, al, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) a.o[i] = fmaf(a.o[i], al, p * k[i]);
    }
}

__global__ __launch_bounds__(256) void shared_simple_kernel(Shared p) {
    const Call &c = p.c;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = (int)(row / c.H), h = (int)(row - (int64_t)t * c.H);
    if (t >= c.n_tok || t < c.q_start[0] || t >= c.q_start[c.B]) return;
    int lo = 0, hi = c.B;  // the request: the last one that starts at or before t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (c.q_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    const Request rq = request(c, lo);
    const float4a x = *reinterpret_cast<const float4a *>(c.q + t * c.q_nb1 + h * c.q_nb2 + 16 * lane);
    float q[4], amax = 0.0f;
    for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(x[i]));
    for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    const float d = (float)(_Float16)(amax / 127.f) * c.qscale, id = amax != 0.0f ? 127.f / amax : 0.0f;
    for (int i = 0; i < 4; ++i) q[i] = rintf(x[i] * id) * d;
    const float slope = c.bias != 0.0f ? slope2(c, h) : 0.0f;
    const int kvh = group_of(c, h), g = p.token_group[t], i = t - rq.q0;
    const int len = g >= 0 && g < p.groups ? (int)min((int64_t)max(p.len[g], 0), p.most_kv) : 0;
    Online a;
    keys(c, p.table + (len ? g * p.table_stride : 0), len, kvh, lane, q, slope, len + rq.pos0 + i, a);
    keys(c, c.table + lo * c.table_stride, sees(rq, i), kvh, lane, q, slope, rq.pos0 + i, a);
    const float *gate = c.gate ? reinterpret_cast<const float *>(c.gate + t * c.gate_nb2 + h * c.gate_nb1) + 4 * lane : nullptr;
    for (int k = 0; k < 4; ++k) {
        const float o = a.l == 0.0f ? 0.0f : a.o[k] / a.l;
        c.dst[((int64_t)t * c.H + h) * kHeadDim + 4 * lane + k] = gate ? gate_by(o, gate[k]) : o;
    }
}

}  // namespace
}  // namespace paged

using namespace paged;

size_t paged_shared_workspace(int64_t n_tok, int64_t H, int64_t Hkv, int64_t B, int64_t groups, int64_t max_q) {
    (void)H, (void)Hkv, (void)B, (void)groups, (void)max_q;
    return n_tok ? 512 : 0;
}

int launch_paged_shared(const SharedArgs &a, hipStream_t s) {
    if (!a.own.ws || a.own.ws_bytes < 512)
        return set_error(SQA_ERR_WORKSPACE, "paged_attn_shared: workspace %zu bytes < 512 needed", a.own.ws ? a.own.ws_bytes : (size_t)0);
    Shared p{};
    p.c = call_of(a.own);
    p.table = (const int32_t *)a.table->data, p.table_stride = (int64_t)a.table->nb[1] / 4;
    p.most_kv = a.table->ne[0] << p.c.lp;
    p.len = (const int32_t *)a.len->data, p.token_group = (const int32_t *)a.token_group->data;
    p.groups = (int)a.table->ne[1];
    const int prof = profile_start("paged_shared", s);
    shared_simple_kernel<<<dim3((unsigned)(((int64_t)p.c.n_tok * p.c.H + 3) / 4)), dim3(256), 0, s>>>(p);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "paged_attn_shared launch");
}

}  // namespace sqa
