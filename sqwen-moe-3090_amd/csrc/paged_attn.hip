// paged_attn.hip - attention of a batch of requests over a paged q4_0 pool: what a
// call launches, its workspace, and the merge of split partials.
//
// Requests of few query rows (up to 16 per KV head; up to 8 where larger ones may be
// in the call) go to paged_decode.hip, the others to paged_chunk.hpp's kernel.
#include <float.h>

#include "paged_merge.hpp"
#include "paged_work.hpp"

namespace sqa {
namespace paged {
namespace {

constexpr int kThreads = 256;

typedef float floatx4 __attribute__((ext_vector_type(4)));
// Merge of a row's partials: out = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), M = max m_s,
// then the gate. m is in base 2 as the kernels hold it: through base e and back, 50 nats lost 2e-6
// of a split's weight. A partial whose m is -inf (no key seen) may hold anything.
__device__ __forceinline__ Row row_of(const Call &c, int t, int h) {
    const int4 w = c.where[t];
    if (t < c.q_start[0] || t >= c.q_start[c.B]) return Row{nullptr, nullptr, 0, 0};  // of no request: w was not written
    return partials(c, w, h);
}

// Few rows of many splits: 16 workgroups per row, 16 dims each; a thread holds one dim
// of every 16th split, all its loads in flight together.
__global__ __launch_bounds__(kThreads) void merge_dims_kernel(Call c) {
    __shared__ float xm[4], xl[4], xo[4][16];
    const int t = blockIdx.x / c.H, h = blockIdx.x - t * c.H;
    const Row r = row_of(c, t, h);
    if (r.n == 0) return;
    const int tid = threadIdx.x, dl = tid & 15, sg = tid >> 4, d = blockIdx.y * 16 + dl;
    float acc[16];
    float2 ml[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int s = sg + 16 * j;
        const bool ok = s < r.n;
        acc[j] = ok ? r.acc[s * r.step + d] : 0.0f;
        ml[j] = ok ? *reinterpret_cast<const float2 *>(r.ml + s * (r.step / 128)) : make_float2(-INFINITY, 0.0f);
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; ++j) m = fmaxf(m, ml[j].x);
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    if ((tid & 63) == 0) xm[tid >> 6] = m;
    __syncthreads();
    const float M = fmaxf(fmaxf(xm[0], xm[1]), fmaxf(xm[2], xm[3]));
    float o = 0.0f, l = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const bool dead = ml[j].x == -INFINITY;
        const float w = dead ? 0.0f : __builtin_amdgcn_exp2f(ml[j].x - M);
        o = dead ? o : fmaf(acc[j], w, o);
        l = dead ? l : fmaf(ml[j].y, w, l);
    }
    o += __shfl_xor(o, 16);
    o += __shfl_xor(o, 32);
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if ((tid & 63) < 16) xo[tid >> 6][dl] = o;
    if ((tid & 63) == 0) xl[tid >> 6] = l;
    __syncthreads();
    if (tid < 16) {
        const float L = (xl[0] + xl[1]) + (xl[2] + xl[3]), O = (xo[0][dl] + xo[1][dl]) + (xo[2][dl] + xo[3][dl]);
        const float o = L == 0.0f ? 0.0f : O / L;
        c.dst[((int64_t)t * c.H + h) * kHeadDim + d] = c.gate ? gate_by(o, gate_row(c, t, h)[d]) : o;
    }
}

// Many rows: a wavefront takes R heads of a token together, 4 dims a lane, so that their
// loads share one memory latency after the other (row entry, (m, l), partials). Bound by
// those three for decode (64 rows of 16 heads: 4.8 us) and by the partials' bytes for
// chunks (972 tokens of 16 heads, 3 splits, gated: 71 MB in 17 us). 64 / R
// splits at a time: lane r * 64 / R + i holds split i's weight for head r.
template <int R>
__global__ __launch_bounds__(kThreads) void merge_rows_kernel(Call c) {
    constexpr int kS = 64 / R, kBatch = R >= 4 ? 2 : 8;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int t = (int)blockIdx.y + (int)(blockIdx.z << 15), h0 = ((int)blockIdx.x * 4 + wave) * R;
    if (t >= c.n_tok || h0 >= c.H) return;
    Row r[R];
#pragma unroll
    for (int k = 0; k < R; ++k) r[k] = row_of(c, t, min(h0 + k, c.H - 1));
    if (r[0].n == 0) return;  // of the token: all heads alike
    const int n = r[0].n, k_own = lane / kS, i_own = lane % kS;
    const float *ml_own = r[0].ml;
#pragma unroll
    for (int k = 1; k < R; ++k) ml_own = k_own == k ? r[k].ml : ml_own;
    floatx4 o[R], g[R];
    float M = -INFINITY, L = 0.0f;  // of head k_own
#pragma unroll
    for (int k = 0; k < R; ++k) {
        o[k] = floatx4{0.f, 0.f, 0.f, 0.f};
        if (c.gate) g[k] = *reinterpret_cast<const float4a *>(gate_row(c, t, min(h0 + k, c.H - 1)) + 4 * lane);
    }
    for (int s0 = 0; s0 < n; s0 += kS) {
        const int s = s0 + i_own;
        const float2 ml = s < n ? *reinterpret_cast<const float2 *>(ml_own + s * (r[0].step / 128)) : make_float2(-INFINITY, 0.0f);
        float m = ml.x;
#pragma unroll
        for (int x = 1; x < kS; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
        const float Mn = fmaxf(M, m), al = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - Mn);
        const float w = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - Mn);
        float l = ml.x == -INFINITY ? 0.0f : ml.y * w;
#pragma unroll
        for (int x = 1; x < kS; x <<= 1) l += __shfl_xor(l, x);
        L = L * al + l;
        M = Mn;
#pragma unroll
        for (int k = 0; k < R; ++k) o[k] *= __int_as_float(__builtin_amdgcn_readlane(__float_as_int(al), k * kS));
        const int end = min(n - s0, kS);
        for (int s1 = 0; s1 < end; s1 += kBatch) {
            floatx4 a[kBatch][R];
            float wt[kBatch][R];
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    wt[j][k] = s1 + j < end ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), k * kS + min(s1 + j, kS - 1))) : 0.0f;
                    if (wt[j][k] != 0.0f)
                        a[j][k] = *reinterpret_cast<const floatx4 *>(r[k].acc + (s0 + s1 + j) * r[k].step + 4 * lane);
                }
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
#pragma unroll
                for (int k = 0; k < R; ++k)
                    if (wt[j][k] != 0.0f) o[k] += a[j][k] * wt[j][k];
        }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
        if (h0 + k >= c.H) break;
        const float Lk = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(L), k * kS));
        const float inv = Lk == 0.0f ? 0.0f : 1.0f / Lk;
        floatx4 x = o[k] * inv;
        if (c.gate) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = gate_by(x[i], g[k][i]);
        }
        *reinterpret_cast<floatx4 *>(c.dst + ((int64_t)t * c.H + h0 + k) * kHeadDim + 4 * lane) = x;
    }
}

}  // namespace

int launch_combine(const Call &c, hipStream_t s) {
    const int prof = profile_start("paged_merge", s);
    const int64_t rows = (int64_t)c.n_tok * c.H;
    // 16 workgroups a row below 128 rows: requests of 8000 keys with 16 rows each, the whole call
    // with these and with a wavefront a row: 16 rows 11.5 and 23.9 us, 64 15.3 and 17.4, 112 20.9
    // and 20.7, 128 22.8 and 21.8, 192 26.9 and 24.8.
    if (rows < 128) {
        merge_dims_kernel<<<dim3((unsigned)rows, 16), dim3(kThreads), 0, s>>>(c);
    } else {
        // four heads a wavefront where that leaves wavefronts enough for the chip
        const bool four = rows > 8192 && c.H >= 16;
        const dim3 grid((unsigned)((c.H + (four ? 16 : 4) - 1) / (four ? 16 : 4)),
                        (unsigned)(c.n_tok < (1 << 15) ? c.n_tok : 1 << 15), (unsigned)((c.n_tok + (1 << 15) - 1) >> 15));
        if (four) merge_rows_kernel<4><<<grid, dim3(kThreads), 0, s>>>(c);
        else merge_rows_kernel<1><<<grid, dim3(kThreads), 0, s>>>(c);
    }
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "paged_attn merge launch");
}

Plan plan_of(int64_t n_tok, int64_t H, int64_t Hkv, int64_t B, int64_t max_q, int64_t groups) {
    Plan p{};
    const int64_t G = H / Hkv, rows = (max_q < n_tok ? max_q : n_tok) * G, cus = device_cu_count();
    const int64_t active = B < n_tok ? B : n_tok;
    p.most_d = rows <= 8 || (rows > 16 && G <= 8) ? 8 : 16;
    if (groups && rows <= 8 && n_tok * G > 8 && n_tok * G <= 16) p.most_d = 16;  // a group may be all the tokens
    p.rows_d = p.most_d;
    const int64_t P = 2 * cus / Hkv;  // pieces that are wanted at most
    const int64_t parts = active + (groups < n_tok ? groups : n_tok);
    p.slots_d = ((P < 1 ? 1 : P) + parts) * Hkv;
    p.least_d = (1 + parts) * Hkv;
    p.where = al256((size_t)n_tok * 16);
    p.slot_d = (size_t)p.rows_d * (kHeadDim + 2) * 4;
    if (rows > p.most_d || (groups && n_tok * G > p.most_d)) {
        p.rows_c = (groups ? n_tok * G : rows) <= 64 ? 64 : 128;
        // whole query tiles and a last one of every request; three rounds where that is less
        const int64_t tile = p.rows_c / G, wgs = (n_tok / tile + active) * Hkv;
        // those of the groups, each of them a slot at least
        p.least_c = groups ? (n_tok / tile + (groups < n_tok ? groups : n_tok)) * Hkv : 0;
        p.grid_c = (wgs + p.least_c + cus > 3 * cus ? wgs + p.least_c + cus : 3 * cus) + 7 & ~(int64_t)7;
        p.slots_c = p.least_c + cus > 3 * cus ? p.least_c + cus : 3 * cus;
        p.work = al256(work_bytes(B + groups));
        p.slot_c = (size_t)p.rows_c * (kHeadDim + 2) * 4;
    }
    return p;
}

size_t least_bytes(const Plan &p) {
    return p.where + p.work + (size_t)p.least_d * p.slot_d + (size_t)p.least_c * p.slot_c + 512;
}
size_t full_bytes(const Plan &p) {
    return p.where + p.work + (size_t)p.slots_d * p.slot_d + (size_t)p.slots_c * p.slot_c + 512;
}

int lay_out(Call &c, const Plan &p, void *ws, size_t ws_bytes, const char *what) {
    const size_t need = least_bytes(p);
    if (!ws || ws_bytes < need)
        return set_error(SQA_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu needed", what, ws ? ws_bytes : (size_t)0, need);
    if (p.grid_c > INT32_MAX) return set_error(SQA_ERR_UNSUPPORTED, "%s: too many query tiles", what);
    size_t left = ws_bytes - 512 - p.where - p.work;
    c.most_d = p.most_d, c.rows_d = p.rows_d, c.rows_c = p.rows_c, c.grid_c = (int)p.grid_c;
    auto take = [&left](int64_t slots, size_t bytes) {
        if (!slots || (size_t)slots > left / bytes) slots = slots ? (int64_t)(left / bytes) : 0;
        left -= (size_t)slots * bytes;
        return (int)slots;
    };
    left -= (size_t)p.least_c * p.slot_c;  // what the chunk kernel cannot do without
    c.slots_d = take(p.slots_d, p.slot_d);
    left += (size_t)p.least_c * p.slot_c;
    c.slots_c = take(p.slots_c, p.slot_c);
    c.room = c.slots_d / c.Hkv;
    c.few_pieces = c.cus / c.Hkv, c.all_pieces = 2 * c.cus / c.Hkv;
    uint8_t *base = reinterpret_cast<uint8_t *>(((uintptr_t)ws + 255) & ~(uintptr_t)255);
    c.where = reinterpret_cast<int4 *>(base);
    c.work = reinterpret_cast<int *>(base + p.where);
    c.acc_d = reinterpret_cast<float *>(base + p.where + p.work);
    c.acc_c = c.acc_d + (size_t)c.slots_d * c.rows_d * kHeadDim;
    c.ml_d = c.acc_c + (size_t)c.slots_c * c.rows_c * kHeadDim;
    c.ml_c = c.ml_d + (size_t)c.slots_d * c.rows_d * 2;
    return SQA_OK;
}

Call call_of(const PagedArgs &a) {
    const sqa_tensor &q = *a.q, &k = *a.k;
    Call c{};
    c.q = (const char *)q.data, c.q_nb1 = (int64_t)q.nb[1], c.q_nb2 = (int64_t)q.nb[2];
    c.k = (const uint8_t *)k.data, c.v = (const uint8_t *)a.v->data;
    c.k_page = (int64_t)k.nb[3], c.v_page = (int64_t)a.v->nb[3];
    c.row_bytes = (int)k.nb[2];
    c.n_pages = (int)k.ne[3], c.page = (int)k.ne[2];
    while ((1 << c.lp) < c.page) ++c.lp;
    c.table = (const int32_t *)a.table->data, c.table_stride = (int64_t)a.table->nb[1] / 4;
    c.most_kv = a.table->ne[0] << c.lp;
    c.B = (int)a.table->ne[1];
    c.q_start = (const int32_t *)a.q_start->data, c.kv_len = (const int32_t *)a.kv_len->data;
    c.prefix = a.prefix ? (const int32_t *)a.prefix->data : nullptr;
    c.n_tok = (int)q.ne[1], c.H = (int)q.ne[2], c.Hkv = (int)k.ne[1], c.G = c.H / c.Hkv;
    c.inv_g = 1.0f / (float)c.G;
    c.qscale = a.scale * kLog2e;
    // (a cap beyond the range is none; the inverse of one below it stays finite, so that 0 stays 0)
    c.cap2 = a.softcap * kLog2e;
    if (c.cap2 > FLT_MAX) c.cap2 = 0.0f;
    c.cap_inv = c.cap2 > 0.0f ? fminf(1.0f / c.cap2, FLT_MAX) : 0.0f;
    c.bias = a.max_bias;
    c.nl2 = 1;
    while (2 * c.nl2 <= c.H) c.nl2 *= 2;
    c.gate = a.gate ? (const char *)a.gate->data : nullptr;
    c.gate_nb1 = a.gate ? (int64_t)a.gate->nb[1] : 0, c.gate_nb2 = a.gate ? (int64_t)a.gate->nb[2] : 0;
    c.dst = (float *)a.dst->data;
    c.cus = device_cu_count();
    return c;
}

}  // namespace paged

using namespace paged;

size_t paged_attn_workspace(int64_t n_tok, int64_t H, int64_t Hkv, int64_t B, int64_t max_q) {
    if (n_tok < 1) return 0;
    const Plan p = plan_of(n_tok, H, Hkv, B, max_q);
    return full_bytes(p);
}

int launch_paged_attn(const PagedArgs &a, hipStream_t s) {
    Call c = call_of(a);
    const Plan p = plan_of(c.n_tok, c.H, c.Hkv, c.B, a.max_q);
    int rc = lay_out(c, p, a.ws, a.ws_bytes, "paged_attn");
    if (rc) return rc;
    rc = launch_few(c, s);
    if (rc) return rc;
    if (p.rows_c) {
        rc = launch_many(c, s);
        if (rc) return rc;
    }
    return launch_combine(c, s);
}

}  // namespace sqa
