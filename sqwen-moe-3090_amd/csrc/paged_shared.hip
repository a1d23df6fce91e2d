// paged_shared.hip - attention of a batch whose groups of requests share long prefixes: what a
// call launches, its workspace, and the merge of the two parts.
//
// A row's own keys go the way of paged_attn (paged_decode.hip, paged_chunk.hpp). The keys of a
// group's prefix meet the rows of all its tokens at once: the many-row kernel of paged_chunk.hpp
// takes tiles of 128 (or 64) rows out of the group's list of members, so that a key is read and
// expanded once for that many rows instead of once for every request's 8. An extra workgroup of
// the few-row launch plans the tiles and splits. Groups of few rows (a token or two) are pieces of
// the few-row kernel, beside the requests. Every row's parts (splits of its own keys and of
// the prefix) then meet in the merge, M the largest of all their maxima:
//   out = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), then the gate.
#include "paged_merge.hpp"
#include "paged_work.hpp"

namespace sqa {
namespace paged {
namespace {

constexpr int kThreads = 256;

// Rows up to which the merge takes a workgroup a row (merge_parts_kernel): 640 rows of some 50
// parts 8.5 us (a wavefront four rows: 25.9), 2048 of 11 parts 11.0 (16.0), 3200 11.1 (11.0),
// 4096 14.6 (12.7), 16384 39.6 (17.8).
constexpr int kFewRows = 3000;

typedef float floatx4 __attribute__((ext_vector_type(4)));

struct Merge {
    Parts parts;
    const int32_t *token_group;
};

// The parts of a row (R heads of a token): splits of its own keys, then of its group's prefix.
template <int R>
struct RowParts {
    Row a[R], b[R];
    int n1, n;
    bool whole;  // the own keys are one part, normalised
    // false: a row of no request, or left as it is
    __device__ __forceinline__ bool find(const Merge &p, int t, int h0) {
        const Parts &c = p.parts;
        const int4 w1 = c.where[t], w2 = c.g_where[t];
        const int g = p.token_group[t];
        if (t < c.q_start[0] || t >= c.q_start[c.B]) return false;  // the entry was not written
        // (where requests' ranges overlap, more of them than there are slots, an entry may be what the
        // workspace held: there is no `whole` without the chunk kernel)
        whole = c.rows_c && (w1.w & 3) == kWhole;
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int h = min(h0 + k, c.H - 1);
            const int64_t at = (int64_t)t * c.H + h;
            a[k] = whole ? Row{c.whole + at * 256, c.stats + at * 2, 0, 1} : partials(c, w1, h);
            b[k] = partials(c, w2, h);
        }
        n1 = a[0].n;
        n = n1 + (g >= 0 && g < c.groups ? b[0].n : 0);
        return n1 != 0;  // (of the token: all heads alike)
    }
    // (m, l) of part s < n, at ml1 and ml2 of the head
    __device__ __forceinline__ float2 stats(const float *ml1, const float *ml2, int s) const {
        const float *at = s < n1 ? ml1 + s * (a[0].step / 128) : ml2 + (s - n1) * (b[0].step / 128);
        return s < n ? *reinterpret_cast<const float2 *>(at) : make_float2(-INFINITY, 0.0f);
    }
    __device__ __forceinline__ const float *acc(int k, int s) const {
        return s < n1 ? a[k].acc + s * a[k].step : b[k].acc + (s - n1) * b[k].step;
    }
};

// Few rows of many parts: a workgroup a row, its wavefronts every fourth part, 4 dims a lane, so
// that 32 parts are on their way together. Every wavefront takes all weights for itself, a part a
// lane: the maximum over all parts first, then the weights, 64 parts at a time.
__global__ __launch_bounds__(kThreads) void merge_parts_kernel(Merge p) {
    constexpr int kBatch = 8;
    __shared__ floatx4 sum[4][64];
    const Parts &c = p.parts;
    const int t = (int)blockIdx.y + (int)(blockIdx.z << 15), h = (int)blockIdx.x;
    if (t >= c.n_tok) return;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    RowParts<1> r;
    if (!r.find(p, t, h)) return;
    const float *gate = c.gate ? gate_row(c, t, h) + threadIdx.x : nullptr;
    const float g = gate ? *gate : 0.0f;
    float2 ml = r.stats(r.a[0].ml, r.b[0].ml, lane);
    float M = ml.x;
    for (int s0 = 64; s0 < r.n; s0 += 64) M = fmaxf(M, r.stats(r.a[0].ml, r.b[0].ml, s0 + lane).x);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    float L = 0.0f;
    for (int s0 = 0; s0 < r.n; s0 += 64) {
        if (s0) ml = r.stats(r.a[0].ml, r.b[0].ml, s0 + lane);
        const float e = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
        const float l = ml.x == -INFINITY ? 0.0f : ml.y * e, w = r.whole && s0 + lane == 0 ? l : e;
        L += l;
        const int end = min(r.n - s0, 64);
        for (int s1 = wave; s1 < end; s1 += 4 * kBatch) {
            floatx4 x[kBatch];
            float wt[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int s = s1 + 4 * j;
                wt[j] = s < end ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), min(s, 63))) : 0.0f;
                if (wt[j] != 0.0f) x[j] = *reinterpret_cast<const floatx4 *>(r.acc(0, s0 + s) + 4 * lane);
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (wt[j] != 0.0f) o += x[j] * wt[j];
        }
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) L += __shfl_xor(L, x);
    sum[wave][lane] = o;
    __syncthreads();
    const float *s = reinterpret_cast<const float *>(sum) + threadIdx.x;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L, x = ((s[0] + s[256]) + (s[512] + s[768])) * inv;
    c.dst[((int64_t)t * c.H + h) * kHeadDim + threadIdx.x] = gate ? gate_by(x, g) : x;
}

// Many rows: a wavefront takes R heads of a token together, 4 dims a lane; 64 / R parts at a
// time: lane r * 64 / R + i holds part i's weight for head r.
template <int R>
__global__ __launch_bounds__(kThreads) void merge_rows_kernel(Merge p) {
    constexpr int kS = 64 / R, kBatch = 2;
    const Parts &c = p.parts;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int t = (int)blockIdx.y + (int)(blockIdx.z << 15), h0 = ((int)blockIdx.x * 4 + wave) * R;
    if (t >= c.n_tok || h0 >= c.H) return;
    RowParts<R> r;
    if (!r.find(p, t, h0)) return;
    const int k_own = lane / kS, i_own = lane % kS;
    const float *ml1 = r.a[0].ml, *ml2 = r.b[0].ml;
#pragma unroll
    for (int k = 1; k < R; ++k) ml1 = k_own == k ? r.a[k].ml : ml1, ml2 = k_own == k ? r.b[k].ml : ml2;
    floatx4 o[R], g4[R];
    float M = -INFINITY, L = 0.0f;  // of head k_own
#pragma unroll
    for (int k = 0; k < R; ++k) {
        o[k] = floatx4{0.f, 0.f, 0.f, 0.f};
        if (c.gate) g4[k] = *reinterpret_cast<const float4a *>(gate_row(c, t, min(h0 + k, c.H - 1)) + 4 * lane);
    }
    for (int s0 = 0; s0 < r.n; s0 += kS) {
        const float2 ml = r.stats(ml1, ml2, s0 + i_own);
        float m = ml.x;
#pragma unroll
        for (int x = 1; x < kS; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
        const float Mn = fmaxf(M, m), al = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - Mn);
        const float e = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - Mn);
        float l = ml.x == -INFINITY ? 0.0f : ml.y * e;
        const float w = r.whole && s0 + i_own == 0 ? l : e;
#pragma unroll
        for (int x = 1; x < kS; x <<= 1) l += __shfl_xor(l, x);
        L = L * al + l;
        M = Mn;
#pragma unroll
        for (int k = 0; k < R; ++k) o[k] *= __int_as_float(__builtin_amdgcn_readlane(__float_as_int(al), k * kS));
        const int end = min(r.n - s0, kS);
        for (int s1 = 0; s1 < end; s1 += kBatch) {
            floatx4 x[kBatch][R];
            float wt[kBatch][R];
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    wt[j][k] = s1 + j < end ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), k * kS + min(s1 + j, kS - 1))) : 0.0f;
                    if (wt[j][k] != 0.0f) x[j][k] = *reinterpret_cast<const floatx4 *>(r.acc(k, s0 + s1 + j) + 4 * lane);
                }
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
#pragma unroll
                for (int k = 0; k < R; ++k)
                    if (wt[j][k] != 0.0f) o[k] += x[j][k] * wt[j][k];
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
            for (int i = 0; i < 4; ++i) x[i] = gate_by(x[i], g4[k][i]);
        }
        *reinterpret_cast<floatx4 *>(c.dst + ((int64_t)t * c.H + h0 + k) * kHeadDim + 4 * lane) = x;
    }
}

// Workspace of a call: the groups' entries, stats and results of requests in one part (where there
// is a chunk kernel), then what a call without groups has.
struct Space {
    Plan plan;
    size_t where, stats, whole;
    size_t more() const { return where + stats + whole + 256; }
};

Space space(int64_t n_tok, int64_t H, int64_t Hkv, int64_t B, int64_t groups, int64_t max_q) {
    Space s{};
    s.plan = plan_of(n_tok, H, Hkv, B, max_q, groups);
    s.where = al256((size_t)n_tok * 16);
    if (s.plan.rows_c) {  // (also where max_q says that no request is the chunk kernel's)
        s.stats = al256((size_t)(n_tok * H) * 8);
        s.whole = al256((size_t)(n_tok * H) * kHeadDim * 4);
    }
    return s;
}

}  // namespace
}  // namespace paged

using namespace paged;

size_t paged_shared_workspace(int64_t n_tok, int64_t H, int64_t Hkv, int64_t B, int64_t groups, int64_t max_q) {
    if (n_tok < 1) return 0;
    const Space s = space(n_tok, H, Hkv, B, groups, max_q);
    return s.more() + full_bytes(s.plan);
}

int launch_paged_shared(const SharedArgs &a, hipStream_t s) {
    const char *what = "paged_attn_shared";
    Merge m{};
    Parts &c = m.parts;
    static_cast<Call &>(c) = call_of(a.own);
    c.groups = (int)a.table->ne[1];
    c.g_table = (const int32_t *)a.table->data, c.g_stride = (int64_t)a.table->nb[1] / 4;
    c.g_most_kv = a.table->ne[0] << c.lp;
    c.g_len = (const int32_t *)a.len->data, c.m_start = (const int32_t *)a.m_start->data;
    c.members = (const int32_t *)a.members->data, c.m_pos = (const int32_t *)a.m_pos->data;
    m.token_group = (const int32_t *)a.token_group->data;

    const Space sp = space(c.n_tok, c.H, c.Hkv, c.B, c.groups, a.own.max_q);
    const size_t least = sp.more() + least_bytes(sp.plan);
    if (!a.own.ws || a.own.ws_bytes < least)
        return set_error(SQA_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu needed", what, a.own.ws ? a.own.ws_bytes : (size_t)0, least);
    uint8_t *base = reinterpret_cast<uint8_t *>(((uintptr_t)a.own.ws + 255) & ~(uintptr_t)255);
    c.g_where = reinterpret_cast<int4 *>(base);
    c.stats = reinterpret_cast<float *>(base + sp.where);
    c.whole = reinterpret_cast<float *>(base + sp.where + sp.stats);
    int rc = lay_out(c, sp.plan, base + sp.more() - 256, a.own.ws_bytes - sp.more(), what);
    if (rc) return rc;

    rc = launch_few(c, s);
    if (!rc && c.rows_c) rc = launch_many(c, s);
    if (rc) return rc;

    const int prof = profile_start("paged_shared_merge", s);
    const bool few = (int64_t)c.n_tok * c.H <= kFewRows;
    const unsigned y = (unsigned)(c.n_tok < (1 << 15) ? c.n_tok : 1 << 15), z = (unsigned)((c.n_tok + (1 << 15) - 1) >> 15);
    if (few) merge_parts_kernel<<<dim3((unsigned)c.H, y, z), dim3(kThreads), 0, s>>>(m);
    else merge_rows_kernel<4><<<dim3((unsigned)((c.H + 15) / 16), y, z), dim3(kThreads), 0, s>>>(m);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "paged_attn_shared merge launch");
}

}  // namespace sqa
