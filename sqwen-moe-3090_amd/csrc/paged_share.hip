// paged_share.hip - which tokens of a step go with which shared prefix.
//
// A request's tokens lie in `members` behind those of lower groups and of the same group's
// earlier requests. One workgroup a request (and one a group, for its first place): it sums
// the lengths of the requests that come before, all of them read again by every workgroup,
// rather than wait for another one's sums; then it writes the request's own tokens.
//
// Bound by latency: arrays, sums, stores. 8 requests 3.0 us, where an empty launch is 2.2; 1024
// with 8192 tokens 4.8 (6.2 with a length loaded behind every group id, and sums through LDS). The
// reads of all by all grow with the square: 4096 requests 20 us, with as many groups 59.
#include "paged_attn.hpp"

namespace sqa {
namespace {

using paged::wave_sum;

struct Range {
    int g, q0, n, kv;
};

// A request's group (n_groups: none, as far as its own arrays say), first token, tokens and length.
__device__ __forceinline__ Range range(const ShareArgs &a, int b) {
    const int g = a.group[b], s0 = a.q_start[b], s1 = a.q_start[b + 1], kv = a.kv_len[b];
    Range r{(uint32_t)g < (uint32_t)a.n_groups && kv > 0 ? g : a.n_groups, min(max(s0, 0), a.T), 0, kv};
    r.n = min(max(s1, r.q0), a.T) - r.q0;
    return r;
}

// 64 threads a workgroup for few requests and tokens: no barrier then.
template <int kThreads>
__global__ __launch_bounds__(kThreads) void paged_share_kernel(ShareArgs a) {
    __shared__ int lens[kThreads], sums[2][kThreads / 64];
    const int tid = threadIdx.x, id = (int)blockIdx.x, G = a.n_groups;
    const bool of_group = id >= a.B, kept = G <= kThreads;
    const Range own = of_group ? Range{id - a.B, 0, 0, 0} : range(a, id);
    const int first = min(max(a.q_start[0], 0), a.T), last = min(max(a.q_start[a.B], 0), a.T);
    Range r = range(a, min(tid, a.B - 1));
    if (kept) lens[tid] = tid < G ? a.shared_len[tid] : 0;
    __syncthreads();
    auto length = [&](int g) { return g < G ? (kept ? lens[g] : a.shared_len[g]) : 0; };
    // tokens of all members, and of those before this request or group (of ranges that overlap the
    // sums may pass T: they stop there)
    int all = 0, before = 0;
    for (int b = tid; b < a.B; b += kThreads) {
        if (b != tid) r = range(a, b);
        const int n = length(r.g) > 0 ? r.n : 0;
        all = min(all + n, a.T);
        before = min(before + (r.g < own.g || (!of_group && r.g == own.g && b < id) ? n : 0), a.T);
    }
    all = min(wave_sum(all), a.T), before = min(wave_sum(before), a.T);
    if (kThreads > 64) {
        if ((tid & 63) == 0) sums[0][tid >> 6] = all, sums[1][tid >> 6] = before;
        __syncthreads();
        all = before = 0;
        for (int w = 0; w < kThreads / 64; ++w) all += sums[0][w], before += sums[1][w];
        all = min(all, a.T), before = min(before, a.T);
    }
    if (of_group) {
        if (tid == 0) a.m_start[own.g] = before;
    } else {
        const int len = length(own.g);
        const bool is = len > 0;
        const int pos0 = (int)min((int64_t)len + own.kv - own.n, (int64_t)INT32_MAX - a.T);
        for (int i = tid; i < own.n; i += kThreads) {
            const int t = own.q0 + i, p = pos0 + i;
            a.token_group[t] = is ? own.g : -1;
            if (!is) continue;
            if (before + i < a.T) a.members[before + i] = t, a.m_pos[before + i] = p;
            if (a.pos)
#pragma unroll
                for (int c = 0; c < 4; ++c) a.pos[(int64_t)c * a.T + t] = p;
        }
    }
    // rows behind the members, and tokens of no request: a part each
    const int r0 = (int)((int64_t)a.T * id / gridDim.x), r1 = (int)((int64_t)a.T * (id + 1) / gridDim.x);
    for (int i = r0 + tid; i < r1; i += kThreads) {
        if (i >= all) a.members[i] = -1, a.m_pos[i] = -1;
        if (i < first || i >= last) a.token_group[i] = -1;
    }
}

}  // namespace

int launch_paged_share(const ShareArgs &a, hipStream_t s) {
    const int prof = profile_start("paged_share", s);
    const dim3 grid((unsigned)(a.B + a.n_groups + 1));
    if (a.B <= 128 && a.T <= 1024) paged_share_kernel<64><<<grid, dim3(64), 0, s>>>(a);
    else paged_share_kernel<256><<<grid, dim3(256), 0, s>>>(a);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "paged_share launch");
}

}  // namespace sqa
