// paged_share.hip - which tokens of a step go with which shared prefix.
//
// A request's tokens lie in `members` behind those of lower groups and of the same group's
// earlier requests. One workgroup a request (and one a group, for its first place): it sums
// the lengths of the requests that come before, all of them read again by every workgroup,
// rather than wait for another one's sums; then it writes the request's own tokens.
#include "paged.hpp"

namespace sqa {
namespace {

constexpr int kThreads = 256;

struct Member {
    int g, q0, n, pos0;  // group (n_groups: none), first token, tokens, position of the first one
};

__device__ __forceinline__ Member member(const ShareArgs &a, int b) {
    const int g = a.group[b], s0 = a.q_start[b], s1 = a.q_start[b + 1], kv = a.kv_len[b];
    Member m{a.n_groups, min(max(s0, 0), a.T), 0, 0};
    m.n = min(max(s1, m.q0), a.T) - m.q0;
    if (g < 0 || g >= a.n_groups || kv <= 0) return m;
    const int len = a.shared_len[g];
    if (len <= 0) return m;
    m.g = g;
    m.pos0 = (int)min((int64_t)len + kv - m.n, (int64_t)INT32_MAX - a.T);
    return m;
}

__global__ __launch_bounds__(kThreads) void paged_share_kernel(ShareArgs a) {
    __shared__ int64_t sums[2][kThreads / 64];
    const int tid = threadIdx.x, id = (int)blockIdx.x;
    const bool of_group = id >= a.B;
    const Member own = of_group ? Member{id - a.B, 0, 0, 0} : member(a, id);
    // tokens of all members, and of those before this request or group
    int64_t all = 0, before = 0;
    for (int b = tid; b < a.B; b += kThreads) {
        const Member m = member(a, b);
        if (m.g == a.n_groups) continue;
        all += m.n;
        if (m.g < own.g || (!of_group && m.g == own.g && b < id)) before += m.n;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) all += __shfl_xor(all, o), before += __shfl_xor(before, o);
    if ((tid & 63) == 0) sums[0][tid >> 6] = all, sums[1][tid >> 6] = before;
    __syncthreads();
    all = before = 0;
    for (int w = 0; w < kThreads / 64; ++w) all += sums[0][w], before += sums[1][w];
    const int M = (int)min(all, (int64_t)a.T);
    if (of_group) {
        if (tid == 0) a.m_start[own.g] = (int)min(before, (int64_t)a.T);
    } else {
        const bool is = own.g < a.n_groups;
        for (int i = tid; i < own.n; i += kThreads) {
            const int t = own.q0 + i, p = own.pos0 + i;
            a.token_group[t] = is ? own.g : -1;
            if (!is) continue;
            if (before + i < a.T) a.members[before + i] = t, a.m_pos[before + i] = p;
            if (a.pos)
#pragma unroll
                for (int c = 0; c < 4; ++c) a.pos[(int64_t)c * a.T + t] = p;
        }
    }
    // rows behind the members, and tokens of no request: a part each
    const int first = min(max(a.q_start[0], 0), a.T), last = min(max(a.q_start[a.B], 0), a.T);
    const int r0 = (int)((int64_t)a.T * id / gridDim.x), r1 = (int)((int64_t)a.T * (id + 1) / gridDim.x);
    for (int r = r0 + tid; r < r1; r += kThreads) {
        if (r >= M) a.members[r] = -1, a.m_pos[r] = -1;
        if (r < first || r >= last) a.token_group[r] = -1;
    }
}

}  // namespace

int launch_paged_share(const ShareArgs &a, hipStream_t s) {
    const int prof = profile_start("paged_share", s);
    paged_share_kernel<<<dim3((unsigned)(a.B + a.n_groups + 1)), dim3(kThreads), 0, s>>>(a);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "paged_share launch");
}

}  // namespace sqa
