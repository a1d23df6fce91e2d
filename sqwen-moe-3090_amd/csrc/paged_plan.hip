// paged_plan.hip - page table, slot map and request bounds of a step, on the GPU.
//
// With new_b = max(n_new[b], 0) and have_b = ceil(past_b / page):
//   end_b  = sum of new up to and with b        (token rows; q_start is its shift)
//   rel_b  = sum of have over ended requests    (pages that come back)
//   need_b = ceil((past_b + new_b) / page) - have_b, 0 where b's tokens fit nowhere
//   upto_b = sum of need up to and with b
// A request is served where it fits and upto_b <= count + rel (or it needs none): in order,
// what a refused one needs stays in the sums of those behind it.
// Three prefix sums over the batch and then work of its own for every token: its
// request by a search in end, its page from the table, or, on a fresh page, from
// the ring at head + upto_b - need_b + i (behind the ring's old pages: from the
// ended request that gives it).
//
// Bound by latency: a dependent chain of loads (lengths, table or ring entry), two scans
// and the launch; a step's arrays are some 10 to 300 KB: 8 requests 3.8 us (4.6 from call to
// call, the host's time), 1024 requests with 8192 tokens 8.5 (8.6); an empty launch takes
// 3.6. 256 threads, so four of 1024 requests each in the scans. Every workgroup takes the
// prefix sums again for itself (B lengths, in LDS) instead of waiting for another
// one's, so one launch does all; tokens, table entries and returned pages are then
// spread over the workgroups, none of which reads what another one writes: a token
// on an old page reads an entry that this step leaves alone, one on a fresh page
// takes the page id where the table's new entry comes from.
#include <mutex>

#include "paged.hpp"

namespace sqa {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMany = 1u << 30;  // token sums stop here (T is at most 2^29)

// v plus the lane's v that a DPP control names (0 where there is none, or the row is masked
// off), saturating at kMany.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t add_dpp(uint32_t v) {
    return min(v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xf, false), kMany);
}

// Inclusive sums over the wavefront: within rows of 16 lanes, then the rows before.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = add_dpp<0x118, 0xf>(add_dpp<0x114, 0xf>(add_dpp<0x112, 0xf>(add_dpp<0x111, 0xf>(v))));
    return add_dpp<0x143, 0xc>(add_dpp<0x142, 0xa>(v));
}

// Inclusive sums over the workgroup's threads of n values at once.
template <int n>
__device__ __forceinline__ void wg_scan(uint32_t (&v)[n], uint32_t (*sums)[4]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < n; ++i) {
        v[i] = wave_scan(v[i]);
        if (lane == 63) sums[i][wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < n; ++i)
#pragma unroll
        for (int w = 0; w < kThreads / 64 - 1; ++w) v[i] = min(v[i] + (w < wave ? sums[i][w] : 0u), kMany);
}

// First index of the n sorted values that is above x (n: none).
__device__ __forceinline__ int above(const uint32_t *v, int n, uint32_t x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__global__ __launch_bounds__(kThreads) void paged_plan_kernel(PlanArgs a) {
    extern __shared__ uint32_t lds[];
    __shared__ uint32_t sums[3][4];
    uint32_t *end = lds, *rel = lds + a.B, *upto = lds + 2 * a.B;
    int32_t *n_past = reinterpret_cast<int32_t *>(lds + 3 * a.B), *n_new = n_past + a.B;
    const int tid = threadIdx.x;
    const int lp = __ffs(a.page) - 1;
    const int64_t most = (int64_t)a.W << lp;
    auto past_of = [&](int b) { return (uint32_t)max(n_past[b], 0); };
    auto new_of = [&](int b) { return (uint32_t)max(n_new[b], 0); };
    auto pages = [&](int64_t n) { return (uint32_t)((n + a.page - 1) >> lp); };
    const int n_pages = a.n_pages;
    int head = a.state[0], count = a.state[1];
    head = head < 0 || head >= n_pages ? 0 : head;
    count = min(max(count, 0), n_pages);

    // the lengths, read once and 4 at a time (by the thread of their run, a latency after the
    // other, 1024 requests took 10.1 us, with the sums by shuffles; now 8.6)
    constexpr int kBatch = 4;
    for (int b = tid; b < a.B; b += kBatch * kThreads) {
        int32_t p[kBatch], n[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int at = min(b + i * kThreads, a.B - 1);
            p[i] = a.n_past[at], n[i] = a.n_new[at];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (b + i * kThreads < a.B) n_past[b + i * kThreads] = p[i], n_new[b + i * kThreads] = n[i];
    }
    __syncthreads();
    // a thread's run of requests, then the sums before it
    const int per = (a.B + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    uint32_t n_tok = 0, n_rel = 0;
    for (int b = b0; b < b1; ++b) {
        n_tok = min(n_tok + min(new_of(b), (uint32_t)a.T + 1), kMany);
        end[b] = n_tok;
        if (n_new[b] < 0) n_rel += min(pages(past_of(b)), (uint32_t)a.W);
        rel[b] = n_rel;
    }
    uint32_t upto_run[2] = {n_tok, n_rel};
    wg_scan(upto_run, sums);
    // sums of the runs before this one: read from the neighbour, not by a subtraction (they saturate)
    __shared__ uint32_t before[2][kThreads + 1];
    before[0][tid + 1] = upto_run[0];
    before[1][tid + 1] = upto_run[1];
    if (tid == 0) before[0][0] = before[1][0] = 0;
    __syncthreads();
    uint32_t n_need = 0;
    for (int b = b0; b < b1; ++b) {
        end[b] = min(end[b] + before[0][tid], kMany);
        rel[b] += before[1][tid];
        const int64_t past = past_of(b), now = past + new_of(b);
        if (n_new[b] >= 0 && now <= most && end[b] <= (uint32_t)a.T) n_need += pages(now) - pages(past);
        upto[b] = n_need;
    }
    uint32_t need_upto[1] = {n_need};
    wg_scan(need_upto, sums + 2);
    for (int b = b0; b < b1; ++b) upto[b] += need_upto[0] - n_need;
    const uint32_t returned = before[1][kThreads];
    const uint32_t avail = min((uint32_t)count + returned, (uint32_t)n_pages);
    __syncthreads();

    auto need_of = [&](int b) { return upto[b] - (b ? upto[b - 1] : 0u); };
    auto served = [&](int b) {
        const int64_t now = (int64_t)past_of(b) + new_of(b);
        return n_new[b] >= 0 && now <= most && end[b] <= (uint32_t)a.T && (need_of(b) == 0 || upto[b] <= avail);
    };
    // page id of the i-th returned page, of the i-th page that leaves the ring
    auto given_back = [&](uint32_t i) {
        const int b = above(rel, a.B, i);
        return a.table[b * a.table_stride + (i - (b ? rel[b - 1] : 0u))];
    };
    auto taken = [&](uint32_t i) {
        if (i >= (uint32_t)count) return given_back(i - (uint32_t)count);
        const uint32_t at = (uint32_t)head + i;
        return a.ring[at < (uint32_t)n_pages ? at : at - (uint32_t)n_pages];
    };

    const int stride = gridDim.x * kThreads, first = blockIdx.x * kThreads + tid;
    for (int t = first; t < a.T; t += stride) {
        const int b = above(end, a.B, (uint32_t)t);
        int64_t slot = -1;
        int32_t p = 0;
        if (b < a.B && served(b)) {
            const uint32_t past = past_of(b);
            p = (int32_t)(past + ((uint32_t)t - (b ? end[b - 1] : 0u)));
            const uint32_t entry = (uint32_t)p >> lp, have = pages(past);
            int32_t *row = a.table + b * a.table_stride;
            int32_t id;
            if (entry >= have) {
                id = taken(upto[b] - need_of(b) + entry - have);
                if ((p & (a.page - 1)) == 0) row[entry] = id;  // a fresh page starts with a new token
            } else {
                id = row[entry];
            }
            if (id >= 0 && id < n_pages) slot = ((int64_t)id << lp) + (p & (a.page - 1));
        }
        a.slots[t] = slot;
#pragma unroll
        for (int k = 0; k < 4; ++k) a.pos[(int64_t)k * a.T + t] = p;
    }
    for (uint32_t i = first; i < avail - min(avail, (uint32_t)count); i += stride) {
        const uint32_t at = (uint32_t)head + (uint32_t)count + i;
        a.ring[at < (uint32_t)n_pages ? at : at - (uint32_t)n_pages] = given_back(i);
    }
    if (blockIdx.x) return;
    uint32_t popped = 0, refused = 0;
    for (int b = b0; b < b1; ++b) {
        const int32_t past = (int32_t)past_of(b), now = past + (int32_t)new_of(b);
        const bool ok = served(b), ended = n_new[b] < 0;
        if (ok && need_of(b)) popped = max(popped, upto[b]);
        refused += !ok && !ended;
        a.q_start[b + 1] = (int32_t)min(end[b], (uint32_t)a.T);
        a.kv_len[b] = ok ? now : 0;
        a.n_past_out[b] = ok ? now : (ended ? 0 : past);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        popped = max(popped, (uint32_t)__shfl_xor((int)popped, o));
        refused += (uint32_t)__shfl_xor((int)refused, o);
    }
    __syncthreads();
    if ((tid & 63) == 0) before[0][tid >> 6] = popped, before[1][tid >> 6] = refused;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 64; ++w) popped = max(popped, before[0][w]), refused += before[1][w];
        const uint32_t at = (uint32_t)head + popped;
        a.state_out[0] = (int32_t)(at < (uint32_t)n_pages ? at : at - (uint32_t)n_pages);
        a.state_out[1] = (int32_t)(avail - popped);
        a.state_out[2] = (int32_t)refused;
        a.state_out[3] = (int32_t)min(end[a.B - 1], (uint32_t)a.T);
        a.q_start[0] = 0;
    }
}

}  // namespace

int launch_paged_plan(const PlanArgs &a, hipStream_t s) {
    int grid = (a.T + kThreads - 1) / kThreads;
    grid = grid < 1 ? 1 : (grid > 256 ? 256 : grid);
    static std::once_flag once;  // the LDS limit is raised once per process
    static hipError_t err = hipSuccess;
    std::call_once(once, [] {
        err = hipFuncSetAttribute((const void *)paged_plan_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 20 * kMaxRequests);
    });
    if (err != hipSuccess) return hip_status(err, "paged_plan LDS attribute");
    const int prof = profile_start("paged_plan", s);
    paged_plan_kernel<<<dim3((unsigned)grid), dim3(kThreads), 20 * (size_t)a.B, s>>>(a);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "paged_plan launch");
}

}  // namespace sqa
