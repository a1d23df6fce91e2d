// paged_work.hpp - how the many-row kernel's work is cut up and ordered, for one
// workgroup of 512 threads. Lengths are known on the GPU only; the plan is made by an
// extra workgroup of the few-row kernel's launch, which runs before, so that the many
// workgroups of the chunk kernel need a few loads to know their part (each making the
// choice for itself took 5 us of every workgroup's time).
#pragma once
#include "paged_attn.hpp"

namespace sqa {
namespace paged {

constexpr int kChunkKeys = 32;   // keys per tile of the chunk kernel
constexpr int kMostSplits = 256; // of a request (the merge's limit)
constexpr int kListed = 4088;    // items up to which the plan is a list in the order of dispatch

// What the plan leaves in the workspace.
struct Work {
    int len;       // key tiles per split, at most
    int items;     // workgroups with work
    int listed;    // whether the list holds them, in the order of dispatch
    int even;      // else: equal parts, renumbered by XCD
};

// A workgroup's part of the call: query tile `tile` of request b's `tiles`, KV head kvh,
// split `split` of `splits`, key tiles [t0, t1); slot: the request's first one (splits > 1).
// b < 0: none.
struct Item {
    int b, kvh, tile, tiles, split, splits, t0, t1, slot;
    Request rq;
    int spare[2];
};
static_assert(sizeof(Item) == 64, "one scalar load");

// Words: Work | list [kListed] of Item | first item of every entry [E + 1] | first slot [E]
constexpr int kListAt = 16, kFirstAt = kListAt + 16 * kListed;
__host__ __device__ inline size_t work_bytes(int64_t B) { return (size_t)(kFirstAt + 2 * B + 4) * 4; }

// Where item `id` of `items` equal parts stands in the order of dispatch: workgroups go
// round-robin to the 8 XCDs, and an XCD gets a run of ids, the query tiles of the same
// keys, which its L2 then serves to all of them.
__device__ __forceinline__ int id_of_workgroup(int lin, int items) {  // -1: none
    const int x = lin & 7, per = items >> 3, rem = items & 7, k = lin >> 3;
    return k >= per + (x < rem ? 1 : 0) ? -1 : x * per + min(x, rem) + k;
}

// Query tiles of a request (0: none of the many-row kernel's) and its key tiles.
__device__ __forceinline__ int chunk_tiles(const Call &c, const Request &r, int qb, int *key_tiles) {
    *key_tiles = 0;
    if (r.n * c.G <= c.most_d) return 0;
    *key_tiles = max((r.kv + kChunkKeys - 1) / kChunkKeys, 1);
    return div_ceil(r.n, qb);
}

// Split `split` of S of kt key tiles.
__device__ __forceinline__ void split_range(int kt, int S, int split, int *t0, int *t1) {
    const int q = div_floor(kt, S), rest = kt - q * S;  // the first `rest` are one longer
    *t0 = split * q + min(split, rest);
    *t1 = *t0 + q + (split < rest);
}

#ifdef SQA_PLAN_CHUNKS

constexpr int kChoices = 16;
// splits of the longest request that are tried
__device__ constexpr int kTried[kChoices] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64, 128};

// Every request is cut into splits of at most `len` key tiles, the same for all, with
// the len of the least estimated time, in tiles of one workgroup (2.4 us): kWg for a
// workgroup's own start and end (11 us), kMerge and kMergeSlot for the merge's start and
// the bytes of a slot. Items go out longest first, one per CU; the time is the work over
// the CUs and a tenth of a part, and at least j + 1 times the (j CUs)-th longest item,
// since j + 1 of the items down to it meet on some CU (counted for lengths of 1/8 to 8/8
// of a part, where there are up to 4 items a CU). Batches of more than kCounted requests, whose items are many, take a quarter
// of a part instead. Against the best of the tried lengths, in a simulation of 129 random
// batches, this costs 0.3% on average and 7% at most.
constexpr float kWg = 4.5f, kMerge = 0.7f, kMergeSlot = 0.014f;
constexpr int kCounted = 64, kLevels = 8, kRounds = 4;
constexpr int kPlanKept = 2300, kTriedAt = 1024;  // entries that LDS holds whole; where the tried lengths stand in it

// Groups of a shared prefix are requests whose tokens all see all keys and whose parts all go
// through the merge.
//
// Run by all 512 threads of one workgroup; lds: 513 + 7 E words for E entries, 513 + E above kPlanKept, and the
// tried lengths.
// Lanes are requests (a run of them above 512), then lengths that are tried, then items.
template <class C>
__device__ __forceinline__ void plan_chunks(const C &c, int *lds) {
    const int E = entries(c);
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, qb = c.rows_c / c.G;
    Work *out = reinterpret_cast<Work *>(c.work);
    int *first = c.work + kFirstAt, *slot = first + E + 1;
    Item *list = reinterpret_cast<Item *>(c.work + kListAt);
    int *sums = lds, *start = lds + 512;                      // start: first item of every request
    Request *known = reinterpret_cast<Request *>(start + E + 1);
    int *slot_of = reinterpret_cast<int *>(known + E);
    int4 *tried = reinterpret_cast<int4 *>(lds + kTriedAt);  // [E][choices] of up to kCounted: tiles, splits, their length, those all see
    const int per = (E + 511) / 512, b0 = min(tid * per, E), b1 = min(b0 + per, E);
    const bool kept = E <= kPlanKept, counted = E <= kCounted;  // in LDS; larger batches read them again
    auto load = [&](int b) {
        return kept ? known[b] : request(c, b);
    };

    int wgs = 0, longest = 0, tokens = 0, members = 0;
    float work = 0.0f;  // key tiles that all query tiles see together
    for (int b = b0; b < b1; ++b) {
        const Request r = request(c, b);
        if (kept) known[b] = r;
        int &count = is_group(c, b) ? members : tokens;
        count = min(count + r.n, c.n_tok + 1);
        int kt;
        const int T = chunk_tiles(c, r, qb, &kt);
        // query tile i of T ends (T - 1 - i) * qb keys before the last one
        const float all = (float)T * (float)kt;
        work += is_group(c, b) ? all : fmaxf(all - 0.5f * (float)T * (float)(T - 1) * (float)qb / kChunkKeys, 0.5f * all);
        wgs += T;
        longest = max(longest, kt);
    }
    wgs = wave_sum(wgs);
    longest = wave_max(longest);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) work += __shfl_xor(work, o);
    tokens = min(wave_sum(tokens), c.n_tok + 1);  // (64 (2^24 + 1) at most)
    members = kIsParts<C> ? min(wave_sum(members), c.n_tok + 1) : 0;
    if (lane == 0) {
        sums[wave] = wgs, sums[8 + wave] = longest, sums[16 + wave] = __float_as_int(work), sums[24 + wave] = tokens;
        sums[32 + wave] = members;
    }
    __syncthreads();
    wgs = longest = tokens = members = 0, work = 0.0f;
    for (int w = 0; w < 8; ++w) {
        wgs += sums[w], longest = max(longest, sums[8 + w]), work += __int_as_float(sums[16 + w]), tokens += sums[24 + w];
        members += sums[32 + w];
    }
    // More tokens than there are: ranges of q_start overlap. The sums of tiles below, and the
    // workgroups and slots that the host provided, are for disjoint ones.
    if (wgs == 0 || tokens > c.n_tok || members > c.n_tok) {
        if (tid == 0) *out = Work{1, 0, 0, 0};
        return;
    }
    work *= (float)c.Hkv;
    __syncthreads();
    // lane j (of 16) estimates length j: query tiles times splits, of all requests and of
    // split ones; 32 requests at a time
    const int j = lane & (kChoices - 1), l_j = max(div_ceil(longest, kTried[j]), 2);
    int n_j = 0, split_j = 0;
    for (int b = 4 * wave + (lane >> 4); b < E; b += 32) {
        int kt;
        const Request r = load(b);
        const int T = chunk_tiles(c, r, qb, &kt), S = div_ceil(kt, l_j), n = T * S;
        if (counted) {
            // (made here, an entry and a length once, not by each of the wavefronts below: the plan of
            // 24 drafts and two groups 11.5 -> 9.4 us, with the slots in LDS)
            const int most = div_ceil(kt, max(S, 1)), past = max(r.kv - r.n, 0);
            tried[b * kChoices + j] = make_int4(T, S, most, min(div_floor(past / kChunkKeys, max(most, 1)), S));
        }
        n_j += n;
        split_j += is_group(c, b) || kt > l_j ? n : 0;
    }
    n_j += __shfl_xor(n_j, 16), split_j += __shfl_xor(split_j, 16);
    n_j += __shfl_xor(n_j, 32), split_j += __shfl_xor(split_j, 32);
    if (lane < kChoices) sums[wave * 32 + lane] = n_j, sums[wave * 32 + 16 + lane] = split_j;
    __syncthreads();
    n_j = split_j = 0;
    for (int w = 0; w < 8; ++w) n_j += sums[w * 32 + j], split_j += sums[w * 32 + 16 + j];
    const int64_t N = (int64_t)n_j * c.Hkv, slots_j = (int64_t)split_j * c.Hkv;
    const int part_j = min(l_j, longest);
    const float part = (float)part_j, cus = (float)c.cus;
    if (counted) {  // wavefront w: query tiles times splits of at least (w + 1) / 8 of a part
        const int x = div_ceil(part_j * (wave + 1), kLevels);
        int n_x = 0;
        for (int b = lane >> 4; b < E && N > c.cus && N <= kRounds * c.cus; b += 4) {
            const int4 v = tried[b * kChoices + j];
            const int T = v.x, S = v.y, most = v.z, whole = v.w;  // most: 0 of an entry without chunks
            if (most < x) continue;
            // splits that the first query tile sees whole, and the others
            n_x += whole * T;
            if (whole == S) continue;
            const Request r = load(b);
            const int kt = max((r.kv + kChunkKeys - 1) / kChunkKeys, 1), past = r.kv - r.n;
            const int prefix = (min(r.prefix, r.kv) + kChunkKeys - 1) / kChunkKeys;
            const int q = most - (most * S > kt), rest = kt - q * S;  // as split_range
            for (int s = whole; s < S; ++s) {
                const int t0 = s * q + min(s, rest), t1 = t0 + q + (s < rest);
                if (t1 - t0 < x) break;
                // tiles that end in or behind the x-th key tile of the split
                const int need = kChunkKeys * (t0 + x - 1) - past + 1;
                n_x += prefix >= t0 + x || need <= 0 ? T : need > r.n ? 0 : T - div_ceil(need, qb) + 1;
            }
        }
        n_x += __shfl_xor(n_x, 16);
        n_x += __shfl_xor(n_x, 32);
        if (lane < kChoices) sums[256 + wave * 16 + lane] = n_x;
        __syncthreads();
    }
    const bool eq = work > 0.85f * (float)N * part;
    float t = fmaxf((work + kWg * (float)N) / cus, part + kWg);
    if (counted) {
        for (int r = 1; r < kRounds && r * c.cus < N && N <= kRounds * c.cus; ++r) {
            int level = 0;
            for (int w = 0; w < kLevels; ++w)
                if ((int64_t)sums[256 + w * 16 + j] * c.Hkv > r * c.cus) level = w + 1;
            if (level) t = fmaxf(t, (float)(r + 1) * (part * (float)level / kLevels + kWg));
        }
        t += N > c.cus ? 0.1f * part : 0.0f;
    } else {
        t = eq ? ceilf((float)N / cus) * (part + kWg) : t + 0.25f * part;
    }
    t += slots_j ? kMerge + kMergeSlot * (float)slots_j : 0.0f;
    // at most kMostSplits per request, slots and workgroups as there are
    const bool fits = j == 0 || (slots_j <= c.slots_c && N <= c.grid_c && longest <= (int64_t)l_j * kMostSplits);
    if (!fits || lane >= kChoices) t = INFINITY;
    float best = t;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) best = fminf(best, __shfl_xor(best, o));
    const int pick = __builtin_ctzll(__ballot(t == best));
    const int len = __shfl(l_j, pick), total = min(__shfl((int)N, pick), c.grid_c);
    const bool even = __shfl((int)eq, pick);
    const int listed = total <= kListed;
    if (tid == 0) *out = Work{len, total, listed, even};
    __syncthreads();

    // first items and slots
    int items = 0, slots = 0;
    for (int b = b0; b < b1; ++b) {
        int kt;
        const int T = chunk_tiles(c, load(b), qb, &kt), S = div_ceil(kt, len), k = T * S * c.Hkv;
        start[b] = items;
        items += k;
        slots += is_group(c, b) || S > 1 ? k : 0;
    }
    const int upto = wave_scan(items), slots_upto = wave_scan(slots);
    if (lane == 63) sums[wave] = upto, sums[8 + wave] = slots_upto;
    __syncthreads();
    int before = upto - items, slots_before = slots_upto - slots;
    for (int w = 0; w < wave; ++w) before += sums[w], slots_before += sums[8 + w];
    for (int b = b0; b < b1; ++b) {
        const int k = (b + 1 < b1 ? start[b + 1] : items) - start[b];
        int kt;
        (void)chunk_tiles(c, load(b), qb, &kt);
        first[b] = start[b] + before;
        slot[b] = slots_before;
        if (kept) slot_of[b] = slots_before;
        slots_before += is_group(c, b) || kt > len ? k : 0;
    }
    __syncthreads();
    for (int b = b0; b < b1; ++b) start[b] += before;
    if (tid == 511) start[E] = before + items, first[E] = before + items;
    if (!listed) return;

    auto item_of = [&](int id, int *own) {
        int lo = 0, hi = E;  // last request whose first item is at most id
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (start[mid] <= id) lo = mid;
            else hi = mid;
        }
        Item it;
        it.b = lo;
        it.rq = load(lo);
        int kt;
        it.tiles = chunk_tiles(c, it.rq, qb, &kt);
        it.splits = div_ceil(kt, len);
        const int k = id - start[lo], q = div_floor(k, it.tiles);
        it.tile = k - q * it.tiles;
        it.kvh = div_floor(q, it.splits);
        it.split = q - it.kvh * it.splits;
        split_range(kt, it.splits, it.split, &it.t0, &it.t1);
        it.slot = kept ? slot_of[lo] : slot[lo];
        it.spare[0] = it.spare[1] = 0;
        const int keys = sees(it.rq, min((it.tile + 1) * qb, it.rq.n) - 1);
        *own = max(min(it.t1, (keys + kChunkKeys - 1) / kChunkKeys) - it.t0, 0);
        return it;
    };
    __syncthreads();  // start and slot are complete
    int own;
    if (even) {
        for (int lin = tid; lin < c.grid_c && (lin >> 3) <= (total >> 3); lin += 512) {
            const int id = id_of_workgroup(lin, total);
            if (id >= 0 && lin < kListed) list[lin] = item_of(id, &own);
        }
        return;
    }
    // counting sort of the items by their length, longest first (the order inside a
    // length is left to chance; no result depends on it)
    constexpr int kBuckets = 64, kKept = 2;  // items that a thread makes once (of more, twice)
    auto bucket_of = [&](int own) {
        return kBuckets - 1 - min((int)((float)own * (float)kBuckets / (float)(len + 1)), kBuckets - 1);
    };
    if (tid < kBuckets) sums[tid] = 0;
    Item it[kKept];
    int bucket[kKept];
#pragma unroll
    for (int u = 0; u < kKept; ++u)
        if (tid + 512 * u < total) {
            it[u] = item_of(tid + 512 * u, &own);
            bucket[u] = bucket_of(own);
        }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kKept; ++u)
        if (tid + 512 * u < total) atomicAdd(&sums[bucket[u]], 1);
    for (int id = tid + 512 * kKept; id < total; id += 512) {
        (void)item_of(id, &own);
        atomicAdd(&sums[bucket_of(own)], 1);
    }
    __syncthreads();
    const int k = sums[lane], at = wave_scan(k) - k;  // every wavefront for itself
    __syncthreads();
    if (wave == 0) sums[lane] = at;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kKept; ++u)
        if (tid + 512 * u < total) list[atomicAdd(&sums[bucket[u]], 1)] = it[u];
    for (int id = tid + 512 * kKept; id < total; id += 512) {
        const Item more = item_of(id, &own);
        list[atomicAdd(&sums[bucket_of(own)], 1)] = more;
    }
}
#endif

}  // namespace paged
}  // namespace sqa
