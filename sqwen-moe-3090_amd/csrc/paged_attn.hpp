// paged_attn.hpp - device code that the attention kernels over a paged pool share:
// the requests of a call, how its keys are split over workgroups, the score options.
#pragma once
#include "paged.hpp"

namespace sqa {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;

// 16 bytes at any 4-byte address (the hardware's loads ask for no more)
typedef float float4a __attribute__((ext_vector_type(4), aligned(4)));

// Forms of an entry of Call::where (its low 2 bits; the others: slots between splits).
// Slot of split i of a token's KV head kvh: first + kvh * heads + i * step, with
// heads 1 (kFew) or slots * step (kMany).
constexpr int kDone = 0;  // nothing to merge: the row is written, or left as it was
constexpr int kFew = 1, kMany = 2;

// What a call's kernels know of it.
struct Call {
    const char *q;  // F32 row (t, h) at q + t * q_nb1 + h * q_nb2
    int64_t q_nb1, q_nb2;
    const uint8_t *k, *v;        // pages of k_page / v_page bytes, rows of row_bytes (all KV heads)
    int64_t k_page, v_page;
    int row_bytes;
    int n_pages, page, lp;       // lp = log2(page)
    const int32_t *table;
    int64_t table_stride;        // entries
    int64_t most_kv;             // keys that a table row can hold
    const int32_t *q_start, *kv_len, *prefix;
    int n_tok, B, H, Hkv, G;
    float inv_g;                 // 1 / G, see group_of
    float qscale;                // softmax scale * log2(e)
    float cap2, cap_inv;         // logit cap * log2(e) and its inverse, 0: none
    float bias;                  // max_bias, 0: none
    int nl2;                     // 2^floor(log2 H)
    const char *gate;
    int64_t gate_nb1, gate_nb2;
    float *dst;
    // workspace: where a token's partials are, and the partials of the two kernels
    int4 *where;                 // [n_tok] {first slot, splits, row of its first head, 4 * step + form}
    float *acc_d, *ml_d;         // [slot][rows_d][256], [slot][rows_d][2]
    float *acc_c, *ml_c;         // [slot][rows_c][256], ...
    int rows_d, rows_c;          // rows of a slot
    int slots_d, slots_c;        // slots of the workspace
    int *work;                   // the many-row kernel's plan (paged_work.hpp)
    int grid_c;                  // its workgroups at most
    int most_d;                  // query rows per KV head that the few-row kernel takes (0: it does not run)
    int room;                    // slots_d / Hkv: pieces that the workspace holds
    int few_pieces, all_pieces;  // pieces that one, two workgroups per CU are
    int cus;
};

// A request's tokens and keys. Anything the arrays may hold leaves rows inside
// [0, n_tok) and keys inside [0, most_kv).
struct Request {
    int q0, n;     // first token row, tokens
    int kv;        // keys that there are
    int pos0;      // position of the first token (may be negative)
    int prefix;    // keys that every token sees
};

__device__ __forceinline__ Request request(const Call &c, int b) {
    Request r;
    const int s0 = c.q_start[b], s1 = c.q_start[b + 1], len = c.kv_len[b];
    r.prefix = c.prefix ? c.prefix[b] : 0;
    r.q0 = min(max(s0, 0), c.n_tok);
    r.n = min(max(s1, r.q0), c.n_tok) - r.q0;
    r.kv = (int)min((int64_t)max(len, 0), c.most_kv);
    r.pos0 = max(len, 0) - r.n;
    return r;
}

// Keys [0, sees) that token i sees.
__device__ __forceinline__ int sees(const Request &r, int i) { return min(max(r.pos0 + i + 1, r.prefix), r.kv); }

// r / G for 0 <= r < 2^20 (the float quotient is nowhere near a whole number but above it).
__device__ __forceinline__ int group_of(const Call &c, int r) { return (int)(((float)r + 0.5f) * c.inv_g); }

// t / n for 0 <= t < 2^30, n > 0: a float quotient, what it left out, and one step either way.
__device__ __forceinline__ int div_floor(int t, int n) {
    const float inv = __builtin_amdgcn_rcpf((float)n);
    int q = (int)((float)t * inv), r = t - q * n;
    const int more = (int)((float)r * inv);
    q += more, r -= more * n;
    if (r < 0) --q, r += n;
    return q + (r >= n);
}
__device__ __forceinline__ int div_ceil(int t, int n) { return div_floor(t + n - 1, n); }  // t + n <= 2^30

// Sum over the wavefront, and inclusive prefix sum, by DPP: row shifts sum each row
// of 16, row broadcasts add the rows before.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }
__device__ __forceinline__ int wave_max(int x) {  // of values >= 0
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xa, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(x, 63);
}

// A wave-uniform value in a scalar register (what comes out of loads and divisions is in
// vector registers, and the compiler would go on there: loops, addresses, page ids).
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The request of a workgroup (b wave-uniform).
__device__ __forceinline__ Request uniform_request(const Call &c, int b) {
    const Request r = request(c, b);
    return Request{uniform(r.q0), uniform(r.n), uniform(r.kv), uniform(r.pos0), uniform(r.prefix)};
}

// Row b of the table, and a page id of it, by the scalar cache (b and i wave-uniform; the
// table is not written during the kernel).
typedef const __attribute__((address_space(4))) int32_t *TableRow;
__device__ __forceinline__ TableRow table_row(const Call &c, int b) {
    const uint64_t at = (uint64_t)(uintptr_t)(c.table + (int64_t)b * c.table_stride);
    return reinterpret_cast<TableRow>(((uint64_t)(uint32_t)uniform((int)(at >> 32)) << 32) | (uint32_t)uniform((int)(uint32_t)at));
}
__device__ __forceinline__ int page_id(TableRow row, int i) { return row[i]; }

// 16 bytes per lane from sbase + voff into LDS at m0v + 16 * lane (asynchronous; the
// caller waits with s_waitcnt vmcnt). sbase and m0v are wave-uniform. The compiler
// does not know what the asm holds, so the waits that it puts between a vector
// instruction that writes a scalar register and a memory instruction that reads it
// (5 states: sbase may come out of v_readfirstlane just before), and between a write of
// m0 and a load into LDS (1), stand in the asm. Without them the load took a base half
// old, half new.
__device__ __forceinline__ void dma16(uint32_t voff, const void *sbase, uint32_t m0v) {
    const uint64_t b = (uint64_t)(uintptr_t)sbase;
    const uint64_t bs = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32) |
                        (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b);
    const uint32_t ms = (uint32_t)__builtin_amdgcn_readfirstlane((int)m0v);
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(bs), "{m0}"(ms) : "memory");
}

// Distance slope of query head h times log2(e).
__device__ __forceinline__ float slope2(const Call &c, int h) {
    const float e = h < c.nl2 ? (float)(h + 1) / (float)c.nl2 : 0.5f * (float)(2 * (h - c.nl2) + 1) / (float)c.nl2;
    return exp2f(-c.bias * e) * kLog2e;
}

// cap2 * tanh(s / cap2) + off of N base-2 logits. Below a quarter, where most logits of
// a capped model lie, by the odd Taylor polynomial to x^9 (the rest is below 2^-26 of x
// there); above it as (e - 1) / (e + 1) with e = exp(2x), whose subtraction loses little
// any more. A step of tanh's own 2^-24 times a cap of 50 would be 3e-6 in a weight, so
// small x must not come out of 1 - 2 / (e + 1).
template <int N>
__device__ __forceinline__ void cap_logits(float (&s)[N], float cap2, float cap_inv, float off) {
    float x[N], top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = s[i] * cap_inv;
        top = fmaxf(top, fabsf(x[i]));  // (passes over a NaN)
        const float y = x[i] * x[i];
        float t = fmaf(y, 0.021869488f, -0.053968254f);
        t = fmaf(y, t, 0.13333333f);
        t = fmaf(y, t, -0.33333333f);
        s[i] = fmaf(cap2, fmaf(x[i] * y, t, x[i]), off);
    }
    if (!__any(top >= 0.25f)) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float z = fminf(fmaxf(x[i], -12.0f), 12.0f);
        const float e = __builtin_amdgcn_exp2f(2.0f * kLog2e * z);
        const float t = (e - 1.0f) * __builtin_amdgcn_rcpf(e + 1.0f);
        s[i] = fabsf(x[i]) >= 0.25f ? fmaf(cap2, t, off) : s[i];  // (NaN stays NaN)
    }
}

// x * sigmoid(g), by the hardware's exp2 and reciprocal (about 1 ulp each)
__device__ __forceinline__ float gate_by(float x, float g) {
    return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g));
}

int launch_few(const Call &c, hipStream_t s);      // paged_decode.hip
int launch_many(const Call &c, hipStream_t s);     // paged_chunk.hip
int launch_combine(const Call &c, hipStream_t s);  // paged_attn.hip

}  // namespace paged
}  // namespace sqa
