// abi_paged.cpp - the extern "C" entry points of a batch over the paged pool:
// argument checks, support queries and dispatch.
#include <math.h>

#include <initializer_list>

#include "checks.hpp"
#include "paged.hpp"

namespace sqa {
namespace {

int check_table(const sqa_tensor *t, const char *what) {
    if (t->type != SQA_TYPE_I32 || t->ne[2] != 1 || t->ne[3] != 1 || t->ne[0] < 1 || t->ne[1] < 1)
        return set_error(SQA_ERR_INVALID, "%s: table must be I32 [W, B]", what);
    if (t->ne[1] > kMaxRequests)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: %lld requests (at most %d)", what, (long long)t->ne[1], kMaxRequests);
    if (t->ne[0] > (1 << 18))
        return set_error(SQA_ERR_UNSUPPORTED, "%s: table rows of %lld pages (at most 2^18)", what, (long long)t->ne[0]);
    if ((t->ne[0] > 1 && t->nb[0] != 4) || t->nb[1] % 4 || (uintptr_t)t->data % 4)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: table rows must be contiguous", what);
    if (!t->data) return set_error(SQA_ERR_INVALID, "%s: null data pointer", what);
    return SQA_OK;
}

int check_paged(const sqa_tensor *q, const sqa_tensor *k, const sqa_tensor *v, const sqa_tensor *table, int64_t max_q,
                float scale, float max_bias, float softcap, const sqa_tensor *dst, const char *what = "paged_attn") {
    if (!q || !k || !v || !table || !dst) return set_error(SQA_ERR_INVALID, "%s: null tensor", what);
    if (q->type != SQA_TYPE_F32 || dst->type != SQA_TYPE_F32)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: q and dst must be F32", what);
    if (k->type != SQA_TYPE_Q4_0 || v->type != SQA_TYPE_Q4_0)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: K and V must be q4_0", what);
    for (int i = 0; i < 4; ++i)
        if (k->ne[i] != v->ne[i]) return set_error(SQA_ERR_INVALID, "%s: K and V pools differ in shape", what);
    if (q->ne[0] != k->ne[0]) return set_error(SQA_ERR_INVALID, "%s: q/k head dims differ", what);
    if (q->ne[0] != kHeadDim)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: head_dim %lld (only 256)", what, (long long)q->ne[0]);
    const int64_t n_tok = q->ne[1], H = q->ne[2], Hkv = k->ne[1], page = k->ne[2], n_pages = k->ne[3];
    if (q->ne[3] != 1 || n_tok < 0 || H < 1 || Hkv < 1 || H % Hkv)
        return set_error(SQA_ERR_INVALID, "%s: n_head %% n_head_kv != 0", what);
    if (H / Hkv > 16 || H > 4096)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: %lld query heads per KV head (at most 16)", what, (long long)(H / Hkv));
    if (n_tok > (1 << 24)) return set_error(SQA_ERR_UNSUPPORTED, "%s: more than 2^24 tokens", what);
    if (!power_of_two(page) || page < 16 || page > (1 << 16))
        return set_error(SQA_ERR_UNSUPPORTED, "%s: page of %lld tokens (a power of two, 16 to 65536)", what, (long long)page);
    if (n_pages < 1 || n_pages > INT32_MAX) return set_error(SQA_ERR_INVALID, "%s: pool without pages", what);
    int rc = check_table(table, what);
    if (rc) return rc;
    if (table->ne[0] * page > INT32_MAX)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: table rows of more than 2^31 tokens", what);
    if (dst->ne[0] != kHeadDim || dst->ne[1] != H || dst->ne[2] != n_tok || dst->ne[3] != 1)
        return set_error(SQA_ERR_INVALID, "%s: dst must be [D, H, n_tok, 1]", what);
    if (n_tok > 0 && (!q->data || !dst->data)) return set_error(SQA_ERR_INVALID, "%s: null data pointer", what);
    if (!k->data || !v->data) return set_error(SQA_ERR_INVALID, "%s: null data pointer", what);
    if (q->nb[0] != 4 || q->nb[1] % 4 || q->nb[2] % 4 || (uintptr_t)q->data % 4)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: q rows must have unit element stride", what);
    const uint64_t row = (uint64_t)kHeadRowBytes * (uint64_t)Hkv;
    if (row * 16 > (1u << 30)) return set_error(SQA_ERR_UNSUPPORTED, "%s: too many KV heads", what);
    for (const sqa_tensor *t : {k, v}) {
        if (t->nb[0] != SQA_Q4_0_BLOCK_BYTES || (Hkv > 1 && t->nb[1] != (uint64_t)kHeadRowBytes) || t->nb[2] != row ||
            (n_pages > 1 && (t->nb[3] < row * (uint64_t)page || t->nb[3] % 16)))
            return set_error(SQA_ERR_UNSUPPORTED, "%s: K/V must be pages of the cache layout (nb = 18, %d, %llu)", what,
                             kHeadRowBytes, (unsigned long long)row);
        if ((uintptr_t)t->data % 16)
            return set_error(SQA_ERR_UNSUPPORTED, "%s: K/V data must be 16-byte aligned", what);
    }
    if (dst->nb[0] != 4 || dst->nb[1] != 4ull * kHeadDim || dst->nb[2] != 4ull * kHeadDim * (uint64_t)H ||
        (uintptr_t)dst->data % 16)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: dst must be contiguous and 16-byte aligned", what);
    if (max_q < 1) return set_error(SQA_ERR_RANGE, "%s: max_q < 1", what);
    if (!isfinite(scale)) return set_error(SQA_ERR_INVALID, "%s: scale not finite", what);
    if (!isfinite(max_bias) || max_bias < 0.0f || !isfinite(softcap) || softcap < 0.0f)
        return set_error(SQA_ERR_INVALID, "%s: max_bias and logit_softcap must be finite and not negative", what);
    return SQA_OK;
}

int check_shared(const sqa_tensor *q, const sqa_tensor *k, const sqa_tensor *v, const sqa_tensor *table,
                 const sqa_tensor *shared_table, int64_t max_q, float scale, float max_bias, float softcap, const sqa_tensor *dst) {
    const char *what = "paged_attn_shared";
    int rc = check_paged(q, k, v, table, max_q, scale, max_bias, softcap, dst, what);
    if (rc) return rc;
    if (!shared_table) return set_error(SQA_ERR_INVALID, "%s: null tensor", what);
    rc = check_table(shared_table, what);
    if (rc) return rc;
    if (shared_table->ne[0] * k->ne[2] > INT32_MAX)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: table rows of more than 2^31 tokens", what);
    return SQA_OK;
}

// The arrays of a call beside q, the pools and the table.
int check_arrays(const sqa_tensor *q, const sqa_tensor *table, const sqa_tensor *q_start, const sqa_tensor *kv_len,
                 const sqa_tensor *prefix, const sqa_tensor *gate, const sqa_tensor *dst, const char *what) {
    const int64_t B = table->ne[1];
    if (!q_start || !kv_len) return set_error(SQA_ERR_INVALID, "%s: null tensor", what);
    if (!dense1(q_start, SQA_TYPE_I32, B + 1, 4) || !dense1(kv_len, SQA_TYPE_I32, B, 4) ||
        (prefix && !dense1(prefix, SQA_TYPE_I32, B, 4)))
        return set_error(SQA_ERR_INVALID, "%s: q_start, kv_len and prefix must be contiguous I32 of B + 1, B and B entries", what);
    if (gate && (gate->type != SQA_TYPE_F32 || gate->ne[0] != dst->ne[0] || gate->ne[1] != dst->ne[1] ||
                 gate->ne[2] != dst->ne[2] || gate->ne[3] != 1 || gate->nb[0] != 4 || gate->nb[1] % 4 || gate->nb[2] % 4 ||
                 (uintptr_t)gate->data % 4 || (q->ne[1] > 0 && !gate->data)))
        return set_error(SQA_ERR_INVALID, "%s: gate must be F32 [D, H, n_tok]", what);
    return SQA_OK;
}

Rows table_rows(const sqa_tensor *t) { return Rows{(uintptr_t)t->data, 4 * (uint64_t)t->ne[0], t->nb[1], t->ne[1]}; }

// Whether dst or the workspace meets another array (`more`: further ones). Some rows of dst, and the
// workspace, are written while others are computed. A row of q or gate is read for no row of dst but
// its own, so that q or gate may be dst itself.
bool clash(const sqa_tensor *q, const sqa_tensor *k, const sqa_tensor *v, const sqa_tensor *table, const sqa_tensor *q_start,
           const sqa_tensor *kv_len, const sqa_tensor *prefix, const sqa_tensor *gate, const sqa_tensor *dst, void *workspace,
           size_t workspace_bytes, std::initializer_list<Rows> more) {
    const int64_t n_tok = q->ne[1], H = q->ne[2], B = table->ne[1];
    auto heads = [&](const sqa_tensor *t, uint64_t token, uint64_t head) {  // its rows, by token or by head
        const uint64_t row = 4 * (uint64_t)kHeadDim, by_token = row + (uint64_t)(H - 1) * head;
        return token >= by_token || n_tok == 1 ? Rows{(uintptr_t)t->data, by_token, token, n_tok}
                                               : Rows{(uintptr_t)t->data, row + (uint64_t)(n_tok - 1) * token, head, H};
    };
    auto same = [&](const sqa_tensor *t, uint64_t token, uint64_t head) {  // dst itself
        return t->data == dst->data && (n_tok == 1 || token == dst->nb[2]) && (H == 1 || head == dst->nb[1]);
    };
    auto pages = [&](const sqa_tensor *t) { return Rows{(uintptr_t)t->data, t->nb[2] * (uint64_t)t->ne[2], t->nb[3], t->ne[3]}; };
    const Rows out = run_of(dst, 4ull * kHeadDim * (uint64_t)(H * n_tok)), rows_q = heads(q, q->nb[1], q->nb[2]);
    const Rows ws{(uintptr_t)workspace, workspace_bytes, 0, workspace ? 1 : 0};
    bool bad = meet(out, ws) || meet(ws, rows_q) || (!same(q, q->nb[1], q->nb[2]) && meet(out, rows_q));
    if (gate) {
        const Rows rows_g = heads(gate, gate->nb[2], gate->nb[1]);
        bad |= meet(ws, rows_g) || (!same(gate, gate->nb[2], gate->nb[1]) && meet(out, rows_g));
    }
    for (const Rows &r : {pages(k), pages(v), table_rows(table), run_of(q_start, 4 * (uint64_t)(B + 1)),
                          run_of(kv_len, 4 * (uint64_t)B), prefix ? run_of(prefix, 4 * (uint64_t)B) : Rows{}})
        bad |= meet(out, r) || meet(ws, r);
    for (const Rows &r : more) bad |= meet(out, r) || meet(ws, r);
    return bad;
}

int check_lora(const sqa_tensor *base, const sqa_tensor *x, const sqa_tensor *gate, const sqa_tensor *a,
               const sqa_tensor *b, const sqa_tensor *dst) {
    const char *what = "lora_add";
    if (!base || !x || !a || !b || !dst) return set_error(SQA_ERR_INVALID, "%s: null tensor", what);
    const int64_t K = x->ne[0], M = x->ne[1], r = a->ne[1], n = a->ne[2], N = b->ne[1];
    if (x->type != SQA_TYPE_F32 || base->type != SQA_TYPE_F32 || dst->type != SQA_TYPE_F32)
        return set_error(SQA_ERR_INVALID, "%s: x, base and dst must be F32", what);
    if (a->type != SQA_TYPE_F16 || b->type != SQA_TYPE_F16)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: a and b must be F16", what);
    if (a->ne[0] != K || b->ne[0] != r || b->ne[2] != n || a->ne[3] != 1 || b->ne[3] != 1)
        return set_error(SQA_ERR_INVALID, "%s: a must be [K, r, n] and b [r, N, n]", what);
    if (K <= 0 || K % 256 || N <= 0 || N % 16 || r <= 0 || r % 8 || r > 128)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: need K %% 256 == 0, N %% 16 == 0, r %% 8 == 0, r <= 128 (K=%lld, N=%lld, r=%lld)",
                         what, (long long)K, (long long)N, (long long)r);
    if (n < 1 || n > INT32_MAX || M < 0 || M > (1 << 24) || K > (1 << 20) || N > (1 << 20))
        return set_error(SQA_ERR_UNSUPPORTED, "%s: sizes out of range", what);
    if (a->nb[0] != 2 || (r > 1 && a->nb[1] != (uint64_t)(2 * K)) || (n > 1 && a->nb[2] != (uint64_t)(2 * K * r)) ||
        b->nb[0] != 2 || b->nb[1] != (uint64_t)(2 * r) || (n > 1 && b->nb[2] != (uint64_t)(2 * r * N)))
        return set_error(SQA_ERR_UNSUPPORTED, "%s: a and b must be contiguous", what);
    if (!a->data || !b->data) return set_error(SQA_ERR_INVALID, "%s: null data pointer", what);
    if ((uintptr_t)a->data % 16 || (uintptr_t)b->data % 16)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: a and b must be 16-byte aligned", what);
    for (const sqa_tensor *t : {x, gate}) {
        if (!t) continue;
        if (t->type != SQA_TYPE_F32 || t->ne[0] != K || t->ne[1] != M || t->ne[2] != 1 || t->ne[3] != 1)
            return set_error(SQA_ERR_INVALID, "%s: x and gate must be F32 [K, M]", what);
        if (t->nb[0] != 4 || t->nb[1] % 4 || (uintptr_t)t->data % 4)
            return set_error(SQA_ERR_UNSUPPORTED, "%s: x and gate must have unit element stride", what);
        if (M > 0 && !t->data) return set_error(SQA_ERR_INVALID, "%s: null data pointer", what);
    }
    for (const sqa_tensor *t : {base, dst}) {
        if (t->ne[0] != N || t->ne[1] != M || t->ne[2] != 1 || t->ne[3] != 1)
            return set_error(SQA_ERR_INVALID, "%s: base and dst must be F32 [N, M]", what);
        if (t->nb[0] != 4 || (M > 1 && t->nb[1] % 16) || (uintptr_t)t->data % 16)
            return set_error(SQA_ERR_UNSUPPORTED, "%s: base and dst rows must be 16-byte aligned", what);
        if (M > 0 && !t->data) return set_error(SQA_ERR_INVALID, "%s: null data pointer", what);
    }
    if (M > 1 && dst->nb[1] < (uint64_t)(4 * N)) return set_error(SQA_ERR_INVALID, "%s: dst rows overlap", what);
    return SQA_OK;
}

}  // namespace
}  // namespace sqa

using namespace sqa;

extern "C" {

int sqa_paged_plan(const sqa_tensor *n_past, const sqa_tensor *n_new, const sqa_tensor *table, const sqa_tensor *ring,
                   const sqa_tensor *state, int32_t page, const sqa_tensor *state_out, const sqa_tensor *n_past_out,
                   const sqa_tensor *q_start, const sqa_tensor *kv_len, const sqa_tensor *slots, const sqa_tensor *pos,
                   void *stream) {
    const char *what = "paged_plan";
    for (const sqa_tensor *t : {n_past, n_new, table, ring, state, state_out, n_past_out, q_start, kv_len, slots, pos})
        if (!t) return set_error(SQA_ERR_INVALID, "%s: null tensor", what);
    const int rc = check_table(table, what);
    if (rc) return rc;
    const int64_t B = table->ne[1], W = table->ne[0], T = slots->ne[0], P = ring->ne[0];
    if (!power_of_two(page) || page < 16 || page > (1 << 16))
        return set_error(SQA_ERR_UNSUPPORTED, "%s: page of %d tokens (a power of two, 16 to 65536)", what, page);
    if (W * page > INT32_MAX) return set_error(SQA_ERR_UNSUPPORTED, "%s: table rows of more than 2^31 tokens", what);
    if (T < 0 || T > (1 << 29)) return set_error(SQA_ERR_UNSUPPORTED, "%s: more than 2^29 token rows", what);
    if (P < 1 || P > (1 << 30)) return set_error(SQA_ERR_INVALID, "%s: ring without pages", what);
    if (!dense1(n_past, SQA_TYPE_I32, B, 4) || !dense1(n_new, SQA_TYPE_I32, B, 4) || !dense1(n_past_out, SQA_TYPE_I32, B, 4) ||
        !dense1(kv_len, SQA_TYPE_I32, B, 4) || !dense1(q_start, SQA_TYPE_I32, B + 1, 4) || !dense1(ring, SQA_TYPE_I32, P, 4) ||
        !dense1(state, SQA_TYPE_I32, 4, 4) || !dense1(state_out, SQA_TYPE_I32, 4, 4) || !dense1(slots, SQA_TYPE_I64, T, 8) ||
        !dense1(pos, SQA_TYPE_I32, 4 * T, 4))
        return set_error(SQA_ERR_INVALID, "%s: arrays must be contiguous, I32 (slots I64), of B, B + 1, 4, T and 4 T entries", what);
    if (B > 1 && table->nb[1] < (uint64_t)(4 * W)) return set_error(SQA_ERR_INVALID, "%s: table rows overlap", what);
    // Every workgroup reads the inputs while others write. (A table's rows with what lies
    // between them; what is written stands first.)
    const sqa_tensor *all[] = {state_out, n_past_out, q_start, kv_len, slots, pos, table, ring, n_past, n_new, state};
    uintptr_t from[11], to[11];
    for (int i = 0; i < 11; ++i) {
        const uint64_t bytes = (uint64_t)all[i]->ne[0] * (i == 4 ? 8 : 4) + (i == 6 ? (uint64_t)(B - 1) * table->nb[1] : 0);
        from[i] = (uintptr_t)all[i]->data;
        to[i] = from[i] + bytes;
    }
    bool clash = false;
    for (int i = 0; i < 8; ++i)
        for (int j = i + 1; j < 11; ++j)
            clash |= (from[i] < to[j]) & (from[j] < to[i]) & (from[i] < to[i]) & (from[j] < to[j]);
    if (clash) return set_error(SQA_ERR_INVALID, "%s: what the plan writes must not overlap its other arrays", what);
    const PlanArgs a{(const int32_t *)n_past->data, (const int32_t *)n_new->data, (int32_t *)table->data,
                     (int64_t)(table->nb[1] / 4), (int32_t *)ring->data, (const int32_t *)state->data,
                     (int32_t *)state_out->data, (int32_t *)n_past_out->data, (int32_t *)q_start->data,
                     (int32_t *)kv_len->data, (int64_t *)slots->data, (int32_t *)pos->data, (int)B, (int)W, page, (int)P,
                     (int)T};
    return launch_paged_plan(a, (hipStream_t)stream);
}

int sqa_supports_paged_attn(const sqa_tensor *q, const sqa_tensor *k, const sqa_tensor *v, const sqa_tensor *table,
                            int64_t max_q, float scale, float max_bias, float logit_softcap, const sqa_tensor *dst) {
    return check_paged(q, k, v, table, max_q, scale, max_bias, logit_softcap, dst) == SQA_OK ? 1 : 0;
}

size_t sqa_paged_attn_workspace_size(const sqa_tensor *q, const sqa_tensor *k, const sqa_tensor *table, int64_t max_q) {
    if (!q || !k || !table || k->ne[1] < 1 || q->ne[1] < 0 || q->ne[2] < 1 || q->ne[2] % k->ne[1] || max_q < 1 ||
        q->ne[2] / k->ne[1] > 16 || table->ne[1] < 1 || table->ne[1] > kMaxRequests)
        return 0;
    return paged_attn_workspace(q->ne[1], q->ne[2], k->ne[1], table->ne[1], max_q);
}

int sqa_paged_attn(const sqa_tensor *q, const sqa_tensor *k, const sqa_tensor *v, const sqa_tensor *table,
                   const sqa_tensor *q_start, const sqa_tensor *kv_len, const sqa_tensor *prefix, int64_t max_q,
                   float scale, float max_bias, float logit_softcap, const sqa_tensor *gate, const sqa_tensor *dst,
                   void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "paged_attn";
    const int rc = check_paged(q, k, v, table, max_q, scale, max_bias, logit_softcap, dst);
    if (rc) return rc;
    if (const int bad = check_arrays(q, table, q_start, kv_len, prefix, gate, dst, what)) return bad;
    if (q->ne[1] == 0) return SQA_OK;
    const size_t most = paged_attn_workspace(q->ne[1], q->ne[2], k->ne[1], table->ne[1], max_q);
    if (clash(q, k, v, table, q_start, kv_len, prefix, gate, dst, workspace, workspace_bytes < most ? workspace_bytes : most, {}))
        return set_error(SQA_ERR_INVALID, "%s: dst and the workspace must not overlap another array, but for a q or gate that is dst itself",
                         what);
    const PagedArgs a{q, k, v, table, q_start, kv_len, prefix, gate, dst, max_q, scale, max_bias, logit_softcap,
                      workspace, workspace_bytes};
    return launch_paged_attn(a, (hipStream_t)stream);
}

int sqa_paged_share(const sqa_tensor *q_start, const sqa_tensor *kv_len, const sqa_tensor *group, const sqa_tensor *shared_len,
                    const sqa_tensor *members, const sqa_tensor *m_start, const sqa_tensor *m_pos,
                    const sqa_tensor *token_group, const sqa_tensor *pos, void *stream) {
    const char *what = "paged_share";
    for (const sqa_tensor *t : {q_start, kv_len, group, shared_len, members, m_start, m_pos, token_group})
        if (!t) return set_error(SQA_ERR_INVALID, "%s: null tensor", what);
    const int64_t B = kv_len->ne[0], G = shared_len->ne[0], T = members->ne[0];
    if (B < 1 || G < 1 || T < 0) return set_error(SQA_ERR_INVALID, "%s: no requests or groups", what);
    if (B > kMaxRequests || G > kMaxRequests)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: %lld requests, %lld groups (at most %d)", what, (long long)B, (long long)G, kMaxRequests);
    if (T > (1 << 24)) return set_error(SQA_ERR_UNSUPPORTED, "%s: more than 2^24 token rows", what);
    if (!dense1(kv_len, SQA_TYPE_I32, B, 4) || !dense1(group, SQA_TYPE_I32, B, 4) || !dense1(q_start, SQA_TYPE_I32, B + 1, 4) ||
        !dense1(shared_len, SQA_TYPE_I32, G, 4) || !dense1(m_start, SQA_TYPE_I32, G + 1, 4) || !dense1(members, SQA_TYPE_I32, T, 4) ||
        !dense1(m_pos, SQA_TYPE_I32, T, 4) || !dense1(token_group, SQA_TYPE_I32, T, 4) || (pos && !dense1(pos, SQA_TYPE_I32, 4 * T, 4)))
        return set_error(SQA_ERR_INVALID, "%s: arrays must be contiguous I32, of B, B + 1, G, G + 1, T and 4 T entries", what);
    // Every workgroup reads the inputs while others write (what is written stands first).
    const sqa_tensor *all[] = {members, m_start, m_pos, token_group, pos, q_start, kv_len, group, shared_len};
    for (int i = 0; i < 5; ++i)
        for (int j = i + 1; j < 9; ++j)
            if (all[i] && all[j] && meet(run_of(all[i], 4 * (uint64_t)all[i]->ne[0]), run_of(all[j], 4 * (uint64_t)all[j]->ne[0])))
                return set_error(SQA_ERR_INVALID, "%s: what the call writes must not overlap its other arrays", what);
    const ShareArgs a{(const int32_t *)q_start->data, (const int32_t *)kv_len->data, (const int32_t *)group->data,
                      (const int32_t *)shared_len->data, (int32_t *)members->data, (int32_t *)m_start->data,
                      (int32_t *)m_pos->data, (int32_t *)token_group->data, pos ? (int32_t *)pos->data : nullptr,
                      (int)B, (int)G, (int)T};
    return launch_paged_share(a, (hipStream_t)stream);
}

int sqa_supports_paged_attn_shared(const sqa_tensor *q, const sqa_tensor *k, const sqa_tensor *v, const sqa_tensor *table,
                                   const sqa_tensor *shared_table, int64_t max_q, float scale, float max_bias,
                                   float logit_softcap, const sqa_tensor *dst) {
    return check_shared(q, k, v, table, shared_table, max_q, scale, max_bias, logit_softcap, dst) == SQA_OK ? 1 : 0;
}

size_t sqa_paged_attn_shared_workspace_size(const sqa_tensor *q, const sqa_tensor *k, const sqa_tensor *table,
                                            const sqa_tensor *shared_table, int64_t max_q) {
    if (sqa_paged_attn_workspace_size(q, k, table, max_q) == 0 || !shared_table || shared_table->ne[1] < 1 ||
        shared_table->ne[1] > kMaxRequests)
        return 0;
    return paged_shared_workspace(q->ne[1], q->ne[2], k->ne[1], table->ne[1], shared_table->ne[1], max_q);
}

int sqa_paged_attn_shared(const sqa_tensor *q, const sqa_tensor *k, const sqa_tensor *v, const sqa_tensor *table,
                          const sqa_tensor *q_start, const sqa_tensor *kv_len, const sqa_tensor *prefix,
                          const sqa_tensor *shared_table, const sqa_tensor *shared_len, const sqa_tensor *members,
                          const sqa_tensor *m_start, const sqa_tensor *m_pos, const sqa_tensor *token_group, int64_t max_q,
                          float scale, float max_bias, float logit_softcap, const sqa_tensor *gate, const sqa_tensor *dst,
                          void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "paged_attn_shared";
    int rc = check_shared(q, k, v, table, shared_table, max_q, scale, max_bias, logit_softcap, dst);
    if (!rc) rc = check_arrays(q, table, q_start, kv_len, prefix, gate, dst, what);
    if (rc) return rc;
    const int64_t n_tok = q->ne[1], B = table->ne[1], G = shared_table->ne[1];
    if (!shared_len || !members || !m_start || !m_pos || !token_group) return set_error(SQA_ERR_INVALID, "%s: null tensor", what);
    if (!dense1(shared_len, SQA_TYPE_I32, G, 4) || !dense1(m_start, SQA_TYPE_I32, G + 1, 4) ||
        !dense1(members, SQA_TYPE_I32, n_tok, 4) || !dense1(m_pos, SQA_TYPE_I32, n_tok, 4) ||
        !dense1(token_group, SQA_TYPE_I32, n_tok, 4))
        return set_error(SQA_ERR_INVALID, "%s: shared_len, m_start, members, m_pos and token_group must be contiguous I32 of G, "
                         "G + 1 and n_tok entries", what);
    if (n_tok == 0) return SQA_OK;
    const size_t most = paged_shared_workspace(n_tok, q->ne[2], k->ne[1], B, G, max_q);
    const uint64_t g4 = 4 * (uint64_t)G, t4 = 4 * (uint64_t)n_tok;
    if (clash(q, k, v, table, q_start, kv_len, prefix, gate, dst, workspace, workspace_bytes < most ? workspace_bytes : most,
              {table_rows(shared_table), run_of(shared_len, g4), run_of(m_start, g4 + 4), run_of(members, t4), run_of(m_pos, t4),
               run_of(token_group, t4)}))
        return set_error(SQA_ERR_INVALID, "%s: dst and the workspace must not overlap another array, but for a q or gate that is dst itself",
                         what);
    const SharedArgs a{{q, k, v, table, q_start, kv_len, prefix, gate, dst, max_q, scale, max_bias, logit_softcap, workspace,
                        workspace_bytes},
                       shared_table, shared_len, members, m_start, m_pos, token_group};
    return launch_paged_shared(a, (hipStream_t)stream);
}

int sqa_supports_lora_add(const sqa_tensor *base, const sqa_tensor *x, const sqa_tensor *gate, const sqa_tensor *a,
                          const sqa_tensor *b, const sqa_tensor *dst) {
    return check_lora(base, x, gate, a, b, dst) == SQA_OK ? 1 : 0;
}

int sqa_lora_add(const sqa_tensor *base, const sqa_tensor *x, const sqa_tensor *gate, const sqa_tensor *a,
                 const sqa_tensor *b, const sqa_tensor *ids, const sqa_tensor *scale, const sqa_tensor *dst,
                 void *stream) {
    const int rc = check_lora(base, x, gate, a, b, dst);
    if (rc) return rc;
    if (!ids || !dense1(ids, SQA_TYPE_I32, x->ne[1], 4))
        return set_error(SQA_ERR_INVALID, "lora_add: ids must be contiguous I32 [M]");
    if (scale && !dense1(scale, SQA_TYPE_F32, a->ne[2], 4))
        return set_error(SQA_ERR_INVALID, "lora_add: scale must be contiguous F32 [n_adapters]");
    if (x->ne[1] == 0) return SQA_OK;
    // Several workgroups read a token's row, or a tile's, while others write their part of it.
    const Rows out = rows_of(dst);
    const bool in_place = base->data == dst->data && (dst->ne[1] == 1 || base->nb[1] == dst->nb[1]);
    const uint64_t r = (uint64_t)a->ne[1], n = (uint64_t)a->ne[2];
    if (meet(out, rows_of(x)) || (gate && meet(out, rows_of(gate))) || (!in_place && meet(out, rows_of(base))) ||
        meet(out, run_of(a, 2 * r * n * (uint64_t)a->ne[0])) || meet(out, run_of(b, 2 * r * n * (uint64_t)b->ne[1])) ||
        meet(out, run_of(ids, 4 * (uint64_t)ids->ne[0])) || (scale && meet(out, run_of(scale, 4 * n))))
        return set_error(SQA_ERR_INVALID, "lora_add: dst must not overlap another array, but for a base that is dst itself");
    return launch_lora_add(*base, *x, gate, *a, *b, *ids, scale, *dst, (hipStream_t)stream);
}

}  // extern "C"
