// paged.hpp - what the kernels over the paged pool share with their entry points.
#pragma once
#include "common.hpp"

namespace sqa {

constexpr int kMaxRequests = 4096;  // places of a batch

struct PagedArgs {
    const sqa_tensor *q, *k, *v, *table, *q_start, *kv_len, *prefix, *gate, *dst;
    int64_t max_q;
    float scale, max_bias, softcap;
    void *ws;
    size_t ws_bytes;
};
size_t paged_attn_workspace(int64_t n_tok, int64_t H, int64_t Hkv, int64_t B, int64_t max_q);
int launch_paged_attn(const PagedArgs &a, hipStream_t s);

struct PlanArgs {
    const int32_t *n_past, *n_new;
    int32_t *table;
    int64_t table_stride;  // in entries
    int32_t *ring;
    const int32_t *state;
    int32_t *state_out, *n_past_out, *q_start, *kv_len;
    int64_t *slots;
    int32_t *pos;
    int B, W, page, n_pages, T;
};
int launch_paged_plan(const PlanArgs &a, hipStream_t s);

int launch_lora_add(const sqa_tensor &base, const sqa_tensor &x, const sqa_tensor *gate, const sqa_tensor &a,
                    const sqa_tensor &b, const sqa_tensor &ids, const sqa_tensor *scale, const sqa_tensor &dst,
                    hipStream_t s);

}  // namespace sqa
