// abi_rows.cpp - the extern "C" entry points of cached rows that are read back or moved:
// argument checks, support queries and dispatch.
#include <math.h>

#include <cmath>

#include "checks.hpp"
#include "rows.hpp"

namespace sqa {
namespace {

// n entries of 8 bytes
int check_index(const sqa_tensor *t, int64_t n, const char *what, const char *name) {
    if (t->type != SQA_TYPE_I64 || t->ne[0] != n || t->ne[1] != 1 || t->ne[2] != 1 || t->ne[3] != 1)
        return set_error(SQA_ERR_INVALID, "%s: %s must be I64 [n_rows]", what, name);
    if (n > 0 && !t->data) return set_error(SQA_ERR_INVALID, "%s: null data pointer", what);
    if (t->nb[0] % 8 || (uintptr_t)t->data % 8 || (n > 1 && (int64_t)t->nb[0] < 0))
        return set_error(SQA_ERR_UNSUPPORTED, "%s: %s strides not supported", what, name);
    return SQA_OK;
}

Rows index_rows(const sqa_tensor *t) { return Rows{(uintptr_t)t->data, 8, t->nb[0], t->ne[0]}; }

int check_get(const sqa_tensor *dst, const sqa_tensor *src, const sqa_tensor *idx) {
    const char *what = "get_rows_q4_0";
    if (!dst || !src || !idx) return set_error(SQA_ERR_INVALID, "%s: null tensor", what);
    if (src->type != SQA_TYPE_Q4_0) return set_error(SQA_ERR_UNSUPPORTED, "%s: src must be q4_0", what);
    if (dst->type != SQA_TYPE_F32 && dst->type != SQA_TYPE_F16)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: dst must be F32 or F16", what);
    const int64_t ne0 = src->ne[0], rows = src->ne[1], n = dst->ne[1];
    if (src->ne[2] != 1 || src->ne[3] != 1 || dst->ne[2] != 1 || dst->ne[3] != 1 || rows < 0 || n < 0)
        return set_error(SQA_ERR_INVALID, "%s: src and dst must be [ne0, rows]", what);
    if (ne0 < 1 || ne0 % SQA_QK4_0 || dst->ne[0] != ne0)
        return set_error(SQA_ERR_INVALID, "%s: rows must be equally long, a multiple of 32 values", what);
    if (ne0 > kMostRowValues || n > kMostRowCount)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: sizes out of range", what);
    const int rc = check_index(idx, n, what, "idx");
    if (rc) return rc;
    const uint64_t e = dst->type == SQA_TYPE_F32 ? 4 : 2;
    if (n > 0 && (!dst->data || (rows > 0 && !src->data))) return set_error(SQA_ERR_INVALID, "%s: null data pointer", what);
    if (src->nb[0] != SQA_Q4_0_BLOCK_BYTES || src->nb[1] % 2 || (uintptr_t)src->data % 2)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: src rows must be contiguous blocks at even addresses", what);
    if (dst->nb[0] != e || dst->nb[1] % e || (uintptr_t)dst->data % e)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: dst rows must have unit element stride", what);
    if (n > 1 && dst->nb[1] < e * (uint64_t)ne0) return set_error(SQA_ERR_INVALID, "%s: dst rows overlap", what);
    return SQA_OK;
}

int check_move(const sqa_tensor *dst, const sqa_tensor *src, const sqa_tensor *to, const sqa_tensor *from,
               const sqa_tensor *delta, const sqa_rope *rope) {
    const char *what = "move_rows_q4_0";
    if (!dst || !src || !to || !from) return set_error(SQA_ERR_INVALID, "%s: null tensor", what);
    if (src->type != SQA_TYPE_Q4_0 || dst->type != SQA_TYPE_Q4_0)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: src and dst must be q4_0", what);
    if (!delta != !rope) return set_error(SQA_ERR_INVALID, "%s: delta and rope go together", what);
    const int64_t D = src->ne[0], heads = src->ne[1], n = to->ne[0];
    for (const sqa_tensor *t : {dst, src}) {
        if (t->ne[0] != D || t->ne[1] != heads || t->ne[2] < 0 || t->ne[3] != 1 || D < 32 || D % 32 || heads < 1)
            return set_error(SQA_ERR_INVALID, "%s: src and dst must be [D, n_head, rows], D a multiple of 32", what);
        if (n > 0 && t->ne[2] > 0 && !t->data) return set_error(SQA_ERR_INVALID, "%s: null data pointer", what);
        const uint64_t row = (uint64_t)(D / SQA_QK4_0 * SQA_Q4_0_BLOCK_BYTES);
        if (t->nb[0] != SQA_Q4_0_BLOCK_BYTES || (heads > 1 && t->nb[1] != row) || t->nb[2] % 2 || (uintptr_t)t->data % 2)
            return set_error(SQA_ERR_UNSUPPORTED, "%s: rows must be contiguous blocks at even addresses", what);
        if (t->ne[2] > 1 && t->nb[2] < row * (uint64_t)heads) return set_error(SQA_ERR_INVALID, "%s: rows overlap", what);
    }
    if (n < 0 || n > kMostRowCount || D > kMostRowValues || heads > kMostRowValues || heads * D > kMostRowValues)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: sizes out of range", what);
    int rc = check_index(to, n, what, "to");
    if (!rc) rc = check_index(from, n, what, "from");
    if (rc) return rc;
    if (!rope) return SQA_OK;
    if (!dense1(delta, SQA_TYPE_I32, 4 * n, 4))
        return set_error(SQA_ERR_INVALID, "%s: delta must be I32 [4 * n_rows] contiguous", what);
    if (D != 64 && D != 128 && D != 256)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: head dim %lld not in {64, 128, 256}", what, (long long)D);
    if (rope->n_rot <= 0 || rope->n_rot % 8 || rope->n_rot > D)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: n_rot %d must be a positive multiple of 8 <= D", what, rope->n_rot);
    int64_t sect = 0;
    for (int k = 0; k < 4; ++k) {
        if (rope->sections[k] < 0) return set_error(SQA_ERR_INVALID, "%s: negative rope section", what);
        sect += rope->sections[k];
    }
    if (sect <= 0 || sect > (1 << 20)) return set_error(SQA_ERR_INVALID, "%s: rope sections' sum out of range", what);
    if (rope->ext_factor != 0.0f)
        return set_error(SQA_ERR_UNSUPPORTED, "%s: ext_factor != 0 (YaRN ramp) is not supported", what);
    if (!std::isfinite(rope->freq_base) || rope->freq_base <= 0.0f || !std::isfinite(rope->freq_scale))
        return set_error(SQA_ERR_INVALID, "%s: freq_base must be positive, freq_scale finite", what);
    // the fastest of the pairs; the kernel's reduction is for angles below 3e9
    const double fast = fmax(1.0, pow((double)rope->freq_base, -2.0 * (rope->n_rot / 2 - 1) / rope->n_rot)) * fabs((double)rope->freq_scale);
    if (!(fast <= kMostFreq))
        return set_error(SQA_ERR_UNSUPPORTED, "%s: rotation pairs of more than %g radians a position", what, kMostFreq);
    return SQA_OK;
}

}  // namespace
}  // namespace sqa

using namespace sqa;

extern "C" {

int sqa_supports_get_rows(const sqa_tensor *dst, const sqa_tensor *src, const sqa_tensor *idx) {
    return check_get(dst, src, idx) == SQA_OK ? 1 : 0;
}

int sqa_get_rows_q4_0(const sqa_tensor *dst, const sqa_tensor *src, const sqa_tensor *idx, void *stream) {
    const int rc = check_get(dst, src, idx);
    if (rc) return rc;
    const uint64_t bytes = (uint64_t)(src->ne[0] / SQA_QK4_0 * SQA_Q4_0_BLOCK_BYTES);
    const Rows out{(uintptr_t)dst->data, dst->nb[0] * (uint64_t)dst->ne[0], dst->nb[1], dst->ne[1]};
    if (meet(out, Rows{(uintptr_t)src->data, bytes, src->nb[1], src->ne[1]}) || meet(out, index_rows(idx)))
        return set_error(SQA_ERR_INVALID, "get_rows_q4_0: dst must not overlap src or idx");
    const GetRows p{(const uint8_t *)src->data, (int64_t)src->nb[1], src->ne[1], (const char *)idx->data,
                    (int64_t)idx->nb[0], (char *)dst->data, (int64_t)dst->nb[1], dst->ne[1],
                    (int)(src->ne[0] / SQA_QK4_0)};
    return launch_get_rows_q4_0(p, dst->type == SQA_TYPE_F16, (hipStream_t)stream);
}

int sqa_supports_move_rows(const sqa_tensor *dst, const sqa_tensor *src, const sqa_tensor *to, const sqa_tensor *from,
                           const sqa_tensor *delta, const sqa_rope *rope) {
    return check_move(dst, src, to, from, delta, rope) == SQA_OK ? 1 : 0;
}

int sqa_move_rows_q4_0(const sqa_tensor *dst, const sqa_tensor *src, const sqa_tensor *to, const sqa_tensor *from,
                       const sqa_tensor *delta, const sqa_rope *rope, void *stream) {
    const char *what = "move_rows_q4_0";
    const int rc = check_move(dst, src, to, from, delta, rope);
    if (rc) return rc;
    const int64_t D = src->ne[0], heads = src->ne[1], n = to->ne[0];
    const uint64_t bytes = (uint64_t)(heads * (D / SQA_QK4_0) * SQA_Q4_0_BLOCK_BYTES);
    const Rows out{(uintptr_t)dst->data, bytes, dst->nb[2], dst->ne[2]}, in{(uintptr_t)src->data, bytes, src->nb[2], src->ne[2]};
    const bool same = dst->data == src->data && (dst->nb[2] == src->nb[2] || dst->ne[2] <= 1 || src->ne[2] <= 1);
    if ((!same && meet(out, in)) || meet(out, index_rows(to)) || meet(out, index_rows(from)) ||
        (delta && meet(out, run_of(delta, 16 * (uint64_t)n))))
        return set_error(SQA_ERR_INVALID, "%s: dst must not overlap another array, but for a src that is dst itself", what);
    MoveRows p{};
    p.src = (const uint8_t *)src->data, p.dst = (uint8_t *)dst->data;
    p.src_nb1 = (int64_t)src->nb[2], p.dst_nb1 = (int64_t)dst->nb[2], p.src_rows = src->ne[2], p.dst_rows = dst->ne[2];
    p.from = (const char *)from->data, p.to = (const char *)to->data;
    p.from_nb0 = (int64_t)from->nb[0], p.to_nb0 = (int64_t)to->nb[0];
    p.n = n, p.heads = (int)heads, p.head_dim = (int)D;
    if (rope) {
        p.delta = (const int32_t *)delta->data;
        p.n_rot = rope->n_rot;
        const int32_t *n = rope->sections, sect = n[0] + n[1] + n[2] + n[3];
        for (int k = 0; k < p.n_rot / 2; ++k) {
            p.freq[k] = (double)rope->freq_scale * pow((double)rope->freq_base, -2.0 * k / p.n_rot);
            const int s = k % sect, c = s % 3;  // the sections' interleaved order, t h w
            p.component[k] = s >= 3 * n[c] ? 3 : (uint8_t)c;
        }
    }
    return launch_move_rows_q4_0(p, (hipStream_t)stream);
}

}  // extern "C"
