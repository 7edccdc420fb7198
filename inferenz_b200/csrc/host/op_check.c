/* op_check.c -- argument checks of the 8-bit floating point operators, and the rule that chooses the grouped product's kernel. Plain C
 * without CUDA, so that both are tested without a device. */
#include "op_check.h"

#include <limits.h>
#include <stdio.h>

#define REFUSE(st, ...)                                                                                                \
    do {                                                                                                               \
        if (err && len) snprintf(err, len, __VA_ARGS__);                                                               \
        return st;                                                                                                     \
    } while (0)

static int io_type(int t) { return t == INZG_T_F32 || t == INZG_T_F16 || t == INZG_T_BF16; }
static int type_bytes(int t) { return t == INZG_T_F32 ? 4 : t == INZG_T_E4M3 ? 1 : 2; }
static int64_t blocks(int64_t v) { return (v + INZG_Q8_BLOCK - 1) / INZG_Q8_BLOCK; }
static int misaligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) != 0; }
/* a pitch that rows of `cols` elements cannot have (0 stands for cols) */
static int bad_ld(int64_t ld, int64_t cols) { return ld != 0 && ld < cols; }
/* rows x pitch past what 64-bit byte offsets hold */
static int too_far(int64_t rows, int64_t ld) { return ld > 0 && rows > INT64_MAX / 8 / ld; }

static inzg_status check_quantized(const char *op, int n, int cols, const void *q, int64_t ldq, const float *s, int64_t lds,
                                   char *err, size_t len) {
    if (!q != !s) REFUSE(INZG_BAD_ARG, "%s: q and s go together", op);
    if (q && (bad_ld(ldq, cols) || bad_ld(lds, blocks(cols)))) REFUSE(INZG_BAD_ARG, "%s: a pitch below its row", op);
    if (q && (too_far(n, ldq) || too_far(n, lds))) REFUSE(INZG_BAD_ARG, "%s: a pitch is out of range", op);
    if (misaligned(s, 4)) REFUSE(INZG_BAD_ARG, "%s: s must be 4-byte aligned", op);
    return INZG_OK;
}

inzg_status inzg__check_rmsnorm_q8(const inzg_rmsnorm_q8_args *a, char *err, size_t len) {
    if (!a) REFUSE(INZG_BAD_ARG, "rmsnorm_q8: no arguments");
    if (a->n < 0 || a->cols <= 0) REFUSE(INZG_BAD_ARG, "rmsnorm_q8: bad n or cols");
    if (a->cols > 32768) REFUSE(INZG_UNSUPPORTED, "rmsnorm_q8: more than 32768 columns");
    if (!io_type(a->type)) REFUSE(INZG_UNSUPPORTED, "rmsnorm_q8: type must be F32, F16 or BF16");
    if (!(a->eps >= 0.0f)) REFUSE(INZG_BAD_ARG, "rmsnorm_q8: eps must not be negative");
    if (bad_ld(a->ldx, a->cols) || bad_ld(a->ldres, a->cols) || bad_ld(a->ldsum, a->cols) || bad_ld(a->ldy, a->cols))
        REFUSE(INZG_BAD_ARG, "rmsnorm_q8: a pitch below its row");
    if (too_far(a->n, a->ldx) || too_far(a->n, a->ldres) || too_far(a->n, a->ldsum) || too_far(a->n, a->ldy))
        REFUSE(INZG_BAD_ARG, "rmsnorm_q8: a pitch is out of range");
    if (a->n == 0) return INZG_OK;
    if (!a->x || !a->w) REFUSE(INZG_BAD_ARG, "rmsnorm_q8: null x or w");
    if (!a->sum && !a->y && !a->q && !a->s) REFUSE(INZG_BAD_ARG, "rmsnorm_q8: no output");
    const size_t b = (size_t)type_bytes(a->type);
    if (misaligned(a->x, b) || misaligned(a->res, b) || misaligned(a->sum, b) || misaligned(a->y, b) || misaligned(a->w, 4))
        REFUSE(INZG_BAD_ARG, "rmsnorm_q8: a pointer is not aligned to its type");
    if (a->sum) {
        const int64_t ls = a->ldsum ? a->ldsum : a->cols;
        if ((a->sum == a->x && ls != (a->ldx ? a->ldx : a->cols)) || (a->sum == a->res && ls != (a->ldres ? a->ldres : a->cols)))
            REFUSE(INZG_BAD_ARG, "rmsnorm_q8: sum in place needs its input's pitch");
    }
    return check_quantized("rmsnorm_q8", a->n, a->cols, a->q, a->ldq, a->s, a->lds, err, len);
}

inzg_status inzg__check_silu_mul_q8(const inzg_silu_mul_q8_args *a, char *err, size_t len) {
    if (!a) REFUSE(INZG_BAD_ARG, "silu_mul_q8: no arguments");
    if (a->n < 0 || a->cols <= 0 || a->cols > INT_MAX / 2 - 256) REFUSE(INZG_BAD_ARG, "silu_mul_q8: bad n or cols");
    if (!io_type(a->type)) REFUSE(INZG_UNSUPPORTED, "silu_mul_q8: type must be F32, F16 or BF16");
    if (bad_ld(a->ldx, 2 * (int64_t)a->cols) || bad_ld(a->ldy, a->cols)) REFUSE(INZG_BAD_ARG, "silu_mul_q8: a pitch below its row");
    if (too_far(a->n, a->ldx) || too_far(a->n, a->ldy)) REFUSE(INZG_BAD_ARG, "silu_mul_q8: a pitch is out of range");
    if (a->n == 0) return INZG_OK;
    if (!a->x) REFUSE(INZG_BAD_ARG, "silu_mul_q8: null x");
    if (!a->y && !a->q && !a->s) REFUSE(INZG_BAD_ARG, "silu_mul_q8: no output");
    const size_t b = (size_t)type_bytes(a->type);
    if (misaligned(a->x, b) || misaligned(a->y, b)) REFUSE(INZG_BAD_ARG, "silu_mul_q8: a pointer is not aligned to its type");
    return check_quantized("silu_mul_q8", a->n, a->cols, a->q, a->ldq, a->s, a->lds, err, len);
}

inzg_status inzg__check_expert_lists(int n, int topk, int n_expert, const void *sel, const void *w, const void *off,
                                     const void *rows, const void *slots, const void *w_out, char *err, size_t len) {
    if (n < 0 || topk <= 0 || n_expert <= 0) REFUSE(INZG_BAD_ARG, "expert_lists: bad n, topk or n_expert");
    if (n_expert > INZG_MAX_GROUPS) REFUSE(INZG_UNSUPPORTED, "expert_lists: more than %d experts", INZG_MAX_GROUPS);
    if ((int64_t)n * topk > INT_MAX / 2) REFUSE(INZG_UNSUPPORTED, "expert_lists: more than 2^30 entries");
    if (!off) REFUSE(INZG_BAD_ARG, "expert_lists: null off");
    if (n && (!sel || !rows || !slots)) REFUSE(INZG_BAD_ARG, "expert_lists: null sel, rows or slots");
    if (!w != !w_out) REFUSE(INZG_BAD_ARG, "expert_lists: w and w_out go together");
    if (misaligned(sel, 4) || misaligned(w, 4) || misaligned(off, 4) || misaligned(rows, 4) || misaligned(slots, 4) ||
        misaligned(w_out, 4))
        REFUSE(INZG_BAD_ARG, "expert_lists: pointers must be 4-byte aligned");
    return INZG_OK;
}

/* what the dense and the grouped product share; `op` names the caller, `wrows` counts the rows of w */
static inzg_status check_product(const char *op, int type, int64_t wrows, int n, int k, int64_t arows, const void *a, int64_t lda,
                                 const float *as, int64_t ldas, const void *w, int64_t ldw, const float *ws,
                                 const void *out, int64_t ldo, int64_t orows, int out_type, char *err, size_t len) {
    const int64_t b = type_bytes(type);
    if (!io_type(out_type)) REFUSE(INZG_UNSUPPORTED, "%s: out_type must be F32, F16 or BF16", op);
    if (wrows > INT_MAX) REFUSE(INZG_UNSUPPORTED, "%s: more than 2^31 - 1 rows of w", op);
    if (bad_ld(lda, k) || bad_ld(ldw, k) || bad_ld(ldo, n) || bad_ld(ldas, blocks(k)))
        REFUSE(INZG_BAD_ARG, "%s: a pitch below its row", op);
    if (too_far(arows, lda) || too_far(wrows, ldw) || too_far(orows, ldo) || too_far(arows, ldas))
        REFUSE(INZG_BAD_ARG, "%s: a pitch is out of range", op);
    if (((lda ? lda : k) * b) % 16 || ((ldw ? ldw : k) * b) % 16)
        REFUSE(INZG_BAD_ARG, "%s: the pitches of a and w must be multiples of 16 bytes", op);
    if ((lda ? lda : k) * b >= (1ll << 40) || (ldw ? ldw : k) * b >= (1ll << 40))
        REFUSE(INZG_UNSUPPORTED, "%s: a pitch of 2^40 bytes or more", op);
    if (!a || !w || !out) REFUSE(INZG_BAD_ARG, "%s: null a, w or out", op);
    if (misaligned(a, 16) || misaligned(w, 16)) REFUSE(INZG_BAD_ARG, "%s: a and w must be 16-byte aligned", op);
    if (misaligned(out, (size_t)type_bytes(out_type))) REFUSE(INZG_BAD_ARG, "%s: out is not aligned to its type", op);
    if (type == INZG_T_E4M3 ? !as || !ws : as || ws) REFUSE(INZG_BAD_ARG, "%s: e4m3 needs both block scales, other types take none", op);
    if (misaligned(as, 4) || misaligned(ws, 4)) REFUSE(INZG_BAD_ARG, "%s: scales must be 4-byte aligned", op);
    return INZG_OK;
}

inzg_status inzg__check_matmul_q8(const inzg_matmul_q8_args *a, char *err, size_t len) {
    if (!a) REFUSE(INZG_BAD_ARG, "matmul_q8: no arguments");
    if (a->m < 0 || a->n <= 0 || a->k <= 0 || a->n > INT_MAX - 256 || a->k > INT_MAX - 256)
        REFUSE(INZG_BAD_ARG, "matmul_q8: bad m, n or k");
    if (a->m > INT_MAX - 256) REFUSE(INZG_UNSUPPORTED, "matmul_q8: too many rows"); /* tiles are rounded up in 32 bits */
    if ((a->m / 16 + (int64_t)1) * (a->n / 128 + (int64_t)1) >= INT_MAX) REFUSE(INZG_UNSUPPORTED, "matmul_q8: too many tiles");
    if (a->m == 0) return INZG_OK;
    return check_product("matmul_q8", INZG_T_E4M3, a->n, a->n, a->k, a->m, a->a, a->lda, a->a_scale, a->lda_scale, a->w, a->ldw,
                         a->w_scale, a->out, a->ldo, a->m, a->out_type, err, len);
}

inzg_status inzg__check_grouped_matmul(const inzg_grouped_matmul_args *a, char *err, size_t len) {
    if (!a) REFUSE(INZG_BAD_ARG, "grouped_matmul: no arguments");
    if (a->type != INZG_T_E4M3 && a->type != INZG_T_BF16 && a->type != INZG_T_F16)
        REFUSE(INZG_UNSUPPORTED, "grouped_matmul: type must be E4M3, BF16 or F16");
    if (a->groups <= 0 || a->n <= 0 || a->k <= 0 || a->n > INT_MAX - 256 || a->k > INT_MAX - 256 || a->a_rows < 0 ||
        a->entries < 0 || a->out_rows_n < 0)
        REFUSE(INZG_BAD_ARG, "grouped_matmul: bad groups, n, k, a_rows, entries or out_rows_n");
    if (a->groups > INZG_MAX_GROUPS) REFUSE(INZG_UNSUPPORTED, "grouped_matmul: more than %d groups", INZG_MAX_GROUPS);
    if (a->entries > INT_MAX - 256) REFUSE(INZG_UNSUPPORTED, "grouped_matmul: too many entries"); /* as for matmul_q8 */
    if ((a->entries / 16 + (int64_t)a->groups) * (a->n / 128 + (int64_t)1) >= INT_MAX)
        REFUSE(INZG_UNSUPPORTED, "grouped_matmul: too many tiles");
    if (a->entries == 0) return INZG_OK;
    if (a->in_rows ? a->a_rows == 0 : a->a_rows < a->entries) REFUSE(INZG_BAD_ARG, "grouped_matmul: fewer rows of a than entries");
    if (a->out_rows ? a->out_rows_n == 0 : a->out_rows_n < a->entries)
        REFUSE(INZG_BAD_ARG, "grouped_matmul: fewer rows of out than entries");
    if (!a->off) REFUSE(INZG_BAD_ARG, "grouped_matmul: null off");
    if (misaligned(a->off, 4) || misaligned(a->in_rows, 4) || misaligned(a->out_rows, 4) || misaligned(a->out_scale, 4))
        REFUSE(INZG_BAD_ARG, "grouped_matmul: index and scale pointers must be 4-byte aligned");
    return check_product("grouped_matmul", a->type, (int64_t)a->groups * a->n, a->n, a->k, a->a_rows, a->a, a->lda, a->a_scale,
                         a->lda_scale, a->w, a->ldw, a->w_scale, a->out, a->ldo, a->out_rows_n, a->out_type, err, len);
}

/* Which kernel, by the entries per group and by how many 32-entry items there are, taken to be one per 32 entries and half a one
 * more per group (measured with k = 2048 and 2560, 32-entry tiles against 128-entry ones, us; bf16 while the whole k was summed in TMEM):
 *   e4m3, 64 groups, n = 1280: 50 a group 44, 52; 62: 52, 53; 69: 55, 53; 80: 58, 52
 *   e4m3, 512 groups, n = 640: 50 a group 150, 173; 62: 180, 190; 70: 192, 190
 *   e4m3, one group, n = 2560: 128 entries 9.8, 16.5; 448: 14.4, 17.2; n = 10240: 96 entries 15.3, 17.2; 128: 18.8, 17.7
 *   bf16, 64 groups, n = 1280: 40 a group 75, 82; 45: 80, 82; 52: 85, 81
 *   bf16, one group, n = 1280: 192 entries 13, 19; n = 40960: 32 entries 42, 53; 64: 71, 57
 * The entries of one group alone fill their tiles: past 32 its bf16 weights are streamed twice. A few items, up to one per SM
 * (e4m3: two), are sooner done in small tiles whatever the groups. `entries` is the caller's upper bound: a rank that lists few of
 * them, or a few groups that have most of them, get the tiles of the mean. */
int inzg__grouped_matmul_tile(int type, int groups, int entries, int n, int num_sms) {
    int64_t few = (entries + 31LL) / 32 + (groups - 1) / 2;
    if (few > entries) few = entries;
    few *= (n + 127LL) / 128;
    if (type != INZG_T_E4M3) return entries <= (groups > 1 ? 40 : 32) * (int64_t)groups || few <= num_sms ? 32 : 128;
    return entries <= 64 * (int64_t)groups || few <= 2 * (int64_t)num_sms ? 32 : 128;
}
