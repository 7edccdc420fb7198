/* op_check.h -- argument checks of the 8-bit floating point operators (include/inzg.h), before anything touches a device.
 * Each returns INZG_OK, or the status of the refusal with its reason in err. */
#ifndef INZG_OP_CHECK_H
#define INZG_OP_CHECK_H

#include <stddef.h>

#include "../../../include/inzg.h"

#ifdef __cplusplus
extern "C" {
#endif

inzg_status inzg__check_rmsnorm_q8(const inzg_rmsnorm_q8_args *a, char *err, size_t len);
inzg_status inzg__check_silu_mul_q8(const inzg_silu_mul_q8_args *a, char *err, size_t len);
inzg_status inzg__check_expert_lists(int n, int topk, int n_expert, const void *sel, const void *w, const void *off,
                                     const void *rows, const void *slots, const void *w_out, char *err, size_t len);
inzg_status inzg__check_matmul_q8(const inzg_matmul_q8_args *a, char *err, size_t len);
inzg_status inzg__check_grouped_matmul(const inzg_grouped_matmul_args *a, char *err, size_t len);

/* entries per tile of the grouped product's kernel for checked arguments: 32 or 128 */
int inzg__grouped_matmul_tile(int type, int groups, int entries, int n, int num_sms);

#ifdef __cplusplus
}
#endif
#endif
