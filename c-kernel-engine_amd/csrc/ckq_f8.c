/* ckq_f8.c - the entry points of e4m3 rows with one scale for each 128 elements, and of tokens sorted by expert: no staging, no state; the launches check
 * what they take. */
#include "ckernel_quant_hip.h"
#include "ckq_launch.h"

int ckq_quantize_f8_dev(ckq_ck_dtype type, const void *x, long ldx, uint8_t *q, long ldq, float *scale, long lds, int rows, int k, void *stream)
{
    return ckq_launch_quantize_f8((int)type, x, ldx, q, ldq, scale, lds, rows, k, stream);
}

int ckq_dequantize_f8_dev(const uint8_t *q, long ldq, const float *scale, long lds, ckq_ck_dtype type, void *y, long ldy, int rows, int k, void *stream)
{
    return ckq_launch_dequantize_f8(q, ldq, scale, lds, (int)type, y, ldy, rows, k, stream);
}

int ckq_swiglu_f8_dev(ckq_ck_dtype type, const void *gate, const void *up, long ld, uint8_t *q, long ldq, float *scale, long lds, int rows, int k, void *stream)
{
    return ckq_launch_swiglu_f8((int)type, gate, up, ld, q, ldq, scale, lds, rows, k, stream);
}

int ckq_gemm_nt_f8_dev(const uint8_t *A, long lda, const float *sa, long ldsa, const uint8_t *B, long ldb, const float *sb, long ldsb, const float *bias,
                       ckq_ck_dtype type, void *C, long ldc, int M, int N, int K, void *stream)
{
    return ckq_launch_gemm_f8(A, lda, sa, ldsa, B, ldb, sb, ldsb, bias, (int)type, C, ldc, M, N, K, stream);
}

int ckq_gemm_nt_f8_experts_dev(const uint8_t *A, long lda, const float *sa, long ldsa, const uint8_t *B, long ldb, long eb, const float *sb, long ldsb, long esb,
                               const float *bias, const int32_t *offsets, int experts, ckq_ck_dtype type, void *C, long ldc, int M, int N, int K, void *stream)
{
    return ckq_launch_gemm_f8_experts(A, lda, sa, ldsa, B, ldb, eb, sb, ldsb, esb, bias, offsets, experts, (int)type, C, ldc, M, N, K, stream);
}

int ckq_moe_sort_dev(const int32_t *ids, int tokens, int choices, int experts, int32_t *offsets, int32_t *order, int32_t *position, void *stream)
{
    return ckq_launch_moe_sort(ids, tokens, choices, experts, offsets, order, position, stream);
}

int ckq_moe_gather_dev(ckq_ck_dtype type, const void *x, long ldx, const int32_t *position, void *y, long ldy, int tokens, int choices, int rows, int k, void *stream)
{
    return ckq_launch_moe_gather((int)type, x, ldx, position, y, ldy, tokens, choices, rows, k, stream);
}

int ckq_moe_gather_f8_dev(ckq_ck_dtype type, const void *x, long ldx, const int32_t *position, uint8_t *q, long ldq, float *scale, long lds,
                          int tokens, int choices, int rows, int k, void *stream)
{
    return ckq_launch_moe_gather_f8((int)type, x, ldx, position, q, ldq, scale, lds, tokens, choices, rows, k, stream);
}

int ckq_moe_combine_dev(ckq_ck_dtype type, const void *y, long ldy, const int32_t *position, const float *weights, void *out, long ldo,
                        int tokens, int choices, int rows, int k, void *stream)
{
    return ckq_launch_moe_combine((int)type, y, ldy, position, weights, out, ldo, tokens, choices, rows, k, stream);
}

int ckq_moe_combine_backward_dev(ckq_ck_dtype type, const void *dout, long ldd, const void *y, long ldy, const int32_t *position, const float *weights,
                                 void *dy, long lddy, float *dweights, int tokens, int choices, int rows, int k, void *stream)
{
    return ckq_launch_moe_combine_backward((int)type, dout, ldd, y, ldy, position, weights, dy, lddy, dweights, tokens, choices, rows, k, stream);
}
