/* ckq_int8.c - the entry points of int8 rows with one scale each: no staging, no state; the launches check what they take. */
#include "ckernel_quant_hip.h"
#include "ckq_launch.h"

int ckq_quantize_i8_dev(ckq_ck_dtype type, const void *x, long ldx, int8_t *q, long ldq, float *scale, int rows, int k, void *stream)
{
    return ckq_launch_quantize_i8((int)type, x, ldx, q, ldq, scale, rows, k, stream);
}

int ckq_dequantize_i8_dev(const int8_t *q, long ldq, const float *scale, ckq_ck_dtype type, void *y, long ldy, int rows, int k, void *stream)
{
    return ckq_launch_dequantize_i8(q, ldq, scale, (int)type, y, ldy, rows, k, stream);
}

int ckq_rmsnorm_i8_dev(ckq_ck_dtype type, const void *x, long ldx, const void *residual, void *sum, long ldr, const float *gamma, float eps,
                       int8_t *q, long ldq, float *scale, int rows, int k, void *stream)
{
    return ckq_launch_rmsnorm_i8((int)type, x, ldx, residual, sum, ldr, gamma, eps, q, ldq, scale, rows, k, stream);
}

int ckq_swiglu_i8_dev(ckq_ck_dtype type, const void *gate, const void *up, long ld, int8_t *q, long ldq, float *scale, int rows, int k, void *stream)
{
    return ckq_launch_swiglu_i8((int)type, gate, up, ld, q, ldq, scale, rows, k, stream);
}

int ckq_gemm_nt_i8_dev(const int8_t *A, long lda, const float *sa, const int8_t *B, long ldb, const float *sb, const float *bias,
                       ckq_ck_dtype type, void *C, long ldc, int M, int N, int K, void *stream)
{
    return ckq_launch_gemm_i8(A, lda, sa, B, ldb, sb, bias, (int)type, C, ldc, M, N, K, stream);
}
