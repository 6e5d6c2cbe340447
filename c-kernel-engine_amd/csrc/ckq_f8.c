/* ckq_f8.c - the entry points of e4m3 rows with one scale for each 128 elements, and of tokens sorted by expert: no staging, no state; the launches check
 * what they take. */
#include <string.h>
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

/* Which of a call's arguments are int: bit i, the i-th. */
#define AT(i) (1u << (i))
static const unsigned ints[] = {
    AT(0) | AT(7) | AT(8), AT(4) | AT(7) | AT(8), AT(0) | AT(8) | AT(9), AT(9) | AT(12) | AT(13) | AT(14), AT(12) | AT(13) | AT(16) | AT(17) | AT(18),
    AT(1) | AT(2) | AT(3), AT(0) | AT(6) | AT(7) | AT(8) | AT(9), AT(0) | AT(8) | AT(9) | AT(10) | AT(11), AT(0) | AT(7) | AT(8) | AT(9) | AT(10),
    AT(0) | AT(10) | AT(11) | AT(12) | AT(13),
};

#define PTR(T, i) ((T *)(uintptr_t)a[i])
#define INT(i)    ((int)a[i])
#define LONG(i)   ((long)a[i])

int ckq_call_dev(const void *call)
{
    static const unsigned char arguments[] = {10, 10, 11, 16, 20, 8, 11, 13, 12, 15};
    int64_t which, a[20];
    if (!call) return CKQ_EINVAL;
    memcpy(&which, call, 8);
    if (which < 0 || which >= (int64_t)sizeof arguments) return CKQ_EINVAL;
    memcpy(a, (const char *)call + 8, 8u * arguments[which]);
    for (int i = 0; i < arguments[which]; ++i)                 /* 2^32 + 16 rows are not 16 */
        if ((ints[which] & AT(i)) && a[i] != (int)a[i]) return CKQ_EINVAL;
    switch (which) {
    case CKQ_CALL_QUANTIZE_F8:
        return ckq_launch_quantize_f8(INT(0), PTR(const void, 1), LONG(2), PTR(uint8_t, 3), LONG(4), PTR(float, 5), LONG(6), INT(7), INT(8), PTR(void, 9));
    case CKQ_CALL_DEQUANTIZE_F8:
        return ckq_launch_dequantize_f8(PTR(const uint8_t, 0), LONG(1), PTR(const float, 2), LONG(3), INT(4), PTR(void, 5), LONG(6), INT(7), INT(8), PTR(void, 9));
    case CKQ_CALL_SWIGLU_F8:
        return ckq_launch_swiglu_f8(INT(0), PTR(const void, 1), PTR(const void, 2), LONG(3), PTR(uint8_t, 4), LONG(5), PTR(float, 6), LONG(7), INT(8), INT(9), PTR(void, 10));
    case CKQ_CALL_GEMM_NT_F8:
        return ckq_launch_gemm_f8(PTR(const uint8_t, 0), LONG(1), PTR(const float, 2), LONG(3), PTR(const uint8_t, 4), LONG(5), PTR(const float, 6), LONG(7), PTR(const float, 8), INT(9),
                                  PTR(void, 10), LONG(11), INT(12), INT(13), INT(14), PTR(void, 15));
    case CKQ_CALL_GEMM_NT_F8_EXPERTS:
        return ckq_launch_gemm_f8_experts(PTR(const uint8_t, 0), LONG(1), PTR(const float, 2), LONG(3), PTR(const uint8_t, 4), LONG(5), LONG(6), PTR(const float, 7), LONG(8), LONG(9),
                                          PTR(const float, 10), PTR(const int32_t, 11), INT(12), INT(13), PTR(void, 14), LONG(15), INT(16), INT(17), INT(18), PTR(void, 19));
    case CKQ_CALL_MOE_SORT:
        return ckq_launch_moe_sort(PTR(const int32_t, 0), INT(1), INT(2), INT(3), PTR(int32_t, 4), PTR(int32_t, 5), PTR(int32_t, 6), PTR(void, 7));
    case CKQ_CALL_MOE_GATHER:
        return ckq_launch_moe_gather(INT(0), PTR(const void, 1), LONG(2), PTR(const int32_t, 3), PTR(void, 4), LONG(5), INT(6), INT(7), INT(8), INT(9), PTR(void, 10));
    case CKQ_CALL_MOE_GATHER_F8:
        return ckq_launch_moe_gather_f8(INT(0), PTR(const void, 1), LONG(2), PTR(const int32_t, 3), PTR(uint8_t, 4), LONG(5), PTR(float, 6), LONG(7), INT(8), INT(9), INT(10), INT(11), PTR(void, 12));
    case CKQ_CALL_MOE_COMBINE:
        return ckq_launch_moe_combine(INT(0), PTR(const void, 1), LONG(2), PTR(const int32_t, 3), PTR(const float, 4), PTR(void, 5), LONG(6), INT(7), INT(8), INT(9), INT(10), PTR(void, 11));
    default:
        return ckq_launch_moe_combine_backward(INT(0), PTR(const void, 1), LONG(2), PTR(const void, 3), LONG(4), PTR(const int32_t, 5), PTR(const float, 6), PTR(void, 7), LONG(8), PTR(float, 9),
                                               INT(10), INT(11), INT(12), INT(13), PTR(void, 14));
    }
}
