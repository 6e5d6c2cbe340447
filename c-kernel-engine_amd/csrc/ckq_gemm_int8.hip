/*
 * ckq_gemm_int8.hip - matrix product of int8 rows with one scale each (one a token, one a channel):
 *
 *   C[m][n] = T((sa[m] * sb[n]) * (float) sum_k A[m][k] B[n][k]  (+ bias[n]))
 *
 * The sum is exact in int32 for k <= 131071 (128 * 128 * k < 2^31), so no order of it, and no split, changes a bit.
 */
#include "ckq_gemm_common.hpp"

template <int T> struct I8Out;
template <> struct I8Out<CKQ_T_F32>  { typedef float type; };
template <> struct I8Out<CKQ_T_BF16> { typedef __bf16 type; };
template <> struct I8Out<CKQ_T_F16>  { typedef _Float16 type; };

struct I8Args {
    const int8_t *A, *B;
    const float  *sa, *sb, *bias;
    void         *C;
    long          lda, ldb, ldc;
    int           M, N, K;
};

__device__ __forceinline__ float i8_scaled(int sum, float sa, float sb) { return (sa * (float)sum) * sb; }

/* A wave has 16 tokens x 16 rows; every lane fetches its own operands, 16 bytes of one row (v_mfma_i32_16x16x64_i8: lane l holds
 * bytes 16 (l / 16) .. of row l % 16 of both operands; result: rows 4 (l / 16) + r of the first, row l % 16 of the second). */
template <class E>
__global__ void __launch_bounds__(256) gemm_i8_simple_kernel(I8Args a)
{
    const int lane = threadIdx.x & 63, wave = wave_in_block();
    const int ntn = (a.N + 15) / 16, ntm = (a.M + 15) / 16;
    const long tile = (long)blockIdx.x * 4 + wave;
    if (tile >= (long)ntn * ntm) return;
    const int n0 = 16 * (int)(tile % ntn), m0 = 16 * (int)(tile / ntn);
    const int r = lane & 15, c = 16 * (lane >> 4);
    const int8_t *pa = a.A + (size_t)min(m0 + r, a.M - 1) * a.lda, *pb = a.B + (size_t)min(n0 + r, a.N - 1) * a.ldb;
    ckq_v4i acc = {0, 0, 0, 0};
    for (int k = 0; k < a.K; k += 64) {
        ckq_v4i va = {0, 0, 0, 0}, vb = {0, 0, 0, 0};
        const int left = a.K - (k + c);
        if (left > 0) {
            va = *reinterpret_cast<const ckq_v4i *>(pa + k + c);
            vb = *reinterpret_cast<const ckq_v4i *>(pb + k + c);
            /* bytes behind the row's last are not zero: take them out of one operand */
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = left - 4 * i;
                va[i] = n >= 4 ? va[i] : n <= 0 ? 0 : va[i] & (int)((1u << (8 * n)) - 1u);
            }
        }
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(vb, va, acc, 0, 0, 0);
    }
    const int m = m0 + r;
    if (m >= a.M) return;
    const float sa = a.sa[m];
    E *out = (E *)a.C + (size_t)m * a.ldc;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = n0 + 4 * (lane >> 4) + i;
        if (n < a.N) {
            float v = i8_scaled(acc[i], sa, a.sb[n]);
            if (a.bias) v += a.bias[n];
            out[n] = (E)v;
        }
    }
}

template <class E>
static int launch_gemm_i8(const I8Args &a, hipStream_t s)
{
    const size_t blocks = ((size_t)((a.M + 15) / 16) * (size_t)((a.N + 15) / 16) + 3) / 4;
    if (blocks > 0x7fffffff) return CKQ_EROWS;
    hipLaunchKernelGGL(gemm_i8_simple_kernel<E>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

extern "C" int ckq_launch_gemm_i8(const int8_t *A, long lda, const float *sa, const int8_t *B, long ldb, const float *sb, const float *bias,
                                  int type, void *C, long ldc, int M, int N, int K, void *stream)
{
    if (!A || !sa || !B || !sb || !C || M <= 0 || N <= 0 || K <= 0 || lda < K || ldb < K || ldc < N) return CKQ_EINVAL;
    const int size = type == CKQ_T_F32 ? 4 : type == CKQ_T_BF16 || type == CKQ_T_F16 ? 2 : 0;
    if (!size) return CKQ_EFORMAT;
    if (((uintptr_t)A | (uintptr_t)B) % 16 || lda % 16 || ldb % 16 || lda > CKQ_I8_PITCH_MAX || ldb > CKQ_I8_PITCH_MAX || K > CKQ_I8_K_MAX) return CKQ_EROWS;
    if ((uintptr_t)C % size || ((uintptr_t)sa | (uintptr_t)sb | (uintptr_t)bias) % 4) return CKQ_EROWS;
    const I8Args a = {A, B, sa, sb, bias, C, lda, ldb, ldc, M, N, K};
    switch (type) {
    case CKQ_T_F32:  return launch_gemm_i8<float>(a, (hipStream_t)stream);
    case CKQ_T_BF16: return launch_gemm_i8<__bf16>(a, (hipStream_t)stream);
    default:         return launch_gemm_i8<_Float16>(a, (hipStream_t)stream);
    }
}
