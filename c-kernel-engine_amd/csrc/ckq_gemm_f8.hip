/*
 * ckq_gemm_f8.hip - matrix product of e4m3 rows, one scale for each 128 elements of a token and each block of 128 x 128 of the weights:
 *
 *   C[m][n] = T(sum_g (sa[g][m] * sb[n / 128][g]) * (sum over k in group g of A[m][k] B[n][k])  (+ bias[n]))
 *
 * and the same of rows sorted by expert, each expert with a matrix of its own.  A group's sum starts from zero; the groups' sums are scaled and
 * added in fp32.
 *
 * Sums.  The matrix cores' e4m3 instructions add eight products at a time after aligning them to the largest of the eight and dropping what is
 * under 2^-13 of it (measured, in all their shapes; between eights they add as fp32 does): a sum of 128 random products is 1.5e-5 of its size off.
 * e4m3 values are exact in fp16, and the fp16 instructions add their products as fp32 does (1e-8), at half the rate.
 */
#include "ckq_gemm_common.hpp"
#include "ckq_int8.hpp"
#include "ckq_rows.hpp"

typedef _Float16 f8_v2h __attribute__((ext_vector_type(2)));
typedef _Float16 f8_v8h __attribute__((ext_vector_type(8)));
typedef float f8_v4f __attribute__((ext_vector_type(4)));

struct F8Args {
    const uint8_t *A, *B;
    const float   *sa, *sb, *bias;
    const int32_t *offsets;                 /* experts: where each one's rows begin, experts + 1 of them; null: one matrix */
    void          *C;
    long           lda, ldsa, ldb, eb, ldsb, esb, ldc;     /* eb, esb: from one expert's matrix and scales to the next */
    int            M, N, K, experts;
};

/* Which rows the t-th tile of BT rows has: expert e, rows m0 .. mend - 1.  All lanes of a wave. */
__device__ __forceinline__ bool f8_rows(const F8Args &a, int t, int BT, int &e, int &m0, int &mend)
{
    if (!a.offsets) {
        e = 0;
        m0 = t * BT;
        mend = a.M;
        return m0 < a.M;
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 64) {
        const int i = min(e0 + lane, a.experts - 1);
        const int lo = max(0, min(a.offsets[i], a.M)), hi = max(lo, min(a.offsets[i + 1], a.M));
        const int n = e0 + lane < a.experts ? (hi - lo + BT - 1) / BT : 0;
        int sum = n;
        for (int d = 1; d < 64; d *= 2) {
            const int other = __shfl_up(sum, d);
            if (lane >= d) sum += other;
        }
        const unsigned long long m = __ballot(before + sum > t);
        if (m) {
            const int l = __ffsll((long long)m) - 1;
            e = __builtin_amdgcn_readfirstlane(e0 + l);
            m0 = __builtin_amdgcn_readlane(lo + (t - before - (sum - n)) * BT, l);
            mend = __builtin_amdgcn_readlane(hi, l);
            return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

/* Sixteen bytes of a row from k on, zeros behind its last. */
__device__ __forceinline__ ckq_v4i f8_chunk(const uint8_t *row, int k, int K)
{
    ckq_v4i v = {0, 0, 0, 0};
    if (k < K) v = *reinterpret_cast<const ckq_v4i *>(row + k);
    if (K - k < 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = K - k - 4 * i;
            v[i] = n >= 4 ? v[i] : n <= 0 ? 0 : v[i] & (int)((1u << (8 * n)) - 1u);
        }
    }
    return v;
}

/* Eight codes as fp16. */
__device__ __forceinline__ f8_v8h f8_half(int lo, int hi)
{
    const f8_v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const f8_v2h c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return f8_v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

/* 16 tokens x 64 rows a wave, operands straight from memory. */
template <class E>
__global__ void __launch_bounds__(256) gemm_f8_kernel(F8Args a, int nnt)
{
    const int lane = threadIdx.x & 63, wave = wave_in_block();
    const int tt = (int)blockIdx.x / nnt, n0 = ((int)blockIdx.x - tt * nnt) * 256 + 64 * wave;
    int e, m0, mend;
    if (!f8_rows(a, tt, 16, e, m0, mend) || n0 >= a.N) return;
    const uint8_t *B = a.B + (size_t)e * a.eb;
    const float *sb = a.sb + (size_t)e * a.esb, *bias = a.bias ? a.bias + (size_t)e * a.N : nullptr;
    const int tok = min(m0 + (lane & 15), mend - 1);
    const uint8_t *pa = a.A + (size_t)tok * a.lda, *pb[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) pb[j] = B + (size_t)min(n0 + 16 * j + (lane & 15), a.N - 1) * a.ldb;
    f8_v4f acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = f8_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    for (int g = 0; g * 128 < a.K; ++g) {
        const int k = 128 * g + 32 * (lane >> 4);
        const ckq_v4i x0 = f8_chunk(pa, k, a.K), x1 = f8_chunk(pa, k + 16, a.K);
        const f8_v8h x[4] = {f8_half(x0[0], x0[1]), f8_half(x0[2], x0[3]), f8_half(x1[0], x1[1]), f8_half(x1[2], x1[3])};
        const float s = a.sa[(size_t)g * a.ldsa + tok] * sb[(size_t)(n0 >> 7) * a.ldsb + g];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const ckq_v4i w0 = f8_chunk(pb[j], k, a.K), w1 = f8_chunk(pb[j], k + 16, a.K);
            f8_v4f p = {0.0f, 0.0f, 0.0f, 0.0f};
            p = __builtin_amdgcn_mfma_f32_16x16x32_f16(f8_half(w0[0], w0[1]), x[0], p, 0, 0, 0);
            p = __builtin_amdgcn_mfma_f32_16x16x32_f16(f8_half(w0[2], w0[3]), x[1], p, 0, 0, 0);
            p = __builtin_amdgcn_mfma_f32_16x16x32_f16(f8_half(w1[0], w1[1]), x[2], p, 0, 0, 0);
            p = __builtin_amdgcn_mfma_f32_16x16x32_f16(f8_half(w1[2], w1[3]), x[3], p, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] = __builtin_fmaf(s, p[i], acc[j][i]);
        }
    }
    if (m0 + (lane & 15) >= mend) return;
    E *out = (E *)a.C + (size_t)tok * a.ldc;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = n0 + 16 * j + 4 * (lane >> 4) + i;
            if (n < a.N) out[n] = (E)(acc[j][i] + (bias ? bias[n] : 0.0f));
        }
}

template <class E>
static int launch_gemm_f8(const F8Args &a, hipStream_t s)
{
    const int ntt = a.offsets ? a.M / 16 + min(a.M, a.experts) : (a.M + 15) / 16, nnt = (a.N + 255) / 256;
    if ((long)ntt * nnt >= 1l << 24) return CKQ_EINVAL;
    return i8_launch(gemm_f8_kernel<E>, dim3((u32)(ntt * nnt)), dim3(256), s, a, nnt);
}

static int f8_gemm(const F8Args &a, int type, void *stream)
{
    if (!a.A || !a.sa || !a.B || !a.sb || !a.C || a.M <= 0 || a.N <= 0 || a.K <= 0 || a.lda < a.K || a.ldb < a.K || a.ldc < a.N || a.ldsa < a.M ||
        a.ldsb < a.K / 128 + (a.K % 128 != 0)) return CKQ_EINVAL;
    const int size = row_size(type);
    if (!size) return CKQ_EFORMAT;
    if (((uintptr_t)a.A | (uintptr_t)a.B) % 16 || a.lda % 16 || a.ldb % 16 || a.eb % 16 || a.lda > CKQ_I8_PITCH_MAX || a.ldb > CKQ_I8_PITCH_MAX) return CKQ_EROWS;
    if ((uintptr_t)a.C % size || ((uintptr_t)a.sa | (uintptr_t)a.sb | (uintptr_t)a.bias | (uintptr_t)a.offsets) % 4) return CKQ_EROWS;
    const hipStream_t s = (hipStream_t)stream;
    return type == CKQ_T_F32 ? launch_gemm_f8<float>(a, s) : type == CKQ_T_BF16 ? launch_gemm_f8<__bf16>(a, s) : launch_gemm_f8<_Float16>(a, s);
}

extern "C" int ckq_launch_gemm_f8(const uint8_t *A, long lda, const float *sa, long ldsa, const uint8_t *B, long ldb, const float *sb, long ldsb, const float *bias,
                                  int type, void *C, long ldc, int M, int N, int K, void *stream)
{
    return f8_gemm({A, B, sa, sb, bias, nullptr, C, lda, ldsa, ldb, 0, ldsb, 0, ldc, M, N, K, 1}, type, stream);
}

extern "C" int ckq_launch_gemm_f8_experts(const uint8_t *A, long lda, const float *sa, long ldsa, const uint8_t *B, long ldb, long eb, const float *sb, long ldsb, long esb,
                                          const float *bias, const int32_t *offsets, int experts, int type, void *C, long ldc, int M, int N, int K, void *stream)
{
    if (!offsets || experts <= 0 || experts > CKQ_MOE_EXPERTS_MAX || eb < 0 || esb < 0) return CKQ_EINVAL;
    return f8_gemm({A, B, sa, sb, bias, offsets, C, lda, ldsa, ldb, eb, ldsb, esb, ldc, M, N, K, experts}, type, stream);
}
