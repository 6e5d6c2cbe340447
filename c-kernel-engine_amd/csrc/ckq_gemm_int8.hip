/*
 * ckq_gemm_int8.hip - matrix product of int8 rows with one scale each (one a token, one a channel):
 *
 *   C[m][n] = T((sa[m] * (float) sum_k A[m][k] B[n][k]) * sb[n]  (+ bias[n]))
 *
 * The sum is exact in int32 for k <= 131071 (128 * 128 * k < 2^31), so no order of it, and no split, changes a bit, and what follows it
 * is the same few fp32 operations everywhere: a token's results have the same bits whichever kernel computes them, alone or
 * among thousands.
 *
 * Three forms:
 * - gemm_i8_stream_kernel, one or two tokens (four of short rows): rows streamed once, v_dot4_i32_i8.  Bound by memory: 11008 x 4096 at one token 7.8 us
 *   with three sets in turn, which the 256 MB cache holds, 5.8 TB/s (a kernel that only reads those bytes takes 7.3), and 8.4 with nine, which it does not.
 * - gemm_i8_split_kernel, a few to some hundred tokens: small tiles, K split among the waves of a block, which exchange their sums once.
 *   Bound by memory where rows are read once (13 x 4096 x 11008 9.5 us, 4.8 TB/s, with three sets in turn, 13.2 with nine), beyond by what a CU can load, 64 bytes a cycle at best (both
 *   operands of every tile: 333 x 1001 x 4847, 231 tiles, 390 KB a CU, 3 us of 9.1, of which a launch takes 3.3).
 * - gemm_i8_tile_kernel, tiles of 64 x 64 to 256 x 256 on all waves of a block, v_mfma_i32_32x32x32_i8.  The largest are bound by the matrix
 *   cores at the clock that the power limit leaves them (8192 x 8192 x 8192: 464 us, 2370 TOPS, matrix cores busy in 71 % of the cycles at
 *   1.6 GHz; the published 5 POP/s are at 2.4).  The smaller ones have a step's copies (40 KB of 128 x 192, 640 cycles at 64 bytes) and reads of LDS beside its multiplications
 *   (768 cycles) and come near the longest of these while few CUs work (0.43 us a step, the multiplications alone 0.37), not with all of them
 *   (512 x 11008 x 4096 0.63: without copies 0.52, without reads too 0.39, the copies alone 0.41); a launch, the first copies and the last stores are 6 of its 26 us.
 * All operands reach the matrix cores through LDS: 16 rows x 64 bytes an instruction, as the matrix cores want them in registers, load at 16 bytes a
 * cycle and CU.
 */
#include "ckq_gemm_common.hpp"
#include "ckq_int8.hpp"
#include <atomic>

struct I8Args {
    const int8_t *A, *B;
    const float  *sa, *sb, *bias;
    void         *C;
    long          lda, ldb, ldc;
    int           M, N, K;
};

/* Uncontracted, so that every kernel has the same bits. */
__device__ __forceinline__ float i8_result(int sum, float sa, float sb, bool with_bias, float bias)
{
#pragma clang fp contract(off)
    const float v = (sa * (float)sum) * sb;
    return with_bias ? v + bias : v;
}

/* ---- tiles through LDS ---------------------------------------------------------------------------------------------- */

/* Which tile the t-th of a launch is: tiles are dealt to the XCDs in equal runs (gemm_deal), and in the order of a run eight token
 * tiles lie beside each other for every tile of rows, so that the tiles an XCD works on at a time share both operands in its L2. */
__device__ __forceinline__ bool i8_which_tile(int t, int ntt, int nnt, int &tt, int &nt)
{
    if (t < 0) return false;
    const int band = t / (8 * nnt), in = t - band * 8 * nnt, wide = min(8, ntt - 8 * band);
    nt = in / wide;
    tt = 8 * band + in - nt * wide;
    return true;
}

typedef float ckq_v4f __attribute__((ext_vector_type(4)));
template <class E> struct __attribute__((packed, aligned(sizeof(E)))) i8_out8 { E v[8]; };

/* Results leave non-temporally: they are not read again by the launch that writes them, and what stays in the L2s is written back
 * when it ends, with nothing beside it (2048 x 8192 x 4096 in bf16, 64.9 -> 60.7 us, of which the results' 33 MB 7 at the rate of a copy). */
typedef u32 i8_u4 __attribute__((ext_vector_type(4)));
typedef i8_u4 __attribute__((aligned(2))) i8_u4_at_2;        /* one store of 16 bytes, wherever it falls */
template <class E> __device__ __forceinline__ void i8_put(E *out, const i8_out8<E> &o)
{
    struct { i8_u4 v[sizeof(o) / 16]; } w = __builtin_bit_cast(decltype(w), o);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(o) / 16); ++i) __builtin_nontemporal_store(w.v[i], reinterpret_cast<i8_u4_at_2 *>(out) + i);
}

/* Eight rows' sums of a token, scaled and stored to C[t][n ..]; sums, scales and bias in LDS. */
template <class E>
__device__ __forceinline__ void i8_store8(const I8Args &a, const void *sums, float sa, const float *sb, const float *bias, int t, int n)
{
    const ckq_v4i *s = reinterpret_cast<const ckq_v4i *>(sums);
    const ckq_v4f *fb = reinterpret_cast<const ckq_v4f *>(sb), *fc = reinterpret_cast<const ckq_v4f *>(bias);
    const int left = a.N - n;
    i8_out8<E> o;
#pragma unroll
    for (int r = 0; r < 8; ++r) o.v[r] = (E)i8_result(s[r >> 2][r & 3], sa, fb[r >> 2][r & 3], a.bias != nullptr, fc[r >> 2][r & 3]);
    if (t >= a.M || left <= 0) return;
    E *out = (E *)a.C + (size_t)t * a.ldc + n;
    if (left >= 8) i8_put(out, o);
    else {
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < left) out[r] = o.v[r];
    }
}

/* WT x WN waves that multiply, each 32 TT tokens x 32 TN rows; NP others that copy, or none (the former do it then); S stages in LDS; FM: see
 * `multiply`. */
template <int WT_, int WN_, int TT_, int TN_, int NP_, int S_, int FM_> struct I8Tile {
    static constexpr int WT = WT_, WN = WN_, TT = TT_, TN = TN_, NP = NP_, S = S_, FM = FM_;
    static constexpr int NW = WT * WN, BT = 32 * TT * WT, BN = 32 * TN * WN, KS = 128, STAGE = (BT + BN) * KS, WAVES = NW + NP;
    static constexpr int NCW = NP ? NP : NW, NCA = BT / 8 / NCW, NCB = BN / 8 / NCW;   /* waves that copy, copies of each a step: eight rows */
    /* the sums on their way out, in the stages' place, 32 tokens a wave and round (see `finish`), all of them in one if they fit */
    static constexpr int PITCH = (NP ? BN : 32 * TN) * 4 + 16, ROUND = 32 * (NP ? WT : NW) * PITCH, AT_ONCE = NP && TT * ROUND <= S * STAGE ? TT : 1;
    static constexpr int SCALES = S * STAGE > ROUND ? S * STAGE : ROUND, LDS = SCALES + 4 * (BT + 2 * BN);
    static_assert(NCW % 2 == 0 && BT % (8 * NCW) == 0 && BN % (8 * NCW) == 0, "whole copies");
    static_assert(BT % 64 == 0 && BN % 64 == 0, "whole copies of the scales");
    static_assert(NP || S == 2, "waves that copy and multiply have a step under way");
    static_assert((S - 1) * (NCA + NCB) < 64 && FM <= TT * TN && LDS <= 160 * 1024, "what a wave can count, a place among the multiplications, one block");
};

template <class E, class T>
__device__ __forceinline__ void i8_tile(const I8Args &a, int m0, int n0, uint8_t *lds)
{
    constexpr int WT = T::WT, WN = T::WN, TT = T::TT, TN = T::TN, NP = T::NP, S = T::S, FM = T::FM, NW = T::NW, BT = T::BT, BN = T::BN, KS = T::KS, STAGE = T::STAGE, NCA = T::NCA;
    constexpr int NCW = T::NCW, NC = T::NCA + T::NCB, NM = TT * TN, NF = TT + TN, PITCH = T::PITCH;
    const int lane = threadIdx.x & 63, wave = wave_in_block(), cw = NP ? wave - NW : wave;
    const ckq_v4i rsa = gemm_buffer((const uint8_t *)a.A + (size_t)m0 * a.lda), rsb = gemm_buffer((const uint8_t *)a.B + (size_t)n0 * a.ldb);
    const u32 base = lds_address(lds);
    const int niter = (a.K + KS - 1) / KS, last = niter - 1, tail = a.K - last * KS;      /* bytes of the last step, 1 .. 128 */

    /* a copy takes eight rows of 128 bytes; the chunk of 16 that a lane fetches is the one that belongs in its place, c ^ (row / 2 % 8):
     * sixteen rows' chunks c, which a phase of a read of 16 bytes a lane takes, then lie on all 64 banks once (c ^ (row % 8): twice, 8.3 cycles a read and not 4.2) */
    u32 ofs[NC];
    const int chunk = (lane & 7) ^ ((4 * cw + (lane >> 4)) & 7);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int row = 8 * (cw + NCW * (i < NCA ? i : i - NCA)) + (lane >> 3);
        ofs[i] = i < NCA ? (u32)min(row, a.M - 1 - m0) * (u32)a.lda : (u32)min(row, a.N - 1 - n0) * (u32)a.ldb;
        ofs[i] += 16u * (u32)chunk;
    }
    auto copy = [&](int i, int it, int buf) {
        /* chunks behind the row's last are read from its start; the tokens' are zeroed (clear_tail) */
        const u32 o = it == last && 16 * chunk >= tail ? ofs[i] - 16u * (u32)chunk : ofs[i];
        const u32 dst = base + (u32)(buf * STAGE + 1024 * (cw + NCW * (i < NCA ? i : i - NCA)) + (i < NCA ? 0 : BT * KS));
        lds_copy16(i < NCA ? rsa : rsb, dst, o, it * KS);
    };
    auto copy_step = [&](int it, int buf) {
#pragma unroll
        for (int c = 0; c < NC; ++c) copy(c, it, buf);
    };
    auto clear_tail = [&](int buf) {                           /* all waves; then they meet */
        for (int e = threadIdx.x; e < BT * 8; e += 64 * T::WAVES) {
            const int row = e >> 3, left = tail - 16 * ((e & 7) ^ ((row >> 1) & 7));
            if (left >= 16) continue;
            ckq_v4i *p = reinterpret_cast<ckq_v4i *>(lds + buf * STAGE + 16 * e);
            ckq_v4i v = *p;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = left - 4 * i;
                v[i] = n >= 4 ? v[i] : n <= 0 ? 0 : v[i] & (int)((1u << (8 * n)) - 1u);
            }
            *p = v;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
    };

    /* the scales and the bias, BT, BN and BN floats, behind the stages: fetched first, used last */
    float *scales = reinterpret_cast<float *>(lds + T::SCALES);
    if (cw >= 0)
        for (int i = cw; i < (BT + 2 * BN) / 64; i += NCW) {
            const bool tok = i < BT / 64, ch = i < (BT + BN) / 64;
            const float *p = tok ? a.sa : ch ? a.sb : a.bias;
            if (!p) continue;
            const int e = 64 * i + lane - (tok ? 0 : ch ? BT : BT + BN);
            lds_copy4(gemm_buffer((const uint8_t *)(p + (tok ? m0 : n0))), base + (u32)T::SCALES + 256u * (u32)i, 4u * (u32)min(e, tok ? a.M - 1 - m0 : a.N - 1 - n0), 0);
        }

    /* The sums through LDS, where nothing is read or copied any more, so that a lane has eight rows' results of one token and a token's leave in whole lines.  The
     * waves that copied store too (four and four waves, 128 x 192: 0.9 us of 27.1 at 512 x 11008 x 4096); eight that are alone have a piece each and wait for no
     * other (256 x 256: 43.2 us, together 45.6 at 512 x 4096 x 4096).  `put` brings a round's sums there. */
    auto finish = [&](auto &&put) {
        constexpr int PER = (NP ? T::BN : 32 * TN) / 8, JOBS = 32 * PER * (NP ? WT * T::AT_ONCE : 1);
#pragma unroll
        for (int round = 0; round < TT; round += T::AT_ONCE) {
            if (NP && round) __syncthreads();
            put(round);
            if (NP) __syncthreads();
            else    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 2
            for (int e = NP ? threadIdx.x : lane; e < JOBS; e += NP ? 64 * T::WAVES : 64) {
                const int row = e / PER, c = 8 * (e % PER) + (NP ? 0 : 32 * TN * (wave % WN)), k = row / (32 * WT), w = NP ? row / 32 % WT : wave / WN;
                const int tok = 32 * (TT * w + round + k) + row % 32;
                i8_store8<E>(a, lds + (NP ? row : 32 * wave + row) * PITCH + 4 * (8 * (e % PER)), scales[tok], scales + BT + c, scales + BT + T::BN + c, m0 + tok, n0 + c);
            }
            if (!NP) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    };

    /* Step `it` has stage it % S.  A step's last operands are read before its last quarter is multiplied; the barrier is there, so
     * that no wave waits with nothing to multiply: all have step it's operands in registers, and step it + 1 has arrived; from there on the
     * stage takes the copies of step it + S. */
    if (NP > 0 && wave >= NW) {
        /* A copy holds its wave until the address unit has taken it, 16 cycles and more, and with it whatever the wave would
         * have multiplied; waves that do nothing else take that from the others (us without | with them: 512 x 11008 x 4096 27.2 | 24.2, 1024 x 4096 x 4096 22.3 |
         * 19.1, 125 x 11008 x 4096 14.8 | 13.0). */
#pragma unroll
        for (int st = 0; st < S; ++st)
            if (st < niter) copy_step(st, st);
        if (niter >= S) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * NC) : "memory");
        else            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (last == 0 && tail < KS) clear_tail(0);
        int buf = 0;
        for (int it = 0; it < niter; ++it) {
            const int next = buf + 1 == S ? 0 : buf + 1;
            if (it + S - 1 < niter) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * NC) : "memory");
            else                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            if (it + 1 == last && tail < KS) clear_tail(next);
            if (it + S < niter) copy_step(it + S, buf);
            buf = next;
        }
        finish([](int) {});
        return;
    }

    /* where a lane's operands are: row lane % 32 of a group of 32, bytes 16 (lane / 32) of the 32 of a multiplication */
    const int wt = wave / WN, wn = wave % WN, half = lane >> 5;
    u32 ra[4], rb[4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        const u32 pos = 16u * (u32)((2 * kk + half) ^ ((lane >> 1) & 7));
        ra[kk] = (u32)(32 * TT * wt + (lane & 31)) * KS + pos;
        rb[kk] = (u32)(BT + 32 * TN * wn + (lane & 31)) * KS + pos;
    }
    ckq_v16i acc[TT][TN];
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = ckq_v16i{};
    ckq_v4i fa[2][TT], fb[2][TN];
    auto fetch = [&](int to, int buf, int kk, int f) {         /* operand f of 32 bytes of K, in the order of their use: a row group, all tokens, the other rows */
        const uint8_t *p = lds + buf * STAGE;
        if (f == 0)       fb[to][0] = *reinterpret_cast<const ckq_v4i *>(p + rb[kk]);
        else if (f <= TT) fa[to][f - 1] = *reinterpret_cast<const ckq_v4i *>(p + ra[kk] + 32 * KS * (f - 1));
        else              fb[to][f - TT] = *reinterpret_cast<const ckq_v4i *>(p + rb[kk] + 32 * KS * (f - TT));
    };
    /* The multiplications of 32 bytes of K; among the first FM of them the reads of the next 32 bytes' operands, and, where these waves
     * copy too, over the first half of a step the copies of the next: a burst of all waves' copies leaves the matrix cores idle for
     * their sum, and the last of them has to arrive in what is left of the step. */
    auto multiply = [&](int from, int quarter, int it, int buf, int fbuf, int fkk) {
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            const int j = m / TT, i = m % TT;
            acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[from][j], fa[from][i], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int f = 0; f < NF; ++f)
                if (f * FM / NF == m && fbuf >= 0) fetch(from ^ 1, fbuf, fkk, f);
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (NP == 0 && c * NM * 2 / NC == quarter * NM + m && it < niter) copy(c, it, buf);
            __builtin_amdgcn_sched_barrier(0);                 /* or the compiler moves the reads to where they are used, and waits for each */
        }
    };

    if (NP == 0) {
        copy_step(0, 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __builtin_amdgcn_s_barrier();
    if (last == 0 && tail < KS) clear_tail(0);
    if (NP == 0 && niter > 1) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (c * 2 < NC) copy(c, 1, 1);
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) fetch(0, 0, 0, f);
    int buf = 0;
    for (int it = 0; it < niter; ++it) {
        const int next = buf + 1 == S ? 0 : buf + 1;
#pragma unroll
        for (int kk = 0; kk < 3; ++kk) multiply(kk & 1, kk + 1, it + 1, next, buf, kk + 1);
        if (NP == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        else         asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (it + 1 == last && tail < KS) clear_tail(next);
        multiply(1, 0, it + 2, buf, it < last ? next : -1, 0);
        buf = next;
    }

    finish([&](int round) {
#pragma unroll
        for (int k = 0; k < T::AT_ONCE; ++k)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const ckq_v16i &c = acc[round + k][j];
                    *reinterpret_cast<ckq_v4i *>(lds + (32 * (NP ? WT * k + wt : wave) + (lane & 31)) * PITCH + 4 * (32 * ((NP ? TN * wn : 0) + j) + 8 * g + 4 * half)) =
                        ckq_v4i{c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]};
                }
    });
}

template <class E, class T>
__global__ void __launch_bounds__(64 * T::WAVES) gemm_i8_tile_kernel(I8Args a, int ntt, int nnt)
{
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::LDS];
    int tt, nt;
    if (i8_which_tile(gemm_deal(blockIdx.x, ntt * nnt), ntt, nnt, tt, nt)) i8_tile<E, T>(a, tt * T::BT, nt * T::BN, lds);
}

/* The first nnt1 columns of tiles of T1, `blocks1` blocks of them, and the rows that they leave in tiles of T2. */
template <class E, class T1, class T2>
__global__ void __launch_bounds__(64 * T1::WAVES) gemm_i8_two_tiles_kernel(I8Args a, int ntt1, int nnt1, int blocks1, int ntt2, int nnt2)
{
    static_assert(T1::WAVES == T2::WAVES, "one size of block");
    __shared__ __attribute__((aligned(16))) uint8_t lds[T1::LDS > T2::LDS ? T1::LDS : T2::LDS];
    int tt, nt;
    if ((int)blockIdx.x < blocks1) {
        if (i8_which_tile(gemm_deal(blockIdx.x, ntt1 * nnt1), ntt1, nnt1, tt, nt)) i8_tile<E, T1>(a, tt * T1::BT, nt * T1::BN, lds);
    } else if (i8_which_tile(gemm_deal(blockIdx.x - blocks1, ntt2 * nnt2), ntt2, nnt2, tt, nt))
        i8_tile<E, T2>(a, tt * T2::BT, nnt1 * T1::BN + nt * T2::BN, lds);
}

template <class E, class T>
static int launch_i8_tiles(const I8Args &a, hipStream_t s)
{
    const int ntt = (a.M + T::BT - 1) / T::BT, nnt = (a.N + T::BN - 1) / T::BN;
    if ((long)ntt * nnt > 0x3fffff) return CKQ_EINVAL;       /* results beyond any memory */
    return i8_launch(gemm_i8_tile_kernel<E, T>, dim3((unsigned)gemm_blocks(ntt, nnt)), dim3(64u * T::WAVES), s, a, ntt, nnt);
}
template <class E, class T1, class T2>
static int launch_i8_two_tiles(const I8Args &a, int nnt1, hipStream_t s)
{
    const int ntt1 = (a.M + T1::BT - 1) / T1::BT, ntt2 = (a.M + T2::BT - 1) / T2::BT, nnt2 = (a.N - nnt1 * T1::BN + T2::BN - 1) / T2::BN;
    if ((long)ntt1 * nnt1 + (long)ntt2 * nnt2 > 0x3fffff) return CKQ_EINVAL;
    const int blocks1 = gemm_blocks(ntt1, nnt1);
    return i8_launch(gemm_i8_two_tiles_kernel<E, T1, T2>, dim3((unsigned)(blocks1 + gemm_blocks(ntt2, nnt2))), dim3(64u * T1::WAVES), s, a, ntt1, nnt1, blocks1, ntt2, nnt2);
}

/* ---- K split among the waves of a block ------------------------------------------------------------------------------ */

/* 16 TG tokens x 16 RN rows a block of NW waves; every wave has all of the tile and each NW-th step of 128 bytes of K, through S stages of
 * its own, so that nothing is waited for but its own copies until the waves' sums meet at the end. */
template <int NW_, int RN_, int TG_, int S_> struct I8Split {
    static constexpr int NW = NW_, RN = RN_, TG = TG_, S = S_, KS = 128;
    static constexpr int BT = 16 * TG, BN = 16 * RN, STAGE = (BT + BN) * KS, PITCH = BN * 4 + 16;
    static constexpr int LDS = NW * (S * STAGE > BT * PITCH ? S * STAGE : BT * PITCH);
    static_assert(LDS <= 160 * 1024, "one block fits");
};

template <class E, class T>
__global__ void __launch_bounds__(64 * T::NW) gemm_i8_split_kernel(I8Args a, int ntt, int nnt)
{
    constexpr int NW = T::NW, RN = T::RN, TG = T::TG, S = T::S, KS = T::KS, BT = T::BT, BN = T::BN, STAGE = T::STAGE, NC = 2 * (RN + TG), PITCH = T::PITCH;
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::LDS];
    const int lane = threadIdx.x & 63, wave = wave_in_block();
    int tt, nt;
    {
        const int t = gemm_deal(blockIdx.x, ntt * nnt);
        if (t < 0) return;
        nt = t / ntt;                                         /* token tiles side by side: they share the rows */
        tt = t - nt * ntt;
    }
    const int m0 = tt * BT, n0 = nt * BN;

    /* what this thread stores in the end, eight rows of a token: their scales and bias are fetched before anything else, or the block would
     * end with a trip to memory */
    constexpr int PER = BN / 8, JOBS = BT * PER;
    static_assert(JOBS <= 64 * NW, "a job a thread");
    const int row = (int)threadIdx.x / PER, col = 8 * ((int)threadIdx.x % PER), t = m0 + row, n8 = n0 + col, left = a.N - n8;
    const bool job = (int)threadIdx.x < JOBS && t < a.M && left > 0;
    float sa = 0.0f, sb[8], bias[8];
    if (job) {
        sa = a.sa[t];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            sb[r] = a.sb[n8 + min(r, left - 1)];
            bias[r] = a.bias ? a.bias[n8 + min(r, left - 1)] : 0.0f;
        }
    }
    const ckq_v4i rsa = gemm_buffer((const uint8_t *)a.A + (size_t)m0 * a.lda), rsb = gemm_buffer((const uint8_t *)a.B + (size_t)n0 * a.ldb);
    const u32 mine = (u32)(wave * S * STAGE);
    const int niter = (a.K + KS - 1) / KS, last = niter - 1, tail = a.K - last * KS, steps = wave < niter ? (niter - 1 - wave) / NW + 1 : 0;

    u32 ofs[NC];
    const int half8 = lane >> 3;                              /* row of a copy's eight */
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int cr = 8 * (i < 2 * TG ? i : i - 2 * TG) + half8, chunk = (lane & 7) ^ ((cr >> 1) & 7);
        ofs[i] = (i < 2 * TG ? (u32)min(cr, a.M - 1 - m0) * (u32)a.lda : (u32)min(cr, a.N - 1 - n0) * (u32)a.ldb) + 16u * (u32)chunk;
    }
    auto copy = [&](int j, int slot) {
        const int it = wave + NW * j;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int cr = 8 * (i < 2 * TG ? i : i - 2 * TG) + half8, chunk = (lane & 7) ^ ((cr >> 1) & 7);
            const u32 o = it == last && 16 * chunk >= tail ? ofs[i] - 16u * (u32)chunk : ofs[i];
            lds_copy16(i < 2 * TG ? rsa : rsb, lds_address(lds) + mine + (u32)(slot * STAGE + 1024 * i), o, it * KS);
        }
    };
    ckq_v4i acc[TG][RN];
#pragma unroll
    for (int i = 0; i < TG; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = ckq_v4i{0, 0, 0, 0};

#pragma unroll
    for (int j = 0; j < S - 1; ++j)
        if (j < steps) copy(j, j);
    int slot = 0;
    for (int j = 0; j < steps; ++j) {
        if (j + S - 1 < steps) {
            copy(j + S - 1, slot == 0 ? S - 1 : slot - 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * NC) : "memory");
        } else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint8_t *p = lds + mine + slot * STAGE;
        const bool cut = wave + NW * j == last && tail < KS;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int c = 4 * kk + (lane >> 4);
            const u32 at = (u32)((lane & 15) * KS + 16 * (c ^ ((lane >> 1) & 7)));
            ckq_v4i fa[TG], fb[RN];
#pragma unroll
            for (int i = 0; i < TG; ++i) fa[i] = *reinterpret_cast<const ckq_v4i *>(p + at + 16 * KS * i);
#pragma unroll
            for (int i = 0; i < RN; ++i) fb[i] = *reinterpret_cast<const ckq_v4i *>(p + at + (BT + 16 * i) * KS);
            if (cut) {                                        /* bytes behind the row's last are anything: not the tokens' */
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int n = tail - 16 * c - 4 * w;
                    const int keep = n >= 4 ? -1 : n <= 0 ? 0 : (int)((1u << (8 * n)) - 1u);
#pragma unroll
                    for (int i = 0; i < TG; ++i) fa[i][w] &= keep;
                }
            }
#pragma unroll
            for (int i = 0; i < TG; ++i)
#pragma unroll
                for (int n = 0; n < RN; ++n) acc[i][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[n], fa[i], acc[i][n], 0, 0, 0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    /* the next copies into this slot come after its reads */
        slot = slot + 1 == S ? 0 : slot + 1;
    }

    /* the waves' sums meet in LDS; eight rows of a token a thread */
    __syncthreads();
    uint8_t *red = lds + wave * BT * PITCH;
#pragma unroll
    for (int i = 0; i < TG; ++i)
#pragma unroll
        for (int n = 0; n < RN; ++n)
            *reinterpret_cast<ckq_v4i *>(red + (16 * i + (lane & 15)) * PITCH + 4 * (16 * n + 4 * (lane >> 4))) = acc[i][n];
    __syncthreads();
    if (!job) return;
    ckq_v4i s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const ckq_v4i *s = reinterpret_cast<const ckq_v4i *>(lds + w * BT * PITCH + row * PITCH + 4 * col);
        s0 += s[0];
        s1 += s[1];
    }
    i8_out8<E> o;
#pragma unroll
    for (int r = 0; r < 8; ++r) o.v[r] = (E)i8_result(r < 4 ? s0[r] : s1[r - 4], sa, sb[r], a.bias != nullptr, bias[r]);
    E *out = (E *)a.C + (size_t)t * a.ldc + n8;
    if (left >= 8) i8_put(out, o);
    else {
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < left) out[r] = o.v[r];
    }
}

template <class E, class T>
static int launch_i8_split(const I8Args &a, hipStream_t s)
{
    const int ntt = (a.M + T::BT - 1) / T::BT, nnt = (a.N + T::BN - 1) / T::BN;
    if ((long)ntt * nnt > 0x3fffff) return CKQ_EINVAL;       /* results beyond any memory */
    return i8_launch(gemm_i8_split_kernel<E, T>, dim3((unsigned)gemm_blocks(ntt, nnt)), dim3(64u * T::NW), s, a, ntt, nnt);
}

/* ---- few tokens: rows streamed ----------------------------------------------------------------------------------------- */

/* MT tokens; a wave has R rows and every KS-th piece of KU KB of K; 4 waves a block.  Rows are loaded non-temporally: a decode step goes through
 * more weights than any cache holds (nine matrices of 11008 x 4096 in turn 8.45 us each and 8.93 otherwise, 4096 x 11008 9.0 and 9.6; three, which fit the
 * 256 MB cache, 8.25 and 8.03). */
template <class E, int MT, int R, int KU, int KS>
__global__ void __launch_bounds__(256) gemm_i8_stream_kernel(I8Args a)
{
    constexpr int G = 4 / KS;
    __shared__ int red[KS > 1 ? 4 * R * MT : 1];
    const int lane = threadIdx.x & 63, wave = wave_in_block();
    const int part = wave % KS, n0 = ((int)blockIdx.x * G + wave / KS) * R;
    if (KS == 1 && n0 >= a.N) return;
    const uint8_t *pb[R], *pa[MT];
#pragma unroll
    for (int r = 0; r < R; ++r) pb[r] = (const uint8_t *)a.B + (size_t)min(n0 + r, a.N - 1) * a.ldb;
#pragma unroll
    for (int t = 0; t < MT; ++t) pa[t] = (const uint8_t *)a.A + (size_t)min(t, a.M - 1) * a.lda;
    /* lane r + R t has row r of token t in the end; its scales and bias come first, or the wave would end with a trip to memory */
    const int n = n0 + lane % R, tok = lane / R;
    const bool job = lane < R * MT && tok < a.M && n < a.N;
    const float sa = a.sa[job ? tok : 0], sb = a.sb[job ? n : 0], bias = a.bias ? a.bias[job ? n : 0] : 0.0f;
    int acc[R][MT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[r][t] = 0;
    for (int k0 = part * KU * 1024; k0 < a.K; k0 += KS * KU * 1024) {
        ckq_v4i w[R][KU], x[MT][KU];
        u32 at[KU];
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            at[u] = (u32)k0 + 1024u * u + 16u * (u32)lane;
            if ((int)at[u] >= a.K) at[u] = 0;                /* counted out below */
        }
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) w[r][u] = __builtin_nontemporal_load(reinterpret_cast<const ckq_v4i *>(pb[r] + at[u]));
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t) x[t][u] = *reinterpret_cast<const ckq_v4i *>(pa[t] + at[u]);
        if (k0 + KU * 1024 > a.K) {
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = a.K - (k0 + 1024 * u + 16 * lane + 4 * i), keep = n >= 4 ? -1 : n <= 0 ? 0 : (int)((1u << (8 * n)) - 1u);
#pragma unroll
                    for (int t = 0; t < MT; ++t) x[t][u][i] &= keep;
                }
        }
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[r][t] = dot4(w[r][u][i], x[t][u][i], acc[r][t]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[r][t] = __builtin_amdgcn_readlane(group_sum<64>(acc[r][t]), 63);
    if (KS > 1) {
        if (lane == 0) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int t = 0; t < MT; ++t) red[(wave * R + r) * MT + t] = acc[r][t];
        }
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int w = 1; w < KS; ++w) acc[r][t] += red[((wave + w) * R + r) * MT + t];
    }
    int sum = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) sum = lane == r + R * t ? acc[r][t] : sum;
    if (!job) return;
    ((E *)a.C)[(size_t)tok * a.ldc + n] = (E)i8_result(sum, sa, sb, a.bias != nullptr, bias);
}

template <class E, int MT, int R, int KU, int KS>
static int launch_i8_stream(const I8Args &a, hipStream_t s)
{
    constexpr int per = 4 / KS * R;
    return i8_launch(gemm_i8_stream_kernel<E, MT, R, KU, KS>, dim3((unsigned)((a.N + per - 1) / per)), dim3(256), s, a);
}

/* ---- which kernel ------------------------------------------------------------------------------------------------------ */

/* Stages and waves as measured, us.  What waves that only copy gain: see i8_tile; none at 256 x 256, where the eight that multiply need 216 registers and a block
 * of twelve waves has 168 each (sixteen waves of 64 x 64 are no faster: 8192 x 8192 x 8192 1.5 % slower).  1024 x 4096 x 4096, 128 x 128: four waves multiplying 64 x 64 each, three stages 21.7, four 22.1,
 * with two to copy 23.4; eight multiplying 32 x 64 22.8.  2048 x 4096 x 4096, 256 x 128: eight and four waves, three stages 35.5, two 37.1.  125 x 11008 x 4096, 64 x 128:
 * four stages 13.2, five 13.4, three 13.9.  500 x 2000 x 2000, 64 x 64: four stages, so that two blocks share a CU, 8.4; six 8.8. */
typedef I8Tile<2, 4, 4, 2, 0, 2, 3> T256x256;
typedef I8Tile<4, 2, 2, 3, 4, 2, 5> T256x192;
typedef I8Tile<4, 2, 2, 2, 4, 3, 2> T256x128;
typedef I8Tile<2, 2, 2, 3, 4, 3, 3> T128x192;
typedef I8Tile<2, 2, 2, 2, 4, 3, 3> T128x128;
typedef I8Tile<2, 2, 1, 2, 4, 4, 2> T64x128;
typedef I8Tile<2, 2, 1, 1, 4, 4, 1> T64x64;                 /* two blocks a CU */
/* Split tiles.  13 x 4096 x 11008: 16 x 16 of eight waves, two stages 10.0, three 10.3, four 10.4; of sixteen 10.5, of four with four stages 10.4; 16 x 32 of four
 * 11.0.  13 x 22016 x 4096: 16 x 32 of four waves, two stages 16.1 (three blocks share a CU), three 17.4, four 19; 16 x 16 19.0.  333 x 1001 x 4847: 32 x 48 of
 * four waves, two stages 9.1, three 9.5, of eight 9.1; 32 x 64 10.1. */
typedef I8Split<4, 3, 2, 2> S32x48;                   /* two blocks a CU */
typedef I8Split<4, 2, 2, 2> S32x32;                   /* two */
typedef I8Split<8, 1, 1, 2> S16x16;                   /* two */
typedef I8Split<4, 2, 1, 2> S16x32;                   /* three */

/* What a launch takes, in us: t0, and for every round of blocks t_tile and as many steps of K as a wave has, each of `step` where all
 * places have a block; a last round of fewer steps faster, for the most part by how many blocks share a CU, a fifth by how many there
 * are in all (L2, power).  Fitted to 512 sizes of 5 to 2048 tokens (64 to 32000 rows, K 64 to 11008; operands from the 256 MB cache, as three
 * sets in turn leave them), each kernel within 4 to 8 % (rms).  Fitted to half of the sizes, the kernel so chosen is on the other half 0.8 % slower than the
 * best of all on average, 1.25 times at worst; without one of them it is 0.9 to 4 % on average.  With weights from memory (28 sizes of 3 to 128 tokens, more sets in turn than the cache holds)
 * 0.9 % and 1.15 times. */
struct I8Cost { int bt, bn, places, split; float t0, t_tile, step; };
static const I8Cost i8_costs[CKQ_I8_TILINGS] = {
    {256, 256, 256, 1, 1.50f, 7.40f, 1.490f},
    {256, 192, 256, 1, 1.50f, 6.74f, 1.173f},
    {256, 128, 256, 1, 1.50f, 5.13f, 0.816f},
    {128, 192, 256, 1, 1.50f, 4.84f, 0.677f},
    {128, 128, 256, 1, 1.50f, 3.45f, 0.522f},
    {64, 128, 256, 1, 1.50f, 2.54f, 0.399f},
    {64, 64, 512, 1, 1.97f, 1.79f, 0.504f},
    {32, 48, 512, 4, 2.16f, 1.14f, 0.890f},
    {32, 32, 512, 4, 2.29f, 1.02f, 0.660f},
    {16, 16, 512, 8, 2.36f, 1.03f, 0.553f},
    {16, 32, 768, 4, 2.72f, 0.64f, 0.799f},
};

static float i8_rounds(const I8Cost &c, long tiles, int K)
{
    const int steps = ((K + 127) / 128 + c.split - 1) / c.split, share = c.places / 256;      /* blocks that share a CU */
    const long full = tiles / c.places, rest = tiles % c.places;
    float t = (float)full * (c.t_tile + (float)steps * c.step);
    if (rest) t += c.t_tile + (float)steps * c.step * (0.2f * (float)rest / (float)c.places + 0.8f * (float)((rest + 255) / 256) / (float)share);
    return t;
}
static long i8_tiles(const I8Cost &c, int M, int N) { return (long)((M + c.bt - 1) / c.bt) * ((N + c.bn - 1) / c.bn); }

/* Columns of 256 x 256 tiles that make whole rounds of the 256 CUs: what they leave goes in tiles of 128 x 192, a shorter last round
 * (2048 x 11008 x 4096: 344 tiles of 256 x 256 in two rounds 102 us; 256 of them and 240 small ones 85). */
static int i8_whole_columns(int M, int N)
{
    const int ntt = (M + 255) / 256, nnt = (N + 255) / 256;
    return (int)((long)ntt * nnt / 256 * 256 / ntt);
}

static std::atomic<int> g_i8_kernel{-1};
extern "C" void ckq_launch_set_i8_kernel(int kernel) { g_i8_kernel.store(kernel < 0 || kernel > CKQ_I8_STREAM ? -1 : kernel); }

/* Rows are streamed (gemm_i8_stream_kernel) for one token or two, and for four where a row is one trip of a wave; at more the dot products, which
 * use four multiplications of an instruction, become the bound (us streamed | split tiles: two tokens, 11008 x 4096 8.5 | 8.8, 151936 x 896 21.1 | 28.7;
 * four, 151936 x 896 24.6 | 29.0, 11008 x 896 4.5 | 3.6, 32000 x 1500 15.5 | 9.7, 11008 x 4096 10.2 | 8.9, 11008 x 11008 23.6 | 25.5). */
static bool i8_streams(int M, int K) { return M <= 2 || (M <= 4 && K <= 1024); }

extern "C" int ckq_launch_i8_kernel(int M, int N, int K)
{
    const int forced = g_i8_kernel.load();
    if (forced >= 0 && (forced != CKQ_I8_STREAM || i8_streams(M, K)) && (forced != CKQ_I8_TWO || i8_whole_columns(M, N) > 0)) return forced;
    if (i8_streams(M, K)) return CKQ_I8_STREAM;
    int best = 0;
    float t = 1e30f;
    for (int i = 0; i < CKQ_I8_TILINGS; ++i) {
        const float ti = i8_costs[i].t0 + i8_rounds(i8_costs[i], i8_tiles(i8_costs[i], M, N), K);
        if (ti < t) { t = ti; best = i; }
    }
    const int cols = i8_whole_columns(M, N);
    if (cols > 0 && 256 * cols < N) {
        const I8Cost &a = i8_costs[CKQ_I8_256x256], &b = i8_costs[CKQ_I8_128x192];
        if (a.t0 + i8_rounds(a, (long)((M + 255) / 256) * cols, K) + i8_rounds(b, i8_tiles(b, M, N - 256 * cols), K) < t) best = CKQ_I8_TWO;
    }
    return best;
}

template <class E>
static int launch_gemm_i8(const I8Args &a, hipStream_t s)
{
    switch (ckq_launch_i8_kernel(a.M, a.N, a.K)) {
    case CKQ_I8_256x256:   return launch_i8_tiles<E, T256x256>(a, s);
    case CKQ_I8_256x192:   return launch_i8_tiles<E, T256x192>(a, s);
    case CKQ_I8_256x128:   return launch_i8_tiles<E, T256x128>(a, s);
    case CKQ_I8_128x192:   return launch_i8_tiles<E, T128x192>(a, s);
    case CKQ_I8_128x128:   return launch_i8_tiles<E, T128x128>(a, s);
    case CKQ_I8_64x128:    return launch_i8_tiles<E, T64x128>(a, s);
    case CKQ_I8_64x64:     return launch_i8_tiles<E, T64x64>(a, s);
    case CKQ_I8_S32x48:    return launch_i8_split<E, S32x48>(a, s);
    case CKQ_I8_S32x32:    return launch_i8_split<E, S32x32>(a, s);
    case CKQ_I8_S16x16:    return launch_i8_split<E, S16x16>(a, s);
    case CKQ_I8_S16x32:    return launch_i8_split<E, S16x32>(a, s);
    case CKQ_I8_TWO:       return launch_i8_two_tiles<E, T256x256, T128x192>(a, i8_whole_columns(a.M, a.N), s);
    }
    /* Rows of up to 1 KB are one trip of a wave: four rows a wave, no exchange.  Longer ones are shared by the waves of a block, so that
     * a launch has its bytes in flight at once however few rows it has.  us at one token, rows x K, (rows a wave, KB a trip, waves of a
     * row) 4, 1, 1 | 4, 1, 2 | 2, 2, 4 | 2, 4, 4: 151936 x 896 20.6 | 20.2 | 46 | 67, 32000 x 2048 12.1 | 10.9 | 11.0 | 11.6, 11008 x 4096 10.7 | 8.8 |
     * 7.8 | 8.4, 4096 x 11008 11.2 | 10.3 | 8.8 | 8.6. */
    const int kb = (a.K + 1023) / 1024;
    if (a.M == 1) return kb <= 1 ? launch_i8_stream<E, 1, 4, 1, 1>(a, s) : kb <= 2 ? launch_i8_stream<E, 1, 4, 1, 2>(a, s)
                       : kb <= 8 ? launch_i8_stream<E, 1, 2, 2, 4>(a, s) : launch_i8_stream<E, 1, 2, 4, 4>(a, s);
    if (a.M == 2) return kb <= 1 ? launch_i8_stream<E, 2, 4, 1, 1>(a, s) : kb <= 2 ? launch_i8_stream<E, 2, 4, 1, 2>(a, s) : launch_i8_stream<E, 2, 2, 2, 4>(a, s);
    return launch_i8_stream<E, 4, 4, 1, 1>(a, s);
}

extern "C" int ckq_launch_gemm_i8(const int8_t *A, long lda, const float *sa, const int8_t *B, long ldb, const float *sb, const float *bias,
                                  int type, void *C, long ldc, int M, int N, int K, void *stream)
{
    if (!A || !sa || !B || !sb || !C || M <= 0 || N <= 0 || K <= 0 || lda < K || ldb < K || ldc < N) return CKQ_EINVAL;
    const int size = type == CKQ_T_F32 ? 4 : type == CKQ_T_BF16 || type == CKQ_T_F16 ? 2 : 0;
    if (!size) return CKQ_EFORMAT;
    if (((uintptr_t)A | (uintptr_t)B) % 16 || lda % 16 || ldb % 16 || lda > CKQ_I8_PITCH_MAX || ldb > CKQ_I8_PITCH_MAX || K > CKQ_I8_K_MAX) return CKQ_EROWS;
    if ((uintptr_t)C % size || ((uintptr_t)sa | (uintptr_t)sb | (uintptr_t)bias) % 4) return CKQ_EROWS;
    /* a launch has fewer than 2^32 threads */
    constexpr int MOST = 1 << 22;
    for (int m = 0; m < M; m += min(MOST, M - m))
        for (int n = 0; n < N; n += min(MOST, N - n)) {
            const I8Args a = {A + (size_t)m * lda, B + (size_t)n * ldb, sa + m, sb + n, bias ? bias + n : nullptr,
                              (char *)C + ((size_t)m * ldc + n) * size, lda, ldb, ldc, min(MOST, M - m), min(MOST, N - n), K};
            const hipStream_t s = (hipStream_t)stream;
            const int rc = type == CKQ_T_F32 ? launch_gemm_i8<float>(a, s) : type == CKQ_T_BF16 ? launch_gemm_i8<__bf16>(a, s) : launch_gemm_i8<_Float16>(a, s);
            if (rc) return rc;
        }
    return 0;
}
