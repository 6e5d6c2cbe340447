/*
 * ckq_gemm_f8.hip - matrix product of e4m3 rows, one scale for each 128 elements of a token and each block of 128 x 128 of the weights:
 *
 *   C[m][n] = T(sum_g (sa[g][m] * sb[n / 128][g]) * (sum over k in group g of A[m][k] B[n][k])  (+ bias[n]))
 *
 * and the same of rows sorted by expert, each expert with a matrix of its own.  A group's sum starts from zero; the groups' sums are scaled and added
 * in fp32.
 *
 * Sums.  The matrix cores' e4m3 instructions add eight products at a time after aligning them to the largest of the eight and dropping what is under
 * 2^-13 of it (measured, in all their shapes; between eights they add as fp32 does): a sum of 128 random products is 1.5e-5 of its size off. e4m3
 * values are exact in fp16, and the fp16 instructions add their products as fp32 does (1e-8), at half the rate.
 *
 * Forms.  One token: rows streamed, bound by reading them (11008 x 4096 from memory 8.4 us, 5.3 TB/s).  A few tokens: K split among the waves of a
 * block, bound by a launch's and a block's start and a wave's steps one after the other (16 tokens 10.8 us, 64 11.8; one token through 8 of 64
 * experts of 2816 x 2048 10.6, 4.4 TB/s).  More: tiles, on the fp16 instructions bound by those and the conversions beside them (matrix cores busy 64
 * %, vector units 63 % of a CU's cycles: 8192^3 930 us, 1180 TFLOP/s, the library's fp16 product without scales 1371), on the e4m3 ones by the power
 * limit and by what keeps scales in fp32 (64 and 49 %: 8192^3 468 us, 2350 TFLOP/s, the library's 2607; 2048 x 11008 x 4096 87 us).
 */
#include "ckq_gemm_common.hpp"
#include "ckq_int8.hpp"
#include "ckq_rows.hpp"
#include <atomic>
#include <math.h>
#include <type_traits>

typedef int   f8_v8i __attribute__((ext_vector_type(8)));
typedef _Float16 f8_v2h __attribute__((ext_vector_type(2)));
typedef _Float16 f8_v8h __attribute__((ext_vector_type(8)));
typedef float f8_v4f __attribute__((ext_vector_type(4)));

struct F8Args {
    const uint8_t *A, *B;
    const float   *sa, *sb, *bias;
    const int32_t *offsets;                 /* experts: where each one's rows begin, experts + 1 of them; null: one matrix */
    void          *C;
    long           lda, ldsa, ldb, eb, ldsb, esb, ebias, ldc;     /* eb, esb, ebias: from one expert's matrix, scales and bias to the next */
    int            M, N, K, experts;
};

/* ---- which tile ---------------------------------------------------------------------------------------------------- */

/* Inclusive sums over a wave's lanes. */
__device__ __forceinline__ int wave_scan(int v)
{
    v += dpp_get<0x111>(v);                                    /* row_shr 1, 2, 4, 8 */
    v += dpp_get<0x112>(v);
    v += dpp_get<0x114>(v);
    v += dpp_get<0x118>(v);
    v += dpp_get<0x142, 0xA>(v);                               /* row_bcast 15, 31 */
    v += dpp_get<0x143, 0xC>(v);
    return v;
}

struct F8Tile { int e, m0, mend, nt; };                        /* expert, rows m0 .. mend - 1 of A, tile of weight rows */

/* Which tile of BT rows x a tile of weight rows the `id`-th block has.  Tiles are dealt to the XCDs in equal runs (gemm_deal), and in the order of
 * a run eight tiles of rows lie beside each other for every tile of weight rows, so that the tiles an XCD works on at a time share both operands
 * in its L2.  Of experts, the tiles that there are are counted first, from the offsets: 64 experts at a time, one a lane. */
__device__ __forceinline__ bool f8_tile(const F8Args &a, int id, int BT, int nnt, F8Tile &w)
{
    const int lane = threadIdx.x & 63;
    int ntt = (a.M + BT - 1) / BT, lo = 0, hi = 0, sum = 0, n = 0;
    auto chunk = [&](int e0) {                                 /* the tiles of experts e0 .. e0 + 63 */
        const int i = min(e0 + lane, a.experts - 1);
        lo = max(0, min(a.offsets[i], a.M));
        hi = max(lo, min(a.offsets[i + 1], a.M));
        n = e0 + lane < a.experts ? (hi - lo + BT - 1) / BT : 0;
        sum = wave_scan(n);
        return __builtin_amdgcn_readlane(sum, 63);
    };
    if (a.offsets) {
        ntt = 0;
        const int most = a.M / BT + min(a.M, a.experts);       /* that the launch counts with: offsets may be anything */
        for (int e0 = 0; e0 < a.experts; e0 += 64) ntt = min(ntt + chunk(e0), most);
    }
    const int t = ntt ? gemm_deal(id, ntt * nnt) : -1;
    if (t < 0) return false;
    const int band = t / (8 * nnt), in = t - band * 8 * nnt, wide = min(8, ntt - 8 * band);
    w.nt = in / wide;
    const int tt = 8 * band + in - w.nt * wide;
    w.e = 0;
    w.m0 = tt * BT;
    w.mend = a.M;
    if (!a.offsets) return true;
    int before = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 64) {
        const int all = a.experts <= 64 ? __builtin_amdgcn_readlane(sum, 63) : chunk(e0);
        if (before + all > tt) {
            const int l = __ffsll((long long)__ballot(before + sum > tt)) - 1;
            w.e = e0 + l;
            w.m0 = __builtin_amdgcn_readlane(lo + (tt - before - (sum - n)) * BT, l);
            w.mend = __builtin_amdgcn_readlane(hi, l);
            return true;
        }
        before += all;
    }
    return false;
}

enum { F8_LAUNCH_MOST = 1 << 23 };                              /* blocks of a launch stay below this: fewer than 2^32 threads */
/* Tiles of rows that there can be: an expert's last one may be one row. */
static long f8_most_tiles(int M, int experts, int BT) { return experts ? (long)M / BT + min(M, experts) : ((long)M + BT - 1) / BT; }
static long f8_most_tiles(const F8Args &a, int BT) { return f8_most_tiles(a.M, a.offsets ? a.experts : 0, BT); }

/* ---- operands and results -------------------------------------------------------------------------------------------- */

/* Eight codes as fp16. */
__device__ __forceinline__ f8_v8h f8_half(int lo, int hi)
{
    const f8_v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const f8_v2h c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return f8_v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <class E> struct __attribute__((packed, aligned(sizeof(E)))) f8_out8 { E v[8]; };

/* Eight rows' results of a token to C[t][n ..].  ONCE: non-temporally, as the large tiles' leave, since what stays in the L2s is written back when
 * the launch ends, with nothing beside it (2048 x 11008 x 4096 in bf16 88.3 -> 81.9 us); a few rows' are read from the caches by what follows (one
 * token through eight experts 28.5 -> 28.0). */
template <class E, bool ONCE>
__device__ __forceinline__ void f8_store8(const F8Args &a, const float *bias, const float (&f)[8], int t, int n)
{
    const int left = a.N - n;
    f8_out8<E> o;
#pragma unroll
    for (int r = 0; r < 8; ++r) o.v[r] = (E)(bias ? f[r] + bias[min(n + r, a.N - 1)] : f[r]);
    E *out = (E *)a.C + (size_t)t * a.ldc + n;
    if (left >= 8) {
        struct { rows_u4 v[sizeof(o) / 16]; } w = __builtin_bit_cast(decltype(w), o);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(o) / 16); ++i) {
            if (ONCE) __builtin_nontemporal_store(w.v[i], reinterpret_cast<rows_u4_at_2 *>(out) + i);
            else      reinterpret_cast<rows_u4_at_2 *>(out)[i] = w.v[i];
        }
    } else {
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (r < left) out[r] = o.v[r];
    }
}

/* Zeros in the bytes behind `tail` of the step of 128 whose `rows` rows lie at p, chunks of 16 swizzled (f8_place): both operands', since a byte there may
 * be a NaN.  `threads` threads. */
__device__ __forceinline__ void f8_clear_tail(uint8_t *p, int rows, int tail, int thread, int threads)
{
    for (int e = thread; e < rows * 8; e += threads) {
        const int row = e >> 3, left = tail - 16 * ((e & 7) ^ ((row >> 1) & 7));
        if (left >= 16) continue;
        ckq_v4i *q = reinterpret_cast<ckq_v4i *>(p + 16 * e);
        ckq_v4i v = *q;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = left - 4 * i;
            v[i] = n >= 4 ? v[i] : n <= 0 ? 0 : v[i] & (int)((1u << (8 * n)) - 1u);
        }
        *q = v;
    }
}

/* ---- tiles on the fp16 instructions ----------------------------------------------------------------------------------- */

/* WT x WN waves, each 32 TT tokens x 32 TN rows.  A step is a group of 128; its codes come to LDS as they are, eight rows of 128 bytes a copy, the
 * chunk of 16 that a lane fetches is the one that belongs in its place, c ^ (row / 2 % 8), so that a read of 16 bytes a lane meets all banks once.
 * Two to four blocks a CU (two, three and four of H128x128, H64x128, H64x64), each other's copies and barriers hidden: 16384 rows of 64 experts x
 * 2816 x 2048 236 | 243 us, 4096 rows 106 | 95 (the first two).  The former's busy CUs have their matrix cores at work 45 % of the time, vector
 * instructions 51, LDS 5 (of 8192^3 64 and 63 %): 5 of a tile's 35 us are its start and end, and about 160 tiles of 128 have the 16384 rows. */
template <int WT_, int WN_, int TT_, int TN_> struct F8Half {
    static constexpr int WT = WT_, WN = WN_, TT = TT_, TN = TN_, NW = WT * WN, BT = 32 * TT * WT, BN = 32 * TN * WN, S = 2;
    static constexpr int CODES = (BT + BN) * 128, STAGE = CODES + 4 * BT + 256, NC = (BT + BN) / 8 / NW, NCA = BT / 8 / NW;
    static constexpr int PITCH = 32 * TN * 4 + 16, OUT = NW * 32 * PITCH, LDS = S * STAGE > OUT ? S * STAGE : OUT;
    static_assert(BT % (8 * NW) == 0 && BN % (8 * NW) == 0 && (BN == 64 || BN == 128), "whole copies; one block of scales");
    static_assert(LDS <= 80 * 1024 && TT <= 2, "two blocks a CU");
};

template <class E, class T>
__global__ void __launch_bounds__(64 * T::NW, 2) gemm_f8_half_kernel(F8Args a, int nnt)
{
    constexpr int WN = T::WN, TT = T::TT, TN = T::TN, NW = T::NW, BT = T::BT, BN = T::BN, STAGE = T::STAGE, NC = T::NC, NCA = T::NCA, PITCH = T::PITCH;
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::LDS];
    F8Tile w;
    if (!f8_tile(a, blockIdx.x, BT, nnt, w)) return;
    const int lane = threadIdx.x & 63, wave = wave_in_block(), n0 = w.nt * BN, mrows = w.mend - w.m0;
    const float *sb = a.sb + (size_t)w.e * a.esb + (size_t)(n0 >> 7) * a.ldsb;
    const ckq_v4i rsa = gemm_buffer(a.A + (size_t)w.m0 * a.lda), rsb = gemm_buffer(a.B + (size_t)w.e * a.eb + (size_t)n0 * a.ldb);
    const u32 base = lds_address(lds);
    const int niter = (a.K + 127) / 128, last = niter - 1, tail = a.K - last * 128;
    u32 ofs[NC];
    const int chunk = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int row = 8 * (wave + NW * (i < NCA ? i : i - NCA)) + (lane >> 3);
        ofs[i] = (i < NCA ? (u32)min(row, mrows - 1) * (u32)a.lda : (u32)min(row, a.N - 1 - n0) * (u32)a.ldb) + 16u * (u32)chunk;
    }
    auto copy = [&](int i, int it, int buf) {                  /* the last: scales */
        if (i == NC) {
            if (wave < BT / 64) lds_copy4(gemm_buffer((const uint8_t *)(a.sa + (size_t)it * a.ldsa + w.m0)), base + (u32)(buf * STAGE + T::CODES + 256 * wave), 4u * (u32)min(64 * wave + lane, mrows - 1), 0);
            if (wave == NW - 1) lds_copy4(gemm_buffer((const uint8_t *)(sb + it)), base + (u32)(buf * STAGE + T::CODES + 4 * BT), 0, 0);
            return;
        }
        /* chunks behind the row's last are read from its start, and zeroed (f8_clear_tail) */
        const u32 o = it == last && 16 * chunk >= tail ? ofs[i] - 16u * (u32)chunk : ofs[i];
        lds_copy16(i < NCA ? rsa : rsb, base + (u32)(buf * STAGE + 1024 * (wave + NW * (i < NCA ? i : i - NCA)) + (i < NCA ? 0 : BT * 128)), o, it * 128);
    };
    auto copy_step = [&](int it, int buf) {
#pragma unroll
        for (int i = 0; i <= NC; ++i) copy(i, it, buf);
    };
    const int wt = wave / WN, wn = wave % WN, half = lane >> 5;
    u32 ra[4], rb[4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        const u32 pos = 16u * (u32)((2 * kk + half) ^ ((lane >> 1) & 7));
        ra[kk] = (u32)(32 * TT * wt + (lane & 31)) * 128 + pos;
        rb[kk] = (u32)(BT + 32 * TN * wn + (lane & 31)) * 128 + pos;
    }
    ckq_v16f acc[TT][TN];
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = ckq_v16f{};
    copy_step(0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    auto clear_tail = [&](int buf) {
        f8_clear_tail(lds + buf * STAGE, BT + BN, tail, threadIdx.x, 64 * NW);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
    };
    if (last == 0 && tail < 128) clear_tail(0);
    if (last > 0) copy_step(1, 1);
    /* All have read this step's operands, and the next ones have arrived: from here on the stage takes the copies of the step after them. */
    auto turn = [&](int it) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (it + 1 == last && tail < 128) clear_tail((it + 1) & 1);
    };
    /* The steps of a wave with LIVE groups of 32 tokens.  Quarters of a step, 32 of its 128: the products of one while the codes of the next
     * become fp16, one operand's half between two multiplications, and those of the one after it leave LDS.  A tile's sums are scaled while the
     * next one's are made, the last tile's in the step after. */
    auto steps = [&](auto live) {
        constexpr int LIVE = decltype(live)::value, NF = LIVE + TN, NM = LIVE * TN;
        f8_v8h h[2][NF][2];                                    /* operands: tokens first, then rows; quarter, halves of 16 */
        ckq_v4i code[NF];
        ckq_v16f part[NM];
        float s[LIVE], tok[LIVE], row = 0.0f, s_last = 0.0f;
        auto read = [&](int f, int it, int kk) { return *reinterpret_cast<const ckq_v4i *>(lds + (it & 1) * STAGE + (f < LIVE ? ra[kk] + 32 * 128 * f : rb[kk] + 32 * 128 * (f - LIVE))); };
#pragma unroll
        for (int f = 0; f < NF; ++f) code[f] = read(f, 0, 0);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            h[0][f][0] = f8_half(code[f][0], code[f][1]);
            h[0][f][1] = f8_half(code[f][2], code[f][3]);
            code[f] = read(f, 0, 1);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) part[NM - 1][r] = 0.0f;
        auto scaled = [&](int t, float by) {                   /* tile t: tokens t % LIVE, rows t / LIVE */
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[t % LIVE][t / LIVE][r] = __builtin_fmaf(by, part[t][r], acc[t % LIVE][t / LIVE][r]);
            asm volatile("" : "+v"(acc[t % LIVE][t / LIVE]));
        };
        for (int it = 0; it < niter; ++it) {
            const float *sc = reinterpret_cast<const float *>(lds + (it & 1) * STAGE + T::CODES);
#pragma unroll
            for (int i = 0; i < LIVE; ++i) tok[i] = sc[32 * (TT * wt + i) + (lane & 31)];
            row = sc[BT];
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                if (kk == 2) turn(it);
#pragma unroll
                for (int m = 0; m < 2 * NM; ++m) {
                    const int t = m >> 1, i = t % LIVE, j = t / LIVE;
                    part[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(h[kk & 1][LIVE + j][m & 1], h[kk & 1][i][m & 1], kk == 0 && (m & 1) == 0 ? ckq_v16f{} : part[t], 0, 0, 0);
                    if (kk == 0 && m == 1 && NM > 1) scaled(NM - 1, s_last);
                    if (kk == 3 && (m & 1) && t > 0) scaled(t - 1, s[(t - 1) % LIVE]);
#pragma unroll
                    for (int u = 0; u < 2 * NF; ++u)           /* the next quarter's operands, all of them among the multiplications */
                        if (u * 2 * NM / (2 * NF) == m) {
                            const int f = u >> 1;
                            h[(kk + 1) & 1][f][u & 1] = f8_half(code[f][2 * (u & 1)], code[f][2 * (u & 1) + 1]);
                            asm volatile("" : "+v"(h[(kk + 1) & 1][f][u & 1]));              /* here, not before its use */
                            if (u & 1) code[f] = read(f, it + (kk >= 2), (kk + 2) & 3);          /* behind the last step: anything */
                        }
                    constexpr int SPAN = 3 * NM;               /* the copies one at a time: a copy holds its wave until the address unit has taken it */
#pragma unroll
                    for (int c = 0; c <= NC; ++c)
                        if (kk >= 2 && c * SPAN / (NC + 1) == (kk - 2) * 2 * NM + m && it + 2 <= last) copy(c, it + 2, it & 1);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (kk == 1) {
#pragma unroll
                    for (int i = 0; i < LIVE; ++i) s[i] = tok[i] * row;
                }
            }
            if (NM == 1) scaled(0, s[0]);
            s_last = s[LIVE - 1];
        }
        if (NM > 1) scaled(NM - 1, s_last);
    };
    const int live = min(TT, (mrows - 32 * TT * wt + 31) >> 5);
    if (live >= TT) steps(std::integral_constant<int, TT>{});
    else if (TT > 1 && live == 1) steps(std::integral_constant<int, 1>{});
    else
        for (int it = 0; it < niter; ++it) {                   /* its tokens are behind the last: it copies */
            turn(it);
            if (it + 2 <= last) copy_step(it + 2, it & 1);
        }
    __syncthreads();
    /* Through LDS, each wave by itself, 32 tokens at a time, so that a lane has eight rows' results of a token and a token's leave in whole lines. */
    const float *bias = a.bias ? a.bias + (size_t)w.e * a.ebias : nullptr;
    uint8_t *mine = lds + wave * 32 * PITCH;
#pragma unroll
    for (int i = 0; i < TT; ++i) {
        if (i >= live) break;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f8_v4f *>(mine + (lane & 31) * PITCH + 4 * (32 * j + 8 * g + 4 * half)) = f8_v4f{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int e = lane; e < 32 * 4 * TN; e += 64) {
            const int row = e / (4 * TN), c = 8 * (e % (4 * TN)), t = w.m0 + 32 * (TT * wt + i) + row, n = n0 + 32 * TN * wn + c;
            float f[8];
            const f8_v4f *q = reinterpret_cast<const f8_v4f *>(mine + row * PITCH + 4 * c);
#pragma unroll
            for (int r = 0; r < 8; ++r) f[r] = q[r >> 2][r & 3];
            if (t < w.mend && n < a.N) f8_store8<E, true>(a, bias, f, t, n);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

template <class E, class T>
static int launch_f8_half(const F8Args &a, hipStream_t s)
{
    const int nnt = (a.N + T::BN - 1) / T::BN;
    const long tiles = f8_most_tiles(a, T::BT) * nnt;
    return i8_launch(gemm_f8_half_kernel<E, T>, dim3((u32)((tiles + 7) & ~7l)), dim3(64u * T::NW), s, a, nnt);
}

/* ---- tiles on the e4m3 instructions ------------------------------------------------------------------------------------ */

/* WT x WN waves that multiply, each 16 TT tokens x 16 TN rows; a group's product is one multiplication, 16 x 16 x 128, whose four sums a lane
 * scales and adds while the next ones are multiplied.  NP others that copy, or none (the former do it then); S stages in LDS; PERCU blocks a CU.
 * With others that copy, whose waits for the address unit hold up no multiplication, us: 512 x 11008 x 4096 36.0 -> 28.4, 1024 x 4096 x 4096 33.0
 * -> 22.8; eight waves of 256 x 256 leave no registers for them. */
template <int WT_, int WN_, int TT_, int TN_, int NP_, int S_, int PERCU_> struct F8Core {
    static constexpr int WT = WT_, WN = WN_, TT = TT_, TN = TN_, NP = NP_, S = S_, PERCU = PERCU_, NW = WT * WN, WAVES = NW + NP, BT = 16 * TT * WT, BN = 16 * TN * WN, NB = (BN + 127) / 128;
    static constexpr int CODES = (BT + BN) * 128, SB = CODES + 4 * BT, STAGE = SB + 256 * NB;
    static constexpr int CW = NP ? NP : NW, NC = (BT + BN) / 8 / CW, NCA = BT / 8 / CW, NS = (BT / 64 + NB + CW - 1) / CW;       /* waves that copy, copies of each a step: eight rows; 64 scales */
    static constexpr int PITCH = 16 * TN * 4 + 16, OUT = NW * 16 * PITCH, LDS = S * STAGE > OUT ? S * STAGE : OUT;
    static constexpr bool EACH = 128 % (16 * TN) != 0;         /* a wave's rows may lie in two blocks of scales: one for each sixteen of them */
    static_assert(TT >= 2 && TN >= 2 && CW % 2 == 0 && BT % (8 * CW) == 0 && BN % (8 * CW) == 0 && BT % 64 == 0 && BN % 64 == 0, "whole copies, whole copies of scales");
    static_assert((NP || S == 2) && (S - 1) * (NC + NS) < 64 && LDS <= 160 * 1024 / PERCU, "waves that copy and multiply have a step under way; what a wave can count; they fit");
};

template <class E, class T>
__device__ __forceinline__ void f8_core_tile(const F8Args &a, const F8Tile &w, int n0, uint8_t *lds)
{
    constexpr int WN = T::WN, TT = T::TT, TN = T::TN, NP = T::NP, S = T::S, NW = T::NW, CW = T::CW, BT = T::BT, BN = T::BN, STAGE = T::STAGE, NC = T::NC, NCA = T::NCA, PITCH = T::PITCH, NS = T::EACH ? TN : 1;
    const int lane = threadIdx.x & 63, wave = wave_in_block(), cw = NP ? wave - NW : wave, mrows = w.mend - w.m0;
    const ckq_v4i rsa = gemm_buffer(a.A + (size_t)w.m0 * a.lda), rsb = gemm_buffer(a.B + (size_t)w.e * a.eb + (size_t)n0 * a.ldb);
    const u32 base = lds_address(lds);
    const int niter = (a.K + 127) / 128, last = niter - 1, tail = a.K - last * 128;
    u32 ofs[NC];
    const int chunk = (lane & 7) ^ ((4 * cw + (lane >> 4)) & 7);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int row = 8 * (cw + CW * (i < NCA ? i : i - NCA)) + (lane >> 3);
        ofs[i] = (i < NCA ? (u32)min(row, mrows - 1) * (u32)a.lda : (u32)min(row, a.N - 1 - n0) * (u32)a.ldb) + 16u * (u32)chunk;
    }
    auto copy = [&](int i, int it, int buf) {
        const u32 o = it == last && 16 * chunk >= tail ? ofs[i] - 16u * (u32)chunk : ofs[i];
        lds_copy16(i < NCA ? rsa : rsb, base + (u32)(buf * STAGE + 1024 * (cw + CW * (i < NCA ? i : i - NCA)) + (i < NCA ? 0 : BT * 128)), o, it * 128);
    };
    auto copy_scales = [&](int it, int buf) {
#pragma unroll
        for (int i = 0; i < T::NS; ++i) {
            const int q = min(cw + CW * i, BT / 64 + T::NB - 1), j = q - BT / 64;         /* every wave has as many, the last ones twice */
            const float *p = j < 0 ? a.sa + (size_t)it * a.ldsa + w.m0 : a.sb + (size_t)w.e * a.esb + (size_t)min((n0 >> 7) + j, (a.N - 1) >> 7) * a.ldsb + it;
            lds_copy4(gemm_buffer((const uint8_t *)p), base + (u32)(buf * STAGE + (j < 0 ? T::CODES + 256 * q : T::SB + 256 * j)), j < 0 ? 4u * (u32)min(64 * q + lane, mrows - 1) : 0u, 0);
        }
    };
    auto copy_step = [&](int it, int buf) {
#pragma unroll
        for (int i = 0; i < NC; ++i) copy(i, it, buf);
        copy_scales(it, buf);
    };
    auto clear_tail = [&](int buf) {                           /* all waves; then they meet */
        f8_clear_tail(lds + buf * STAGE, BT + BN, tail, threadIdx.x, 64 * T::WAVES);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
    };
    /* Step `it` has stage it % S.  A step's last operands are read before its last tokens are multiplied; the barrier is there: all have step it's
     * operands in registers, and step it + 1 has arrived; from there on the stage takes the copies of step it + S. */
    if (NP > 0 && wave >= NW) {
        constexpr int EACH_STEP = NC + T::NS;
#pragma unroll
        for (int st = 0; st < S; ++st)
            if (st < niter) copy_step(st, st);
        if (niter >= S) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * EACH_STEP) : "memory");
        else            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (last == 0 && tail < 128) clear_tail(0);
        int buf = 0;
        for (int it = 0; it < niter; ++it) {
            const int next = buf + 1 == S ? 0 : buf + 1;
            if (it + S - 1 < niter) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * EACH_STEP) : "memory");
            else                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            if (it + 1 == last && tail < 128) clear_tail(next);
            if (it + S < niter) copy_step(it + S, buf);
            buf = next;
        }
        __syncthreads();
        return;
    }
    const int wt = wave / WN, wn = wave % WN;
    u32 ra[2], rb[2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
        const u32 pos = 16u * (u32)((4 * kk + (lane >> 4)) ^ ((lane >> 1) & 7));
        ra[kk] = (u32)(16 * TT * wt + (lane & 15)) * 128 + pos;
        rb[kk] = (u32)(BT + 16 * TN * wn + (lane & 15)) * 128 + pos;
    }
    auto read = [&](int buf, const u32 (&r)[2], int f) {
        const uint8_t *p = lds + buf * STAGE + 16 * 128 * f;
        const ckq_v4i lo = *reinterpret_cast<const ckq_v4i *>(p + r[0]), hi = *reinterpret_cast<const ckq_v4i *>(p + r[1]);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    f8_v4f acc[TT][TN];
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f8_v4f{0.0f, 0.0f, 0.0f, 0.0f};

    if (NP == 0) {
        copy_step(0, 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __builtin_amdgcn_s_barrier();
    if (last == 0 && tail < 128) clear_tail(0);
    f8_v8i fa[3], fb[TN];
    float sa[TT], sb[NS];
    int sb_at[NS];                                             /* which of the tile's blocks of scales */
#pragma unroll
    for (int j = 0; j < NS; ++j) sb_at[j] = BT + 64 * (((n0 & 127) + 16 * (TN * wn + j)) >> 7);
    auto read_scales = [&](int buf) {
        const float *sc = reinterpret_cast<const float *>(lds + buf * STAGE + T::CODES);
#pragma unroll
        for (int j = 0; j < NS; ++j) sb[j] = sc[sb_at[j]];
#pragma unroll
        for (int i = 0; i < TT; ++i) sa[i] = sc[16 * (TT * wt + i) + (lane & 15)];
    };
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[j] = read(0, rb, j);
    fa[0] = read(0, ra, 0);
    fa[1] = read(0, ra, 1);
    read_scales(0);
    const f8_v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    int buf = 0;
    for (int it = 0; it < niter; ++it) {
        const int next = buf + 1 == S ? 0 : buf + 1;
        f8_v4f part[3];
        auto scaled = [&](int m) {                             /* the sums of the m-th multiplication of the step */
            const float s = sa[m / TN] * sb[m % TN % NS];
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[m / TN][m % TN][r] = __builtin_fmaf(s, part[m % 3][r], acc[m / TN][m % TN][r]);
            asm volatile("" : "+v"(acc[m / TN][m % TN]));     /* here, and not all of them behind the last branch of the step */
        };
#pragma unroll
        for (int i = 0; i < TT; ++i) {
            if (i + 2 < TT) fa[(i + 2) % 3] = read(buf, ra, i + 2);
            if (i + 1 == TT) {
                if (NP == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                else         asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                if (it + 1 == last && tail < 128) clear_tail(next);
            }
            const f8_v8i now = fa[i % 3];
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int m = i * TN + j;
                part[m % 3] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], now, zero, 0, 0, 0, 0, 0, 0);
                if (m > 1) scaled(m - 2);
                if (i + 1 == TT) {                             /* behind the last step's: anything */
                    fb[j] = read(next, rb, j);
                    if (j == 0) fa[0] = read(next, ra, 0);
                    if (j == 1) fa[1] = read(next, ra, 1);
                }
                /* the copies of the next step, one at a time: a copy holds its wave until the address unit has taken it */
                constexpr int SPAN = TT * TN * 3 / 8;
                if (NP == 0 && m == 0 && it < last) copy_scales(it + 1, next);
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    if (NP == 0 && c * SPAN / NC == m && it < last) copy(c, it + 1, next);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        scaled(TT * TN - 2);
        scaled(TT * TN - 1);
        read_scales(next);
        buf = next;
    }
    const float *bias = a.bias ? a.bias + (size_t)w.e * a.ebias : nullptr;
    uint8_t *mine = lds + wave * 16 * PITCH;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TT; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) *reinterpret_cast<f8_v4f *>(mine + (lane & 15) * PITCH + 4 * (16 * j + 4 * (lane >> 4))) = acc[i][j];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int e = lane; e < 16 * 2 * TN; e += 64) {
            const int row = e / (2 * TN), c = 8 * (e % (2 * TN)), t = w.m0 + 16 * (TT * wt + i) + row, n = n0 + 16 * TN * wn + c;
            float f[8];
            const f8_v4f *q = reinterpret_cast<const f8_v4f *>(mine + row * PITCH + 4 * c);
#pragma unroll
            for (int r = 0; r < 8; ++r) f[r] = q[r >> 2][r & 3];
            if (t < w.mend && n < a.N) f8_store8<E, true>(a, bias, f, t, n);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

template <class E, class T>
__global__ void __launch_bounds__(64 * T::WAVES, T::WAVES * T::PERCU / 4) gemm_f8_core_kernel(F8Args a, int nnt)
{
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::LDS];
    F8Tile w;
    if (f8_tile(a, blockIdx.x, T::BT, nnt, w)) f8_core_tile<E, T>(a, w, w.nt * T::BN, lds);
}

/* One matrix: the first nnt1 columns of tiles of T1, `blocks1` blocks of them, and the rows that they leave in tiles of T2. */
template <class E, class T1, class T2>
__global__ void __launch_bounds__(64 * T1::WAVES, T1::WAVES / 4) gemm_f8_two_kernel(F8Args a, int nnt1, int blocks1, int nnt2)
{
    static_assert(T1::WAVES == T2::WAVES && T1::PERCU == 1, "one size of block");
    __shared__ __attribute__((aligned(16))) uint8_t lds[T1::LDS > T2::LDS ? T1::LDS : T2::LDS];
    F8Tile w;
    if ((int)blockIdx.x < blocks1) {
        if (f8_tile(a, blockIdx.x, T1::BT, nnt1, w)) f8_core_tile<E, T1>(a, w, w.nt * T1::BN, lds);
    } else if (f8_tile(a, blockIdx.x - blocks1, T2::BT, nnt2, w))
        f8_core_tile<E, T2>(a, w, nnt1 * T1::BN + w.nt * T2::BN, lds);
}
template <class E, class T1, class T2>
static int launch_f8_two(const F8Args &a, int nnt1, hipStream_t s)
{
    const int nnt2 = (a.N - nnt1 * T1::BN + T2::BN - 1) / T2::BN;
    const long blocks1 = (f8_most_tiles(a, T1::BT) * nnt1 + 7) & ~7l, blocks2 = (f8_most_tiles(a, T2::BT) * nnt2 + 7) & ~7l;
    return i8_launch(gemm_f8_two_kernel<E, T1, T2>, dim3((u32)(blocks1 + blocks2)), dim3(64u * T1::WAVES), s, a, nnt1, (int)blocks1, nnt2);
}

template <class E, class T>
static int launch_f8_core(const F8Args &a, hipStream_t s)
{
    const int nnt = (a.N + T::BN - 1) / T::BN;
    const long tiles = f8_most_tiles(a, T::BT) * nnt;
    return i8_launch(gemm_f8_core_kernel<E, T>, dim3((u32)((tiles + 7) & ~7l)), dim3(64u * T::WAVES), s, a, nnt);
}

/* ---- K split among the waves of a block -------------------------------------------------------------------------------- */

/* 16 TG tokens x 16 RN rows a block of NW waves; every wave has all of the tile and each NW-th group of K, through S stages of its own, so that
 * nothing is waited for but its own copies until the waves' sums meet at the end, in the order of the waves.  333 x 1001 x 4847, us: 16 x 32 on
 * four waves 14.7, 32 x 32 on four 13.9, 48 x 32 on seven 11.3 (one round of the CUs), 64 x 32 on six 13.2; operands straight to registers, 16
 * rows x 64 bytes a load, take twice as long to come: 16.9. */
template <int NW_, int RN_, int TG_, int S_> struct F8Split {
    static constexpr int NW = NW_, RN = RN_, TG = TG_, S = S_, BT = 16 * TG, BN = 16 * RN, CODES = (BT + BN) * 128, STAGE = CODES + 512, PITCH = BN * 4 + 16, NC = 2 * (RN + TG);
    static constexpr int LDS = NW * (S * STAGE > BT * PITCH ? S * STAGE : BT * PITCH);
    static_assert(LDS <= 160 * 1024 && BT <= 64 && 128 % BN == 0, "one block fits; one copy of scales, one block of them");
};

template <class E, class T>
__global__ void __launch_bounds__(64 * T::NW) gemm_f8_split_kernel(F8Args a, int nnt)
{
    constexpr int NW = T::NW, RN = T::RN, TG = T::TG, S = T::S, BT = T::BT, BN = T::BN, STAGE = T::STAGE, NC = T::NC, PITCH = T::PITCH;
    __shared__ __attribute__((aligned(16))) uint8_t lds[T::LDS];
    F8Tile w;
    if (!f8_tile(a, blockIdx.x, BT, nnt, w)) return;
    const int lane = threadIdx.x & 63, wave = wave_in_block(), n0 = w.nt * BN, mrows = w.mend - w.m0;
    const float *sb = a.sb + (size_t)w.e * a.esb + (size_t)(n0 >> 7) * a.ldsb;
    const ckq_v4i rsa = gemm_buffer(a.A + (size_t)w.m0 * a.lda), rsb = gemm_buffer(a.B + (size_t)w.e * a.eb + (size_t)n0 * a.ldb);
    uint8_t *mine = lds + wave * S * STAGE;
    const u32 base = lds_address(mine);
    const int niter = (a.K + 127) / 128, last = niter - 1, tail = a.K - last * 128, steps = wave < niter ? (niter - 1 - wave) / NW + 1 : 0;
    u32 ofs[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int cr = 8 * (i < 2 * TG ? i : i - 2 * TG) + (lane >> 3), chunk = (lane & 7) ^ ((cr >> 1) & 7);
        ofs[i] = (i < 2 * TG ? (u32)min(cr, mrows - 1) * (u32)a.lda : (u32)min(cr, a.N - 1 - n0) * (u32)a.ldb) + 16u * (u32)chunk;
    }
    auto copy = [&](int j, int slot) {
        const int it = wave + NW * j;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int cr = 8 * (i < 2 * TG ? i : i - 2 * TG) + (lane >> 3), chunk = (lane & 7) ^ ((cr >> 1) & 7);
            const u32 o = it == last && 16 * chunk >= tail ? ofs[i] - 16u * (u32)chunk : ofs[i];
            lds_copy16(i < 2 * TG ? rsa : rsb, base + (u32)(slot * STAGE + 1024 * i), o, it * 128);
        }
        lds_copy4(gemm_buffer((const uint8_t *)(a.sa + (size_t)it * a.ldsa + w.m0)), base + (u32)(slot * STAGE + T::CODES), 4u * (u32)min(lane, mrows - 1), 0);
        lds_copy4(gemm_buffer((const uint8_t *)(sb + it)), base + (u32)(slot * STAGE + T::CODES + 256), 0, 0);
    };
    f8_v4f acc[TG][RN];
#pragma unroll
    for (int i = 0; i < TG; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = f8_v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < S - 1; ++j)
        if (j < steps) copy(j, j);
    int slot = 0;
    for (int j = 0; j < steps; ++j) {
        const int it = wave + NW * j;
        if (j + S - 1 < steps) {
            copy(j + S - 1, slot == 0 ? S - 1 : slot - 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * (NC + 2)) : "memory");
        } else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        uint8_t *p = mine + slot * STAGE;
        if (it == last && tail < 128) {
            f8_clear_tail(p, BT + BN, tail, lane, 64);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        const float *sc = reinterpret_cast<const float *>(p + T::CODES);
        float s[TG];
#pragma unroll
        for (int i = 0; i < TG; ++i) s[i] = sc[16 * i + (lane & 15)] * sc[64];
        f8_v4f part[TG][RN];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int c = 4 * kk + (lane >> 4);
            const u32 at = (u32)((lane & 15) * 128 + 16 * (c ^ ((lane >> 1) & 7)));
            f8_v8h fa[TG][2], fb[RN][2];
#pragma unroll
            for (int i = 0; i < TG; ++i) {
                const ckq_v4i v = *reinterpret_cast<const ckq_v4i *>(p + at + 16 * 128 * i);
                fa[i][0] = f8_half(v[0], v[1]);
                fa[i][1] = f8_half(v[2], v[3]);
            }
#pragma unroll
            for (int i = 0; i < RN; ++i) {
                const ckq_v4i v = *reinterpret_cast<const ckq_v4i *>(p + at + (BT + 16 * i) * 128);
                fb[i][0] = f8_half(v[0], v[1]);
                fb[i][1] = f8_half(v[2], v[3]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < TG; ++i)
#pragma unroll
                    for (int n = 0; n < RN; ++n)
                        part[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb[n][h], fa[i][h], kk == 0 && h == 0 ? f8_v4f{0.0f, 0.0f, 0.0f, 0.0f} : part[i][n], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < TG; ++i)
#pragma unroll
            for (int n = 0; n < RN; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][n][r] = __builtin_fmaf(s[i], part[i][n][r], acc[i][n][r]);
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
            *reinterpret_cast<f8_v4f *>(red + (16 * i + (lane & 15)) * PITCH + 4 * (16 * n + 4 * (lane >> 4))) = acc[i][n];
    __syncthreads();
    constexpr int PER = BN / 8, JOBS = BT * PER;
    static_assert(JOBS <= 64 * NW, "a job a thread");
    const int row = (int)threadIdx.x / PER, col = 8 * ((int)threadIdx.x % PER), t = w.m0 + row, n = n0 + col;
    if ((int)threadIdx.x >= JOBS || t >= w.mend || n >= a.N) return;
    float f[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) f[r] = 0.0f;
#pragma unroll
    for (int v = 0; v < NW; ++v) {
        const f8_v4f *q = reinterpret_cast<const f8_v4f *>(lds + v * BT * PITCH + row * PITCH + 4 * col);
#pragma unroll
        for (int r = 0; r < 8; ++r) f[r] += q[r >> 2][r & 3];
    }
    f8_store8<E, false>(a, a.bias ? a.bias + (size_t)w.e * a.ebias : nullptr, f, t, n);
}

template <class E, class T>
static int launch_f8_split(const F8Args &a, hipStream_t s)
{
    const int nnt = (a.N + T::BN - 1) / T::BN;
    const long tiles = f8_most_tiles(a, T::BT) * nnt;
    return i8_launch(gemm_f8_split_kernel<E, T>, dim3((u32)((tiles + 7) & ~7l)), dim3(64u * T::NW), s, a, nnt);
}

/* ---- one token: rows streamed ------------------------------------------------------------------------------------------ */

/* A wave has R rows and every KS-th piece of KU KB of K; 4 waves a block.  A lane has sixteen elements of a group at a time: their products in
 * pairs (v_dot2_f32_f16), times the group's scales, onto its sum.  Rows are loaded non-temporally: a decode step goes through more weights than
 * any cache holds. */
template <class E, int R, int KU, int KS>
__global__ void __launch_bounds__(256) gemm_f8_stream_kernel(F8Args a)
{
    constexpr int G = 4 / KS;
    static_assert(R <= 64 && 128 % R == 0, "a result a lane; rows in one block of scales");
    __shared__ float red[KS > 1 ? 4 * R : 1];
    const int lane = threadIdx.x & 63, wave = wave_in_block(), part = wave % KS, n0 = ((int)blockIdx.x * G + wave / KS) * R, last_group = (a.K - 1) >> 7;
    if (KS == 1 && n0 >= a.N) return;
    const uint8_t *pb[R];
    const float *sb = a.sb + (size_t)(min(n0, a.N - 1) >> 7) * a.ldsb;
#pragma unroll
    for (int r = 0; r < R; ++r) pb[r] = a.B + (size_t)min(n0 + r, a.N - 1) * a.ldb;
    float acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = 0.0f;
    for (int k0 = part * KU * 1024; k0 < a.K; k0 += KS * KU * 1024) {
        ckq_v4i v[R][KU], x[KU];
        float s[KU];
        u32 at[KU];
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            at[u] = (u32)k0 + 1024u * u + 16u * (u32)lane;
            if ((int)at[u] >= a.K) at[u] = 0;                /* zeroed below */
        }
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) v[r][u] = __builtin_nontemporal_load(reinterpret_cast<const ckq_v4i *>(pb[r] + at[u]));
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const int g = min((k0 >> 7) + 8 * u + (lane >> 3), last_group);
            x[u] = *reinterpret_cast<const ckq_v4i *>(a.A + at[u]);
            s[u] = a.sa[(size_t)g * a.ldsa] * sb[g];
        }
        if (k0 + KU * 1024 > a.K) {
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {                  /* both sides: a byte behind the last may be a NaN */
                    const int n = a.K - (k0 + 1024 * u + 16 * lane + 4 * i), keep = n >= 4 ? -1 : n <= 0 ? 0 : (int)((1u << (8 * n)) - 1u);
                    x[u][i] &= keep;
#pragma unroll
                    for (int r = 0; r < R; ++r) v[r][u][i] &= keep;
                }
        }
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            f8_v2h h[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[u][i], 1.0f, false);
                h[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[u][i], 1.0f, true);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sum = __builtin_amdgcn_fdot2(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[r][u][i], 1.0f, false), h[2 * i], sum, false);
                    sum = __builtin_amdgcn_fdot2(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[r][u][i], 1.0f, true), h[2 * i + 1], sum, false);
                }
                acc[r] = __builtin_fmaf(s[u], sum, acc[r]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, group_sum<64>(acc[r])), 63));
    if (KS > 1) {
        if (lane == 0) {
#pragma unroll
            for (int r = 0; r < R; ++r) red[wave * R + r] = acc[r];
        }
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int v = 1; v < KS; ++v) acc[r] += red[(wave + v) * R + r];
    }
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) sum = lane == r ? acc[r] : sum;
    const int n = n0 + lane;
    if (lane < R && n < a.N) ((E *)a.C)[n] = (E)(a.bias ? sum + a.bias[n] : sum);
}

template <class E, int R, int KU, int KS>
static int launch_f8_stream(const F8Args &a, hipStream_t s)
{
    constexpr int per = 4 / KS * R;
    return i8_launch(gemm_f8_stream_kernel<E, R, KU, KS>, dim3((u32)((a.N + per - 1) / per)), dim3(256), s, a);
}
/* us, rows x K, (rows a wave, KB a trip, waves of a row): 11008 x 4096, 4, 1, 2 9.66 | 4, 1, 4 9.23 | 2, 2, 2 9.18 | 2, 1, 4 9.82 | 1, 2, 4 13.2;
 * 4096 x 11008, 4, 1, 4 9.97 | 2, 1, 4 9.32 | 2, 4, 4 10.0; 11008 x 2048, 4, 1, 2 5.76 | 2, 2, 2 5.88; 4000 x 1000, 4, 1, 1 2.94 | 4, 1, 4 3.23. */
template <class E>
static int launch_f8_stream(const F8Args &a, hipStream_t s)
{
    const int kb = (a.K + 1023) / 1024;
    return kb <= 1 ? launch_f8_stream<E, 4, 1, 1>(a, s) : kb <= 2 ? launch_f8_stream<E, 4, 1, 2>(a, s) : kb <= 4 ? launch_f8_stream<E, 2, 2, 2>(a, s) : launch_f8_stream<E, 2, 1, 4>(a, s);
}

/* ---- which kernel ------------------------------------------------------------------------------------------------------ */

typedef F8Half<2, 2, 2, 2> H128x128;
typedef F8Half<2, 2, 1, 2> H64x128;
typedef F8Half<2, 2, 1, 1> H64x64;
typedef F8Split<7, 2, 3, 2> S48x32w7;
typedef F8Split<4, 2, 2, 2> S32x32;
typedef F8Split<8, 2, 1, 2> S16x32w8;
typedef F8Split<4, 2, 1, 2> S16x32;
typedef F8Split<2, 2, 1, 2> S16x32w2;
typedef F8Split<8, 1, 1, 2> S16x16;
typedef F8Core<2, 4, 8, 4, 0, 2, 1> C256x256;
typedef F8Core<4, 2, 4, 4, 4, 3, 1> C256x128;
typedef F8Core<2, 2, 4, 6, 4, 3, 1> C128x192;
typedef F8Core<2, 2, 4, 4, 4, 4, 1> C128x128;
typedef F8Core<2, 2, 2, 4, 4, 4, 1> C64x128;
typedef F8Core<2, 2, 2, 2, 4, 4, 2> C64x64;

/* What a launch takes, in us: t0, and for every round of blocks t_tile and as many steps of K as a wave has, each of `step` where all places have
 * a block; in a last round of fewer blocks less, `share` of it by how many share a CU, the rest by how many there are in all, but no less than a
 * block alone takes, `alone`.  Fitted to 800 random products of one matrix (2 to 4096 tokens, 32 to 32000 rows, K 32 to 11008; three sets in
 * turn): the kernel so chosen is 0.8 % (fp32 results) and 0.7 % (16 bits) slower than the fastest on average, 1.2 times at worst, as much on one
 * half of them when fitted to the other; over experts (500 random products, 2 to 128 of them, none of which it was fitted to) 1.8 % and 1.4 times. */
struct F8Cost { int bt, bn, places, split; float t0, t_tile, step, share, alone; };
static const F8Cost f8_costs[CKQ_F8_TILINGS] = {
    {128, 128, 512, 1, 1.48f, 5.25f, 1.886f, 0.90f, 0.28f}, {64, 128, 768, 1, 1.41f, 3.69f, 1.596f, 1.00f, 0.45f}, {64, 64, 1024, 1, 1.78f, 2.53f, 1.301f, 1.00f, 0.40f},
    {48, 32, 256, 7, 1.99f, 2.53f, 0.976f, 0.86f, 0.0f},    {32, 32, 512, 4, 2.00f, 2.14f, 0.743f, 1.00f, 0.72f},  {16, 32, 256, 8, 1.95f, 1.86f, 0.662f, 0.78f, 0.0f},
    {16, 32, 768, 4, 2.27f, 1.53f, 0.809f, 1.00f, 0.56f},   {16, 32, 1536, 2, 2.02f, 1.69f, 0.828f, 1.00f, 0.54f}, {16, 16, 512, 8, 2.07f, 1.57f, 0.654f, 1.00f, 0.57f},
    {256, 256, 256, 1, 0.00f, 8.83f, 1.854f, 0.64f, 0.0f},  {256, 128, 256, 1, 0.00f, 7.22f, 0.895f, 0.65f, 0.0f}, {128, 128, 256, 1, 1.51f, 4.98f, 0.562f, 0.68f, 0.0f},
    {64, 128, 256, 1, 1.73f, 3.30f, 0.374f, 0.73f, 0.0f},   {64, 64, 512, 1, 1.92f, 2.40f, 0.404f, 1.00f, 0.58f},  {128, 192, 256, 1, 1.28f, 6.69f, 0.720f, 0.70f, 0.0f},
};
static const F8Cost f8_cost_rest = {128, 192, 256, 1, 0.00f, 11.29f, 0.486f, 0.95f, 0.0f};         /* beside tiles of 256 x 256 */

static float f8_rounds(const F8Cost &c, float tiles, int K)
{
    const int steps = ((K + 127) / 128 + c.split - 1) / c.split;
    const float places = (float)c.places, full = floorf(tiles / places), rest = tiles - full * places;
    float t = full * (c.t_tile + (float)steps * c.step);
    if (rest > 0.0f) t += c.t_tile + (float)steps * c.step * fmaxf(c.alone, (1.0f - c.share) * rest / places + c.share * ceilf(rest / 256.0f) * 256.0f / places);
    return t;
}
/* Tiles of M rows; of experts, which have what only the device knows, as many as if each row went to any of them alike. */
static float f8_row_tiles(int bt, int M, int experts)
{
    if (!experts) return (float)((M + (long)bt - 1) / bt);
    const float used = (float)experts * (1.0f - powf(1.0f - 1.0f / (float)experts, (float)M)), rows = (float)M / used;
    return rows > 0.75f * (float)bt ? used * fmaxf(1.0f, rows / (float)bt + 0.5f) : used;
}
static float f8_tiles(const F8Cost &c, int M, int N, int experts) { return f8_row_tiles(c.bt, M, experts) * (float)((N + (long)c.bn - 1) / c.bn); }

/* Columns of 256 x 256 tiles that make whole rounds of the 256 CUs: what they leave goes in tiles of 128 x 192, a shorter last round (2048 x 11008
 * x 4096: 344 tiles of 256 x 256 in two rounds 105 us; 256 of them and 240 small ones 87). */
static int f8_whole_columns(int M, int N)
{
    const long ntt = (M + 255l) / 256, nnt = (N + 255l) / 256;
    return (int)(ntt * nnt / 256 * 256 / ntt);
}

/* Whether a kernel takes a product in one launch. */
static bool f8_fits(int kernel, int M, int N, int experts)
{
    if (kernel == CKQ_F8_STREAM) return N <= 1 << 23;
    const int bt = kernel == CKQ_F8_TWO ? 128 : f8_costs[kernel].bt, bn = kernel == CKQ_F8_TWO ? 192 : f8_costs[kernel].bn;
    const long wide = (N + (long)bn - 1) / bn, tiles = kernel == CKQ_F8_TWO ? (f8_most_tiles(M, experts, bt) + 2) * (wide + 2) : f8_most_tiles(M, experts, bt) * wide;
    return tiles < F8_LAUNCH_MOST - 16;
}

static std::atomic<int> g_f8_kernel{-1};
extern "C" void ckq_launch_set_f8_kernel(int kernel) { g_f8_kernel.store(kernel < 0 || kernel > CKQ_F8_STREAM ? -1 : kernel); }

/* The e4m3 instructions' sums, 1.5e-5 off on random products and by 2^-13 of the largest of each eight at most for every other one of them, are
 * taken where the result is rounded to 16 bits (bf16 2^-9, fp16 2^-12 off) and nothing but that: not for fp32 results, not where the caller says
 * so (CKQ_SUMS_FP32), and not over experts, whose first product's results go through another quantizer, where each change of a value moves some of
 * them by a sixteenth (an MLP with 32 experts in fp16: 0.0017 off the definition, with fp32 sums 0.0003).  Random products of one matrix gain 5.8
 * % by them on average, 2048 x 11008 x 4096 174 -> 87 us. */
/* -1: none takes it in one launch. */
extern "C" int ckq_launch_f8_kernel(int type, int M, int N, int K, int experts)
{
    const bool cores = type != CKQ_T_F32 && !(type & CKQ_SUMS_FP32) && !experts;
    int forced = g_f8_kernel.load();
    if ((type & CKQ_SUMS_FP32) && forced >= CKQ_F8_C256x256 && forced <= CKQ_F8_TWO) forced = -1;
    const int cols = experts ? 0 : f8_whole_columns(M, N);
    if (forced >= 0 && (forced != CKQ_F8_STREAM || (M == 1 && !experts)) && (forced != CKQ_F8_TWO || cols > 0)) return f8_fits(forced, M, N, experts) ? forced : -1;
    if (M == 1 && !experts) return f8_fits(CKQ_F8_STREAM, M, N, 0) ? CKQ_F8_STREAM : -1;
    int best = -1;
    float t = 1e30f;
    for (int i = 0; i < (cores ? CKQ_F8_TILINGS : CKQ_F8_C256x256); ++i) {
        /* of an expert's last tile of 128, groups of 32 tokens that are not there cost nothing (160 products of 256 to 65536 rows over 8 to 128
         * experts: 1.3 % from the fastest on average without the factor, 1.0 with it) */
        const float ti = (f8_costs[i].t0 + f8_rounds(f8_costs[i], f8_tiles(f8_costs[i], M, N, experts), K)) * (experts && i == CKQ_F8_H128x128 ? 0.95f : 1.0f);
        if (ti < t && f8_fits(i, M, N, experts)) { t = ti; best = i; }
    }
    if (best >= 0 && cores && cols > 0 && 256 * cols < N) {
        const F8Cost &a = f8_costs[CKQ_F8_C256x256], &b = f8_cost_rest;
        if (a.t0 + f8_rounds(a, (float)((M + 255l) / 256) * (float)cols, K) + f8_rounds(b, f8_tiles(b, M, N - 256 * cols, 0), K) < t && f8_fits(CKQ_F8_TWO, M, N, 0)) best = CKQ_F8_TWO;
    }
    return best;
}

/* What one launch does not take goes in halves, of the tokens or of the weights' rows, which are whole tiles and blocks of scales; over experts of
 * the latter only. */
template <class E>
static int launch_gemm_f8(const F8Args &a, int type, hipStream_t s)
{
    switch (ckq_launch_f8_kernel(type, a.M, a.N, a.K, a.offsets ? a.experts : 0)) {
    case CKQ_F8_H128x128:    return launch_f8_half<E, H128x128>(a, s);
    case CKQ_F8_H64x128:     return launch_f8_half<E, H64x128>(a, s);
    case CKQ_F8_H64x64:      return launch_f8_half<E, H64x64>(a, s);
    case CKQ_F8_S48x32w7:    return launch_f8_split<E, S48x32w7>(a, s);
    case CKQ_F8_S32x32:      return launch_f8_split<E, S32x32>(a, s);
    case CKQ_F8_S16x32w8:    return launch_f8_split<E, S16x32w8>(a, s);
    case CKQ_F8_S16x32:      return launch_f8_split<E, S16x32>(a, s);
    case CKQ_F8_S16x32w2:    return launch_f8_split<E, S16x32w2>(a, s);
    case CKQ_F8_S16x16:      return launch_f8_split<E, S16x16>(a, s);
    case CKQ_F8_C256x256:    return launch_f8_core<E, C256x256>(a, s);
    case CKQ_F8_C256x128:    return launch_f8_core<E, C256x128>(a, s);
    case CKQ_F8_C128x128:    return launch_f8_core<E, C128x128>(a, s);
    case CKQ_F8_C64x128:     return launch_f8_core<E, C64x128>(a, s);
    case CKQ_F8_C64x64:      return launch_f8_core<E, C64x64>(a, s);
    case CKQ_F8_C128x192:    return launch_f8_core<E, C128x192>(a, s);
    case CKQ_F8_TWO:         return launch_f8_two<E, C256x256, C128x192>(a, f8_whole_columns(a.M, a.N), s);
    case CKQ_F8_STREAM:      return launch_f8_stream<E>(a, s);
    default:                 break;
    }
    F8Args first = a, second = a;
    if (!a.offsets && a.M > a.N) {
        first.M = (a.M / 2 + 127) & ~127;
        if (first.M >= a.M) return CKQ_EINVAL;
        second.M = a.M - first.M;
        second.A += (size_t)first.M * a.lda;
        second.sa += first.M;
        second.C = (E *)a.C + (size_t)first.M * a.ldc;
    } else {
        first.N = (a.N / 2 + 127) & ~127;
        if (first.N >= a.N) return CKQ_EINVAL;
        second.N = a.N - first.N;
        second.B += (size_t)first.N * a.ldb;
        second.sb += (size_t)(first.N / 128) * a.ldsb;
        if (a.bias) second.bias += first.N;
        second.C = (E *)a.C + first.N;
    }
    const int rc = launch_gemm_f8<E>(first, type, s);
    return rc ? rc : launch_gemm_f8<E>(second, type, s);
}

static int f8_gemm(const F8Args &a, int type, void *stream)
{
    if (!a.A || !a.sa || !a.B || !a.sb || !a.C || a.M <= 0 || a.N <= 0 || a.K <= 0 || a.lda < a.K || a.ldb < a.K || a.ldc < a.N || a.ldsa < a.M ||
        a.ldsb < a.K / 128 + (a.K % 128 != 0)) return CKQ_EINVAL;
    const int t = type & ~CKQ_SUMS_FP32, size = row_size(t);
    if (!size) return CKQ_EFORMAT;
    if (((uintptr_t)a.A | (uintptr_t)a.B) % 16 || a.lda % 16 || a.ldb % 16 || a.eb % 16 || a.lda > CKQ_I8_PITCH_MAX || a.ldb > CKQ_I8_PITCH_MAX) return CKQ_EROWS;
    if ((uintptr_t)a.C % size || ((uintptr_t)a.sa | (uintptr_t)a.sb | (uintptr_t)a.bias | (uintptr_t)a.offsets) % 4) return CKQ_EROWS;
    const hipStream_t s = (hipStream_t)stream;
    return t == CKQ_T_F32 ? launch_gemm_f8<float>(a, type, s) : t == CKQ_T_BF16 ? launch_gemm_f8<__bf16>(a, type, s) : launch_gemm_f8<_Float16>(a, type, s);
}

extern "C" int ckq_launch_gemm_f8(const uint8_t *A, long lda, const float *sa, long ldsa, const uint8_t *B, long ldb, const float *sb, long ldsb, const float *bias,
                                  int type, void *C, long ldc, int M, int N, int K, void *stream)
{
    return f8_gemm({A, B, sa, sb, bias, nullptr, C, lda, ldsa, ldb, 0, ldsb, 0, 0, ldc, M, N, K, 1}, type, stream);
}

extern "C" int ckq_launch_gemm_f8_experts(const uint8_t *A, long lda, const float *sa, long ldsa, const uint8_t *B, long ldb, long eb, const float *sb, long ldsb, long esb,
                                          const float *bias, const int32_t *offsets, int experts, int type, void *C, long ldc, int M, int N, int K, void *stream)
{
    if (!offsets || experts <= 0 || experts > CKQ_MOE_EXPERTS_MAX || M > CKQ_MOE_SLOTS_MAX || eb < 0 || esb < 0) return CKQ_EINVAL;
    return f8_gemm({A, B, sa, sb, bias, offsets, C, lda, ldsa, ldb, eb, ldsb, esb, N, ldc, M, N, K, experts}, type, stream);
}
