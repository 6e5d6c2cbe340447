/*
 * ckq_int8_rows.hip - rows in 8 bits with one scale each: the activations (and, when a model is loaded, the
 * weights) of the int8 matmul of ckq_gemm_int8.hip, and the rows read back.
 *
 *   v       = x                                        quantize
 *           = h * r * gamma,  h = T(x + residual),  r = 1 / sqrt(sum h^2 / k + eps)    rmsnorm
 *           = gate / (1 + exp(-gate)) * up             swiglu
 *   a       = max(max_i |v_i|, 2^-100)                 (a row of zeros divides by nothing)
 *   q_i     = rne(v_i * (127 / a)),  scale = a / 127
 *
 * All of it in fp32.  The norm's factor r is the same for a whole row, so the largest |h * gamma| is looked for in
 * the pass that sums the squares, and r comes into the two factors of the row afterwards: one reduction across the
 * waves where the order of the formula would need two.  A row with an infinity or a NaN in v has that as its scale
 * and zeros as its quants, so that whatever is computed from it is not a number either; the maximum is taken over
 * bit patterns, where NaN > inf > everything else, and no order of lanes or waves can lose one.
 */
#include "ckq_device.hpp"
#include "ckq_int8.hpp"
#include "ckq_launch.h"
#include "ckq_rows.hpp"
#include <algorithm>

enum { ROWS_QUANTIZE, ROWS_RMSNORM, ROWS_SWIGLU };

struct RowsArgs {
    const void  *x;          /* rows; gate */
    const void  *y;          /* rmsnorm: residual or null; swiglu: up */
    void        *h;          /* rmsnorm: x + residual, where there is one */
    const float *gamma;
    int8_t      *q;
    float       *scale;
    long         ldx, ldy, ldh, ldq;
    float        eps;
    int          rows, k;
};

/* What the values of a vector (eight elements) are made of. */
template <class E> struct RowParts { raw8<E> x, y; raw8<float> g; };

template <int OP, bool ONCE, class E>
__device__ __forceinline__ void row_fetch(RowParts<E> &p, const RowsArgs &a, const E *x, const E *y, int v)
{
    const int left = a.k - 8 * v;
    p.x = fetch8<ONCE>(x + 8 * v, left);
    if (OP != ROWS_QUANTIZE && y) p.y = fetch8<ONCE>(y + 8 * v, left);
    if (OP == ROWS_RMSNORM) p.g = fetch8<false>(a.gamma + 8 * v, left);
}

/* The same of a row of eight elements and more: its last vector, where it is not whole, is cut out of the row's last eight elements, so that every lane has the same
 * loads.  (Some of those eight may be written by the lane before it, if the sum goes where x is: these are dropped.) */
template <int OP, bool ONCE, class E>
__device__ __forceinline__ void row_fetch_even(RowParts<E> &p, const RowsArgs &a, const E *x, const E *y, int v)
{
    const int at = min(8 * v, a.k - 8), drop = 8 * v - at;
    p.x = fetch8<ONCE>(x + at, 8);
    if (OP != ROWS_QUANTIZE && y) p.y = fetch8<ONCE>(y + at, 8);
    if (OP == ROWS_RMSNORM) p.g = fetch8<false>(a.gamma + at, 8);
    if ((a.k & 7) && drop) {
        drop_first(p.x, drop);
        if (OP != ROWS_QUANTIZE && y) drop_first(p.y, drop);
        if (OP == ROWS_RMSNORM) drop_first(p.g, drop);
    }
}

/* The values themselves, rmsnorm's without the row's factor r; `ss` collects the squares.  x + residual goes to h, where it is not null. */
template <int OP, class E>
__device__ __forceinline__ void row_values(float (&f)[8], const RowParts<E> &p, bool with_y, E *h, int left, float &ss)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = raw_value<E>(p.x, i);
    if (OP == ROWS_SWIGLU) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = row_swiglu(f[i], raw_value<E>(p.y, i));
    }
    if (OP == ROWS_RMSNORM) {
        if (with_y) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = (float)(E)(f[i] + raw_value<E>(p.y, i));         /* the norm is of the stream as it is stored */
            if (h) store8(h, f, left);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            ss = __builtin_fmaf(f[i], f[i], ss);
            f[i] *= raw_value<float>(p.g, i);
        }
    }
}

__device__ __forceinline__ u32 top_bits(const float (&f)[8], u32 top)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(u32, f[i]) & 0x7fffffffu);
    return top;
}

__device__ __forceinline__ u32 wave_top(u32 v)
{
    v = max(v, (u32)dpp_get<0xB1>((int)v));
    v = max(v, (u32)dpp_get<0x4E>((int)v));
    v = max(v, (u32)dpp_get<0x141>((int)v));
    v = max(v, (u32)dpp_get<0x140>((int)v));
    v = max(v, (u32)dpp_get<0x142, 0xA>((int)v));
    v = max(v, (u32)dpp_get<0x143, 0xC>((int)v));
    return (u32)__builtin_amdgcn_readlane((int)v, 63);
}
/* Of the first sixteen lanes alone. */
__device__ __forceinline__ u32 row_top(u32 v)
{
    v = max(v, (u32)dpp_get<0xB1>((int)v));
    v = max(v, (u32)dpp_get<0x4E>((int)v));
    v = max(v, (u32)dpp_get<0x141>((int)v));
    v = max(v, (u32)dpp_get<0x140>((int)v));
    return (u32)__builtin_amdgcn_readlane((int)v, 0);
}
__device__ __forceinline__ float wave_sum(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, group_sum<64>(v)), 63));
}

__device__ __forceinline__ u32 rounded_bits(float e, float inv)
{
#pragma clang fp contract(off)
    const float p = e * inv;
    return __builtin_bit_cast(u32, p + 12582912.0f);
}

/* NV > 0: `wpr` waves have a row, each thread at most NV vectors of it, held in registers between the two passes (k <= 512 wpr NV);
 * NV = 0: rows of any length, read again for the second pass: those longer than 32768, of sixteen waves each, and those shorter than eight.
 *
 * A row's squares are added in an order that its length alone decides, so that its results have the same bits alone and in any batch, though the
 * number of rows decides how many waves share it: each group of 512 elements by one wave, in the tree of its lanes; groups whose numbers differ by a multiple of
 * sixteen in turn; these sums, at most sixteen, in turn.  (NV = 0: each thread's elements, its wave's threads, the waves.)  It costs a wave of several groups a reduction for each of
 * them, nothing that shows beside the memory (us with one reduction a wave | now: norm in bf16 of 2048 x 4096 11.2 | 11.2, of 2048 x 8192 25.5 | 24.7, of one row of
 * 4096 2.73 | 2.69).
 */
template <int OP, class E, int NV>
__global__ void __launch_bounds__(1024) rows_i8_kernel(RowsArgs a, int wpr)
{
    __shared__ __attribute__((aligned(16))) float red_ss[NV == 4 ? 32 : 16];
    __shared__ u32   red_top[16];
    const int lane = threadIdx.x & 63, wave = wave_in_block(), nw = blockDim.x >> 6;
    const int row = __builtin_amdgcn_readfirstlane(wpr == 1 ? (int)blockIdx.x * nw + wave : (int)blockIdx.x);
    const bool live = row < a.rows;                          /* wpr == 1: waves behind the last row have nothing to do */
    if (wpr == 1 && !live) return;
    const E *x = (const E *)a.x + (size_t)row * a.ldx;
    const E *y = a.y ? (const E *)a.y + (size_t)row * a.ldy : nullptr;
    E *h = a.h ? (E *)a.h + (size_t)row * a.ldh : nullptr;
    const int nvec = (a.k >> 3) + ((a.k & 7) != 0), first = wpr == 1 ? lane : (int)threadIdx.x, step = 64 * wpr;

    float f[NV > 0 ? NV : 1][8], sq[NV > 0 ? NV : 1], ss = 0.0f;
    u32 top = 0;
#pragma unroll
    for (int i = 0; i < (NV > 0 ? NV : 1); ++i) sq[i] = 0.0f;
    if (NV > 0) {
        /* A vector's loads are under way together, gamma's too, before the store to h (which may be x or the residual, so that the compiler moves none
         * across it): one row of 4096 3.0 -> 2.7 us.  Those of two vectors and more only in the quantizer (2048 x 11008 in fp32 18.6 -> 17.6): elsewhere
         * their registers cost waves (norm of 2048 x 4096 in bf16 10.8 -> 12.6, SwiGLU of 2048 x 11008 20.1 -> 21.6). */
        constexpr int CH = OP == ROWS_QUANTIZE && NV > 0 ? NV : 1;
        /* What is quantized and a SwiGLU's halves are read for the last time, non-temporally, which leaves the caches to the quants: SwiGLU between the
         * two matmuls of an MLP of 4096 x 11008, at 2048 tokens 36 -> 25 us, at 4096 60 -> 42, the same at 128 to 1024 and at 8192; quantizer and what reads the quants, 11008 x 4096
         * in fp32 70 -> 64.  What lies in a cache anyway loses 2 to 4 % (SwiGLU of 512 x 11008 and its
         * reader, three sets in turn, 12.2 -> 12.7).  A residual stream has later readers (norm of 2048 x 4096 and its reader 17.6 -> 22.7). */
        constexpr bool ONCE = OP != ROWS_RMSNORM;
#pragma unroll
        for (int c = 0; c < NV; c += CH) {
            if (CH == 1) {
                const int v = first + c * step;
                if (v < nvec) {
                    RowParts<E> p;
                    row_fetch_even<OP, ONCE>(p, a, x, y, v);
                    row_values<OP>(f[c], p, y != nullptr, h ? h + 8 * v : nullptr, a.k - 8 * v, sq[c]);
                    top = top_bits(f[c], top);
                }
                continue;
            }
            RowParts<E> p[CH];
#pragma unroll
            for (int i = 0; i < CH; ++i)
                if (first + (c + i) * step < nvec) row_fetch<OP, ONCE>(p[i], a, x, y, first + (c + i) * step);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int v = first + (c + i) * step;
                if (v < nvec) {
                    row_values<OP>(f[c + i], p[i], y != nullptr, h ? h + 8 * v : nullptr, a.k - 8 * v, sq[c + i]);
                    top = top_bits(f[c + i], top);
                }
            }
        }
    } else
        for (int v = first; v < nvec; v += step) {
            RowParts<E> p;
            row_fetch<OP, false>(p, a, x, y, v);
            row_values<OP>(f[0], p, y != nullptr, h ? h + 8 * v : nullptr, a.k - 8 * v, sq[0]);
            top = top_bits(f[0], top);
        }

    top = wave_top(top);
    if (OP == ROWS_RMSNORM) {
#pragma unroll
        for (int i = 0; i < (NV > 0 ? NV : 1); ++i) sq[i] = wave_sum(sq[i]);
    }
    if (wpr == 1 || wpr == 16) {                             /* a wave has all groups of a row, or those that differ by multiples of sixteen */
#pragma unroll
        for (int i = 0; i < (NV > 0 ? NV : 1); ++i) ss += sq[i];
    }
    if (wpr > 1) {
        const int groups = wpr == 16 ? 16 : (NV > 0 ? NV : 1) * wpr;                  /* more than 16: three a wave of eight */
        if (lane == 0) {
            red_top[wave] = top;
            if (OP == ROWS_RMSNORM && wpr == 16) red_ss[wave] = ss;
            if (OP == ROWS_RMSNORM && wpr < 16) {
#pragma unroll
                for (int i = 0; i < (NV > 0 ? NV : 1); ++i) red_ss[wave + i * wpr] = sq[i];
            }
        }
        __syncthreads();
        /* the reads together: a loop over the waves waits for each by itself */
        const u32 tops = (lane & 15) < nw ? red_top[lane & 15] : 0u;
        if (OP == ROWS_RMSNORM) {
            const rows_f4 *red = reinterpret_cast<const rows_f4 *>(red_ss);
            rows_f4 col[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) col[i] = red[i];
            if (NV == 4 && groups > 16) {
#pragma unroll
                for (int i = 0; i < 4; ++i) col[i] += red[4 + i];
            }
            ss = col[0][0] + col[0][1];
            if (groups > 2) ss = ss + col[0][2] + col[0][3];
            if (groups > 4) ss = ss + col[1][0] + col[1][1] + col[1][2] + col[1][3];
            if (groups > 8) {
#pragma unroll
                for (int i = 0; i < 8; ++i) ss += col[2 + i / 4][i % 4];
            }
        }
        top = row_top(tops);
    }

    const float ftop = __builtin_bit_cast(float, top);
    const float r = OP == ROWS_RMSNORM ? 1.0f / sqrtf(ss / (float)a.k + a.eps) : 1.0f;
    /* an infinity or a NaN in the row; the squares' sum beyond fp32 (r = 0); a row of zeros and no eps (r infinite) */
    bool finite = ftop * r < __builtin_inff() && r > 0.0f;
    float amax = fmaxf(ftop * r, 0x1p-100f), inv = fminf(127.0f / amax * r, 0x1.fffffep127f);      /* gamma of zeros: 0 * inv has to be 0 */
    int8_t *q = a.q + (size_t)row * a.ldq;
    auto put = [&](const float (&e)[8], int v) {
        /* e inv in fp32, plus 1.5 * 2^23: the nearest integer (ties to even) in the low bits, |e inv| <= 127 (1 + 2^-22).  Not in one multiply-add,
         * which would round 63.5 less a rounding of inv the other way: quants are those of the formula in fp32, operation by operation. */
        u32 b[8], p[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = rounded_bits(e[i], inv);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            p[i] = !finite ? 0u : __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0c0c0400u) | __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x04000c0cu);
        const int left = a.k - 8 * v;
        if (left >= 8) {
            row8q o;
            o.v[0] = p[0];
            o.v[1] = p[1];
            *reinterpret_cast<row8q *>(q + 8 * v) = o;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) q[8 * v + i] = (int8_t)sbyte(p[i >> 2], i & 3);
        }
    };
    if (OP == ROWS_RMSNORM && (r > 0x1p26f || (r > 0.0f && top != 0 && ftop < 0x1p-100f))) {
        /* So small (rms and sqrt(eps) under 2^-26, or sum * gamma under 2^-100) that squares or sum * gamma may be below what fp32 holds: the row again from memory, the
         * larger of its largest element and sqrt(eps) made one half to one, in the order of the formula.  All waves of a row come here or none. */
        const E *src = y ? (const E *)h : x;
        const int groups = (nvec + 63) >> 6, w0 = wpr == 1 ? 0 : wave;
        auto each = [&](int g, auto &&use) {                 /* this lane's vector of a group, if there is one: its elements, and gamma's */
            const int v = 64 * g + lane;
            if (v >= nvec) return;
            const int left = a.k - 8 * v;
            use(fetch8<false>(src + 8 * v, left), fetch8<false>(a.gamma + 8 * v, left), v);
        };
        auto meet = [&](u32 t) {                             /* largest of the row */
            t = wave_top(t);
            if (wpr == 1) return t;
            __syncthreads();                                 /* what was there has been read */
            if (lane == 0) red_top[wave] = t;
            __syncthreads();
            return row_top((lane & 15) < nw ? red_top[lane & 15] : 0u);
        };
        u32 t = 0;
        for (int g = w0; g < groups; g += wpr)
            each(g, [&](const raw8<E> &e, const raw8<float> &, int) {
#pragma unroll
                for (int i = 0; i < 8; ++i) t = max(t, __builtin_bit_cast(u32, raw_value<E>(e, i)) & 0x7fffffffu);
            });
        const float big = fmaxf(__builtin_bit_cast(float, meet(t)), sqrtf(a.eps));
        const int up = max(0, -__builtin_amdgcn_frexp_expf(big));
        float sum = 0.0f;
        for (int c = w0; c < 16; c += wpr) {                 /* in the order of above */
            float part = 0.0f;
            for (int g = c; g < groups; g += 16) {
                float s = 0.0f;
                each(g, [&](const raw8<E> &e, const raw8<float> &, int) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float b = __builtin_ldexpf(raw_value<E>(e, i), up);
                        s = __builtin_fmaf(b, b, s);
                    }
                });
                part += wave_sum(s);
            }
            if (wpr == 1) sum += part;
            else if (lane == 0) red_ss[c] = part;
        }
        if (wpr > 1) {
            __syncthreads();
            for (int c = 0; c < 16; ++c) sum += red_ss[c];
        }
        const float rs = 1.0f / sqrtf(sum / (float)a.k + __builtin_ldexpf(a.eps, 2 * up));
        auto values = [&](float (&o)[8], const raw8<E> &e, const raw8<float> &g) {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __builtin_ldexpf(raw_value<E>(e, i), up) * rs * raw_value<float>(g, i);
        };
        t = 0;
        for (int g = w0; g < groups; g += wpr)
            each(g, [&](const raw8<E> &e, const raw8<float> &gm, int) {
                float o[8];
                values(o, e, gm);
                t = top_bits(o, t);
            });
        t = meet(t);
        const float most = __builtin_bit_cast(float, t);
        finite = big > 0.0f && most < __builtin_inff();      /* zeros and no eps: no norm */
        amax = fmaxf(most, 0x1p-100f);
        inv = 127.0f / amax;
        if (first == 0) a.scale[row] = finite ? amax / 127.0f : big > 0.0f ? most : __builtin_nanf("");
        for (int g = w0; g < groups; g += wpr)
            each(g, [&](const raw8<E> &e, const raw8<float> &gm, int v) {
                float o[8];
                values(o, e, gm);
                put(o, v);
            });
        return;
    }
    if (first == 0) a.scale[row] = finite ? amax / 127.0f : top >= 0x7f800000u ? ftop : r > 0.0f ? ftop * r : __builtin_nanf("");
    if (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int v = first + i * step;
            if (v < nvec) put(f[i], v);
        }
    } else
        for (int v = first; v < nvec; v += step) {
            RowParts<E> p;
            /* x + residual again from where this thread has stored it: x or the residual may be gone by now */
            const bool stored = OP == ROWS_RMSNORM && y;
            row_fetch<OP, false>(p, a, stored ? (const E *)h : x, OP == ROWS_RMSNORM ? nullptr : y, v);
            row_values<OP>(f[0], p, false, (E *)nullptr, a.k - 8 * v, ss);
            put(f[0], v);
        }
}

/* Waves of a row: as few as leave a thread three vectors (24 elements), so that loads, reduction and stores of several rows share
 * a CU; where every row has a CU to itself, as many as leave it one.  us with 2 | 4 | 8 | 16 waves a row: norm of 2048 x 4096 in bf16 13.2 |
 * 11.9 | 13.2 | 15.4 (10.8 with four since), SwiGLU of 2048 x 11008 31.0 | 21.3 | 20.4 | 20.9, quantizer of 11008 x 4096 in fp32 34.1 | 32.1 | 31.8 | 38.0 and of
 * 11008 x 896 9.3 | 10.2 | 14.9 | 29.3 (one wave 8.7); SwiGLU of 93 x 4863 in fp32 5.1 | 4.3 | 4.2 | 3.7.  Bound by memory beyond a few hundred
 * rows: 4.9 to 7 TB/s of what is read and written (a copy has 4.8 beyond the caches), and by the latency of one trip below. */
static int rows_waves(int nvec, int rows)
{
    int wpr = 1;
    while (wpr < 16 && nvec > 64 * wpr * (rows <= 256 ? 1 : 3)) wpr *= 2;
    return wpr;
}

template <int OP, class E>
static int launch_rows(RowsArgs a, hipStream_t s)
{
    const int nvec = a.k / 8 + (a.k % 8 != 0);
    const int wpr = rows_waves(nvec, a.rows), per = a.k < 8 ? 5 : (nvec - 1) / (64 * wpr) + 1;    /* 5: any length */
    const dim3 block(wpr == 1 ? 256u : 64u * (unsigned)wpr);
    /* a launch has fewer than 2^32 threads */
    for (;;) {
        const int left = a.rows, now = min(left, 1 << 21);
        a.rows = now;
        const dim3 grid((unsigned)(wpr == 1 ? (now + 3) / 4 : now));
        const int rc = per <= 1 ? i8_launch(rows_i8_kernel<OP, E, 1>, grid, block, s, a, wpr) : per <= 2 ? i8_launch(rows_i8_kernel<OP, E, 2>, grid, block, s, a, wpr)
                     : per <= 4 ? i8_launch(rows_i8_kernel<OP, E, 4>, grid, block, s, a, wpr) : i8_launch(rows_i8_kernel<OP, E, 0>, grid, block, s, a, wpr);
        if (rc || left == now) return rc;
        a.x = (const E *)a.x + (size_t)now * a.ldx;
        if (a.y) a.y = (const E *)a.y + (size_t)now * a.ldy;
        if (a.h) a.h = (E *)a.h + (size_t)now * a.ldh;
        a.q += (size_t)now * a.ldq;
        a.scale += now;
        a.rows = left - now;
    }
}

template <int OP>
static int launch_rows(int type, const RowsArgs &a, void *stream)
{
    switch (type) {
    case CKQ_T_F32:  return launch_rows<OP, float>(a, (hipStream_t)stream);
    case CKQ_T_BF16: return launch_rows<OP, __bf16>(a, (hipStream_t)stream);
    case CKQ_T_F16:  return launch_rows<OP, _Float16>(a, (hipStream_t)stream);
    default:         return CKQ_EFORMAT;
    }
}

extern "C" int ckq_launch_quantize_i8(int type, const void *x, long ldx, int8_t *q, long ldq, float *scale, int rows, int k, void *stream)
{
    if (!x || !q || !scale || rows <= 0 || k <= 0 || ldx < k || ldq < k) return CKQ_EINVAL;
    if (!row_size(type)) return CKQ_EFORMAT;
    if ((uintptr_t)x % row_size(type) || (uintptr_t)scale % 4) return CKQ_EROWS;
    const RowsArgs a = {x, nullptr, nullptr, nullptr, q, scale, ldx, 0, 0, ldq, 0.0f, rows, k};
    return launch_rows<ROWS_QUANTIZE>(type, a, stream);
}

extern "C" int ckq_launch_rmsnorm_i8(int type, const void *x, long ldx, const void *residual, void *sum, long ldr, const float *gamma, float eps,
                                     int8_t *q, long ldq, float *scale, int rows, int k, void *stream)
{
    if (!x || !gamma || !q || !scale || rows <= 0 || k <= 0 || ldx < k || ldq < k) return CKQ_EINVAL;
    if (sum == x && ldr != ldx && rows > 1) return CKQ_EINVAL;        /* rows would be overwritten before they are read */
    if (!residual != !sum || (residual && ldr < k) || !(eps >= 0.0f && eps < __builtin_inff())) return CKQ_EINVAL;
    if (!row_size(type)) return CKQ_EFORMAT;
    if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)sum) % row_size(type) || ((uintptr_t)scale | (uintptr_t)gamma) % 4) return CKQ_EROWS;
    const RowsArgs a = {x, residual, sum, gamma, q, scale, ldx, ldr, ldr, ldq, eps, rows, k};
    return launch_rows<ROWS_RMSNORM>(type, a, stream);
}

extern "C" int ckq_launch_swiglu_i8(int type, const void *gate, const void *up, long ld, int8_t *q, long ldq, float *scale, int rows, int k, void *stream)
{
    if (!gate || !up || !q || !scale || rows <= 0 || k <= 0 || ld < k || ldq < k) return CKQ_EINVAL;
    if (!row_size(type)) return CKQ_EFORMAT;
    if (((uintptr_t)gate | (uintptr_t)up) % row_size(type) || (uintptr_t)scale % 4) return CKQ_EROWS;
    const RowsArgs a = {gate, up, nullptr, nullptr, q, scale, ld, ld, 0, ldq, 0.0f, rows, k};
    return launch_rows<ROWS_SWIGLU>(type, a, stream);
}

/* y = T(scale * q), sixteen elements a thread, so that a load is as wide as it can be (eight: 2048 x 4096 to bf16 6.9 us, 5.5 now; 11008 x 4096
 * 25.0 and 22.2).  Bound by memory: 1 byte read and the type's written, 4.6 to 6.1 TB/s. */
struct __attribute__((packed, aligned(1))) row16q { u32 v[4]; };
template <class E>
__global__ void __launch_bounds__(256) dequantize_i8_kernel(const int8_t *__restrict__ q, long ldq, const float *__restrict__ scale,
                                                            E *__restrict__ y, long ldy, u32 rows, int k, u32 nvec)
{
    const u32 t = blockIdx.x * 256 + threadIdx.x, row = t / nvec, v = t - row * nvec;      /* fewer than 2^32 threads */
    if (row >= rows) return;
    const int8_t *p = q + (size_t)row * ldq + 16 * (size_t)v;
    E *o = y + (size_t)row * ldy + 16 * (size_t)v;
    const int left = k - 16 * (int)v;
    const float s = scale[row];
    float f[2][8];
    if (left >= 16) {
        const row16q r = *reinterpret_cast<const row16q *>(p);
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i >> 3][i & 7] = s * (float)sbyte(r.v[i >> 2], i & 3);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i >> 3][i & 7] = i < left ? s * (float)p[i] : 0.0f;
    }
    store8(o, f[0], left);
    if (left > 8) store8(o + 8, f[1], left - 8);
}

extern "C" int ckq_launch_dequantize_i8(const int8_t *q, long ldq, const float *scale, int type, void *y, long ldy, int rows, int k, void *stream)
{
    if (!q || !scale || !y || rows <= 0 || k <= 0 || ldq < k || ldy < k) return CKQ_EINVAL;
    if (!row_size(type)) return CKQ_EFORMAT;
    if ((uintptr_t)y % row_size(type) || (uintptr_t)scale % 4) return CKQ_EROWS;
    const u32 nvec = (u32)(k / 16 + (k % 16 != 0));
    const hipStream_t s = (hipStream_t)stream;
    /* a launch has fewer than 2^32 threads */
    const int most = (int)std::min<size_t>(rows, std::max<size_t>(1, ((size_t)1 << 31) / nvec));
    for (int row = 0; row < rows;) {
        const int n = min(rows - row, most);
        const int8_t *qr = q + (size_t)row * ldq;
        const dim3 grid((unsigned)(((size_t)n * nvec + 255) / 256)), block(256);
        const int rc = type == CKQ_T_F32  ? i8_launch(dequantize_i8_kernel<float>, grid, block, s, qr, ldq, scale + row, (float *)y + (size_t)row * ldy, ldy, (u32)n, k, nvec)
                     : type == CKQ_T_BF16 ? i8_launch(dequantize_i8_kernel<__bf16>, grid, block, s, qr, ldq, scale + row, (__bf16 *)y + (size_t)row * ldy, ldy, (u32)n, k, nvec)
                                          : i8_launch(dequantize_i8_kernel<_Float16>, grid, block, s, qr, ldq, scale + row, (_Float16 *)y + (size_t)row * ldy, ldy, (u32)n, k, nvec);
        if (rc) return rc;
        row += n;
    }
    return 0;
}
