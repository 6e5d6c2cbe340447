/* ckq_rows.hpp - what the kernels of rows share: vectors of eight elements of a row that starts anywhere an element can, SwiGLU of one. */
#pragma once
#include "ckq_device.hpp"
#include "ckq_launch.h"

template <int T> struct RowType;
template <> struct RowType<CKQ_T_F32>  { typedef float type; };
template <> struct RowType<CKQ_T_BF16> { typedef __bf16 type; };
template <> struct RowType<CKQ_T_F16>  { typedef _Float16 type; };

/* Eight consecutive elements; rows start anywhere an element can (the loads and stores take that as they are). */
template <class E> struct __attribute__((packed, aligned(sizeof(E)))) row8 { E v[8]; };
template <class E> struct __attribute__((packed, aligned(sizeof(E)))) row4 { E v[4]; };
template <class E> struct __attribute__((packed, aligned(sizeof(E)))) row2 { E v[2]; };
struct __attribute__((packed, aligned(1))) row8q { u32 v[2]; };

/* The same as loaded, in whole registers. */
template <class E> struct raw8 { u32 w[2 * sizeof(E)]; };
typedef float rows_f4 __attribute__((ext_vector_type(4)));
typedef u32 rows_u4 __attribute__((ext_vector_type(4)));
typedef rows_u4 __attribute__((aligned(2))) rows_u4_at_2;    /* one load of 16 bytes, wherever it falls */
template <bool ONCE, class E>                                /* ONCE: read for the last time, kept in no cache */
__device__ __forceinline__ raw8<E> fetch8(const E *p, int left)
{
    raw8<E> r;
    if (left >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(E) / 2; ++i) {
            const rows_u4_at_2 *at = reinterpret_cast<const rows_u4_at_2 *>(p) + i;
            const rows_u4 v = ONCE ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[4 * i + j] = v[j];
        }
        return r;
    }
#pragma unroll
    for (int i = 0; i < 2 * (int)sizeof(E); ++i) r.w[i] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < left) {
            if constexpr (sizeof(E) == 4) r.w[i] = __builtin_bit_cast(u32, p[i]);
            else                          r.w[i / 2] |= (u32)__builtin_bit_cast(uint16_t, p[i]) << (16 * (i & 1));
        }
    return r;
}
/* The elements from `drop` (0 .. 7) on, and zeros. */
template <class E>
__device__ __forceinline__ void drop_first(raw8<E> &r, int drop)
{
    constexpr int N = 2 * sizeof(E), PER = 4 / sizeof(E);    /* dwords, elements of one */
    if (PER == 2 && (drop & 1)) {
#pragma unroll
        for (int i = 0; i < N; ++i) r.w[i] = r.w[i] >> 16 | (i + 1 < N ? r.w[i + 1] << 16 : 0u);
    }
#pragma unroll
    for (int by = 1; by < N; by *= 2)
        if (drop & (by * PER)) {
#pragma unroll
            for (int i = 0; i < N; ++i) r.w[i] = i + by < N ? r.w[i + by] : 0u;
        }
}
/* The same as fetch8; EIGHT: of a row of at least eight elements, without a branch and loads of their own for its last: the row's last eight,
 * those before them dropped (drop_rest). */
template <bool EIGHT, class E>
__device__ __forceinline__ raw8<E> fetch8_of(const E *p, int left)
{
    return EIGHT ? fetch8<false>(p + min(0, left - 8), 8) : fetch8<false>(p, left);
}
template <bool EIGHT, class E>
__device__ __forceinline__ void drop_rest(raw8<E> &r, int left)
{
    if (EIGHT && left < 8) {
        drop_first(r, min(8 - left, 7));
        if (left <= 0) {
#pragma unroll
            for (int i = 0; i < 2 * (int)sizeof(E); ++i) r.w[i] = 0;
        }
    }
}
template <class E>
__device__ __forceinline__ float raw_value(const raw8<E> &r, int i)
{
    if constexpr (sizeof(E) == 4) return __builtin_bit_cast(float, r.w[i]);
    else return (float)__builtin_bit_cast(E, (uint16_t)(r.w[i / 2] >> (16 * (i & 1))));
}
template <class E, bool ONCE = false>                        /* ONCE: not kept in a cache */
__device__ __forceinline__ void store_eight(E *p, const float (&f)[8])
{
    row8<E> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = (E)f[i];
    if (ONCE) {
        struct { rows_u4 v[sizeof(E) / 2]; } w = __builtin_bit_cast(decltype(w), r);
#pragma unroll
        for (int i = 0; i < (int)sizeof(E) / 2; ++i) __builtin_nontemporal_store(w.v[i], reinterpret_cast<rows_u4_at_2 *>(p) + i);
    } else
        *reinterpret_cast<row8<E> *>(p) = r;
}
template <class E>
__device__ __forceinline__ void store8(E *p, const float (&f)[8], int left)
{
    if (left >= 8) {
        store_eight(p, f);
        asm volatile("");                                    /* or what both branches store is moved behind them, in pieces */
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = (E)f[i];
    }
}
/* The same, a row's last elements four, two and one at a time (RMSNorm with a residual in fp32, 2048 x 11008, is 3 % slower with it). */
template <class E, bool ONCE = false>
__device__ __forceinline__ void store8_pieces(E *p, const float (&f)[8], int left)
{
    if (left >= 8) {
        store_eight<E, ONCE>(p, f);
        asm volatile("");
    } else if (left > 0) {
        E e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = (E)f[i];
        if (left & 4) {
            *reinterpret_cast<row4<E> *>(p) = row4<E>{{e[0], e[1], e[2], e[3]}};
            p += 4;
#pragma unroll
            for (int i = 0; i < 3; ++i) e[i] = e[i + 4];
        }
        if (left & 2) {
            *reinterpret_cast<row2<E> *>(p) = row2<E>{{e[0], e[1]}};
            p += 2;
            e[0] = e[2];
        }
        if (left & 1) *p = e[0];
    }
}

/* gate / (1 + exp(-gate)) * up.  v_exp_f32 and v_rcp_f32, an ulp each: what they and the exponent's rounding are off is (2 + |gate|) 2^-23 of a
 * value that is about to be rounded to one part in 254 of the row's largest or to four bits (integer and fraction of the exponent apart, it would
 * be an ulp or two at any gate: int8 rows, 512 x 4864 5.35 -> 5.82 us, 2048 x 11008 23.5 -> 24.2).  A quarter of both sides of the fraction, so
 * that the reciprocal of no finite sum is below the normal numbers, where the instruction has zeros: those values count where up is large enough. */
__device__ __forceinline__ float row_swiglu(float gate, float up)
{
    const float e = __builtin_amdgcn_exp2f(gate * -1.44269504f);
    return 0.25f * gate * __builtin_amdgcn_rcpf(__builtin_fmaf(0.25f, e, 0.25f)) * up;
}

/* Bytes of an element; 0: no type of a row. */
static inline int row_size(int type) { return type == CKQ_T_F32 ? 4 : type == CKQ_T_BF16 || type == CKQ_T_F16 ? 2 : 0; }
