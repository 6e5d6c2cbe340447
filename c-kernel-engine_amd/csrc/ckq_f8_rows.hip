/*
 * ckq_f8_rows.hip - rows in e4m3 with one scale for each 128 elements: the activations of the fp8 matmuls of ckq_gemm_f8.hip, and
 * the rows read back.
 *
 *   v       = x                                        quantize; a token's row for each of its experts: gather
 *           = gate / (1 + exp(-gate)) * up             swiglu
 *   a       = max(max_i |v_i|, 2^-100)                 over a group of 128 elements (a group of zeros divides by nothing)
 *   q_i     = e4m3(448 v_i / a),  scale = a / 448
 *
 * The quotient is rounded correctly: 448 v / a of values with eight or eleven bits is often halfway between two codes, and a
 * product with 448 / a, which is rounded, would put half of those ties on the wrong side.  With a = a' 2^e, a' in [1, 2): n = 448 * 2^-e v
 * is exact for bf16 and fp16 (448 = 7 * 64), and a quotient from the correctly rounded inverse of a' and one
 * residual step is the correctly rounded one (Markstein, 1990).  Three operations an element more than the product.  Of an fp32 v, n
 * has up to 27 bits: what its rounding takes, which a multiply-add gives exactly, goes into the residual (without it, of fp32 rows one code in
 * some millions, and one in twenty next to a tie, is the wrong neighbour).  SwiGLU's v is off by more than that to begin with.
 *
 * A group with an infinity or a NaN in v has that as its scale and zeros as its codes; the maximum is taken over bit patterns, where
 * NaN > inf > everything else.
 */
#include "ckq_device.hpp"
#include "ckq_int8.hpp"
#include "ckq_launch.h"
#include "ckq_rows.hpp"
#include <algorithm>

enum { F8_QUANTIZE, F8_SWIGLU, F8_GATHER };

struct F8RowsArgs {
    const void  *x, *y;      /* rows; swiglu: gate, up */
    const int   *position;   /* gather: where each of a token's `choices` rows goes, [rows][choices] */
    uint8_t     *q;
    float       *scale;
    long         ldx, ldq, lds;
    int          rows, k, choices, most;     /* gather: positions from `most` on are none */
};

struct __attribute__((packed, aligned(1))) row16f8 { u32 v[4]; };
typedef u32 __attribute__((aligned(1))) u32_at_1;
typedef uint16_t __attribute__((aligned(1))) u16_at_1;

/* Sixteen values of a group, a' and 448 * 2^-e of it: their codes.  LONG: values of more bits than the product with c keeps. */
template <bool LONG>
__device__ __forceinline__ row16f8 f8_codes(const float (&v)[16], float a1, float c, bool finite)
{
#pragma clang fp contract(off)
    const float inv = 1.0f / a1;
    row16f8 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float n = v[4 * i + j] * c, q = n * inv, rest = __builtin_fmaf(-a1, q, n);
            t[j] = __builtin_fmaf(LONG ? rest + __builtin_fmaf(v[4 * i + j], c, -n) : rest, inv, q);
        }
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], w, true);
        o.v[i] = finite ? (u32)w : 0u;
    }
    return o;
}

/* Eight lanes have a group, sixteen elements each; a block has 2^rs rows beside each other and 32 >> rs groups of each: a row's codes leave in
 * whole lines, a group's scales side by side.  Bound by memory: 2048 x 11008 in bf16 68 MB in 13.4 to 15 us (4.5 to 5.1 TB/s; loads past the
 * caches, half a line each, 16.2), few rows by a launch (2). */
template <int OP, class E, bool EIGHT>
__global__ void __launch_bounds__(256) rows_f8_kernel(F8RowsArgs a, int rs, u32 group_tiles)
{
    const u32 rt = blockIdx.x / group_tiles, gt = blockIdx.x - rt * group_tiles;
    const int team = threadIdx.x >> 3, l = threadIdx.x & 7;
    const int row = (int)(rt << rs) + (team & ((1 << rs) - 1)), g = (int)gt * (32 >> rs) + (team >> rs);
    const long at = 128l * g + 16 * l;
    if (row >= a.rows || 128l * g >= a.k) return;              /* all eight lanes */
    const int left = (int)(a.k - at);
    const E *x = (const E *)a.x + (size_t)row * a.ldx + at;
    int to[8];                                                 /* gather: where the first eight go, under way with the row itself */
    if (OP == F8_GATHER) {
#pragma unroll
        for (int j = 0; j < 8; ++j) to[j] = a.position[(size_t)row * a.choices + min(j, a.choices - 1)];
    }
    raw8<E> r0 = fetch8_of<EIGHT>(x, left), r1 = fetch8_of<EIGHT>(x + 8, left - 8);
    float v[16];
    if (OP == F8_SWIGLU) {
        const E *y = (const E *)a.y + (size_t)row * a.ldx + at;
        raw8<E> u0 = fetch8_of<EIGHT>(y, left), u1 = fetch8_of<EIGHT>(y + 8, left - 8);
        if (left < 16) {
            drop_rest<EIGHT>(r0, left);
            drop_rest<EIGHT>(r1, left - 8);
            drop_rest<EIGHT>(u0, left);
            drop_rest<EIGHT>(u1, left - 8);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = row_swiglu(raw_value<E>(r0, i), raw_value<E>(u0, i));
            v[i + 8] = row_swiglu(raw_value<E>(r1, i), raw_value<E>(u1, i));
        }
    } else {
        if (left < 16) {
            drop_rest<EIGHT>(r0, left);
            drop_rest<EIGHT>(r1, left - 8);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = raw_value<E>(r0, i);
            v[i + 8] = raw_value<E>(r1, i);
        }
    }
    u32 top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __builtin_bit_cast(u32, v[i]) & 0x7fffffffu);
    top = max(top, (u32)dpp_get<0xB1>((int)top));
    top = max(top, (u32)dpp_get<0x4E>((int)top));
    top = max(top, (u32)dpp_get<0x141>((int)top));
    const bool finite = top < 0x7f800000u;
    const u32 bits = finite ? max(top, 0x0d800000u) : 0x3f800000u;                       /* 2^-100 at least */
    const float scale = finite ? __builtin_bit_cast(float, bits) / 448.0f : __builtin_bit_cast(float, top);
    const row16f8 o = f8_codes<sizeof(E) == 4 && OP != F8_SWIGLU>(v, __builtin_bit_cast(float, (bits & 0x7fffffu) | 0x3f800000u),
                               __builtin_bit_cast(float, ((262u - (bits >> 23)) << 23) | 0x600000u), finite);
    auto put = [&](int to) {
        uint8_t *q = a.q + (size_t)to * a.ldq + at;
        if (left >= 16) *reinterpret_cast<row16f8 *>(q) = o;
        else if (left > 0) {                                   /* eight, four, two and one */
            u32 v0 = o.v[0], v1 = o.v[1];
            if (left & 8) {
                *reinterpret_cast<row8q *>(q) = row8q{{v0, v1}};
                v0 = o.v[2];
                v1 = o.v[3];
                q += 8;
            }
            if (left & 4) {
                *reinterpret_cast<u32_at_1 *>(q) = v0;
                v0 = v1;
                q += 4;
            }
            if (left & 2) {
                *reinterpret_cast<u16_at_1 *>(q) = (uint16_t)v0;
                v0 >>= 16;
                q += 2;
            }
            if (left & 1) *q = (uint8_t)v0;
        }
        if (l == 0) a.scale[(size_t)g * a.lds + to] = scale;
    };
    if (OP != F8_GATHER) put(row);
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < a.choices && (u32)to[j] < (u32)a.most) put(to[j]);
        for (int j = 8; j < a.choices; ++j) {
            const int more = a.position[(size_t)row * a.choices + j];
            if ((u32)more < (u32)a.most) put(more);
        }
    }
}

/* As many rows beside each other as there are, 32 at most: the scales of a group leave side by side. */
static int f8_rows_shift(int rows, int k)
{
    int rs = 0;
    while (rs < 5 && (1 << rs) < rows && k <= 1 << 24) ++rs;      /* a launch has fewer than 2^32 threads */
    return rs;
}
/* Rows that one launch takes, for the same reason. */
static int f8_rows_most(int rows, int rs, u32 group_tiles) { return (int)std::min<size_t>(rows, ((size_t)1 << 23) / group_tiles << rs); }

template <int OP, class E>
static int launch_rows_f8(F8RowsArgs a, hipStream_t s)
{
    const int rs = f8_rows_shift(a.rows, a.k), groups = a.k / 128 + (a.k % 128 != 0), per = 32 >> rs;
    const u32 group_tiles = (u32)((groups + per - 1) / per);
    const int most = f8_rows_most(a.rows, rs, group_tiles);
    for (int rows = a.rows;;) {
        const int now = min(rows, most);
        a.rows = now;
        const int rc = i8_launch(a.k >= 8 ? rows_f8_kernel<OP, E, true> : rows_f8_kernel<OP, E, false>, dim3((u32)((now + (1 << rs) - 1) >> rs) * group_tiles), dim3(256), s, a, rs, group_tiles);
        if (rc || rows == now) return rc;
        rows -= now;
        a.x = (const E *)a.x + (size_t)now * a.ldx;
        if (a.y) a.y = (const E *)a.y + (size_t)now * a.ldx;
        if (OP == F8_GATHER) a.position += (size_t)now * a.choices;
        else {
            a.q += (size_t)now * a.ldq;
            a.scale += now;
        }
    }
}

template <int OP>
static int launch_rows_f8(int type, const F8RowsArgs &a, void *stream)
{
    switch (type) {
    case CKQ_T_F32:  return launch_rows_f8<OP, float>(a, (hipStream_t)stream);
    case CKQ_T_BF16: return launch_rows_f8<OP, __bf16>(a, (hipStream_t)stream);
    case CKQ_T_F16:  return launch_rows_f8<OP, _Float16>(a, (hipStream_t)stream);
    default:         return CKQ_EFORMAT;
    }
}

extern "C" int ckq_launch_quantize_f8(int type, const void *x, long ldx, uint8_t *q, long ldq, float *scale, long lds, int rows, int k, void *stream)
{
    if (!x || !q || !scale || rows <= 0 || k <= 0 || ldx < k || ldq < k || lds < rows) return CKQ_EINVAL;
    if (!row_size(type)) return CKQ_EFORMAT;
    if ((uintptr_t)x % row_size(type) || (uintptr_t)scale % 4) return CKQ_EROWS;
    const F8RowsArgs a = {x, nullptr, nullptr, q, scale, ldx, ldq, lds, rows, k, 0, 0};
    return launch_rows_f8<F8_QUANTIZE>(type, a, stream);
}

extern "C" int ckq_launch_swiglu_f8(int type, const void *gate, const void *up, long ld, uint8_t *q, long ldq, float *scale, long lds, int rows, int k, void *stream)
{
    if (!gate || !up || !q || !scale || rows <= 0 || k <= 0 || ld < k || ldq < k || lds < rows) return CKQ_EINVAL;
    if (!row_size(type)) return CKQ_EFORMAT;
    if (((uintptr_t)gate | (uintptr_t)up) % row_size(type) || (uintptr_t)scale % 4) return CKQ_EROWS;
    const F8RowsArgs a = {gate, up, nullptr, q, scale, ld, ldq, lds, rows, k, 0, 0};
    return launch_rows_f8<F8_SWIGLU>(type, a, stream);
}

extern "C" int ckq_launch_moe_gather_f8(int type, const void *x, long ldx, const int32_t *position, uint8_t *q, long ldq, float *scale, long lds,
                                        int tokens, int choices, int rows, int k, void *stream)
{
    if (!x || !position || !q || !scale || tokens <= 0 || choices <= 0 || rows <= 0 || k <= 0 || ldx < k || ldq < k || lds < rows) return CKQ_EINVAL;
    if (!row_size(type)) return CKQ_EFORMAT;
    if ((uintptr_t)x % row_size(type) || ((uintptr_t)scale | (uintptr_t)position) % 4) return CKQ_EROWS;
    const F8RowsArgs a = {x, nullptr, position, q, scale, ldx, ldq, lds, tokens, k, choices, rows};
    return launch_rows_f8<F8_GATHER>(type, a, stream);
}

/* y = T(scale * q), sixteen elements a thread, in pieces that are sixteen bytes of y: eight lanes store a line (2048 x 11008 to bf16 12.2 us, 5.5
 * TB/s, to fp32 20.1; sixteen beside each other 14.0 and 32.5). */
template <class E>
__global__ void __launch_bounds__(256) dequantize_f8_kernel(const uint8_t *__restrict__ q, long ldq, const float *__restrict__ scale, long lds,
                                                            E *__restrict__ y, long ldy, int rows, int k, int rs, u32 group_tiles)
{
    constexpr int V = 16 / sizeof(E), NP = 16 / V;
    const u32 rt = blockIdx.x / group_tiles, gt = blockIdx.x - rt * group_tiles;
    const int team = threadIdx.x >> 3, l = threadIdx.x & 7;
    const int row = (int)(rt << rs) + (team & ((1 << rs) - 1)), g = (int)gt * (32 >> rs) + (team >> rs);
    const long at = 128l * g;
    if (row >= rows || at >= k) return;
    const int left = (int)min(128l, k - at) - V * l;           /* of piece i: 8 V i less */
    const uint8_t *p = q + (size_t)row * ldq + at + V * l;
    E *o = y + (size_t)row * ldy + at + V * l;
    const float s = scale[(size_t)g * lds + row];
    struct __attribute__((packed, aligned(1))) codes { u32 v[V / 4]; } r[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int n = left - 8 * V * i;
        if (n >= V) r[i] = *reinterpret_cast<const codes *>(p + 8 * V * i);
        else {
#pragma unroll
            for (int j = 0; j < V / 4; ++j) r[i].v[j] = 0;
#pragma unroll
            for (int j = 0; j < V - 1; ++j)
                if (j < n) r[i].v[j >> 2] |= (u32)p[8 * V * i + j] << (8 * (j & 3));
        }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int n = left - 8 * V * i;
        struct __attribute__((packed, aligned(sizeof(E)))) piece { E v[V]; } f;
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)r[i].v[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)r[i].v[j], true);
            f.v[4 * j] = (E)(s * lo[0]);
            f.v[4 * j + 1] = (E)(s * lo[1]);
            f.v[4 * j + 2] = (E)(s * hi[0]);
            f.v[4 * j + 3] = (E)(s * hi[1]);
        }
        E *to = o + 8 * V * i;
        if (n >= V) {
            *reinterpret_cast<piece *>(to) = f;
            asm volatile("");                                /* or what both branches store is moved behind them, in pieces */
        } else {
#pragma unroll
            for (int j = 0; j < V - 1; ++j)
                if (j < n) to[j] = f.v[j];
        }
    }
}

extern "C" int ckq_launch_dequantize_f8(const uint8_t *q, long ldq, const float *scale, long lds, int type, void *y, long ldy, int rows, int k, void *stream)
{
    if (!q || !scale || !y || rows <= 0 || k <= 0 || ldq < k || ldy < k || lds < rows) return CKQ_EINVAL;
    if (!row_size(type)) return CKQ_EFORMAT;
    if ((uintptr_t)y % row_size(type) || (uintptr_t)scale % 4) return CKQ_EROWS;
    const int rs = f8_rows_shift(rows, k), groups = k / 128 + (k % 128 != 0), per = 32 >> rs;
    const u32 group_tiles = (u32)((groups + per - 1) / per);
    const int most = f8_rows_most(rows, rs, group_tiles);
    const hipStream_t s = (hipStream_t)stream;
    for (int row = 0; row < rows;) {
        const int n = min(rows - row, most);
        const uint8_t *qr = q + (size_t)row * ldq;
        const dim3 grid((u32)((n + (1 << rs) - 1) >> rs) * group_tiles), block(256);
        const int rc = type == CKQ_T_F32  ? i8_launch(dequantize_f8_kernel<float>, grid, block, s, qr, ldq, scale + row, lds, (float *)y + (size_t)row * ldy, ldy, n, k, rs, group_tiles)
                     : type == CKQ_T_BF16 ? i8_launch(dequantize_f8_kernel<__bf16>, grid, block, s, qr, ldq, scale + row, lds, (__bf16 *)y + (size_t)row * ldy, ldy, n, k, rs, group_tiles)
                                          : i8_launch(dequantize_f8_kernel<_Float16>, grid, block, s, qr, ldq, scale + row, lds, (_Float16 *)y + (size_t)row * ldy, ldy, n, k, rs, group_tiles);
        if (rc) return rc;
        row += n;
    }
    return 0;
}
