/*
 * ckq_moe.hip - tokens sorted by expert and back.  Token t has `choices` slots, s = t * choices + j, each with the number of an expert
 * (none: anything outside 0 .. experts - 1) and, on the way back, a weight.
 *
 *   sort      slots in the order of their experts, those of one expert as they come: offsets[e] = slots of experts under e,
 *             order[p] = slot, position[s] = p (none: -1, and -1 in order from offsets[experts] on)
 *   gather    y[position[s]] = x[s / choices]
 *   combine   out[t] = T(sum_j w[s] y[position[s]]), in fp32, j in turn; without weights, the gradient of gather
 *   backward  dy[position[s]] = T(w[s] dout[t]),  dw[s] = sum_i dout[t][i] y[position[s]][i]
 *
 * No atomics: every result has one order of operations, whatever runs when.  Bound by memory but for a few tokens, where a launch is.
 */
#include "ckq_device.hpp"
#include "ckq_int8.hpp"
#include "ckq_launch.h"
#include "ckq_rows.hpp"
#include <algorithm>

/* ---- sort ---------------------------------------------------------------------------------------------------------- */

/* A block has an expert, the last one what has none.  Each goes through all slots: it counts those that belong before its own, and its own in each
 * wave's run of slots, whose places follow from that; then it writes its own.  No scratch memory, one launch, and the slots' order is kept without
 * a sort.  A wave takes 64 NV slots at a time into registers, one a lane and load; what it has compared it counts in scalar registers, two vector
 * instructions a slot.  Runs of up to 64 NV slots are read once.  65536 slots of 128 experts, us: one slot a lane and load, a load at a time,
 * 41.6; four a lane, counted in vector registers, 19.8; this 11 to 13 (16384 of 64 5.5, 8 slots 3.0: a launch), of which most are the instructions
 * of both passes. */
template <int NV>
__global__ void __launch_bounds__(1024) moe_sort_kernel(const int32_t *__restrict__ ids, int slots, int run, int experts, int32_t *__restrict__ offsets, int32_t *__restrict__ order,
                                                        int32_t *__restrict__ position)
{
    __shared__ int before[16], mine[16];
    const int lane = threadIdx.x & 63, wave = wave_in_block(), nw = blockDim.x >> 6;
    const u32 e = blockIdx.x;
    const int first = min(wave * run, slots), end = min(first + run, slots);
    u32 key[NV];                                               /* none: `experts`; behind the end: more than that.  No branch depends on either */
    auto load = [&](int s0) {
        const __amdgpu_buffer_rsrc_t rest = __builtin_amdgcn_make_buffer_rsrc((void *)(ids + s0), 0, (int)(4u * (u32)(slots - s0)), 0x00020000);      /* zeros behind the last */
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] = __builtin_amdgcn_raw_buffer_load_b32(rest, 4 * lane + 256 * i, 0, 0);
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] = min(key[i], (u32)experts);
        if (end - s0 < 64 * NV)
#pragma unroll
            for (int i = 0; i < NV; ++i) key[i] = s0 + 64 * i + lane < end ? key[i] : ~0u;
    };
    int less = 0, same = 0;
    for (int s0 = first; s0 < end; s0 += 64 * NV) {
        load(s0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            less += __popcll(__ballot(key[i] < e));
            same += __popcll(__ballot(key[i] == e));
        }
    }
    if (lane == 0) {
        before[wave] = less;
        mine[wave] = same;
    }
    __syncthreads();
    int at = 0, all = 0;
    for (int w = 0; w < nw; ++w) {
        all += before[w];
        at += before[w] + (w < wave ? mine[w] : 0);
    }
    at = __builtin_amdgcn_readfirstlane(at);
    if (threadIdx.x == 0) offsets[e] = all;
    if (same == 0) return;
    const bool some = e < (u32)experts;
    for (int s0 = first; s0 < end; s0 += 64 * NV) {
        if (end - first > 64 * NV) load(s0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            asm volatile("" : "+v"(key[i]));                  /* compared again: 64 masks kept from above are more registers than there are */
            const unsigned long long m = __ballot(key[i] == e);
            if (m == 0) continue;
            const int s = s0 + 64 * i + lane, p = __builtin_amdgcn_mbcnt_hi((u32)(m >> 32), __builtin_amdgcn_mbcnt_lo((u32)m, (u32)at));
            if (key[i] == e) {
                order[p] = some ? s : -1;
                position[s] = some ? p : -1;
            }
            at += __popcll(m);
        }
    }
}

extern "C" int ckq_launch_moe_sort(const int32_t *ids, int tokens, int choices, int experts, int32_t *offsets, int32_t *order, int32_t *position, void *stream)
{
    if (!ids || !offsets || !order || !position || tokens <= 0 || choices <= 0 || experts <= 0) return CKQ_EINVAL;
    if ((long)tokens * choices > CKQ_MOE_SLOTS_MAX || experts > CKQ_MOE_EXPERTS_MAX) return CKQ_EINVAL;
    if (((uintptr_t)ids | (uintptr_t)offsets | (uintptr_t)order | (uintptr_t)position) % 4) return CKQ_EROWS;
    const int slots = tokens * choices, run = ((slots - 1) / 1024 + 1) * 64;             /* of sixteen waves */
    const dim3 grid((u32)experts + 1);
    const hipStream_t s = (hipStream_t)stream;
    if (slots <= 4096) return i8_launch(moe_sort_kernel<4>, grid, dim3(64u * (u32)((slots - 1) / 256 + 1)), s, ids, slots, 256, experts, offsets, order, position);
    /* Read once where sixteen waves hold all slots and a CU has one block; else twice, by blocks of which a CU has two.  us, once | twice: 65536
     * slots of 128 experts 10.9 | 11.9, of 256 14.6 | 11.5, 262144 of 128 (either way twice) 36.7 | 35.4. */
    return i8_launch(slots > 16384 && slots <= 65536 && experts < 256 ? moe_sort_kernel<64> : moe_sort_kernel<16>, grid, dim3(1024), s, ids, slots, run, experts, offsets, order, position);
}

/* ---- rows there and back ------------------------------------------------------------------------------------------- */

struct MoeArgs {
    const void    *x;        /* gather: tokens' rows; combine: experts' rows; backward: the gradient of combine's output */
    const void    *y;        /* backward: experts' rows */
    void          *out;
    const int32_t *position;
    const float   *w;        /* or null */
    float         *dw;
    long           ldx, ldy, ldo;
    int            tokens, choices, rows, k;
};

/* Eight slots' places at a time are read before anything is done with them. */
template <class F>
__device__ __forceinline__ void moe_places(const MoeArgs &a, size_t t, F &&use)
{
    const int32_t *position = a.position + t * a.choices;
    for (int j0 = 0; j0 < a.choices; j0 += 8) {
        int p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = j0 + j < a.choices ? position[j0 + j] : -1;
        use(j0, p);
    }
}

/* Where a thread's eight elements begin: a row's last thread has its last eight, some of which the one before has too (the same values), so that
 * none has loads of its own. */
__device__ __forceinline__ long moe_at(const MoeArgs &a, u32 v) { return max(0l, min(8 * (long)v, (long)a.k - 8)); }

/* Eight elements a thread.  Bound by the rows it writes (8192 tokens of 8 slots x 2048 in bf16: 302 MB in 52 us, 5.8 TB/s).  ONCE here and in the
 * backward pass: what is written leaves non-temporally (moe_past_cache). */
template <class E, bool ONCE>
__global__ void __launch_bounds__(256) moe_gather_kernel(MoeArgs a, u32 nvec)
{
    const u32 i = blockIdx.x * 256 + threadIdx.x, t = i / nvec, v = i - t * nvec;
    if (t >= (u32)a.tokens) return;
    const long at = moe_at(a, v);
    const int left = (int)(a.k - at);
    const raw8<E> r = fetch8<false>((const E *)a.x + (size_t)t * a.ldx + at, left);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = raw_value<E>(r, j);
    moe_places(a, t, [&](int, const int (&p)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if ((u32)p[j] < (u32)a.rows) store8_pieces<E, ONCE>((E *)a.out + (size_t)p[j] * a.ldo + at, f, left);
    });
}

/* Eight elements a thread, the rows of eight slots on their way together (one token of 8 slots x 2048 6.8 us one after the other, 3.7 together),
 * non-temporally, being read for the last time, which leaves the caches to what is beside them (with a gather before it, 8192 tokens of 8 slots x
 * 2048 in bf16 132 -> 115 us; alone 52, 5.8 TB/s); fp32 not, whose loads take half a line each (119 -> 116). */
template <class E>
__global__ void __launch_bounds__(256) moe_combine_kernel(MoeArgs a, u32 nvec)
{
    const u32 i = blockIdx.x * 256 + threadIdx.x, t = i / nvec, v = i - t * nvec;
    if (t >= (u32)a.tokens) return;
    const long at = moe_at(a, v);
    const int left = (int)(a.k - at);
    const E *y = (const E *)a.x + at;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.0f;
    moe_places(a, t, [&](int j0, const int (&p)[8]) {
        float w[8];
        raw8<E> r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = a.w && j0 + j < a.choices ? a.w[(size_t)t * a.choices + j0 + j] : 1.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j0 + j < a.choices) r[j] = fetch8<sizeof(E) == 2>(y + (size_t)((u32)p[j] < (u32)a.rows ? p[j] : 0) * a.ldx, left);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if ((u32)p[j] < (u32)a.rows) {
#pragma unroll
                for (int c = 0; c < 8; ++c) f[c] = __builtin_fmaf(w[j], raw_value<E>(r[j], c), f[c]);
            }
    });
    store8_pieces((E *)a.out + (size_t)t * a.ldo + at, f, left);
}

/* A block has a token, its slots eight at a time: bound by the rows read and written (4096 tokens of 8 slots x 2048 in bf16, 285 MB in 58 us, 4.9
 * TB/s).  What vectors of eight leave of a row is read and written an element a lane, beside them: 93 tokens of 8 slots x 1001 in fp32 8.6 -> 6.0
 * us, 2048 of 8 x 2047 in bf16 50 -> 37.  Sums of dw: each thread's elements in turn, the tree of a wave's lanes, the waves in turn. */
template <class E, bool ONCE>
__global__ void __launch_bounds__(256) moe_combine_backward_kernel(MoeArgs a)
{
    __shared__ float red[4][8];
    const size_t t = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = wave_in_block();
    const E *d = (const E *)a.x + t * a.ldx;
    moe_places(a, t, [&](int j0, const int (&p)[8]) {
        float w[8], sum[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = j0 + j < a.choices ? a.w[t * a.choices + j0 + j] : 0.0f;
            sum[j] = 0.0f;
        }
        const int rest = a.k & 7, last = (int)threadIdx.x - 192;       /* the last wave, which short rows leave idle, has what no vector holds, an element a lane */
        if (last >= 0 && last < rest) {
            const long at = a.k - rest + last;
            const float g = (float)d[at];
            E y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j0 + j < a.choices) y[j] = ((const E *)a.y)[(size_t)((u32)p[j] < (u32)a.rows ? p[j] : 0) * a.ldy + at];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if ((u32)p[j] < (u32)a.rows) {
                    sum[j] = g * (float)y[j];
                    ((E *)a.out)[(size_t)p[j] * a.ldo + at] = (E)(w[j] * g);
                }
        }
        for (long v = 8l * threadIdx.x; v < a.k - rest; v += 2048) {
            const raw8<E> g = fetch8<false>(d + v, 8);
            raw8<E> y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j0 + j < a.choices) y[j] = fetch8<ONCE>((const E *)a.y + (size_t)((u32)p[j] < (u32)a.rows ? p[j] : 0) * a.ldy + v, 8);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if ((u32)p[j] < (u32)a.rows) {
                    float f[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        sum[j] = __builtin_fmaf(raw_value<E>(g, c), raw_value<E>(y[j], c), sum[j]);
                        f[c] = w[j] * raw_value<E>(g, c);
                    }
                    store_eight<E, ONCE>((E *)a.out + (size_t)p[j] * a.ldo + v, f);
                }
        }
        if (j0) __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j0 + j >= a.choices) break;
            const float s = group_sum<64>(sum[j]);
            if (lane == 63) red[wave][j] = s;
        }
        __syncthreads();
        if ((int)threadIdx.x < 8 && j0 + (int)threadIdx.x < a.choices)
            a.dw[t * a.choices + j0 + threadIdx.x] = red[0][threadIdx.x] + red[1][threadIdx.x] + red[2][threadIdx.x] + red[3][threadIdx.x];
    });
}

/* The launches of all tokens: one has fewer than 2^32 threads.  (min and max without std:: are those of int, on the host.) */
template <class E, class L>
static int moe_each(MoeArgs a, bool out_by_token, size_t threads, L &&launch)
{
    const int most = (int)std::min<size_t>(a.tokens, std::max<size_t>(1, ((size_t)1 << 31) / threads));
    for (int left = a.tokens;;) {
        const int now = min(left, most);
        a.tokens = now;
        const int rc = launch(a);
        if (rc || left == now) return rc;
        left -= now;
        a.position += (size_t)now * a.choices;
        if (a.w) a.w += (size_t)now * a.choices;
        if (a.dw) a.dw += (size_t)now * a.choices;
        if (out_by_token) a.out = (E *)a.out + (size_t)now * a.ldo;
        else              a.x = (const E *)a.x + (size_t)now * a.ldx;
    }
}

/* Whether what is written, a row for each slot, is more than the 256 MB cache holds beside the rest: then it leaves non-temporally, and its reader
 * finds it in memory either way.  us, kept | not: gather and the combine of its rows, bf16 x 2048, 67 MB 25.6 | 28.5, 134 MB 47.0 | 51.7, 252 MB
 * 115 | 100; the backward pass and the combine of its rows, 134 MB 73.0 | 80.6.  Not where a line leaves in pieces, that memory would get one by
 * one: fp32, whose threads store two pieces of 32 bytes one after the other (gather and combine of 537 MB 257 | 360, backward and combine of rows
 * x 2047 364 | 383), and gather's rows that do not begin at 16 bytes (bf16 x 2047 126 | 137). */
static bool moe_past_cache(const MoeArgs &a, size_t size, bool gather)
{
    return size == 2 && (size_t)a.tokens * a.choices * a.k * size > (size_t)192 << 20 && !(gather && ((uintptr_t)a.out % 16 || a.ldo % 8));
}

enum { MOE_GATHER, MOE_COMBINE, MOE_BACKWARD };
template <int OP, class E>
static int launch_moe(const MoeArgs &a, hipStream_t s)
{
    const u32 nvec = (u32)(a.k / 8 + (a.k % 8 != 0));
    const bool once = moe_past_cache(a, sizeof(E), OP == MOE_GATHER);
    return moe_each<E>(a, OP == MOE_COMBINE, OP == MOE_BACKWARD ? 256 : nvec, [&](const MoeArgs &b) {
        if (OP == MOE_BACKWARD) return i8_launch(once ? moe_combine_backward_kernel<E, sizeof(E) == 2> : moe_combine_backward_kernel<E, false>, dim3((u32)b.tokens), dim3(256), s, b);
        const dim3 grid((u32)(((size_t)b.tokens * nvec + 255) / 256));
        return i8_launch(OP == MOE_COMBINE ? moe_combine_kernel<E> : once ? moe_gather_kernel<E, sizeof(E) == 2> : moe_gather_kernel<E, false>, grid, dim3(256), s, b, nvec);
    });
}
template <int OP>
static int launch_moe(int type, const MoeArgs &a, void *stream)
{
    if (a.tokens <= 0 || a.choices <= 0 || a.rows <= 0 || a.k <= 0) return CKQ_EINVAL;
    const int size = row_size(type);
    if (!size) return CKQ_EFORMAT;
    if (((uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.out) % size || ((uintptr_t)a.position | (uintptr_t)a.w | (uintptr_t)a.dw) % 4) return CKQ_EROWS;
    const hipStream_t s = (hipStream_t)stream;
    return type == CKQ_T_F32 ? launch_moe<OP, float>(a, s) : type == CKQ_T_BF16 ? launch_moe<OP, __bf16>(a, s) : launch_moe<OP, _Float16>(a, s);
}

extern "C" int ckq_launch_moe_gather(int type, const void *x, long ldx, const int32_t *position, void *y, long ldy, int tokens, int choices, int rows, int k, void *stream)
{
    if (!x || !position || !y || ldx < k || ldy < k) return CKQ_EINVAL;
    return launch_moe<MOE_GATHER>(type, {x, nullptr, y, position, nullptr, nullptr, ldx, 0, ldy, tokens, choices, rows, k}, stream);
}

extern "C" int ckq_launch_moe_combine(int type, const void *y, long ldy, const int32_t *position, const float *weights, void *out, long ldo,
                                      int tokens, int choices, int rows, int k, void *stream)
{
    if (!y || !position || !out || ldy < k || ldo < k) return CKQ_EINVAL;
    return launch_moe<MOE_COMBINE>(type, {y, nullptr, out, position, weights, nullptr, ldy, 0, ldo, tokens, choices, rows, k}, stream);
}

extern "C" int ckq_launch_moe_combine_backward(int type, const void *dout, long ldd, const void *y, long ldy, const int32_t *position, const float *weights,
                                               void *dy, long lddy, float *dweights, int tokens, int choices, int rows, int k, void *stream)
{
    if (!dout || !y || !position || !weights || !dy || !dweights || ldd < k || ldy < k || lddy < k) return CKQ_EINVAL;
    if (dy == y && lddy != ldy && rows > 1) return CKQ_EINVAL;        /* rows would be overwritten before they are read */
    return launch_moe<MOE_BACKWARD>(type, {dout, y, dy, position, weights, dweights, ldd, ldy, lddy, tokens, choices, rows, k}, stream);
}
