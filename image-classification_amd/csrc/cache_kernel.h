// cache_kernel.h -- a bank of key / value rows held in 4 bits: quantising append, softmax attention, eviction.
//
// Held format (OCP microscaling FP4).  A row of `dim` values is padded with zeros to W = 32 NB in {64, 128, 256} and cut
// into blocks of 32.  A block has one scale 2^e, e the smallest integer with max|x| <= 7 * 2^e (7 = the half step above
// the largest element 6, so that the largest value of a block is never further off than half a step of its binade), clamped
// to [-126, 125] and stored as the byte e + 127.  Elements are x / 2^e on E2M1 (0 .5 1 1.5 2 3 4 6, sign bit), nearest even,
// saturating; two a byte, the even one in the low four bits.  Every element times its scale is exact in bf16, which is what
// the matrix cores read: v_cvt_scalef32_pk_bf16_fp4 turns two elements and their scale into two bf16 in one instruction.
// A row (of one head) whose key or value has a NaN or an infinity is held as NaN whole: scale bytes 255 on its key (0 on its
// value, so that a product with a probability of zero stays zero), elements 0.
//
//   key, value              [batch][heads][rows][W / 2]   bytes
//   key_scale, value_scale  [batch][heads][W / 32][rows]  bytes: rows innermost, so that a lane of the value product gets the
//                                                         scales of its four neighbouring rows with one 4-byte load
//   weight (float32), position (int32)  [batch][heads][rows];  length, seen (int32)  [batch];  rows: a multiple of 64
//
// Matrix-core layout (v_mfma_f32_16x16x32_bf16; lane = 16 j + c; A: row c, 8 k-values of group j; B: column c, the same;
// result: column c, rows 4 j + r).  Both products are computed transposed, so that the probabilities never leave their lane:
//   S^T = K Q^T: A = 16 rows of the bank, B = 16 query rows.  The order of the k index (head dims) is free as long as both
//     sides agree: lane group j owns the dims [j W/4, (j+1) W/4), i.e. W/8 contiguous bytes of a row = one wide load, and
//     MFMA step i takes its 8 dims j W/4 + 8 i ...
//   O^T = V^T P^T: B = the probabilities as S^T left them (lane: query row c; 8 bank rows 16 a + 4 j + r of a unit of 32 as
//     the 8 k-values, a = 0, 1), A = 8 values of one channel: lane c owns the 2 NB channels [c W/16, (c+1) W/16), i.e. NB
//     contiguous bytes of each of its 8 rows, and MFMA step i takes channel c W/16 + i.
#ifndef MI_CACHE_KERNEL_H
#define MI_CACHE_KERNEL_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace mi {

typedef __attribute__((ext_vector_type(8))) __bf16 cb16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 cb16x2;
typedef __attribute__((ext_vector_type(4))) float cf32x4;
typedef __attribute__((ext_vector_type(16))) float cf32x16;

enum { CACHE_F32 = 0, CACHE_BF16 = 1, CACHE_F16 = 2 };

constexpr float CACHE_LOG2E = 1.4426950408889634f;

struct CacheView {
    uint8_t *key, *key_scale, *value, *value_scale;
    float *weight;
    int *position, *length, *seen;
    int batch, heads, dim, rows, limit;      // rows: allocated (multiple of 64); limit: most rows that are used
};

// Rows in use of a sequence, whatever its buffer holds (a restored state may be anything).
__device__ __forceinline__ int rows_used(const CacheView &c, int b) { return min(max(c.length[b], 0), c.limit); }

// ---------------------------------------------------------------------------------------------------- element access
template <int DT>
__device__ __forceinline__ void load8(const void *p, float (&x)[8])
{
    if constexpr (DT == CACHE_F32) {
        const float4 a = ((const float4 *)p)[0], b = ((const float4 *)p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 a = *(const uint4 *)p;
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == CACHE_BF16) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const uint16_t l = (uint16_t)w[i], h = (uint16_t)(w[i] >> 16);
                x[2 * i] = (float)__builtin_bit_cast(_Float16, l);
                x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, h);
            }
        }
    }
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    cb16x2 r;
    r[0] = (__bf16)a;
    r[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, r);
}

// Eight float32 rounded once to the caller's type (float16: saturating is not wanted, infinities stay infinities).
template <int DT>
__device__ __forceinline__ void store8(void *p, const float (&x)[8])
{
    if constexpr (DT == CACHE_F32) {
        ((float4 *)p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        ((float4 *)p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == CACHE_BF16) {
                w[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
            } else {
                const _Float16 l = (_Float16)x[2 * i], h = (_Float16)x[2 * i + 1];
                w[i] = (uint32_t)__builtin_bit_cast(uint16_t, l) | ((uint32_t)__builtin_bit_cast(uint16_t, h) << 16);
            }
        }
        *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// N = 2, 4 or 8 of them.
template <int DT, int N>
__device__ __forceinline__ void store_n(void *p, const float (&x)[N])
{
    if constexpr (N == 8) store8<DT>(p, x);
    else if constexpr (DT == CACHE_F32) {
#pragma unroll
        for (int i = 0; i < N; i += 2) ((float2 *)p)[i / 2] = make_float2(x[i], x[i + 1]);
    } else {
        uint32_t w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            if constexpr (DT == CACHE_BF16) w[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
            else {
                const _Float16 l = (_Float16)x[2 * i], h = (_Float16)x[2 * i + 1];
                w[i] = (uint32_t)__builtin_bit_cast(uint16_t, l) | ((uint32_t)__builtin_bit_cast(uint16_t, h) << 16);
            }
        }
        if constexpr (N == 4) *(uint2 *)p = make_uint2(w[0], w[1]);
        else *(uint32_t *)p = w[0];
    }
}

template <int DT>
__host__ __device__ constexpr int elem_bytes() { return DT == CACHE_F32 ? 4 : 2; }

// ------------------------------------------------------------------------------------------------------ append (push)
struct PushParams {
    CacheView c;
    const char *key, *value;
    long long key_s[3], value_s[3];          // byte strides: sequence, head, row
    const int *counts;                       // real rows of each sequence, or null: all T
    int T;
    char *held_key, *held_value;             // [batch][heads][T][dim] of the input type, or null
};

// The scale byte of a block whose largest magnitude is `top`: top = 1.f * 2^(E - 127) <= 1.75 * 2^(e + 2).
__device__ __forceinline__ int scale_byte(float top)
{
    const uint32_t b = __float_as_uint(top);
    const int byte = (int)(b >> 23) - 2 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return byte < 1 ? 1 : byte > 252 ? 252 : byte;
}

__device__ __forceinline__ int push_count(const PushParams &p, int b, int len)
{
    int n = p.counts ? p.counts[b] : p.T;
    n = n < 0 ? 0 : n > p.T ? p.T : n;
    const int room = p.c.limit - len;
    return n < room ? n : room < 0 ? 0 : room;
}

// A lane takes 8 dims of one side (key or value) of one row: W / 8 lanes a side, 2 W / 8 a row; a block of 32 is 4 lanes.
// WHOLE: a workgroup has a sequence to itself (few rows, as in decoding) and lengthens it at its end, which saves the launch of
// cache_advance_kernel (64 sequences, one row of 8 heads: 4.3 + 1.7 us with it).
template <int DT, int W, bool WHOLE>
__global__ __launch_bounds__(256) void cache_push_kernel(PushParams p)
{
    constexpr int SIDE = W / 8, ROW = 2 * SIDE;
    constexpr int TURN = 256 / ROW, TURNS = 4;                   // rows a turn; turns of a workgroup that shares a sequence
    const int lane = threadIdx.x & 63, c = threadIdx.x % SIDE, side = threadIdx.x / SIDE & 1;
    // WHOLE: rows of all heads of sequence blockIdx.x; otherwise a stretch of one head's
    const int chunks = WHOLE ? 1 : (p.T + TURN * TURNS - 1) / (TURN * TURNS);
    const int group = (int)(blockIdx.x / chunks), b = WHOLE ? (int)blockIdx.x : group / p.c.heads;
    const int first = WHOLE ? 0 : (int)(blockIdx.x % chunks) * TURN * TURNS, last = WHOLE ? p.c.heads * p.T : min(p.T, first + TURN * TURNS);
    const int len = rows_used(p.c, b), n = push_count(p, b, len);
#pragma unroll WHOLE ? 1 : TURNS
    for (int r0 = first; r0 < last; r0 += TURN) {
        const int r = r0 + threadIdx.x / ROW;
        const bool in = r < last;
        const int h = WHOLE ? (in ? r / p.T : 0) : group - b * p.c.heads, t = WHOLE ? (in ? r - h * p.T : 0) : r;
        const bool real = in && t < n;
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (real && c * 8 < p.c.dim) {
            const char *src = side ? p.value + b * p.value_s[0] + h * p.value_s[1] + t * p.value_s[2]
                                   : p.key + b * p.key_s[0] + h * p.key_s[1] + t * p.key_s[2];
            load8<DT>(src + (long long)c * 8 * elem_bytes<DT>(), x);
        }
        float top = 0.f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            bad |= (__float_as_uint(x[i]) & 0x7f800000u) == 0x7f800000u;
            top = fmaxf(top, fabsf(x[i]));
        }
        top = fmaxf(top, __shfl_xor(top, 1));
        top = fmaxf(top, __shfl_xor(top, 2));
        const unsigned long long who = __ballot(bad);
        const unsigned long long mine = ROW == 64 ? ~0ull : ((1ull << (ROW & 63)) - 1) << (lane / ROW * ROW);
        const bool poison = (who & mine) != 0;
        const int byte = scale_byte(top);
        uint32_t code = 0;
        if (!poison) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = ldexpf(x[i], 127 - byte);        // a power of two: exact
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[0], y[1], 1.0f, 0);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[2], y[3], 1.0f, 1);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[4], y[5], 1.0f, 2);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[6], y[7], 1.0f, 3);
        }
        if (real) {
            const long long bh = (long long)b * p.c.heads + h;
            const long long slot = (long long)len + t;
            *(uint32_t *)((side ? p.c.value : p.c.key) + (bh * p.c.rows + slot) * (W / 2) + c * 4) = code;
            if ((c & 3) == 0)
                (side ? p.c.value_scale : p.c.key_scale)[(bh * (W / 32) + c / 4) * p.c.rows + slot] = (uint8_t)(!poison ? byte : side ? 0 : 255);
            if (c == 0) {
                if (side) p.c.position[bh * p.c.rows + slot] = p.c.seen[b] + t;
                else p.c.weight[bh * p.c.rows + slot] = 0.f;
            }
        }
        char *held = side ? p.held_value : p.held_key;
        if (held && in && c * 8 < p.c.dim) {
            float v[8];
            const float s = ldexpf(1.f, byte - 127);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int four = (int)(code >> (4 * i)) & 15, low = four & 7;
                const float a = (low < 4 ? 0.5f * (float)low : low < 6 ? (float)(low - 2) : (float)(2 * low - 8)) * s;
                // a float16 above 57344 is held as 2^16, past its largest number: the copy is the nearest that there is
                const float near = DT == CACHE_F16 ? fminf(a, 65504.f) : a;
                v[i] = poison ? __uint_as_float(0x7fc00000u) : !real ? 0.f : four > 7 ? -near : near;
            }
            const long long at_row = ((long long)b * p.c.heads + h) * p.T + t;
            store8<DT>(held + (at_row * p.c.dim + c * 8) * elem_bytes<DT>(), v);
        }
    }
    if constexpr (WHOLE) {
        __syncthreads();
        if (threadIdx.x == 0) {
            p.c.length[b] = len + n;
            p.c.seen[b] += n;
        }
    }
}

// After the rows are written: every sequence is longer by what it got.
__global__ void cache_advance_kernel(PushParams p)
{
    const int b = blockIdx.x * 64 + threadIdx.x;
    if (b >= p.c.batch) return;
    const int len = rows_used(p.c, b), n = push_count(p, b, len);
    p.c.length[b] = len + n;
    p.c.seen[b] += n;
}

// How many rows the longest sequence would have after a push: what the host looks at where its own bound says it may not fit.
__global__ __launch_bounds__(256) void cache_longest_kernel(PushParams p, int *out)
{
    __shared__ int s_most[4];
    int most = 0;
    for (int b = threadIdx.x; b < p.c.batch; b += 256) {
        int n = p.counts ? p.counts[b] : p.T;
        n = n < 0 ? 0 : n > p.T ? p.T : n;
        most = max(most, (int)min((uint32_t)rows_used(p.c, b) + (uint32_t)n, 0x7fffffffu));     // up to 2^30 each
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = max(most, __shfl_xor(most, d));
    if ((threadIdx.x & 63) == 0) s_most[threadIdx.x >> 6] = most;
    __syncthreads();
    if (threadIdx.x == 0) *out = max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3]));
}

// Clears *out where the last rows of a (sequence, head) are not the rows pushed last, in their order: what causal attention of several
// rows goes by.  A sequence of which no row was evicted is in order.
__global__ void cache_order_start_kernel(int *out) { *out = 1; }

__global__ __launch_bounds__(256) void cache_order_kernel(PushParams p, int *out)
{
    const long long bh = blockIdx.x;
    const int b = (int)(bh / p.c.heads), len = rows_used(p.c, b), seen = p.c.seen[b];
    int n = p.counts ? p.counts[b] : p.T;
    n = n > p.T ? p.T : n;
    if (n <= 1 || seen == len) return;
    for (int slot = max(0, len - n) + (int)threadIdx.x; slot < len; slot += 256)
        if (p.c.position[bh * p.c.rows + slot] != seen - len + slot) *out = 0;
}

// Every sequence is cut to at most its entry of `lengths` (or `length`): of each head the rows pushed last leave.  Where no row of the
// sequence was ever evicted, or what leaves lies behind the new length in the order of its pushes, that is all there is to do.  An
// eviction puts rows from above into freed slots, so that a row's slot says nothing of its age: then the rows with the largest positions
// leave, and the slots that they free below the new length take the rows that stay from above it, both in ascending order (as an
// eviction does; no row is read that another one is written to).  Positions go on from the cut, and in any case behind all that stay.
// A workgroup a sequence, a wave a head: the order is looked at in 4 bytes a head and row that leaves (2.6 us for 64 sequences of 8 heads).
// Only where it does not hold is a head gone over, without a barrier, in two passes where an eviction has kept all that leaves (a call that
// takes 5 of 2048 rows back: 24 us for 64 sequences of 8 heads; of 131 k rows 530 us for one.  With a workgroup on one head after the
// other and the edge found by digits, counted with atomics: 440 and 3800 us).
constexpr int TRIM_THREADS = 1024, TRIM_RING = 512;
constexpr int TRIM_NO_TIES = 0x7fffffff;

struct TrimShared {
    int holes[TRIM_THREADS / 64][TRIM_RING], tails[TRIM_THREADS / 64][64];
    int last;
};

// How many of the first `len` rows f says yes to (its argument: a row's position, in unsigned order).
template <typename F>
__device__ __forceinline__ int count_rows(const int *pos, int len, F f)
{
    int n = 0;
    for (int i0 = (threadIdx.x & 63) * 4; i0 < len; i0 += 1024) {
        int4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = i0 + 256 * k < len ? *(const int4 *)(pos + i0 + 256 * k) : make_int4(0, 0, 0, 0);      // (rows are allocated in 64s)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = i0 + 256 * k, y[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) n += i + e < len && f((uint32_t)y[e] ^ 0x80000000u);
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
    return n;
}

// One wave: lets the len - n youngest of the `len` rows of one head leave and puts the others into slots 0 .. n.  Returns the largest
// position that stays, where it may be seen - (len - n) or more, else -1.
__device__ __forceinline__ int trim_head(const CacheView &c, long long bh, int width, int len, int n, int seen, int *holes, int *tails)
{
    const int lane = threadIdx.x & 63, gone = len - n;
    int *const pos = c.position + bh * c.rows;
    bool moved = false;
    for (int i = n + lane; i < len; i += 64) moved |= pos[i] != seen - len + i;
    if (!__any(moved)) return -1;
    // rows behind `edge` leave, and of those on it all but the `tied` lowest slots
    uint32_t edge = ((uint32_t)(seen - gone) ^ 0x80000000u) - 1;
    int tied = TRIM_NO_TIES, last = -1;
    if (count_rows(pos, len, [&](uint32_t u) { return u > edge; }) != gone) {
        // this head has evicted some of the rows pushed last: the gone-th largest position, by bits from the top
        edge = 0;
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
            if (count_rows(pos, len, [&](uint32_t u) { return u >= (edge | bit); }) >= gone) edge |= bit;
        const int behind = count_rows(pos, len, [&](uint32_t u) { return u > edge; });
        tied = count_rows(pos, len, [&](uint32_t u) { return u == edge; }) - (gone - behind);
        if (tied > 0) last = (int)(edge ^ 0x80000000u);
        else
            for (int i = lane; i < len; i += 64)
                if (((uint32_t)pos[i] ^ 0x80000000u) < edge) last = max(last, pos[i]);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) last = max(last, __shfl_xor(last, d));
    }
    const unsigned long long below = (1ull << lane) - 1;
    const auto leaves = [&](bool in, uint32_t u, int &on) {        // of 64 neighbours, asked in ascending order; `on`: rows on the edge so far
        if (tied == TRIM_NO_TIES) return in && u > edge;
        const unsigned long long who = __ballot(in && u == edge);
        const int before = on + __popcll(who & below);
        on += __popcll(who);
        return in && (u > edge || (u == edge && before >= tied));
    };
    int on_hole = 0, on_tail = tied == TRIM_NO_TIES ? 0 : count_rows(pos, n, [&](uint32_t u) { return u == edge; });
    const int words = width / 32, parts = 4 * words + 2;          // 16 bytes of key or value, or a byte of their scales, for each 32 dims
    int found = 0, filled = 0, hole0 = 0;                          // freed slots found, and taken; where the search goes on
    for (int t0 = n; t0 < len; t0 += 64) {
        const bool in = t0 + lane < len, stays = in && !leaves(in, in ? (uint32_t)pos[t0 + lane] ^ 0x80000000u : 0u, on_tail);
        const unsigned long long who = __ballot(stays);
        if (!who) continue;
        const int want = __popcll(who);
        if (stays) tails[__popcll(who & below)] = t0 + lane;
        while (found < filled + want && hole0 < n) {               // as many freed slots as rows that stay: fewer than 64 + 256 wait
            uint32_t u[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = hole0 + 64 * k + lane < n ? (uint32_t)pos[hole0 + 64 * k + lane] ^ 0x80000000u : 0u;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int slot = hole0 + 64 * k + lane;
                const bool hole = leaves(slot < n, u[k], on_hole);
                const unsigned long long free = __ballot(hole);
                if (hole) holes[(found + __popcll(free & below)) % TRIM_RING] = slot;
                found += __popcll(free);
            }
            hole0 += 256;
        }
        __threadfence_block();                                     // lists of the wave's own: written before they are read
        const int moves = min(want, found - filled);
        for (int i = lane; i < moves * parts; i += 64) {
            const int k = i / parts, part = i - k * parts, src = tails[k], dst = holes[(filled + k) % TRIM_RING];
            if (part < 2 * words) {
                uint8_t *side = (part < words ? c.key : c.value) + bh * c.rows * (width / 2) + part % words * 16;
                *(uint4 *)(side + (long long)dst * (width / 2)) = *(const uint4 *)(side + (long long)src * (width / 2));
            } else if (part < 4 * words) {
                uint8_t *side = (part < 3 * words ? c.key_scale : c.value_scale) + (bh * words + part % words) * c.rows;
                side[dst] = side[src];
            } else if (part == 4 * words) c.weight[bh * c.rows + dst] = c.weight[bh * c.rows + src];
            else pos[dst] = pos[src];
        }
        filled += moves;
        __threadfence_block();                                     // and read before the next ones are written
    }
    return last;
}

__global__ __launch_bounds__(TRIM_THREADS) void cache_trim_kernel(CacheView c, const int *lengths, int length, int width)
{
    __shared__ TrimShared sh;
    const int b = blockIdx.x, wave = threadIdx.x >> 6;
    int n = lengths ? lengths[b] : length;
    n = n < 0 ? 0 : n;
    const int len = rows_used(c, b), gone = len - n, seen = c.seen[b];
    if (gone <= 0) return;
    if (threadIdx.x == 0) sh.last = -1;
    __syncthreads();
    if (n > 0 && seen != len)
        for (int h = wave; h < c.heads; h += TRIM_THREADS / 64) {
            const int last = trim_head(c, (long long)b * c.heads + h, width, len, n, seen, sh.holes[wave], sh.tails[wave]);
            if (last >= 0 && (threadIdx.x & 63) == 0) atomicMax(&sh.last, last);
        }
    __syncthreads();
    if (threadIdx.x == 0) {
        c.length[b] = n;
        c.seen[b] = max(seen - gone, sh.last + 1);
    }
}

// ------------------------------------------------------------------------------------------------ 4 bits to bf16
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float scale_of(uint32_t word, int e) { return __uint_as_float(((word >> (8 * e)) & 255u) << 23); }

template <int I>
__device__ __forceinline__ uint32_t cvt2(uint32_t w, float s)
{
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, I));
}

__device__ __forceinline__ cb16x8 cvt8(uint32_t w, float s)
{
    const uint4 v = make_uint4(cvt2<0>(w, s), cvt2<1>(w, s), cvt2<2>(w, s), cvt2<3>(w, s));
    return __builtin_bit_cast(cb16x8, v);
}

// ---------------------------------------------------------------------------------------------------------- read back
// Rows [0, limit) of every sequence and head as bf16 (exact); rows behind the last one are zeros.  A lane takes 8 dims of a row; a
// workgroup CACHE_READ_TURNS * 2048 / W rows of one head, so that nothing is divided by (with a row found by 64-bit divisions: 93 us for
// 2064 rows of 256 heads, 128 wide).
constexpr int CACHE_READ_TURNS = 8;

template <int W>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheView c, uint4 *key, uint4 *value, int chunks)
{
    constexpr int SIDE = W / 8, ROW = 2 * SIDE, TURN = 256 / ROW;
    const long long bh = blockIdx.x / chunks;
    const int d = threadIdx.x % SIDE, side = threadIdx.x / SIDE & 1, first = (int)(blockIdx.x % chunks) * TURN * CACHE_READ_TURNS;
    if (d * 8 >= c.dim) return;
    const int len = rows_used(c, (int)(bh / c.heads));
    const uint8_t *codes = (side ? c.value : c.key) + bh * c.rows * (W / 2) + d * 4;
    const uint8_t *scales = (side ? c.value_scale : c.key_scale) + (bh * (W / 32) + d / 4) * c.rows, *nans = c.key_scale + (bh * (W / 32) + d / 4) * c.rows;
    uint4 *out = (side ? value : key) + bh * c.limit * (c.dim / 8) + d;
#pragma unroll
    for (int turn = 0; turn < CACHE_READ_TURNS; ++turn) {
        const int slot = first + turn * TURN + threadIdx.x / ROW;
        if (slot >= c.limit) continue;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (slot < len) {
            v = __builtin_bit_cast(uint4, cvt8(*(const uint32_t *)(codes + (long long)slot * (W / 2)), scale_of(scales[slot])));
            if (nans[slot] == 255) v = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
        }
        out[(long long)slot * (c.dim / 8)] = v;
    }
}

// ---------------------------------------------------------------------------------------------------------- attention
struct CacheAttendParams {
    CacheView c;
    const char *q;
    long long q_s[3];                        // byte strides: sequence, query head, row
    char *out;
    long long out_s[3];
    const int *counts;                       // real query rows of each sequence, or null: all T
    int T, G, causal;                        // G query heads read one head of the bank
    int R, tiles;                            // R = T G rows per (sequence, head), row = t G + g; tiles of 16 MT or 32 WAVES of them
    int nsplit;                              // pieces that the bank's rows are cut into
    int mixed;                               // tiled form: pieces in another order for each tile
    float c2;                                // scale * log2(e)
    float *part;                             // nsplit > 1: [split][batch heads][R][W] partial sums ...
    float2 *part_ml;                         //             ... and [split][batch heads][R] (maximum, sum), maximum in log2 units
    int chunks;                              // weights: workgroups along the bank's rows of a (sequence, head); each takes every chunks-th stretch
    int rsplit;                              // weights, many query rows: pieces of the query rows ...
    float *part_w;                           //          ... and their sums, [piece][batch heads][rows]
    float2 *norm;                            // [batch heads][R] what turns a score into a probability (weights wanted), or null:
                                             // p = exp2(s c2 - x) y.  (As one number, the log of the denominator, it would
                                             // cost a rounding of 2^-19 of each p where scores are 16 to 32.)
    float *scores;                           // [batch heads][R][rows] scores before the scale (few query rows, weights wanted), or null
};

// How many slots a query row sees: the last n rows of a sequence are the n query rows themselves when `causal`.
__device__ __forceinline__ int visible(int t, int n, int len, int causal)
{
    if (t >= n) return 0;
    const int v = causal ? len - n + t + 1 : len;
    return v < 0 ? 0 : v;
}

__device__ __forceinline__ int real_rows(const int *counts, int b, int T)
{
    int n = counts ? counts[b] : T;
    return n < 0 ? 0 : n > T ? T : n;
}

// 8 values as 1..3 bf16 pieces whose sum is the value: 8 bits of significand each (bf16: exact with one, float16: with two,
// float32: with three; the first is at most the largest bf16, which the largest float32 would round past).  One piece of an infinity or
// NaN is that value itself, those after it are zero.
// Probabilities need no such care: what is left of a NaN is a NaN.
template <int P, bool CARE = true>
__device__ __forceinline__ void split_pieces(const float (&x)[8], cb16x8 (&out)[P])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float v = x[i];
#pragma unroll
        for (int k = 0; k < P; ++k) {
            constexpr float MOST = 0x1.fep127f;      // the largest bf16
            const bool first = CARE && P == 3 && k == 0;          // (an infinity or NaN is left to the second piece)
            const __bf16 h = (__bf16)(first ? __builtin_amdgcn_fmed3f(v, -MOST, MOST) : v);
            out[k][i] = h;
            v = v - (float)h;
            if (CARE && !first && (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) v = 0.f;
        }
    }
}

template <int DT> struct Pieces { static constexpr int N = DT == CACHE_F32 ? 3 : DT == CACHE_F16 ? 2 : 1; };

// NB words of 8 elements / NB bytes of 2 elements at p, as words (one load each).
template <int NB>
__device__ __forceinline__ void load_key(const uint8_t *p, uint32_t (&w)[NB])
{
    if constexpr (NB == 2) {
        const uint2 v = *(const uint2 *)p;
        w[0] = v.x, w[1] = v.y;
    } else {                                 // 4, 8 or 16 words
#pragma unroll
        for (int i = 0; i < NB / 4; ++i) {
            const uint4 v = ((const uint4 *)p)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    }
}

template <int NB> struct ValueWords { static constexpr int N = NB == 8 ? 2 : 1; };
template <int NB>
__device__ __forceinline__ void load_value(const uint8_t *p, uint32_t (&w)[ValueWords<NB>::N])
{
    if constexpr (NB == 2) w[0] = *(const uint16_t *)p;
    else if constexpr (NB == 4) w[0] = *(const uint32_t *)p;
    else {
        const uint2 v = *(const uint2 *)p;
        w[0] = v.x, w[1] = v.y;
    }
}

// One unit of 32 bank rows as a wave's lanes hold it.
template <int NB>
struct Unit {
    uint32_t k[2][NB];                       // rows 16 a + c, dims of group j
    uint32_t ks[2][NB == 8 ? 2 : 1];
    uint32_t v[8][ValueWords<NB>::N];        // rows 16 a + 4 j + r (e = 4 a + r), channels of lane c
    uint32_t vs[2];
};

template <int NB>
struct UnitAt {                              // addresses of one lane within one (sequence, head)
    const uint8_t *k, *ks, *v, *vs;
    long long scale_ld;
    __device__ __forceinline__ UnitAt(const CacheView &c, long long bh, int lane)
    {
        constexpr int W = 32 * NB;
        const int j = lane >> 4, cc = lane & 15;
        k = c.key + bh * c.rows * (W / 2) + (long long)cc * (W / 2) + j * 4 * NB;
        ks = c.key_scale + (bh * NB + j * NB / 4) * c.rows + cc;
        v = c.value + bh * c.rows * (W / 2) + (long long)(4 * j) * (W / 2) + cc * NB;
        vs = c.value_scale + (bh * NB + cc * NB / 16) * c.rows + 4 * j;
        scale_ld = c.rows;
    }
    __device__ __forceinline__ void load_k(long long u0, uint32_t (&kk)[2][NB], uint32_t (&kks)[2][NB == 8 ? 2 : 1]) const
    {
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            load_key<NB>(k + (u0 + 16 * a) * (16 * NB), kk[a]);
            kks[a][0] = ks[u0 + 16 * a];
            if constexpr (NB == 8) kks[a][1] = ks[scale_ld + u0 + 16 * a];
        }
    }
    __device__ __forceinline__ void load(long long u0, Unit<NB> &u) const
    {
        load_k(u0, u.k, u.ks);
        load_v(u0, u);
    }
    __device__ __forceinline__ void load_v(long long u0, Unit<NB> &u) const
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) load_value<NB>(v + (u0 + 16 * (e >> 2) + (e & 3)) * (16 * NB), u.v[e]);
#pragma unroll
        for (int a = 0; a < 2; ++a) u.vs[a] = *(const uint32_t *)(vs + u0 + 16 * a);
    }
};

// 16 bank rows (tile a of a unit) as the A operand of step i.  A row held as NaN carries it in its first element: that is
// enough to make its score NaN for every query row that sees it.
template <int NB>
__device__ __forceinline__ cb16x8 key_operand(const uint32_t (&k)[NB], const uint32_t (&ks)[NB == 8 ? 2 : 1], int i)
{
    const uint32_t byte = ks[NB == 8 ? i / 4 : 0];
    cb16x8 f = cvt8(k[i], scale_of(byte));
    if (i == 0) {
        uint4 v = __builtin_bit_cast(uint4, f);
        v.x = byte == 255 ? 0x7fc07fc0u : v.x;
        f = __builtin_bit_cast(cb16x8, v);
    }
    return f;
}

// Query rows of one tile of 16 as B operands: lane c = row, group j = dims.
template <int DT, int NB, int P>
__device__ __forceinline__ void load_query(const CacheAttendParams &p, int b, int h, int row, int j, bool real, cb16x8 (&q)[NB][P])
{
    const int t = row / p.G, g = row - t * p.G;
    const char *src = p.q + b * p.q_s[0] + (long long)(h * p.G + g) * p.q_s[1] + t * p.q_s[2];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        const int d = j * 8 * NB + i * 8;
        if (real && d < p.c.dim) load8<DT>(src + (long long)d * elem_bytes<DT>(), x);
        split_pieces<P>(x, q[i]);
    }
}

__device__ __forceinline__ float across_j_max(float x)
{
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float across_j_sum(float x)
{
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// A running sum of probabilities with what its roundings lost beside it: added one by one to the sum of a row that one slot dominates,
// thousands of small ones would vanish (attention sums 3e-6 off for a row on 16 k slots).
struct LongSum {
    float sum = 0.f, lost = 0.f;
    __device__ __forceinline__ void add(float x)
    {
        const float t = sum + x;
        lost += fabsf(sum) >= fabsf(x) ? (sum - t) + x : (x - t) + sum;
        sum = t;
    }
    __device__ __forceinline__ void scale(float f) { sum *= f, lost *= f; }
    __device__ __forceinline__ float value() const { return sum + lost; }
};

// Streaming form: a workgroup has MT tiles of 16 query rows of one (sequence, head) and one piece of its bank rows; its four
// waves take every fourth unit of 32 rows each, straight from memory into registers, and are joined at the end.
template <int DT, int NB, int MT>
__global__ __launch_bounds__(256, 2) void cache_attend_kernel(CacheAttendParams p)
{
    constexpr int W = 32 * NB, PQ = Pieces<DT>::N, PP = DT == CACHE_F32 ? 3 : 2, LD = W + 4;
    // Query operands stay in registers where they fit beside the sums of two waves a SIMD, else in shared memory, which the sums of
    // the four waves use after the loop.
    constexpr bool Q_LDS = NB == 8 || MT * NB * (PQ + 2) >= 32;
    constexpr bool TIGHT = MT * NB >= 8;     // conversions stay with their product: moved ahead of it by the scheduler they spill
    constexpr int O_BYTES = 4 * 16 * LD * 4, Q_BYTES = Q_LDS ? MT * NB * PQ * 1024 : 0;
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ alignas(16) char s_both[O_BYTES > Q_BYTES ? O_BYTES : Q_BYTES];
    float (&s_o)[4][16][LD] = *(float (*)[4][16][LD])s_both;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, j = lane >> 4;
    long long id = blockIdx.x;
    const int split = (int)(id % p.nsplit);
    id /= p.nsplit;
    const int tile = (int)(id % p.tiles);
    const long long bh = id / p.tiles;
    const int b = (int)(bh / p.c.heads), h = (int)(bh % p.c.heads);
    const int len = rows_used(p.c, b);
    const int n = real_rows(p.counts, b, p.T);

    cb16x8 q[Q_LDS ? 1 : MT][NB][PQ];
    int lim[MT], most = 0, least = 0x7fffffff;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = (tile * MT + m) * 16 + c;
        const bool in = row < p.R;
        lim[m] = in ? visible(row / p.G, n, len, p.causal) : 0;
        load_query<DT, NB, PQ>(p, b, h, in ? row : 0, j, lim[m] > 0, q[Q_LDS ? 0 : m]);
        if constexpr (Q_LDS) {                                    // every wave has them all: each leaves a quarter
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (i % 4 == wave % 4 || NB < 4) {
#pragma unroll
                    for (int k = 0; k < PQ; ++k) ((uint4 *)s_both)[((m * NB + i) * PQ + k) * 64 + lane] = __builtin_bit_cast(uint4, q[0][i][k]);
                }
        }
        most = max(most, lim[m]);
        least = min(least, lim[m]);
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        most = max(most, __shfl_xor(most, d));
        least = min(least, __shfl_xor(least, d));
    }
    most = __builtin_amdgcn_readfirstlane(most);
    least = __builtin_amdgcn_readfirstlane(least);

    // this piece: whole units of 32 rows of what the tile sees
    const int units = (most + 31) / 32, per = (units + p.nsplit - 1) / p.nsplit;
    const int first = split * per, last = min(units, first + per);

    cf32x4 o[MT][2 * NB];
    float mx[MT], ref[MT];                   // maximum, its share of the exponent
    LongSum sum[MT];                         // of this lane's probabilities
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        mx[m] = -INFINITY;
        ref[m] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) o[m][i] = cf32x4{0, 0, 0, 0};
    }
    if constexpr (Q_LDS) __syncthreads();
    const UnitAt<NB> at(p.c, bh, lane);
    const auto query = [&](int m, int i, int k) __attribute__((always_inline)) {
        if constexpr (Q_LDS) return __builtin_bit_cast(cb16x8, ((const uint4 *)s_both)[((m * NB + i) * PQ + k) * 64 + lane]);
        else return q[m][i][k];
    };
    const auto compute = [&](int u0, Unit<NB> &u, int next) __attribute__((always_inline)) {
        cf32x4 s[MT][2], small[PQ > 1 ? MT : 1][2];               // products of the query's first piece, and of the others
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int m = 0; m < MT; ++m) s[m][a] = small[PQ > 1 ? m : 0][a] = cf32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const cb16x8 kf[2] = {key_operand<NB>(u.k[0], u.ks[0], i), key_operand<NB>(u.k[1], u.ks[1], i)};
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int k = 0; k < PQ; ++k) {
                    const cb16x8 qf = query(m, i, k);
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        cf32x4 &to = k ? small[PQ > 1 ? m : 0][a] : s[m][a];
                        to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[a], qf, to, 0, 0, 0);
                    }
                }
            if constexpr (TIGHT) __builtin_amdgcn_sched_barrier(0);
        }
        if (next < last) at.load_k((long long)next * 32, u.k, u.ks);
        if constexpr (PQ > 1) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int a = 0; a < 2; ++a) s[m][a] += small[m][a];
        }
        cb16x8 pf[MT][PP];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (u0 + 32 > least) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (u0 + 16 * (e >> 2) + 4 * j + (e & 3) >= lim[m]) s[m][e >> 2][e & 3] = -INFINITY;
            }
            if (p.scores && c < p.R) {
#pragma unroll
                for (int a = 0; a < 2; ++a) *(cf32x4 *)(p.scores + (bh * p.R + c) * p.c.rows + u0 + 16 * a + 4 * j) = s[m][a];
            }
            float top = s[m][0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) top = fmaxf(top, s[m][e >> 2][e & 3]);
            if (__any(top > mx[m])) {                     // after the first units the maximum hardly ever moves
                const float now = fmaxf(mx[m], across_j_max(top));
                ref[m] = now == -INFINITY ? 0.f : now * p.c2;
                const float shrink = __builtin_amdgcn_exp2f(fmaf(mx[m], p.c2, -ref[m]));
                mx[m] = now;
                sum[m].scale(shrink);
#pragma unroll
                for (int i = 0; i < 2 * NB; ++i) o[m][i] *= shrink;
            }
            float x[8], part = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(fmaf(s[m][e >> 2][e & 3], p.c2, -ref[m]));
                part += x[e];
            }
            sum[m].add(part);
            split_pieces<PP, false>(x, pf[m]);
        }
#pragma unroll
        for (int i2 = 0; i2 < NB; ++i2) {                 // channels 2 i2, 2 i2 + 1 of each lane
            uint32_t pair[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float sc = scale_of(u.vs[e >> 2], e & 3);
                const uint32_t w = u.v[e][NB == 8 ? i2 / 4 : 0];
                pair[e] = i2 % 4 == 0 ? cvt2<0>(w, sc) : i2 % 4 == 1 ? cvt2<1>(w, sc) : i2 % 4 == 2 ? cvt2<2>(w, sc) : cvt2<3>(w, sc);
            }
            uint4 lo, hi;
            lo.x = __builtin_amdgcn_perm(pair[1], pair[0], 0x05040100u), hi.x = __builtin_amdgcn_perm(pair[1], pair[0], 0x07060302u);
            lo.y = __builtin_amdgcn_perm(pair[3], pair[2], 0x05040100u), hi.y = __builtin_amdgcn_perm(pair[3], pair[2], 0x07060302u);
            lo.z = __builtin_amdgcn_perm(pair[5], pair[4], 0x05040100u), hi.z = __builtin_amdgcn_perm(pair[5], pair[4], 0x07060302u);
            lo.w = __builtin_amdgcn_perm(pair[7], pair[6], 0x05040100u), hi.w = __builtin_amdgcn_perm(pair[7], pair[6], 0x07060302u);
            const cb16x8 ve = __builtin_bit_cast(cb16x8, lo), vo = __builtin_bit_cast(cb16x8, hi);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int k = 0; k < PP; ++k) {
                    o[m][2 * i2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ve, pf[m][k], o[m][2 * i2], 0, 0, 0);
                    o[m][2 * i2 + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo, pf[m][k], o[m][2 * i2 + 1], 0, 0, 0);
                }
            if constexpr (TIGHT) __builtin_amdgcn_sched_barrier(0);
        }
        if (next < last) at.load_v((long long)next * 32, u);
    };
    // DEPTH units are on their way or in hand, and the next one's keys and values follow as soon as their registers are free: a unit
    // is computed about as fast as memory answers.
    constexpr int DEPTH = MT * NB <= 4 ? 3 : NB < 8 && DT == CACHE_BF16 ? 2 : 1;
    Unit<NB> u[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (first + wave + 4 * d < last) at.load((long long)(first + wave + 4 * d) * 32, u[d]);
    for (int un = first + wave; un < last; un += 4 * DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (un + 4 * d >= last) break;
            compute((un + 4 * d) * 32, u[d], un + 4 * (d + DEPTH));
        }
    }

    // join the four waves, one tile of 16 rows at a time (what the loop read of shared memory is read: the barrier below)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const float l = across_j_sum(sum[m].value());
        __syncthreads();
        if (j == 0) {
            s_m[wave][c] = mx[m];
            s_l[wave][c] = l;
        }
        __syncthreads();
        float top = s_m[0][c];
#pragma unroll
        for (int w = 1; w < 4; ++w) top = fmaxf(top, s_m[w][c]);
        const float f = __builtin_amdgcn_exp2f(fmaf(mx[m], p.c2, top == -INFINITY ? 0.f : -(top * p.c2)));
        // channel of o[i][r]: (4 j + r) * 2 NB + i: 2 NB neighbours for each r
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) s_o[wave][c][(4 * j + r) * 2 * NB + i] = o[m][i][r] * f;
        __syncthreads();
        const int row0 = (tile * MT + m) * 16;
        for (int at8 = threadIdx.x; at8 < 16 * (W / 8); at8 += 256) {
            const int rr = at8 / (W / 8), d = at8 % (W / 8) * 8, row = row0 + rr;
            if (row >= p.R) continue;
            float big = s_m[0][rr];
            for (int w = 1; w < 4; ++w) big = fmaxf(big, s_m[w][rr]);
            const float rref = big == -INFINITY ? 0.f : big * p.c2;
            float den = 0.f;
            for (int w = 0; w < 4; ++w) den += s_l[w][rr] * __builtin_amdgcn_exp2f(fmaf(s_m[w][rr], p.c2, -rref));
            float x[8];
            for (int i = 0; i < 8; ++i) x[i] = (s_o[0][rr][d + i] + s_o[1][rr][d + i]) + (s_o[2][rr][d + i] + s_o[3][rr][d + i]);
            if (p.nsplit > 1) {
                const long long g = ((long long)split * p.c.batch * p.c.heads + bh) * p.R + row;
                store8<CACHE_F32>(p.part + g * W + d, x);
                if (d == 0) p.part_ml[g] = make_float2(den == 0.f ? -INFINITY : rref, den);
            } else {
                // a row that sees nothing is zero; one that sees nothing but NaN, or whose scores are all -inf (0 / 0), is NaN
                const int t = row / p.G, g = row - t * p.G;
                const bool none = visible(t, n, len, p.causal) <= 0;
                const float inv = 1.f / den;
                for (int i = 0; i < 8; ++i) x[i] = none ? 0.f : x[i] * inv;
                if (d < p.c.dim) store8<DT>(p.out + b * p.out_s[0] + (long long)(h * p.G + g) * p.out_s[1] + t * p.out_s[2] + (long long)d * elem_bytes<DT>(), x);
                if (p.norm && d == 0) p.norm[bh * p.R + row] = make_float2(rref, none ? 0.f : inv);
            }
        }
    }
}

// Tiled form, for many query rows: each of a workgroup's WAVES waves has 32 of them, and the workgroup walks over the bank in tiles
// of 16 WAVES rows, which its waves turn into bf16 once, in shared memory, in the order in which the matrix cores read them (a
// fragment: 64 lanes x 16 bytes).  v_mfma_f32_32x32x16_bf16 (lane = 32 l + c; A: row c, 8 k-values of half l; result: column c,
// rows 8 (r / 4) + 4 l + r % 4), transposed products as above:
//   key fragment (32 bank rows tt, step i): bank row 32 tt + c, the 8 dims l W/2 + 8 i ...
//   value fragment (16 bank rows s, ct): channel c NB + ct, bank rows 16 s + 4 l + {0..3, 8..11}: the rows of which lane (c, l) of
//   S^T has the probabilities of query row c in registers 8 (s % 2) ...
template <int NB>
struct TileRegs {                            // what a wave turns into fragments: NB of the 2 NB steps of 32 keys, 16 values
    uint32_t k[NB], ks[NB == 8 ? 2 : 1], v[8], vs[2];
};

template <int NB>
struct TileAt {
    const uint8_t *k, *ks, *v, *vs;
    long long scale_ld;
    __device__ __forceinline__ TileAt(const CacheView &c, long long bh, int lane, int wave)
    {
        constexpr int W = 32 * NB;
        const int l = lane >> 5, cc = lane & 31, half = wave & 1, row = 32 * (wave >> 1) + cc;
        k = c.key + (bh * c.rows + row) * (W / 2) + l * (W / 4) + half * 4 * NB;
        ks = c.key_scale + (bh * NB + (l * 2 * NB + half * NB) / 4) * c.rows + row;
        v = c.value + (bh * c.rows + 16 * wave + 4 * l) * (W / 2) + cc * (NB / 2);
        vs = c.value_scale + (bh * NB + cc * NB / 32) * c.rows + 16 * wave + 4 * l;
        scale_ld = c.rows;
    }
    __device__ __forceinline__ void load(long long u0, TileRegs<NB> &t) const
    {
        load_key<NB>(k + u0 * (16 * NB), t.k);
        t.ks[0] = ks[u0];
        if constexpr (NB == 8) t.ks[1] = ks[scale_ld + u0];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint8_t *at = v + (u0 + 8 * (e >> 2) + (e & 3)) * (16 * NB);
            t.v[e] = NB == 2 ? *at : NB == 4 ? *(const uint16_t *)at : *(const uint32_t *)at;
        }
        t.vs[0] = *(const uint32_t *)(vs + u0);
        t.vs[1] = *(const uint32_t *)(vs + u0 + 8);
    }
};

__device__ __forceinline__ uint4 transpose_pairs(const uint32_t (&pair)[8], uint32_t sel)
{
    return make_uint4(__builtin_amdgcn_perm(pair[1], pair[0], sel), __builtin_amdgcn_perm(pair[3], pair[2], sel),
                      __builtin_amdgcn_perm(pair[5], pair[4], sel), __builtin_amdgcn_perm(pair[7], pair[6], sel));
}

template <int NB>
__device__ __forceinline__ void store_tile(const TileRegs<NB> &t, uint4 *keys, uint4 *values, int lane, int wave)
{
    const int half = wave & 1, tt = wave >> 1;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const uint32_t byte = t.ks[NB == 8 ? i / 4 : 0];
        uint4 f = __builtin_bit_cast(uint4, cvt8(t.k[i], scale_of(byte)));
        if (i == 0) f.x = byte == 255 ? 0x7fc07fc0u : f.x;
        keys[(tt * 2 * NB + half * NB + i) * 64 + lane] = f;
    }
    float sc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sc[e] = scale_of(t.vs[e >> 2], e & 3);
#pragma unroll
    for (int i2 = 0; i2 < NB / 2; ++i2) {
        uint32_t pair[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            pair[e] = i2 == 0 ? cvt2<0>(t.v[e], sc[e]) : i2 == 1 ? cvt2<1>(t.v[e], sc[e]) : i2 == 2 ? cvt2<2>(t.v[e], sc[e]) : cvt2<3>(t.v[e], sc[e]);
        values[(wave * NB + 2 * i2) * 64 + lane] = transpose_pairs(pair, 0x05040100u);
        values[(wave * NB + 2 * i2 + 1) * 64 + lane] = transpose_pairs(pair, 0x07060302u);
    }
}

// 32 query rows as B operands: lane c = row, half l = dims l W/2 + 8 i.
template <int DT, int NB, int P>
__device__ __forceinline__ void load_query32(const CacheAttendParams &p, int b, int h, int row, int l, bool real, int i, cb16x8 (&q)[P])
{
    const int t = row / p.G, g = row - t * p.G, d = l * 16 * NB + i * 8;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (real && d < p.c.dim)
        load8<DT>(p.q + b * p.q_s[0] + (long long)(h * p.G + g) * p.q_s[1] + t * p.q_s[2] + (long long)d * elem_bytes<DT>(), x);
    split_pieces<P>(x, q);
}

// How much a score may pass the reference of the exponent (in powers of two) before sums are rescaled: float32 and bf16 have the
// range, and with it the reference hardly ever moves after the first tile.
constexpr float CACHE_SLACK = 16.f;

// Pieces of the probabilities: one for bf16 (2^-8 of each p at most, as much as the result's own rounding may be), as many as the
// query's for the others.  The denominator sums them unrounded: attention sums are divided by it too.
template <int DT, int NB, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 ? 2 : NB == 8 || DT == CACHE_F32 ? 1 : 2) void cache_attend_tile_kernel(CacheAttendParams p)
{
    constexpr int W = 32 * NB, SK = 2 * NB, PQ = Pieces<DT>::N, PP = PQ, ROWS = 32 * WAVES, TOKENS = 16 * WAVES, SUB = TOKENS / 32;
    constexpr int KF = SUB * SK, VF = WAVES * NB;                 // fragments of a tile
    constexpr int RING = 4;                  // operands on their way: read right before its use, one waits for shared memory longer than for the matrix core
    extern __shared__ uint4 s_tile[];        // [2][KF + VF][64]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, l = lane >> 5;
    // Heads innermost (a head's bank stays in one die's cache where heads are a multiple of 8), the longest rows first.  Workgroups
    // go to the eight dies in turn: where pieces differ in length (the first one of causal rows is the longest), their order changes
    // with the tile, by a number whose parity no die has one of; an even number of them would leave half of the dies the long ones.
    const int bhs = p.c.batch * p.c.heads;
    const long long bh = blockIdx.x % bhs;
    const int rest = (int)(blockIdx.x / bhs), turn = rest / p.nsplit, tile = p.tiles - 1 - turn;
    const int split = (rest % p.nsplit + (p.mixed ? __popc(turn) : 0)) % p.nsplit;
    const int b = (int)(bh / p.c.heads), h = (int)(bh % p.c.heads);
    const int len = rows_used(p.c, b);
    const int n = real_rows(p.counts, b, p.T);

    const int row = tile * ROWS + wave * 32 + c;
    const bool real = row < p.R && row / p.G < n;
    const int lim = real ? visible(row / p.G, n, len, p.causal) : 0x7fffffff;      // rows that are not real need no mask: nothing is kept of them
    const unsigned long long seeing = __ballot(real && lim > 0);  // rows that see anything: for the end, in two scalar registers
    // the workgroup's first row sees least of its real ones, the last one most
    const int t_first = tile * ROWS / p.G, t_last = min(min(tile * ROWS + ROWS - 1, p.R - 1) / p.G, n - 1);
    const int least = t_last < t_first ? 0 : visible(t_first, n, len, p.causal), most = t_last < t_first ? 0 : visible(t_last, n, len, p.causal);
    // pieces are as long for every tile (causal: the first tiles have fewer of them)
    const int units = (most + TOKENS - 1) / TOKENS, per = ((len + TOKENS - 1) / TOKENS + p.nsplit - 1) / p.nsplit, first = split * per, last = min(units, first + per);

    cb16x8 q[SK][PQ];
#pragma unroll
    for (int i = 0; i < SK; ++i) load_query32<DT, NB, PQ>(p, b, h, real ? row : 0, l, real, i, q[i]);
    cf32x16 o[NB], s[SUB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    float ref = -INFINITY, top = -INFINITY;                       // reference of the exponent (log2 units), largest score of a tile
    LongSum total;

    if (first < last) {
        const TileAt<NB> at(p.c, bh, lane, wave & 3);
        TileRegs<NB> t;
        // four waves have 64 rows of a tile; where those lie past the allocation (a multiple of 64), its last 64 stand in: they are masked
        const auto load = [&](int un) __attribute__((always_inline)) { at.load(min(min(un, last - 1) * TOKENS + 64 * (wave >> 2), p.c.rows - 64), t); };
        const auto leave = [&](int un) __attribute__((always_inline)) {
            uint4 *to = s_tile + ((un - first) & 1) * (KF + VF) * 64;
            store_tile<NB>(t, to, to + KF * 64, lane, wave);
        };
        // scores of a tile and the largest of them
        const auto product = [&](int un, auto masked) __attribute__((always_inline)) {
            const uint4 *keys = s_tile + ((un - first) & 1) * (KF + VF) * 64;
            cf32x16 small[PQ > 1 ? SUB : 1];                      // products of the query's smaller pieces
#pragma unroll
            for (int tt = 0; tt < SUB; ++tt)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[tt][r] = small[PQ > 1 ? tt : 0][r] = 0.f;
            const auto operand = [&](int f) __attribute__((always_inline)) { return __builtin_bit_cast(cb16x8, keys[(f % SUB * SK + f / SUB) * 64 + lane]); };
            cb16x8 ring[RING];
#pragma unroll
            for (int f = 0; f < RING; ++f) ring[f] = operand(f);
#pragma unroll
            for (int f = 0; f < SUB * SK; ++f) {
                const int i = f / SUB, tt = f % SUB;
#pragma unroll
                for (int k = 0; k < PQ; ++k) {
                    cf32x16 &to = k ? small[PQ > 1 ? tt : 0] : s[tt];
                    to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[f % RING], q[i][k], to, 0, 0, 0);
                }
                if (f + RING < SUB * SK) ring[f % RING] = operand(f + RING);
                if constexpr (NB > 2) __builtin_amdgcn_sched_barrier(0);      // (64 dims: 406 us for 8192 rows in this order, 345 us in the compiler's)
            }
            if constexpr (PQ > 1) {
#pragma unroll
                for (int tt = 0; tt < SUB; ++tt) s[tt] += small[tt];
            }
            if constexpr (decltype(masked)::value) {
                const int left = lim - un * TOKENS - 4 * l;
#pragma unroll
                for (int r = 0; r < 16 * SUB; ++r)
                    if (32 * (r >> 4) + 8 * ((r & 15) >> 2) + (r & 3) >= left) s[r >> 4][r & 15] = -INFINITY;
            }
            top = s[0][0];
#pragma unroll
            for (int r = 1; r < 16 * SUB; ++r) top = fmaxf(top, s[r >> 4][r & 15]);
        };
        const auto moved = [&]() __attribute__((always_inline)) { return __any(fmaf(top, p.c2, -CACHE_SLACK) > ref); };
        const auto rescale = [&]() __attribute__((always_inline)) {
            const float now = fmaxf(ref, fmaxf(top, __shfl_xor(top, 32)) * p.c2);
            const float shrink = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref - now);
            ref = now;
            total.scale(shrink);
#pragma unroll
            for (int i = 0; i < NB; ++i) o[i] *= shrink;
        };
        const auto apply = [&](int un) __attribute__((always_inline)) {
            const uint4 *values = s_tile + ((un - first) & 1) * (KF + VF) * 64 + KF * 64;
            const float off = ref == -INFINITY ? 0.f : -ref;
            float sum = 0.f;
            const auto operand = [&](int f) __attribute__((always_inline)) { return __builtin_bit_cast(cb16x8, values[f * 64 + lane]); };
            cb16x8 ring[RING];
#pragma unroll
            for (int f = 0; f < RING; ++f) ring[f] = operand(f);
#pragma unroll
            for (int sq = 0; sq < 2 * SUB; ++sq) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(fmaf(s[sq >> 1][(sq & 1) * 8 + e], p.c2, off));
                    sum += x[e];
                }
                cb16x8 pf[PP];
                split_pieces<PP, false>(x, pf);
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const int f = sq * NB + i;
#pragma unroll
                    for (int k = 0; k < PP; ++k) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[f % RING], pf[k], o[i], 0, 0, 0);
                    if (f + RING < 2 * SUB * NB) ring[f % RING] = operand(f + RING);
                }
            }
            total.add(sum);
        };
        load(first);
        leave(first);
        load(first + 1);
        __syncthreads();
        // Tiles that every row of the workgroup sees whole, then those on the border.  A step ends with the scores of the next
        // tile, so that rescaling, a rare case, lies outside of the inner loops (inside, it cost 64 register copies a tile).
        const int whole = max(first, min(last, least / TOKENS));
        int un = first;
        if (first < whole) product(un, std::false_type());
        else product(un, std::true_type());
        if (moved()) rescale();
        while (un + 1 < whole) {
            do {
                apply(un);
                ++un;
                leave(un);
                load(un + 1);
                __syncthreads();
                product(un, std::false_type());
            } while (un + 1 < whole && !moved());
            if (moved()) rescale();
        }
        while (un + 1 < last) {
            do {
                apply(un);
                ++un;
                leave(un);
                load(un + 1);
                __syncthreads();
                product(un, std::true_type());
            } while (un + 1 < last && !moved());
            if (moved()) rescale();
        }
        apply(un);
    }
    float sum = total.value();
    sum += __shfl_xor(sum, 32);
    if (row >= p.R) return;
    const bool none = !(seeing >> lane & 1);                      // (a row that sees nothing but NaN, or scores of -inf, is NaN)
    const int tq = row / p.G, g = row - tq * p.G;
    if (p.nsplit > 1) {
        const long long gr = ((long long)split * bhs + bh) * p.R + row;
        float *to = p.part + gr * W;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float x[NB];
#pragma unroll
            for (int i = 0; i < NB; ++i) x[i] = o[i][r];
            store_n<CACHE_F32, NB>(to + (8 * (r >> 2) + 4 * l + (r & 3)) * NB, x);
        }
        if (l == 0) p.part_ml[gr] = make_float2(none || sum == 0.f ? -INFINITY : ref == -INFINITY ? 0.f : ref, sum);
        return;
    }
    const float inv = 1.f / sum;
    char *to = p.out + b * p.out_s[0] + (long long)(h * p.G + g) * p.out_s[1] + tq * p.out_s[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int d = (8 * (r >> 2) + 4 * l + (r & 3)) * NB;
        if (d >= p.c.dim) continue;
        float x[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) x[i] = none ? 0.f : o[i][r] * inv;
        store_n<DT, NB>(to + (long long)d * elem_bytes<DT>(), x);
    }
    if (p.norm && l == 0) p.norm[bh * p.R + row] = make_float2(ref == -INFINITY ? 0.f : ref, none ? 0.f : inv);
}

// Joins the pieces of a row: W / 8 lanes side by side in a piece.  More than 8 pieces: one workgroup a row, 2048 / W pieces at a time
// (a lane group a row took 152 us for 256 pieces of 32 rows, a chain of dependent loads; this 6 us).  Otherwise a lane group a row
// (65536 rows in 2 pieces, 128 wide: 72 us with a workgroup a row).
constexpr int CACHE_MAX_SPLIT = 256, CACHE_FEW_SPLITS = 8;

template <int DT, int W>
__device__ __forceinline__ void store_joined(const CacheAttendParams &p, long long g0, int d, float (&x)[8], float big, float den)
{
    const long long bh = g0 / p.R;
    const int row = (int)(g0 % p.R), b = (int)(bh / p.c.heads), h = (int)(bh % p.c.heads), t = row / p.G, g = row - t * p.G;
    float inv = 1.f / den, off = big;
    if (big == -INFINITY) {                  // no piece has sums: the row sees nothing (zero), or all of its scores are -inf (0 / 0)
        const bool none = visible(t, real_rows(p.counts, b, p.T), rows_used(p.c, b), p.causal) <= 0;
        inv = none ? 0.f : __uint_as_float(0x7fc00000u), off = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= inv;
    if (d < p.c.dim) store8<DT>(p.out + b * p.out_s[0] + (long long)(h * p.G + g) * p.out_s[1] + t * p.out_s[2] + (long long)d * elem_bytes<DT>(), x);
    if (p.norm && d == 0) p.norm[g0] = make_float2(off, inv);
}

template <int DT, int W>
__global__ __launch_bounds__(256) void cache_join_few_kernel(CacheAttendParams p)
{
    const long long all = (long long)p.c.batch * p.c.heads * p.R, g0 = ((long long)blockIdx.x * 256 + threadIdx.x) / (W / 8);
    const int d = threadIdx.x % (W / 8) * 8;
    if (g0 >= all) return;
    float2 ml[CACHE_FEW_SPLITS];
    float big = -INFINITY;
#pragma unroll
    for (int s = 0; s < CACHE_FEW_SPLITS; ++s) {
        ml[s] = s < p.nsplit ? p.part_ml[s * all + g0] : make_float2(-INFINITY, 0.f);
        big = fmaxf(big, ml[s].x);
    }
    float den = 0.f, x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < CACHE_FEW_SPLITS; ++s) {
        if (ml[s].x == -INFINITY) continue;               // a piece that saw nothing has no sums to read
        const float f = __builtin_amdgcn_exp2f(ml[s].x - big);
        den += ml[s].y * f;
        float y[8];
        load8<CACHE_F32>(p.part + (s * all + g0) * W + d, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += y[i] * f;
    }
    store_joined<DT, W>(p, g0, d, x, big, den);
}

template <int DT, int W>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheAttendParams p)
{
    constexpr int LANES = W / 8, GROUPS = 256 / LANES;
    __shared__ float s_f[CACHE_MAX_SPLIT];
    __shared__ float s_x[GROUPS][W];
    const long long all = (long long)p.c.batch * p.c.heads * p.R, g0 = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, d = tid % LANES * 8, group = tid / LANES;
    // every wave finds the maximum and the denominator for itself
    float2 ml[CACHE_MAX_SPLIT / 64];
    float big = -INFINITY;
#pragma unroll
    for (int k = 0; k < CACHE_MAX_SPLIT / 64; ++k) {
        const int s = k * 64 + lane;
        ml[k] = s < p.nsplit ? p.part_ml[s * all + g0] : make_float2(-INFINITY, 0.f);
        big = fmaxf(big, ml[k].x);
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) big = fmaxf(big, __shfl_xor(big, m));
    float den = 0.f;
#pragma unroll
    for (int k = 0; k < CACHE_MAX_SPLIT / 64; ++k) {
        // a piece that saw nothing has no sums to read
        const float f = ml[k].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[k].x - big);
        den += ml[k].y * f;
        if (tid < 64) s_f[k * 64 + lane] = ml[k].x == -INFINITY ? -1.f : f;
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) den += __shfl_xor(den, m);
    __syncthreads();
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int s = group; s < p.nsplit; s += GROUPS) {
        const float f = s_f[s];
        if (f < 0.f) continue;                            // (a NaN goes on)
        float y[8];
        load8<CACHE_F32>(p.part + (s * all + g0) * W + d, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += y[i] * f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s_x[group][d + i] = x[i];
    __syncthreads();
    if (group) return;
    for (int g = 1; g < GROUPS && g < p.nsplit; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += s_x[g][d + i];
    store_joined<DT, W>(p, g0, d, x, big, den);
}

// Attention sums: weight[slot] += sum over the query rows of their probabilities.  A wave has one unit of 32 bank rows and goes over
// all rows that may see it, so that every sum has one owner and one order.
template <int DT, int NB>
__global__ __launch_bounds__(256) void cache_weigh_kernel(CacheAttendParams p)
{
    constexpr int PQ = Pieces<DT>::N;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, j = lane >> 4;
    const long long bh = blockIdx.x / p.chunks;
    const int b = (int)(bh / p.c.heads), h = (int)(bh % p.c.heads);
    const int len = rows_used(p.c, b);
    const int n = real_rows(p.counts, b, p.T);
    const UnitAt<NB> at(p.c, bh, lane);
    for (int u0 = (int)(blockIdx.x % p.chunks) * 128 + wave * 32; u0 < len; u0 += p.chunks * 128) {
        uint32_t kk[2][NB], ks[2][NB == 8 ? 2 : 1];
        at.load_k(u0, kk, ks);
        float w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        // rows before the first that sees slot u0 are left out
        const int t0 = p.causal ? max(0, u0 - (len - n)) : 0;
        for (int row0 = (int)((long long)t0 * p.G / 16 * 16); row0 < n * p.G; row0 += 16) {
            const int row = row0 + c;
            const bool in = row < p.R;
            const int lim = in ? visible(row / p.G, n, len, p.causal) : 0;
            cb16x8 q[NB][PQ];
            load_query<DT, NB, PQ>(p, b, h, in ? row : 0, j, lim > 0, q);
            const float2 norm = lim > 0 ? p.norm[bh * p.R + row] : make_float2(0.f, 0.f);
            cf32x4 s[2] = {cf32x4{0, 0, 0, 0}, cf32x4{0, 0, 0, 0}}, small[2] = {cf32x4{0, 0, 0, 0}, cf32x4{0, 0, 0, 0}};
#pragma unroll
            for (int a = 0; a < 2; ++a) {
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const cb16x8 kf = key_operand<NB>(kk[a], ks[a], i);
#pragma unroll
                    for (int k = 0; k < PQ; ++k) {
                        cf32x4 &to = k ? small[a] : s[a];
                        to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[i][k], to, 0, 0, 0);
                    }
                }
                if constexpr (PQ > 1) s[a] += small[a];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], p.c2, -norm.x)) * norm.y;
                w[e] += u0 + 16 * (e >> 2) + 4 * j + (e & 3) < lim ? x : 0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) w[e] += __shfl_xor(w[e], d);
            const int slot = u0 + 16 * (e >> 2) + 4 * j + (e & 3);
            if (c == e && slot < len) p.c.weight[bh * p.c.rows + slot] += w[e];
        }
    }
}

// The same for many query rows: each of a workgroup's eight waves keeps 32 bank rows as operands, and all go over the query rows in
// tiles of 64 that they share through shared memory.  The scores of a tile are computed while the exponentials of the one before
// are: what bounds it is three vector instructions a score beside 8 / 32 of a matrix one.  Where bank rows are few, the query rows
// are cut into `rsplit` pieces, whose sums are added up after.  (1000 rows of 16 heads on 16 000: 255 us with 64 bank rows a wave,
// 207 us with tiles of 32 and four waves a SIMD, in both each wave's products and exponentials in turn.)
template <int DT, int NB>
__global__ __launch_bounds__(512, 2) void cache_weigh_tile_kernel(CacheAttendParams p)
{
    constexpr int W = 32 * NB, SK = 2 * NB, PQ = Pieces<DT>::N, RT = 2 * SK * PQ > 64 ? 1 : 2, QROWS = 32 * RT;
    constexpr int MINE = RT * SK / 8;                             // fragments of a query tile (RT SK) that a wave loads
    static_assert(MINE * 8 == RT * SK && (RT == 1 || SK == 4 * MINE), "eight waves, each with steps of one 32 rows");
    __shared__ uint4 s_q[2][RT * SK * PQ][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, l = lane >> 5;
    const int bhs = p.c.batch * p.c.heads;
    const long long bh = blockIdx.x % bhs;
    const int rest = (int)(blockIdx.x / bhs), piece = rest % p.rsplit, chunk = rest / p.rsplit;
    const int b = (int)(bh / p.c.heads), h = (int)(bh % p.c.heads);
    const int len = rows_used(p.c, b);
    const int n = real_rows(p.counts, b, p.T);
    const int tiles = (int)(((long long)n * p.G + QROWS - 1) / QROWS), per = (tiles + p.rsplit - 1) / p.rsplit;
    // A wave loads fragments of one 32 rows of a tile (its row c), steps `step` on; dims that pad a row read its first ones, which
    // meet zeros of the bank.
    const int mine32 = RT == 2 ? wave >> 2 : 0, step = wave * MINE % SK, real_rows_all = n * p.G;
    const char *const query = p.q + b * p.q_s[0] + (long long)h * p.G * p.q_s[1];
    const int dt = QROWS / p.G, dg = QROWS - dt * p.G;            // from a tile's row to the next one's, without a division
    const long long ahead = dt * p.q_s[2] + dg * p.q_s[1], wrap = p.q_s[2] - p.G * p.q_s[1];
    const char *const final = query + (long long)max(n - 1, 0) * p.q_s[2] + (p.G - 1) * p.q_s[1];
    int at_dim[MINE];
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
        const int d = l * 16 * NB + (step + m) * 8;
        at_dim[m] = d < p.c.dim ? d * elem_bytes<DT>() : 0;
    }
    const float2 *const norms = p.norm + bh * p.R;
    for (int w0 = chunk * 256; w0 < len; w0 += p.chunks * 256) {
        const int u0 = w0 + wave * 32;
        cb16x8 kf[SK];
        {
            const long long at = min(u0 + c, p.c.rows - 1);       // rows past the allocation: any row, left out below
            uint32_t w[SK];
            load_key<SK>(p.c.key + (bh * p.c.rows + at) * (W / 2) + l * (W / 4), w);
#pragma unroll
            for (int i = 0; i < SK; ++i) {
                const uint32_t byte = p.c.key_scale[(bh * NB + (l * SK + i) / 4) * p.c.rows + at];
                uint4 f = __builtin_bit_cast(uint4, cvt8(w[i], scale_of(byte)));
                if (i == 0) f.x = byte == 255 ? 0x7fc07fc0u : f.x;
                kf[i] = __builtin_bit_cast(cb16x8, f);
            }
        }
        float w[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) w[r] = 0.f;
        // tiles before the first row that sees slot w0 are left out; those before the first that sees all slots of the workgroup
        // are masked (rows that are not real count zero times)
        const int t_lo = p.causal ? max(0, w0 - (len - n)) : 0, t_all = p.causal ? max(0, w0 + 255 - (len - n)) : 0;
        const int first = max(piece * per, (int)min((long long)tiles, (long long)t_lo * p.G / QROWS)), last = min(tiles, (piece + 1) * per);
        const int border = max(first, (int)min((long long)last, ((long long)t_all * p.G + QROWS - 1) / QROWS));
        if (first < last) {
            int next = first * QROWS;                             // the tile that is loaded next, by its first row
            int g = (next + 32 * mine32 + c) % p.G;
            const char *row = query + (long long)((next + 32 * mine32 + c) / p.G) * p.q_s[2] + g * p.q_s[1];
            uint4 mine[MINE * PQ];
            float2 norm[3][RT];                                   // of the tile in hand, the next, the one loaded
            // Rows past the last real one repeat it and count zero times.
            const auto fetch = [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int a = 0; a < RT; ++a) {
                    const int r = next + 32 * a + c;
                    norm[2][a] = norms[min(r, real_rows_all - 1)];
                    norm[2][a].x = -norm[2][a].x;
                    norm[2][a].y = r < real_rows_all ? norm[2][a].y : 0.f;
                }
                const char *from = next + 32 * mine32 + c < real_rows_all ? row : final;
#pragma unroll
                for (int m = 0; m < MINE; ++m) {
                    if constexpr (DT == CACHE_BF16) {
                        const uint4 x = *(const uint4 *)(from + at_dim[m]);
                        mine[m] = make_uint4(x.x, x.y, x.z, x.w);             // (copied whole, the array went to memory)
                    } else {
                        float x[8];
                        load8<DT>(from + at_dim[m], x);
                        cb16x8 q[PQ];
                        split_pieces<PQ>(x, q);
#pragma unroll
                        for (int k = 0; k < PQ; ++k) mine[m * PQ + k] = __builtin_bit_cast(uint4, q[k]);
                    }
                }
                next += QROWS;
                g += dg;
                row += ahead;
                if (g >= p.G) g -= p.G, row += wrap;
            };
            const auto leave = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
                for (int m = 0; m < MINE * PQ; ++m) s_q[(tile - first) & 1][wave * MINE * PQ + m][lane] = mine[m];
#pragma unroll
                for (int a = 0; a < RT; ++a) norm[0][a] = norm[1][a], norm[1][a] = norm[2][a];
            };
            // Scores of tile `tile + 1` (past the last one: of whatever is there, never used) into `ahead`, beside the exponentials of
            // tile `tile`, whose scores are in `s` (NOW false: without them).  The order is fixed: a matrix instruction, the operand four
            // further on, and the vector instructions that fit beside; left alone, the compiler reads each operand right before its use
            // and puts all of one kind before all of the other, and a wave issues in order.  The smaller pieces of the query come first.
            constexpr int FRAGS = RT * SK * PQ, RING = 4;
            const auto both = [&](int tile, cf32x16 (&s)[RT], cf32x16 (&ahead)[RT], auto now, auto masked) __attribute__((always_inline)) {
                const uint4 (*const from)[64] = s_q[(tile + 1 - first) & 1];
                const auto operand = [&](int f) __attribute__((always_inline)) {      // f: piece (descending), step, 32 rows
                    const int k = PQ - 1 - f / (RT * SK), i = f / RT % SK, a = f % RT;
                    return __builtin_bit_cast(cb16x8, from[(a * SK + i) * PQ + k][lane]);
                };
                cb16x8 ring[RING];
#pragma unroll
                for (int f = 0; f < RING; ++f) ring[f] = operand(f);
                int left[RT];                                     // slots from this lane's first that its row of the tile sees
#pragma unroll
                for (int a = 0; a < RT; ++a) {
                    left[a] = 0;
                    if constexpr (decltype(masked)::value) left[a] = visible((tile * QROWS + 32 * a + c) / p.G, n, len, p.causal) - u0 - 4 * l;
#pragma unroll
                    for (int r = 0; r < 16; ++r) ahead[a][r] = 0.f;
                }
#pragma unroll
                for (int f = 0; f < FRAGS; ++f) {
                    ahead[f % RT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[f / RT % SK], ring[f % RING], ahead[f % RT], 0, 0, 0);
                    if (f + RING < FRAGS) ring[f % RING] = operand(f + RING);
                    if constexpr (decltype(now)::value) {
#pragma unroll
                        for (int e = f * 16 * RT / FRAGS; e < (f + 1) * 16 * RT / FRAGS; ++e) {
                            const int a = e / 16, r = e % 16;
                            const float x = __builtin_amdgcn_exp2f(fmaf(s[a][r], p.c2, norm[0][a].x)), more = fmaf(x, norm[0][a].y, w[r]);
                            if constexpr (decltype(masked)::value) w[r] = 8 * (r >> 2) + (r & 3) < left[a] ? more : w[r];
                            else w[r] = more;
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            const auto step = [&](int tile, cf32x16 (&s)[RT], cf32x16 (&ahead)[RT], auto masked) __attribute__((always_inline)) {
                both(tile, s, ahead, std::true_type(), masked);
                leave(tile);                                      // tile + 2, into the buffer that this tile had
                fetch();
                __syncthreads();
            };
            cf32x16 s0[RT], s1[RT];
            int tile = first;
            const auto run = [&](int end, auto masked) __attribute__((always_inline)) {
                for (; tile + 1 < end; tile += 2) {
                    step(tile, s0, s1, masked);
                    step(tile + 1, s1, s0, masked);
                }
                if (tile < end) {
                    step(tile, s0, s1, masked);
                    ++tile;
#pragma unroll
                    for (int a = 0; a < RT; ++a) s0[a] = s1[a];
                }
            };
            __syncthreads();
            fetch();
            leave(first);
            fetch();
            leave(first + 1);
            fetch();
            __syncthreads();
            both(first - 1, s1, s0, std::false_type(), std::false_type());
            __syncthreads();                                      // the first step writes where this one read
            run(border, std::true_type());
            run(last, std::false_type());
        }
        float *to = p.rsplit > 1 ? p.part_w + ((long long)piece * bhs + bh) * p.c.rows : p.c.weight + bh * p.c.rows;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) w[r] += __shfl_xor(w[r], d);
            const int slot = u0 + 8 * (r >> 2) + 4 * l + (r & 3);
            if (c == r && slot < len) {
                if (p.rsplit > 1) to[slot] = w[r];
                else to[slot] += w[r];
            }
        }
    }
}

__global__ __launch_bounds__(256) void cache_weigh_add_kernel(CacheAttendParams p)
{
    const int bhs = p.c.batch * p.c.heads;
    const long long bh = blockIdx.x % bhs;
    const int len = rows_used(p.c, (int)(bh / p.c.heads));
    const int step = (int)(gridDim.x / bhs) * 256;
    for (int slot = (int)(blockIdx.x / bhs) * 256 + threadIdx.x; slot < len; slot += step) {
        float w = p.c.weight[bh * p.c.rows + slot];
        for (int s = 0; s < p.rsplit; ++s) w += p.part_w[((long long)s * bhs + bh) * p.c.rows + slot];
        p.c.weight[bh * p.c.rows + slot] = w;
    }
}

// The same where the attention kernel left its scores behind: four slots a thread, R scores each.
__global__ __launch_bounds__(256) void cache_weigh_scores_kernel(CacheAttendParams p)
{
    const long long bh = blockIdx.x / p.chunks;
    const int b = (int)(bh / p.c.heads);
    const int len = rows_used(p.c, b);
    const int n = real_rows(p.counts, b, p.T);
    for (int slot = ((int)(blockIdx.x % p.chunks) * 256 + threadIdx.x) * 4; slot < len; slot += p.chunks * 1024) {
        float w[4] = {0, 0, 0, 0};
        for (int row = 0; row < p.R; ++row) {
            const int lim = visible(row / p.G, n, len, p.causal);
            if (lim <= slot) continue;                    // (scores of a unit that no row of the tile sees were never written)
            const float2 norm = p.norm[bh * p.R + row];
            const cf32x4 s = *(const cf32x4 *)(p.scores + (bh * p.R + row) * p.c.rows + slot);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[e], p.c2, -norm.x)) * norm.y;
                w[e] += slot + e < lim ? x : 0.f;
            }
        }
        float *to = p.c.weight + bh * p.c.rows + slot;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (slot + e < len) to[e] += w[e];
    }
}

// ------------------------------------------------------------------------------------------------------------ eviction
struct EvictParams {
    CacheView c, into;
    int keep, recent, in_place;
    int *count;                              // [batch heads] rows to copy
    int2 *pairs;                             // [batch heads][keep] (destination slot, source slot)
};

// Order of the rows: recent ones first, then by weight (NaN above +inf, -0 = +0), ties to the lower slot.
__device__ __forceinline__ uint32_t evict_rank(float w, int position, int from)
{
    if (position >= from) return 0xffffffffu;
    if (w != w) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

constexpr int EVICT_THREADS = 1024, EVICT_BINS = 2048;
constexpr int EVICT_LIST = 2048;             // rows of one bin of the first digit that are gathered for the other two
constexpr int EVICT_RESIDENT = 32768;        // ranks of so many rows fit the shared memory beside the histogram and that list

struct EvictShared {
    int hist[EVICT_BINS];
    uint32_t list[EVICT_LIST];
    int2 wave[EVICT_THREADS / 64];
    int pick[3], listed;
};

// Exclusive prefix sums of two numbers over the waves of the workgroup (one value a wave, from any lane of it).
__device__ __forceinline__ int2 wave_scan2(int2 v, EvictShared &sh, int2 &all)
{
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave[wave] = v;
    __syncthreads();
    int2 before = make_int2(0, 0);
    all = make_int2(0, 0);
#pragma unroll
    for (int i = 0; i < EVICT_THREADS / 64; ++i) {
        if (i < wave) before.x += sh.wave[i].x, before.y += sh.wave[i].y;
        all.x += sh.wave[i].x, all.y += sh.wave[i].y;
    }
    return before;
}

__device__ __forceinline__ int wave_sum(int x)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
    return x;
}

// One digit of a lane's rank into the histogram.  Equal neighbours (rows that nothing attended to yet) are counted once for the wave,
// not 64 times in turn.
__device__ __forceinline__ void count_digit(EvictShared &sh, bool in, int digit)
{
    const unsigned long long who = __ballot(in);
    if (!who) return;
    const int first = __builtin_amdgcn_readlane(digit, __ffsll((long long)who) - 1);
    const unsigned long long same = __ballot(in && digit == first);
    if ((threadIdx.x & 63) == 0) atomicAdd(&sh.hist[first], __popcll(same));
    if (in && digit != first) atomicAdd(&sh.hist[digit], 1);
}

__device__ __forceinline__ void clear_digits(EvictShared &sh)
{
    for (int i = threadIdx.x; i < EVICT_BINS; i += EVICT_THREADS) sh.hist[i] = 0;
    __syncthreads();
}

// The bin that holds the left-th largest (bins from the top, two a thread): its digit, how many of it stay, how many it has.
__device__ __forceinline__ void pick_digit(EvictShared &sh, int left)
{
    __syncthreads();
    const int lane = threadIdx.x & 63, top = EVICT_BINS - 1 - 2 * threadIdx.x, a = sh.hist[top], b = sh.hist[top - 1];
    int sum = a + b;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(sum, d);
        if (lane >= d) sum += v;
    }
    int2 all;
    const int above = wave_scan2(make_int2(__builtin_amdgcn_readlane(sum, 63), 0), sh, all).x + sum - a - b;
    if (above < left && above + a + b >= left) {
        const bool second = above + a < left;
        sh.pick[0] = second ? top - 1 : top;
        sh.pick[1] = left - above - (second ? a : 0);
        sh.pick[2] = second ? b : a;
    }
    __syncthreads();
}

// Calls f(row, its rank) for all rows of a stretch, 64 neighbours a wave at a time, four ranks on their way; rows past the end have
// rank 0 and are told by their number.
template <int STEP, typename Rank, typename F>
__device__ __forceinline__ void for_ranks(int lo, int hi, Rank rank, F f)
{
    const int lane = threadIdx.x & 63;
    for (int i0 = lo; i0 < hi; i0 += 4 * STEP) {
        uint32_t r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = i0 + k * STEP + lane < hi ? rank(i0 + k * STEP + lane) : 0u;
#pragma unroll
        for (int k = 0; k < 4; ++k) f(i0 + k * STEP + lane, r[k]);
    }
}

// The rank that the keep-th row has, by digits of 11, 11 and 10 bits (the first one may be counted already), then the lists of what has
// to be copied: wave w goes over the w-th sixteenth of the slots and counts with ballots.
template <typename Rank>
__device__ __forceinline__ void select_rows(const EvictParams &p, long long bh, int n, Rank rank, EvictShared &sh, bool counted)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, keep = p.keep;
    int2 *pairs = p.pairs + bh * keep;
    if (!counted) {
        clear_digits(sh);
        for_ranks<EVICT_THREADS>(wave * 64, n, rank, [&](int i, uint32_t r) { count_digit(sh, i < n, (int)(r >> 21)); });
    }
    pick_digit(sh, keep);
    uint32_t prefix = (uint32_t)sh.pick[0] << 21;
    int left = sh.pick[1];
    const int listed = sh.pick[2];
    const bool gather = listed <= EVICT_LIST;
    if (tid == 0) sh.listed = 0;
    clear_digits(sh);
    if (gather) {                            // the rows of that bin, in any order: the other digits look at them alone
        for_ranks<EVICT_THREADS>(wave * 64, n, rank, [&](int i, uint32_t r) {
            const bool in = i < n && (r & 0xffe00000u) == prefix;
            const unsigned long long who = __ballot(in);
            if (!who) return;
            int at = 0;
            if (lane == 0) at = atomicAdd(&sh.listed, __popcll(who));
            at = __builtin_amdgcn_readfirstlane(at) + __popcll(who & ((1ull << lane) - 1));
            if (in) sh.list[at] = r;
        });
        __syncthreads();
    }
#pragma unroll
    for (int pass = 1; pass < 3; ++pass) {
        const int shift = pass == 1 ? 10 : 0;
        const uint32_t mask = pass == 1 ? 2047u : 1023u, known = pass == 1 ? 0xffe00000u : 0xfffffc00u;
        if (pass == 2) clear_digits(sh);
        const auto count = [&](int i, int end, uint32_t r) { count_digit(sh, i < end && (r & known) == prefix, (int)((r >> shift) & mask)); };
        if (gather) for_ranks<EVICT_THREADS>(wave * 64, listed, [&](int i) { return sh.list[i]; }, [&](int i, uint32_t r) { count(i, listed, r); });
        else for_ranks<EVICT_THREADS>(wave * 64, n, rank, [&](int i, uint32_t r) { count(i, n, r); });
        pick_digit(sh, left);
        prefix |= (uint32_t)sh.pick[0] << shift;
        left = sh.pick[1];
    }
    // rows above the edge stay, and of those on it the `left` lowest slots: in the usual case all of them
    const uint32_t edge = prefix;
    const bool all_ties = sh.pick[2] == left;
    const int seg = ((n + EVICT_THREADS - 1) / EVICT_THREADS) * 64, lo = min(n, wave * seg), hi = min(n, lo + seg);
    const unsigned long long below = (1ull << lane) - 1;
    int2 all;
    int eq0 = 0;
    if (!all_ties) {
        int eq = 0;
        for_ranks<64>(lo, hi, rank, [&](int i, uint32_t r) { eq += i < hi && r == edge; });
        eq0 = wave_scan2(make_int2(wave_sum(eq), 0), sh, all).x;
    }
    int at = eq0;                            // rows on the edge before this wave's next 64
    const auto kept_at = [&](int i, uint32_t r) {
        if (all_ties) return i < hi && r >= edge;
        const unsigned long long on = __ballot(i < hi && r == edge);
        const bool kept = i < hi && (r > edge || (r == edge && at + __popcll(on & below) < left));
        at += __popcll(on);
        return kept;
    };
    int holes = 0, tails = 0;                // freed slots below keep, kept rows from there on
    for_ranks<64>(lo, hi, rank, [&](int i, uint32_t r) {
        const bool kept = kept_at(i, r);
        holes += i < hi && i < keep && !kept;
        tails += i >= keep && kept;
    });
    const int2 off = wave_scan2(make_int2(wave_sum(holes), wave_sum(tails)), sh, all);
    const int base = p.in_place ? 0 : keep - all.x;               // pairs before those of the freed slots: rows that stay where they are
    if (tid == 0) p.count[bh] = p.in_place ? all.x : keep;
    at = eq0, holes = off.x, tails = off.y;
    for_ranks<64>(lo, hi, rank, [&](int i, uint32_t r) {
        const bool kept = kept_at(i, r);
        const int i0 = __builtin_amdgcn_readfirstlane(i);
        if (i0 < keep) {
            const unsigned long long h = __ballot(i < hi && i < keep && !kept);
            const int nh = holes + __popcll(h & below);
            if (h >> lane & 1) pairs[base + nh].x = i;
            else if (base && i < keep && kept) pairs[i - nh] = make_int2(i, i);
            holes += __popcll(h);
        }
        if (i0 + 63 >= keep) {
            const unsigned long long t = __ballot(i >= keep && kept);
            if (t >> lane & 1) pairs[base + tails + __popcll(t & below)].y = i;
            tails += __popcll(t);
        }
    });
}

// One workgroup per (sequence, head).  The freed slots below `keep` take, in ascending order, the kept rows from above: in place
// no row is read that another one is written to, and no more rows move than left.  Ranks are built in one pass over weights and
// positions, all of its loads at once, and stay in shared memory where they fit; `resident` of them do.  (32 banks of 24 k rows: 203 us
// with a pass over memory for each of four digits and a thread a stretch of slots, 38 us with ranks in shared memory and loads one
// after the other.)
__global__ __launch_bounds__(EVICT_THREADS) void cache_select_kernel(EvictParams p, int resident)
{
    extern __shared__ uint32_t s_rank[];
    __shared__ EvictShared sh;
    const long long bh = blockIdx.x;
    const int b = (int)(bh / p.c.heads), tid = threadIdx.x;
    const int n = rows_used(p.c, b);
    if (n <= p.keep) {
        if (!p.in_place)
            for (int i = tid; i < n; i += EVICT_THREADS) p.pairs[bh * p.keep + i] = make_int2(i, i);
        if (tid == 0) p.count[bh] = p.in_place ? 0 : n;
        return;
    }
    const int from = p.c.seen[b] - p.recent;
    const float *w = p.c.weight + bh * p.c.rows;
    const int *pos = p.c.position + bh * p.c.rows;
    if (n <= resident) {
        constexpr int LOADS = EVICT_RESIDENT / (EVICT_THREADS * 4);
        float4 x[LOADS];
        int4 y[LOADS];
#pragma unroll
        for (int k = 0; k < LOADS; ++k) {                         // rows are allocated in 64s: whole vectors
            const int i = (tid + k * EVICT_THREADS) * 4;
            x[k] = i < n ? *(const float4 *)(w + i) : make_float4(0, 0, 0, 0);
            y[k] = i < n ? *(const int4 *)(pos + i) : make_int4(0, 0, 0, 0);
        }
        clear_digits(sh);
#pragma unroll
        for (int k = 0; k < LOADS; ++k) {
            const int i = (tid + k * EVICT_THREADS) * 4;
            if (__builtin_amdgcn_readfirstlane(i) >= n) break;
            const uint4 r = make_uint4(evict_rank(x[k].x, y[k].x, from), evict_rank(x[k].y, y[k].y, from), evict_rank(x[k].z, y[k].z, from), evict_rank(x[k].w, y[k].w, from));
            if (i < n) *(uint4 *)(s_rank + i) = r;
            count_digit(sh, i < n, (int)(r.x >> 21));
            count_digit(sh, i + 1 < n, (int)(r.y >> 21));
            count_digit(sh, i + 2 < n, (int)(r.z >> 21));
            count_digit(sh, i + 3 < n, (int)(r.w >> 21));
        }
        select_rows(p, bh, n, [&](int i) { return s_rank[i]; }, sh, true);
    } else
        select_rows(p, bh, n, [&](int i) { return evict_rank(w[i], pos[i], from); }, sh, false);
}

// Copies the rows of the lists.  W / 8 lanes a row: a quarter of them for each of key, value, their scales; 16 bytes a lane.
template <int W>
__global__ __launch_bounds__(256) void cache_move_kernel(EvictParams p, int chunks)
{
    constexpr int ROW = W / 8, Q = ROW / 4;
    const long long bh = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x % chunks), b = (int)(bh / p.c.heads);
    const int count = p.count[bh];
    const int lane = threadIdx.x % ROW, part = lane / Q, c = lane % Q;
    for (int i = chunk * (256 / ROW) + threadIdx.x / ROW; i < count; i += chunks * (256 / ROW)) {
        const int2 pr = p.pairs[bh * p.keep + i];
        const long long src = bh * p.c.rows + pr.y, dst = bh * p.into.rows + pr.x;
        if (part == 0) ((uint4 *)(p.into.key + dst * (W / 2)))[c] = ((const uint4 *)(p.c.key + src * (W / 2)))[c];
        else if (part == 1) ((uint4 *)(p.into.value + dst * (W / 2)))[c] = ((const uint4 *)(p.c.value + src * (W / 2)))[c];
        else {
            const uint8_t *from = part == 2 ? p.c.key_scale : p.c.value_scale;
            uint8_t *to = part == 2 ? p.into.key_scale : p.into.value_scale;
            to[(bh * (W / 32) + c) * p.into.rows + pr.x] = from[(bh * (W / 32) + c) * p.c.rows + pr.y];
            if (c == 0) {
                if (part == 2) p.into.weight[dst] = p.c.weight[src];
                else p.into.position[dst] = p.c.position[src];
            }
        }
    }
    if (chunk == 0 && threadIdx.x == 0 && bh % p.c.heads == 0) {
        const int n = rows_used(p.c, b);
        p.into.length[b] = n < p.keep ? n : p.keep;
        if (!p.in_place) p.into.seen[b] = p.c.seen[b];
    }
}

}  // namespace mi
#endif
