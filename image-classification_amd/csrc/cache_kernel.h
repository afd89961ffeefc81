// cache_kernel.h -- a bank of key / value rows held in 4 bits: quantising append, softmax attention, eviction.
//
// Held format (OCP microscaling FP4).  A row of `dim` values is padded with zeros to W = 64 NB / 2 ... in {64, 128, 256} and
// cut into blocks of 32.  A block has one scale 2^e, e the smallest integer with max|x| <= 7 * 2^e (7 = the half step above
// the largest element 6, so that the largest value of a block is never further off than half a step of its binade), clamped
// to [-126, 125] and stored as the byte e + 127.  Elements are x / 2^e on E2M1 (0 .5 1 1.5 2 3 4 6, sign bit), nearest even,
// saturating; two a byte, the even one in the low four bits.  Every element times its scale is exact in bf16, which is what
// the matrix cores read: v_cvt_scalef32_pk_bf16_fp4 turns two elements and their scale into two bf16 in one instruction.
// A row (of one head) whose key or value has a NaN or an infinity is held as NaN whole: scale bytes 255, elements 0.
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

namespace mi {

typedef __attribute__((ext_vector_type(8))) __bf16 cb16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 cb16x2;
typedef __attribute__((ext_vector_type(4))) float cf32x4;

enum { CACHE_F32 = 0, CACHE_BF16 = 1, CACHE_F16 = 2 };

constexpr float CACHE_LOG2E = 1.4426950408889634f;

struct CacheView {
    uint8_t *key, *key_scale, *value, *value_scale;
    float *weight;
    int *position, *length, *seen;
    int batch, heads, dim, rows, limit;      // rows: allocated (multiple of 64); limit: most rows that are used
};

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
template <int DT, int W>
__global__ __launch_bounds__(256) void cache_push_kernel(PushParams p)
{
    constexpr int SIDE = W / 8, ROW = 2 * SIDE;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long r = at / ROW;
    const int c = (int)(at % SIDE), side = (int)(at / SIDE) & 1;
    const long long all = (long long)p.c.batch * p.c.heads * p.T;
    const bool in = r < all;
    const long long rr = in ? r : 0;
    const int t = (int)(rr % p.T), h = (int)(rr / p.T % p.c.heads), b = (int)(rr / p.T / p.c.heads);
    const int len = p.c.length[b], n = push_count(p, b, len);
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
    const int lane = threadIdx.x & 63;
    const unsigned long long who = __ballot(bad);
    const unsigned long long mine = ROW == 64 ? ~0ull : ((1ull << (ROW & 63)) - 1) << (lane / ROW * ROW);
    const bool poison = (who & mine) != 0;
    const int byte = scale_byte(top);
    uint32_t code = 0;
    if (!poison) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = ldexpf(x[i], 127 - byte);            // a power of two: exact
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
            (side ? p.c.value_scale : p.c.key_scale)[(bh * (W / 32) + c / 4) * p.c.rows + slot] = (uint8_t)(poison ? 255 : byte);
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
            v[i] = poison ? __uint_as_float(0x7fc00000u) : !real ? 0.f : four > 7 ? -a : a;
        }
        store8<DT>(held + (r * p.c.dim + c * 8) * elem_bytes<DT>(), v);
    }
}

// After the rows are written: every sequence is longer by what it got.
__global__ void cache_advance_kernel(PushParams p)
{
    const int b = blockIdx.x * 64 + threadIdx.x;
    if (b >= p.c.batch) return;
    const int n = push_count(p, b, p.c.length[b]);
    p.c.length[b] += n;
    p.c.seen[b] += n;
}

// Every sequence is cut to at most its entry of `lengths` (or `length`); positions go on from where the cut left them.
__global__ void cache_trim_kernel(CacheView c, const int *lengths, int length)
{
    const int b = blockIdx.x * 64 + threadIdx.x;
    if (b >= c.batch) return;
    int n = lengths ? lengths[b] : length;
    n = n < 0 ? 0 : n;
    const int gone = c.length[b] - n;
    if (gone > 0) {
        c.length[b] = n;
        c.seen[b] -= gone;
    }
}

// ---------------------------------------------------------------------------------------------------------- read back
// Rows [0, limit) of every sequence and head as bf16 (exact); rows behind the last one are zeros.  A lane takes 8 dims.
template <int W>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheView c, uint4 *key, uint4 *value)
{
    constexpr int SIDE = W / 8, ROW = 2 * SIDE;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long r = at / ROW;
    const int d = (int)(at % SIDE), side = (int)(at / SIDE) & 1;
    if (r >= (long long)c.batch * c.heads * c.limit || d * 8 >= c.dim) return;
    const long long bh = r / c.limit, slot = r % c.limit;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (slot < c.length[bh / c.heads]) {
        const uint32_t code = *(const uint32_t *)((side ? c.value : c.key) + (bh * c.rows + slot) * (W / 2) + d * 4);
        const uint32_t byte = (side ? c.value_scale : c.key_scale)[(bh * (W / 32) + d / 4) * c.rows + slot];
        const float s = __uint_as_float(byte << 23);
        v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 0));
        v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 1));
        v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 2));
        v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, 3));
        if (byte == 255) v = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
    }
    (side ? value : key)[r * (c.dim / 8) + d] = v;
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
    int R, tiles;                            // R = T G rows per (sequence, head), row = t G + g; tiles of MT * 16 of them
    int nsplit;                              // pieces that the bank's rows are cut into
    float c2;                                // scale * log2(e)
    float *part;                             // nsplit > 1: [split][batch heads][R][W] partial sums ...
    float2 *part_ml;                         //             ... and [split][batch heads][R] (maximum, sum), maximum in log2 units
    int chunks;                              // weights: workgroups a (sequence, head), each takes every chunks-th 128 rows
    float *lse;                              // [batch heads][R] log2 of the softmax denominator (weights wanted), or null
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
// float32: with three).  A piece of an infinity or NaN is that value itself, the rest zero.
template <int P>
__device__ __forceinline__ void split_pieces(const float (&x)[8], cb16x8 (&out)[P])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float v = x[i];
#pragma unroll
        for (int k = 0; k < P; ++k) {
            const __bf16 h = (__bf16)v;
            out[k][i] = h;
            v = v - (float)h;
            if ((__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) v = 0.f;
        }
    }
}

template <int DT> struct Pieces { static constexpr int N = DT == CACHE_F32 ? 3 : DT == CACHE_F16 ? 2 : 1; };

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
// a value's scale is kept finite: a NaN row has reached the result through its key, and 0 * inf must not reach other rows
__device__ __forceinline__ float value_scale_of(uint32_t word, int e)
{
    const uint32_t bits = e == 3 ? (word >> 1) & 0x7f800000u : (word << (23 - 8 * e)) & 0x7f800000u;
    return __uint_as_float(bits < 0x7f000000u ? bits : 0x7f000000u);
}

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

// NB words of 8 elements / NB bytes of 2 elements at p, as words (one load each).
template <int NB>
__device__ __forceinline__ void load_key(const uint8_t *p, uint32_t (&w)[NB])
{
    if constexpr (NB == 2) {
        const uint2 v = *(const uint2 *)p;
        w[0] = v.x, w[1] = v.y;
    } else {
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
    if (i % 4 == 0 && byte == 255) {
        uint4 v = __builtin_bit_cast(uint4, f);
        v = make_uint4(0x7fc07fc0u, 0, 0, 0);
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

// Streaming form: a workgroup has MT tiles of 16 query rows of one (sequence, head) and one piece of its bank rows; its four
// waves take every fourth unit of 32 rows each, straight from memory into registers, and are joined at the end.
template <int DT, int NB, int MT>
__global__ __launch_bounds__(256) void cache_attend_kernel(CacheAttendParams p)
{
    constexpr int W = 32 * NB, PQ = Pieces<DT>::N, PP = DT == CACHE_F32 ? 3 : 2, LD = W + 4;
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ float s_o[4][16][LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, j = lane >> 4;
    long long id = blockIdx.x;
    const int split = (int)(id % p.nsplit);
    id /= p.nsplit;
    const int tile = (int)(id % p.tiles);
    const long long bh = id / p.tiles;
    const int b = (int)(bh / p.c.heads), h = (int)(bh % p.c.heads);
    int len = p.c.length[b];
    len = len > p.c.limit ? p.c.limit : len;
    const int n = real_rows(p.counts, b, p.T);

    cb16x8 q[MT][NB][PQ];
    int lim[MT], most = 0, least = 0x7fffffff;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = (tile * MT + m) * 16 + c;
        const bool in = row < p.R;
        lim[m] = in ? visible(row / p.G, n, len, p.causal) : 0;
        load_query<DT, NB, PQ>(p, b, h, in ? row : 0, j, lim[m] > 0, q[m]);
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
    float mx[MT], sum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        mx[m] = -INFINITY;
        sum[m] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) o[m][i] = cf32x4{0, 0, 0, 0};
    }
    const UnitAt<NB> at(p.c, bh, lane);
    for (int un = first + wave; un < last; un += 4) {
        const int u0 = un * 32;
        Unit<NB> u;
        at.load(u0, u);
        cf32x4 s[MT][2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
#pragma unroll
            for (int m = 0; m < MT; ++m) s[m][a] = cf32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const cb16x8 kf = key_operand<NB>(u.k[a], u.ks[a], i);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int k = 0; k < PQ; ++k) s[m][a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[m][i][k], s[m][a], 0, 0, 0);
            }
        }
        cb16x8 pf[MT][PP];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (u0 + 32 > least) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (u0 + 16 * (e >> 2) + 4 * j + (e & 3) >= lim[m]) s[m][e >> 2][e & 3] = -INFINITY;
            }
            float top = s[m][0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) top = fmaxf(top, s[m][e >> 2][e & 3]);
            const float now = fmaxf(mx[m], across_j_max(top));
            const float ref = now == -INFINITY ? 0.f : now * p.c2;
            const float shrink = __builtin_amdgcn_exp2f(fmaf(mx[m], p.c2, -ref));
            mx[m] = now;
            float x[8], part = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(fmaf(s[m][e >> 2][e & 3], p.c2, -ref));
                part += x[e];
            }
            sum[m] = sum[m] * shrink + part;
            split_pieces<PP>(x, pf[m]);
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) o[m][i] *= shrink;
        }
#pragma unroll
        for (int i2 = 0; i2 < NB; ++i2) {                 // channels 2 i2, 2 i2 + 1 of each lane
            uint32_t pair[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float sc = value_scale_of(u.vs[e >> 2], e & 3);
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
        }
    }

    // join the four waves, one tile of 16 rows at a time
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const float l = across_j_sum(sum[m]);
        __syncthreads();
        if (j == 0) {
            s_m[wave][c] = mx[m];
            s_l[wave][c] = l;
        }
        __syncthreads();
        float top = s_m[0][c];
#pragma unroll
        for (int w = 1; w < 4; ++w) top = fmaxf(top, s_m[w][c]);
        const float ref = top == -INFINITY ? 0.f : top * p.c2;
        const float f = __builtin_amdgcn_exp2f(fmaf(mx[m], p.c2, -ref));
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
                if (d == 0) p.part_ml[g] = make_float2(big == -INFINITY ? -INFINITY : rref, den);
            } else {
                const float inv = big == -INFINITY ? 0.f : 1.f / den;
                for (int i = 0; i < 8; ++i) x[i] = big == -INFINITY ? 0.f : x[i] * inv;
                const int t = row / p.G, g = row - t * p.G;
                if (d < p.c.dim) store8<DT>(p.out + b * p.out_s[0] + (long long)(h * p.G + g) * p.out_s[1] + t * p.out_s[2] + (long long)d * elem_bytes<DT>(), x);
                if (p.lse && d == 0) p.lse[bh * p.R + row] = big == -INFINITY ? INFINITY : rref + __builtin_amdgcn_logf(den);
            }
        }
    }
}

// Joins the pieces of a row: W / 8 lanes a row, 8 channels a lane.
template <int DT, int W>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheAttendParams p)
{
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long all = (long long)p.c.batch * p.c.heads * p.R, g0 = at / (W / 8);
    const int d = (int)(at % (W / 8)) * 8;
    if (g0 >= all) return;
    float big = -INFINITY;
    for (int s = 0; s < p.nsplit; ++s) big = fmaxf(big, p.part_ml[s * all + g0].x);
    float den = 0.f, x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int s = 0; s < p.nsplit; ++s) {
        const float2 ml = p.part_ml[s * all + g0];
        if (ml.x == -INFINITY) continue;                  // nothing seen there: its sums may be left unread
        const float f = __builtin_amdgcn_exp2f(ml.x - big);
        den += ml.y * f;
        float y[8];
        load8<CACHE_F32>(p.part + (s * all + g0) * W + d, y);
        for (int i = 0; i < 8; ++i) x[i] += y[i] * f;
    }
    const float inv = 1.f / den;
    for (int i = 0; i < 8; ++i) x[i] = big == -INFINITY ? 0.f : x[i] * inv;
    const long long bh = g0 / p.R;
    const int row = (int)(g0 % p.R), b = (int)(bh / p.c.heads), h = (int)(bh % p.c.heads), t = row / p.G, g = row - t * p.G;
    if (d < p.c.dim) store8<DT>(p.out + b * p.out_s[0] + (long long)(h * p.G + g) * p.out_s[1] + t * p.out_s[2] + (long long)d * elem_bytes<DT>(), x);
    if (p.lse && d == 0) p.lse[g0] = big == -INFINITY ? INFINITY : big + __builtin_amdgcn_logf(den);
}

// Attention sums: weight[slot] += sum over the query rows of exp(s - lse).  A wave has one unit of 32 bank rows and goes over
// all rows that may see it, so that every sum has one owner and one order.
template <int DT, int NB>
__global__ __launch_bounds__(256) void cache_weigh_kernel(CacheAttendParams p)
{
    constexpr int PQ = Pieces<DT>::N;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, j = lane >> 4;
    const long long bh = blockIdx.x / p.chunks;
    const int b = (int)(bh / p.c.heads), h = (int)(bh % p.c.heads);
    int len = p.c.length[b];
    len = len > p.c.limit ? p.c.limit : len;
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
            const float lse = lim > 0 ? p.lse[bh * p.R + row] : INFINITY;
            cf32x4 s[2] = {cf32x4{0, 0, 0, 0}, cf32x4{0, 0, 0, 0}};
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const cb16x8 kf = key_operand<NB>(kk[a], ks[a], i);
#pragma unroll
                    for (int k = 0; k < PQ; ++k) s[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[i][k], s[a], 0, 0, 0);
                }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], p.c2, -lse));
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

constexpr int EVICT_THREADS = 1024;

// Exclusive prefix sum over the workgroup of two counts at once; totals in `all`.
__device__ __forceinline__ int2 block_scan2(int2 v, int2 *s_wave, int2 &all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int2 x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int a = __shfl_up(x.x, d), e = __shfl_up(x.y, d);
        if (lane >= d) x.x += a, x.y += e;
    }
    __syncthreads();
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    int2 before = make_int2(0, 0);
    all = make_int2(0, 0);
    for (int i = 0; i < EVICT_THREADS / 64; ++i) {
        if (i < wave) before.x += s_wave[i].x, before.y += s_wave[i].y;
        all.x += s_wave[i].x, all.y += s_wave[i].y;
    }
    return make_int2(before.x + x.x - v.x, before.y + x.y - v.y);
}

// One workgroup per (sequence, head): radix select of the keep-th rank, then the lists of what has to be copied.  The freed
// slots below `keep` take, in ascending order, the kept rows from above it: in place no row is read that another one is
// written to, and no more rows move than left.
__global__ __launch_bounds__(EVICT_THREADS) void cache_select_kernel(EvictParams p)
{
    __shared__ int s_hist[256];
    __shared__ int2 s_wave[EVICT_THREADS / 64];
    __shared__ uint32_t s_prefix;
    __shared__ int s_left;
    const long long bh = blockIdx.x;
    const int b = (int)(bh / p.c.heads), tid = threadIdx.x;
    int n = p.c.length[b];
    n = n > p.c.limit ? p.c.limit : n;
    const int from = p.c.seen[b] - p.recent, keep = p.keep;
    const float *w = p.c.weight + bh * p.c.rows;
    const int *pos = p.c.position + bh * p.c.rows;
    int2 *pairs = p.pairs + bh * keep;
    if (n <= keep) {
        if (!p.in_place)
            for (int i = tid; i < n; i += EVICT_THREADS) pairs[i] = make_int2(i, i);
        if (tid == 0) p.count[bh] = p.in_place ? 0 : n;
        return;
    }
    if (tid == 0) s_prefix = 0, s_left = keep;
    uint32_t known = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) s_hist[tid] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix;
        for (int i = tid; i < n; i += EVICT_THREADS) {
            const uint32_t r = evict_rank(w[i], pos[i], from);
            if ((r & known) == prefix) atomicAdd(&s_hist[(r >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int left = s_left, d = 255;
            while (d > 0 && s_hist[d] < left) left -= s_hist[d--];
            s_left = left;
            s_prefix = prefix | ((uint32_t)d << shift);
        }
        known |= 255u << shift;
        __syncthreads();
    }
    const uint32_t edge = s_prefix;
    const int ties = s_left;                 // rows of rank `edge` that stay: the lowest slots
    const int per = (n + EVICT_THREADS - 1) / EVICT_THREADS, lo = min(n, tid * per), hi = min(n, lo + per);
    int eq = 0;
    for (int i = lo; i < hi; ++i) eq += evict_rank(w[i], pos[i], from) == edge;
    int2 all;
    const int before = block_scan2(make_int2(eq, 0), s_wave, all).x;
    int2 mine = make_int2(0, 0);             // (freed slots below keep, kept rows above it)
    int at = before;
    for (int i = lo; i < hi; ++i) {
        const uint32_t r = evict_rank(w[i], pos[i], from);
        const bool kept = r > edge || (r == edge && at++ < ties);
        if (i < keep) mine.x += !kept;
        else mine.y += kept;
    }
    int2 off = block_scan2(mine, s_wave, all);
    if (tid == 0) p.count[bh] = p.in_place ? all.x : keep;
    at = before;
    // in place: pair i = (i-th freed slot, i-th kept row above); otherwise pair s = (s, its source), via the free tail of the
    // list: the kept rows above are first written where only freed slots are looked up, so they go through shared memory
    for (int i = lo; i < hi; ++i) {
        const uint32_t r = evict_rank(w[i], pos[i], from);
        const bool kept = r > edge || (r == edge && at++ < ties);
        if (p.in_place) {
            if (i < keep) {
                if (!kept) pairs[off.x++].x = i;
            } else if (kept) pairs[off.y++].y = i;
        } else if (i < keep) {
            pairs[i].x = i;
            if (kept) pairs[i].y = i;
        }
    }
    if (p.in_place) return;
    // the i-th freed slot of all: its owner waits for the i-th kept row above, in rounds of one list in shared memory
    __shared__ int s_src[4096];
    const int2 total = all;
    for (int base = 0; base < total.x; base += 4096) {
        __syncthreads();
        int y = off.y;
        at = before;
        for (int i = lo; i < hi; ++i) {
            const uint32_t r = evict_rank(w[i], pos[i], from);
            const bool kept = r > edge || (r == edge && at++ < ties);
            if (i >= keep && kept) {
                if (y >= base && y < base + 4096) s_src[y - base] = i;
                ++y;
            }
        }
        __syncthreads();
        int x = off.x;
        at = before;
        for (int i = lo; i < hi && i < keep; ++i) {
            const uint32_t r = evict_rank(w[i], pos[i], from);
            const bool kept = r > edge || (r == edge && at++ < ties);
            if (!kept) {
                if (x >= base && x < base + 4096) pairs[i].y = s_src[x - base];
                ++x;
            }
        }
    }
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
        int n = p.c.length[b];
        n = n > p.c.limit ? p.c.limit : n;
        p.into.length[b] = n < p.keep ? n : p.keep;
        if (!p.in_place) p.into.seen[b] = p.c.seen[b];
    }
}

}  // namespace mi
#endif
