// The rotation of query and key rows at their positions, shared by the kernel that only rotates
// and the append that rotates on the way (both in ma_pages.hip).
//
// A pair (x, y) of channels at position p turns by the angle whose cosine and sine row p of the
// table holds: x' = x c - y s, y' = y c + x s.  Products and sums are rounded to f32 one by one (no
// fused multiply-add), the result once to its type: the bits are those of the same four
// operations anywhere else, so a key has one stored form however it was rotated.
#pragma once

#include "ma_pages.h"

namespace ma {

// cosines [dim / 2] and sines [dim / 2] of a row; dim a multiple of 16, rows 16-byte aligned
struct RotaryDev {
    const float *table;
    const int32_t *first;      // position of every request's token 0
    int64_t s_row;
    int rows, dim;
    bool next;                 // channels 2 i and 2 i + 1 are a pair (else i and i + dim / 2)
    int32_t *status;           // (or NULL: nobody asks)
    const int32_t *count;
};

inline RotaryDev rotary_dev(const ma_rotary *r, const int32_t *lengths) {
    return RotaryDev{r->table, r->first ? r->first : lengths, r->s_row, r->rows, r->dim, r->interleaved != 0,
                     r->status, r->count};
}

// of n new tokens from position first on, is one outside the table?  (One thread a request, behind its rows.)
constexpr int ROTARY_OUTSIDE = 32;
__device__ __forceinline__ void rotary_note(const RotaryDev &r, int first, int n) {
    if (r.status && n > 0 && (first < 0 || (int64_t)first + n > r.rows)) atomicOr(r.status, ROTARY_OUTSIDE);
}

// the table's row of request b's token t (positions beyond the table: its last row)
__device__ __forceinline__ const float *rotary_row(const RotaryDev &r, int first, int t) {
    const int64_t pos = min(max((int64_t)first + t, (int64_t)0), (int64_t)r.rows - 1);
    return r.table + pos * r.s_row;
}

template <int DT>
__device__ __forceinline__ void rotary_unpack(uint32_t w, float &a, float &b) {
    if constexpr (DT == MA_BF16) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    } else {
        a = ma_f16_to_f32((uint16_t)w);
        b = ma_f16_to_f32((uint16_t)(w >> 16));
    }
}
template <int DT>
__device__ __forceinline__ uint32_t rotary_pack(float a, float b) {
    if constexpr (DT == MA_BF16) return ma_pack_bf16x2(a, b);
    const f16x2_t v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
}

// x c + y s, each operation rounded
__device__ __forceinline__ float rotary_turn(float x, float c, float y, float s) {
#pragma clang fp contract(off)
    const float a = x * c, b = y * s;
    return a + b;
}

// two channels x and their partners y (the first of the pairs: with -s)
template <int DT>
__device__ __forceinline__ uint32_t rotary_halves(uint32_t x, uint32_t y, float c0, float c1, float s0, float s1) {
    float x0, x1, y0, y1;
    rotary_unpack<DT>(x, x0, x1);
    rotary_unpack<DT>(y, y0, y1);
    return rotary_pack<DT>(rotary_turn(x0, c0, y0, s0), rotary_turn(x1, c1, y1, s1));
}
// two channels that are a pair
template <int DT>
__device__ __forceinline__ uint32_t rotary_pair(uint32_t w, float c, float s) {
    float x, y;
    rotary_unpack<DT>(w, x, y);
    return rotary_pack<DT>(rotary_turn(x, c, -y, s), rotary_turn(y, c, x, s));
}

// 8 pairs: channels a, b of 16 bytes each, i and i + dim / 2 or 16 neighbours
template <int DT>
__device__ __forceinline__ void rotary_unit(uint4 &a, uint4 &b, const float (&c)[8], const float (&s)[8], bool next) {
    uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (next) {
            aw[i] = rotary_pair<DT>(aw[i], c[i], s[i]);
            bw[i] = rotary_pair<DT>(bw[i], c[4 + i], s[4 + i]);
        } else {
            const uint32_t x = aw[i], y = bw[i];
            aw[i] = rotary_halves<DT>(x, y, c[2 * i], c[2 * i + 1], -s[2 * i], -s[2 * i + 1]);
            bw[i] = rotary_halves<DT>(y, x, c[2 * i], c[2 * i + 1], s[2 * i], s[2 * i + 1]);
        }
    }
    a = uint4{aw[0], aw[1], aw[2], aw[3]};
    b = uint4{bw[0], bw[1], bw[2], bw[3]};
}

// Rows of up to 2 heads of one request at their positions: a thread takes 16 channels (8 pairs,
// or 16 that are not turned) of one token, and reads its cosines and sines once for both.  in and out
// may be the same rows.
//
// bound: the bytes, 4 D a row and 4 dim a position.  4 096 tokens of 4 requests (32 query and 8 KV heads,
// D 128): 344 MB in 62.6 us, 5.5 TB/s, where a copy of as many bytes reaches 5.3 (one head a thread 66.3, four 63.8, eight 67.3); a token of 64
// requests (28 and 4 heads) 4.2 us, which is a launch and two loads in a row (4.1, 4.6, 6.3).
constexpr int ROTARY_HEADS = 2;
struct RotaryRows {
    const uint16_t *in;
    uint16_t *out;
    int64_t s_ib, s_ih, s_it, s_ob, s_oh, s_ot;
    int heads;
};
template <int D, int DT>
__device__ __forceinline__ void rotary_heads(const RotaryDev &r, const RotaryRows &x, int first, int b, int h0, int t, int unit) {
    const int half = r.dim / 2;
    const bool turn = 16 * unit < r.dim;
    // (channels behind the turned ones are copied, 16 together)
    const int c0 = turn && !r.next ? 8 * unit : 16 * unit, c1 = turn && !r.next ? c0 + half : c0 + 8;
    const uint16_t *in = x.in + (int64_t)b * x.s_ib + (int64_t)h0 * x.s_ih + (int64_t)t * x.s_it;
    uint16_t *out = x.out + (int64_t)b * x.s_ob + (int64_t)h0 * x.s_oh + (int64_t)t * x.s_ot;
    const int n = min(x.heads - h0, ROTARY_HEADS);
    uint4 a[ROTARY_HEADS], z[ROTARY_HEADS];
#pragma unroll
    for (int i = 0; i < ROTARY_HEADS; ++i) {     // (behind the last head: the last one again, which is not stored)
        const uint16_t *src = in + (int64_t)min(i, n - 1) * x.s_ih;
        a[i] = pg_load16(src + c0);
        z[i] = pg_load16(src + c1);
    }
    if (turn) {
        const float *row = rotary_row(r, first, t) + 8 * unit;
        float c[8], s[8];
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const f32x4_t cv = *(const f32x4_t *)(row + i), sv = *(const f32x4_t *)(row + half + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) c[i + k] = cv[k], s[i + k] = sv[k];
        }
#pragma unroll
        for (int i = 0; i < ROTARY_HEADS; ++i) rotary_unit<DT>(a[i], z[i], c, s, r.next);
    }
#pragma unroll
    for (int i = 0; i < ROTARY_HEADS; ++i)
        if (i < n) {
            pg_store16(out + (int64_t)i * x.s_oh + c0, a[i]);
            pg_store16(out + (int64_t)i * x.s_oh + c1, z[i]);
        }
}

}  // namespace ma
