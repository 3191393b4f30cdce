// The paged 4-bit store shared by the page kernels (ma_pages.hip) and the attention over
// pages (ma_paged_attn.hip).
//
// A page holds page_tokens tokens (a multiple of 32) of every KV head: per head, one record
// of 40 D bytes for each group of 32 tokens,
//   [K codes 16 D][V codes 16 D][ks 2 D][kz 2 D][vs 2 D][vz 2 D]          (f16 parameters)
// in the order in which v_mfma_f32_16x16x32 takes its operands, so that a wave reads a
// group's codes as whole contiguous 16-byte (8-byte) lanes and never moves one between lanes:
//   K codes  [mt 2][h 4][m 16][cb D/32] words of 8 channels: lane (h, m) of the A operand of
//            S^T = K Q^T, rows m of token tile mt <-> token 8 (m/4) + 4 mt + m%4, channels
//            (D/4) h + 8 cb + (0..7)
//   V codes  [half D/64][h 4][m 16][4] words of 8 tokens: lane (h, m) of the A operand of
//            O^T = V^T P^T, row m of channel tile ct = 4 half + (0..3) <-> channel (D/16) m + ct,
//            tokens 8 h + (0..7) -- the tokens whose scores lane (., h) of the S^T result holds
//   ks, kz   [D] per channel; vs, vz [D/32][32] per (channel group, token)
// Nibbles of a word from the lowest up: elements 0 2 4 6 1 3 5 7.  Masking a word with
// 0x000f000f (0x00f000f0, and both again after >> 8) leaves the element pairs (0,1), (2,3),
// (4,5), (6,7) in the two halves of a register.
#pragma once

#include "ma_common.h"

namespace ma {

constexpr int PG_GROUP = 32;   // tokens of a record

typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;

// 16 (8) bytes at any 2-byte-aligned address (the global memory path takes them)
struct __attribute__((packed, aligned(2))) pg_u4 { uint32_t x, y, z, w; };
struct __attribute__((packed, aligned(2))) pg_u2 { uint32_t x, y; };
struct __attribute__((packed, aligned(1))) pg_b8 { uint32_t x, y; };

__device__ __forceinline__ uint4 pg_load16(const void *p) {
    const pg_u4 v = *(const pg_u4 *)p;
    return uint4{v.x, v.y, v.z, v.w};
}
__device__ __forceinline__ uint2 pg_load8(const void *p) {
    const pg_u2 v = *(const pg_u2 *)p;
    return uint2{v.x, v.y};
}
__device__ __forceinline__ void pg_store16(void *p, uint4 v) { *(pg_u4 *)p = pg_u4{v.x, v.y, v.z, v.w}; }
__device__ __forceinline__ void pg_store8(void *p, uint2 v) { *(pg_u2 *)p = pg_u2{v.x, v.y}; }

// the store as the kernels hold it (strides of pool in bytes, of the tails in elements)
struct PagesDev {
    uint8_t *pool;
    uint16_t *kt, *vt;
    const int32_t *table, *lengths;
    const uint8_t *mask;
    int64_t s_page, s_head, s_tb, s_th, s_tt, s_table, s_mb, s_mh;
    int num_pages, width, page_tokens, mask_tokens;
};

inline PagesDev pages_dev(const ma_pages *p) {
    PagesDev d;
    d.pool = (uint8_t *)p->pool;
    d.kt = (uint16_t *)p->k_tail;
    d.vt = (uint16_t *)p->v_tail;
    d.table = p->table;
    d.lengths = p->lengths;
    d.mask = p->mask;
    d.s_page = p->s_pool[0];
    d.s_head = p->s_pool[1];
    d.s_tb = p->s_tail[0];
    d.s_th = p->s_tail[1];
    d.s_tt = p->s_tail[2];
    d.s_table = p->s_table;
    d.s_mb = p->s_mask[0];
    d.s_mh = p->s_mask[1];
    d.num_pages = p->num_pages;
    d.width = p->width;
    d.page_tokens = p->page_tokens;
    d.mask_tokens = p->mask_tokens;
    return d;
}

// stored tokens of request b that its table row can hold (a longer length reads no further)
__device__ __forceinline__ int pg_length(const PagesDev &p, int b) {
    const int64_t cap = (int64_t)p.width * p.page_tokens;
    const int n = max(p.lengths[b], 0);
    return n < cap ? n : (int)cap;
}

// the record of group g of (b, head h), or NULL where the table names no page of the pool
__device__ __forceinline__ const uint8_t *pg_record(const PagesDev &p, int page_id, int gi, int h, int rec) {
    if (page_id < 0 || page_id >= p.num_pages) return nullptr;
    return p.pool + (int64_t)page_id * p.s_page + (int64_t)h * p.s_head + (int64_t)gi * rec;
}

// the nonzero bytes of x, as 4 bits
__device__ __forceinline__ uint32_t pg_byte_bits(uint32_t x) {
    x |= x >> 4;
    x |= x >> 2;
    x |= x >> 1;
    return ((x & 0x01010101u) * 0x10204080u) >> 28;
}
// the seen ones of 8 tokens from position pos on, of a request with a mask
__device__ __forceinline__ uint32_t pg_mask_bits(const PagesDev &p, int b, int h, int pos) {
    const uint8_t *m = p.mask + (int64_t)b * p.s_mb + (int64_t)h * p.s_mh;
    const int n = p.mask_tokens;
    if (n >= 8) {     // 8 bytes that the mask has, moved to where they belong
        const int at = min(pos, n - 8), out = min(pos - at, 8);
        const pg_b8 v = *(const pg_b8 *)(m + (uint32_t)at);
        return (pg_byte_bits(v.x) | pg_byte_bits(v.y) << 4) >> out;
    }
    uint32_t bits = 0;
    for (int i = 0; i < 8; ++i)
        if (pos + i < n && m[pos + i]) bits |= 1u << i;
    return bits;
}

// inclusive prefix sum over the wave of values >= 0: by lane moves where 32 bits hold every sum
__device__ __forceinline__ int64_t pg_wave_scan(int64_t x, int lane) {
    if (!__any(x >= (int64_t)1 << 25)) return (int64_t)ma_wave_prefix_u32((uint32_t)x);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// host: the checks every entry point over a store makes
int pg_check(const ma_pages *p, int B, int H, int D, const char *who);

}  // namespace ma
