// Attention of a block of queries of every request over [its pages of 4-bit K/V | its 16-bit
// tail | the block's own keys], for ragged requests whose lengths lie on the device.
//
// The work is a line of items: a group of 32 packed tokens, the tail, or 32 keys of the
// block, of one segment = (request, KV head, row group); a row is one of the R = (Hq / H) T
// pairs of a query head of the KV head and a position.  Every workgroup takes an equal stretch
// of the line, whatever segments it crosses, so ragged lengths need no plan and no read-back:
// it finds its first request by a scan of the lengths.  A segment that lies in one stretch is
// written out; one cut between workgroups leaves f32 partials (row maximum, sum, unnormalised
// output), which paged_merge_kernel joins in a fixed order: the same call gives the same bits.
//
// Over selected blocks of a request's tokens the lists say what is read, about as much for every segment:
// no line is cut there, a segment has a fixed number of workgroups (own_part).
//
// Two kernels walk the line.  Up to 32 rows (single tokens, short blocks) are bound by the
// cache's bytes: there every wave unpacks records into its own registers.  More rows are bound
// by the matrix cores: there a record is unpacked once, into LDS, for up to 256 rows.
//
// Per item and wave: S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32, K and V as A
// operands.  A lane of S^T holds 8 tokens of one query row, which is the B operand that P^T
// needs: nothing moves between lanes.  Codes become f16 in place (mask into the mantissa of
// 1024 or 64, subtract, one fused multiply-add by scale and zero: one rounding of 2^-11
// relative, where a bf16 copy of the cache has 2^-8); scores, maxima, sums and outputs are
// f32; weights are rounded to f16 (2^-11; their range: P_MAX below) for the second product, and
// their sum is that of what is multiplied.  Together 3.5e-4 of a result in the 2-norm, where bf16
// results are rounded by 1.6e-3: what the matrix cores' full rate costs.  f16 results are rounded by
// 2.1e-4 alone, so for them keys, values and weights are sums of two f16 (2.1e-4 in all; more than 32
// rows: values are one, whose second half has no room in the LDS at D 128: 3.0e-4).
// The tail and the block's keys are read as they are, the weight a sum of two of their type.
#include "ma_pages.h"

using namespace ma;

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 b16x8_t;

constexpr int WAVES = 4;
// Weights are 2^(score - reference) and become f16, which holds 11 bits from 2^-14 to 2^16 and
// nothing below 2^-25.  A row's reference therefore follows its items.  It begins where a score of 0
// weighs 2^P_NEW.  Where the largest weight of an item's 32 tokens (of a lane's 8, as it is looked at)
// would lie above 2^P_MAX or below 2^P_MIN (of the first item: 2^P_FIRST), the reference is moved to
// where it is 2^P_NEW (those found below 2^P_LOW then, so that the next items lie well inside).  Most
// items, and most first ones, leave the reference and the accumulators alone.  A weight then carries
// at most 2^-25 absolute, 2^-17 of the largest of its item, beside f16's 2^-11 relative, however far
// another item's score is above: with the row's maximum as the only reference, a key that leads by 17
// nats and has no value of its own left the others no digits.  Beside such a key, in its own item, what
// is below 2^-25 of it can be lost (2^-17 where all before it was dead).  The reference goes down only while the sum stays below P_SUM, which
// leaves the accumulators 2^67 of room.  Following costs 32 tokens of 8 requests 51.2 -> 52.7 us, 512
// tokens of 2 requests 217 -> 222, one token of 64 requests nothing.
constexpr float P_MAX = 15.0f, P_MIN = -8.0f, P_FIRST = 0.0f, P_LOW = 0.0f, P_NEW = 7.0f;
constexpr float P_SUM = 0x1p60f;
constexpr float NO_MAX = -1e30f;

struct AttnArgs {
    ma_tensor4 q, kc, vc, out;
    PagesDev p;
    const int32_t *new_lens;
    int B, H, G, T, R, RG, HR, causal, W;   // HR = H * RG
    int max_len;              // tokens that a table row can name
    int rows0, dense;         // items that a segment's 16-bit rows are worth: rows0, and 1 << dense each
    float sl2;                // scale * log2(e)
    float *wm, *wl, *wo;      // partials of slots [2 W]: per row reference and sum, unnormalised rows
    int4 *desc;               // [B, H, RG]: what note_segment says of every segment
    // Over selected blocks (SEL): every run of `run` positions has a list of its own, rows are those of
    // a run (R = G run), and RG = runs * RGR.
    const int32_t *blocks;    // [B, H, runs, count]
    int count, m, run, RGR;   // entries of a list, groups of a block
    int parts, wide;          // workgroups of a segment; they have 8 waves (few rows)
};

// values that every lane holds alike, as scalars
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// What a request has: new tokens, stored tokens, whole groups, tail, and the items of one of its
// segments.  The first START items of a segment are no work: they stand for its start and end
// (queries, table, first loads; joining, writing), so that stretches of equal length are of
// equal time; rows0 in front of its 16-bit rows stand for those rows' first loads.  A request
// without new tokens has none.
//
// START 1, 8, 12, 16, 20: one token of 64 ragged requests 58, 52.4, 52.8, 52.4, 54.1 us, of 2 long
// ones 66.8 to 67.3; of many rows 9 % slower with 1, 4 to 16 within 2 % of one another.
constexpr int START = 8;
struct Items {
    int n, len, ng, rem, items;      // ng: packed items
};
// Over selected blocks (SEL) the packed items are the groups of as many of the list's entries as the
// request has blocks; an entry that names none, and groups behind the request's last, are items that
// nothing is seen of.  seen: the block's keys that any row of the segment sees.
template <bool SEL>
__device__ __forceinline__ Items items_from(const AttnArgs &a, int n, int len, int seen = 0) {
    Items r;
    r.n = n;
    r.len = len;
    r.ng = len / PG_GROUP;
    if (SEL)         // (of a block longer than the request, the request's)
        r.ng = (int)min((unsigned)a.count, ((unsigned)r.ng + (unsigned)a.m - 1) / (unsigned)a.m) * min(a.m, r.ng);
    r.rem = len % PG_GROUP;
    const int cur = a.kc.ptr ? ((SEL ? seen : n) + PG_GROUP - 1) / PG_GROUP : 0;
    const int rows = (r.rem ? 1 : 0) + cur;
    r.items = n ? (SEL ? 0 : START) + r.ng + (rows ? a.rows0 + (rows << a.dense) : 0) : 0;
    return r;
}
__device__ __forceinline__ Items items_of(const AttnArgs &a, int b) {
    return items_from<false>(a, a.new_lens ? min(max(a.new_lens[b], 0), a.T) : a.T, min(max(a.p.lengths[b], 0), a.max_len));
}
// ... of a request that the whole wave looks at
__device__ __forceinline__ Items items_at(const AttnArgs &a, int b) {
    const Items r = items_of(a, b);
    return items_from<false>(a, uniform(r.n), uniform(r.len));
}
// positions of a segment's rows: row = query head * positions + position
template <bool SEL>
__device__ __forceinline__ int positions(const AttnArgs &a) { return SEL ? a.run : a.T; }

// The lane's number, as a value that nothing is known of: what is computed from it stays where
// it is used, where the compiler would otherwise keep every address of the rare paths in
// registers across the main loop (it spilled 170 of them).
__device__ __forceinline__ int hidden(int lane) {
    asm volatile("" : "+v"(lane));
    return lane;
}

// (x & mask) | bits in one instruction (its constants lie in registers)
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "s"(mask), "v"(bits));
    return r;
}
// pairs of codes as f16 (exact), the k-th pair of a code word
__device__ __forceinline__ f16x2_t code_pair(uint32_t w, int k) {
    const uint32_t x = k & 2 ? w >> 8 : w;
    if (k & 1)     // 64 + code
        return __builtin_bit_cast(f16x2_t, and_or(x, 0x00f000f0u, 0x54005400u)) - (f16x2_t){(_Float16)64.0f, (_Float16)64.0f};
    return __builtin_bit_cast(f16x2_t, and_or(x, 0x000f000fu, 0x64006400u)) -      // 1024 + code
           (f16x2_t){(_Float16)1024.0f, (_Float16)1024.0f};
}

// the 8 values of a code word; s, z: their parameters, pair by pair
__device__ __forceinline__ f16x8_t word_values(uint32_t w, uint4 s, uint4 z) {
    const uint32_t sw[4] = {s.x, s.y, s.z, s.w}, zw[4] = {z.x, z.y, z.z, z.w};
    f16x8_t r;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const f16x2_t v = __builtin_elementwise_fma(code_pair(w, k), __builtin_bit_cast(f16x2_t, sw[k]),
                                                    __builtin_bit_cast(f16x2_t, zw[k]));
        r[2 * k] = v[0];
        r[2 * k + 1] = v[1];
    }
    return r;
}

// f16 results: a value in two parts.  Few rows: code * scale with the scale's upper 7 bits and with
// its lower 4, both exact, the zero being a product of its own.
__device__ __forceinline__ f16x2_t as_f16x2(uint32_t w) { return __builtin_bit_cast(f16x2_t, w); }
__device__ __forceinline__ void split_scale(uint4 s, uint4 &hi, uint4 &lo) {
    hi = uint4{s.x & 0xfff0fff0u, s.y & 0xfff0fff0u, s.z & 0xfff0fff0u, s.w & 0xfff0fff0u};
    auto rest = [](uint32_t x, uint32_t y) { return __builtin_bit_cast(uint32_t, as_f16x2(x) - as_f16x2(y)); };
    lo = uint4{rest(s.x, hi.x), rest(s.y, hi.y), rest(s.z, hi.z), rest(s.w, hi.w)};
}
__device__ __forceinline__ void word_products(uint32_t w, uint4 s_hi, uint4 s_lo, f16x8_t &hi, f16x8_t &lo) {
    const uint32_t hw[4] = {s_hi.x, s_hi.y, s_hi.z, s_hi.w}, lw[4] = {s_lo.x, s_lo.y, s_lo.z, s_lo.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const f16x2_t c = code_pair(w, k), x = c * as_f16x2(hw[k]), y = c * as_f16x2(lw[k]);
        hi[2 * k] = x[0], hi[2 * k + 1] = x[1];
        lo[2 * k] = y[0], lo[2 * k + 1] = y[1];
    }
}
// Many rows: the value rounded, and what the rounding left (product and sum with their errors).
__device__ __forceinline__ void word_values2(uint32_t w, uint4 s, uint4 z, f16x8_t &hi, f16x8_t &lo) {
#pragma clang fp contract(off)
    const uint32_t sw[4] = {s.x, s.y, s.z, s.w}, zw[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const f16x2_t c = code_pair(w, k), a = as_f16x2(sw[k]), b = as_f16x2(zw[k]);
        const f16x2_t x = c * a, dx = __builtin_elementwise_fma(c, a, -x);
        const f16x2_t v = x + b, y = v - x, dv = (x - (v - y)) + (b - y), r = dv + dx;
        hi[2 * k] = v[0], hi[2 * k + 1] = v[1];
        lo[2 * k] = r[0], lo[2 * k + 1] = r[1];
    }
}

__device__ __forceinline__ f32x4_t mfma16(f16x8_t a, f16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma16(b16x8_t a, b16x8_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// maximum / sum over the four lanes that hold a row (lane ^ 16, lane ^ 32)
__device__ __forceinline__ float max_rows(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return ma_max_xor32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_rows(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return ma_sum_xor32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// A record, and 16 (8) bytes of it at a scalar base and a lane's 32-bit offset.  The address
// space is in the type: as a plain pointer put together from lanes' halves it would be read by
// flat loads, whose results come in no order.
typedef const __attribute__((address_space(1))) uint8_t *rec_t;
typedef __attribute__((ext_vector_type(4))) uint32_t w4_t;
typedef __attribute__((ext_vector_type(2))) uint32_t w2_t;
__device__ __forceinline__ uint4 rec16(rec_t base, uint32_t off) {
    const w4_t v = *(const __attribute__((address_space(1))) w4_t *)(base + off);
    return uint4{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ uint2 rec8(rec_t base, uint32_t off) {
    const w2_t v = *(const __attribute__((address_space(1))) w2_t *)(base + off);
    return uint2{v[0], v[1]};
}

// one record's words of a wave
template <int D>
struct RawK {
    uint4 s[D / 32], z[D / 32];
    uint32_t k[2][D / 32];
};
template <int D>
struct RawV {
    uint4 s, z, v[D / 64];
};

template <int D>
__device__ __forceinline__ void load_k(RawK<D> &w, rec_t rec, int lane_) {
    const uint32_t lane = (uint32_t)hidden(lane_), par = (D / 2) * (lane >> 4);
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        if constexpr (D == 128) {
            const uint4 c = rec16(rec + 1024 * mt, 16 * lane);
            w.k[mt][0] = c.x; w.k[mt][1] = c.y; w.k[mt][2] = c.z; w.k[mt][3] = c.w;
        } else {
            const uint2 c = rec8(rec + 512 * mt, 8 * lane);
            w.k[mt][0] = c.x; w.k[mt][1] = c.y;
        }
    }
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb) {
        w.s[cb] = rec16(rec + 32 * D + 16 * cb, par);
        w.z[cb] = rec16(rec + 34 * D + 16 * cb, par);
    }
}
template <int D>
__device__ __forceinline__ void load_v(RawV<D> &w, rec_t rec, int lane_) {
    const uint32_t lane = (uint32_t)hidden(lane_);
    const uint32_t par = 2 * (32 * ((D / 16) * (lane & 15u) / 32) + 8 * (lane >> 4));
#pragma unroll
    for (int half = 0; half < D / 64; ++half) w.v[half] = rec16(rec + 16 * D + 1024 * half, 16 * lane);
    w.s = rec16(rec + 36 * D, par);
    w.z = rec16(rec + 38 * D, par);
}
// the values' words in the keys' registers, for a wave that unpacks one or the other: the same
// loads at other places, so that neither is copied (poff: place of a lane's parameters)
template <int D>
__device__ __forceinline__ void load_either(RawK<D> &w, rec_t rec, int lane, bool v, int poff_) {
    const uint32_t off = (uint32_t)hidden(lane) * (D == 128 ? 16 : 8), poff = (uint32_t)hidden(poff_);
    const rec_t codes = rec + (v ? 16 * D : 0), par = rec + (v ? 36 * D : 32 * D);
    if constexpr (D == 128) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            const uint4 c = rec16(codes + 1024 * mt, off);
            w.k[mt][0] = c.x; w.k[mt][1] = c.y; w.k[mt][2] = c.z; w.k[mt][3] = c.w;
        }
    } else {   // (values: 16 bytes of a lane, as two words and two words)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            const uint2 c = rec8(codes + (v ? 8 * mt : 512 * mt), v ? 2 * off : off);
            w.k[mt][0] = c.x; w.k[mt][1] = c.y;
        }
    }
    w.s[0] = rec16(par, poff);
    w.z[0] = rec16(par + 2 * D, poff);
    if (!v) {
#pragma unroll
        for (int cb = 1; cb < D / 32; ++cb) {
            w.s[cb] = rec16(par + 16 * cb, poff);
            w.z[cb] = rec16(par + (2 * D + 16 * cb), poff);
        }
    }
}
template <int D>
__device__ __forceinline__ RawV<D> v_from(const RawK<D> &w) {
    RawV<D> v;
#pragma unroll
    for (int x = 0; x < D / 64; ++x) {
        const uint32_t *y = &w.k[0][0] + 4 * x;
        v.v[x] = uint4{y[0], y[1], y[2], y[3]};
    }
    v.s = w.s[0];
    v.z = w.z[0];
    return v;
}
template <int D>
__device__ __forceinline__ uint32_t v_word(const RawV<D> &w, int ct) {
    const uint4 x = w.v[ct / 4];
    return (ct & 3) == 0 ? x.x : (ct & 3) == 1 ? x.y : (ct & 3) == 2 ? x.z : x.w;
}

__device__ __forceinline__ uint32_t halves_of(uint32_t bits) {   // bit 0 -> low half, bit 1 -> high half
    return (bits & 1u ? 0xffffu : 0u) | (bits & 2u ? 0xffff0000u : 0u);
}
// a dead token's value is 0 whatever its parameters say; live: bit i = token i of the lane's 8
template <int D>
__device__ __forceinline__ void clear_dead(RawV<D> &w, uint32_t live) {
    const uint32_t h0 = halves_of(live), h1 = halves_of(live >> 2), h2 = halves_of(live >> 4), h3 = halves_of(live >> 6);
    w.s = uint4{w.s.x & h0, w.s.y & h1, w.s.z & h2, w.s.w & h3};
    w.z = uint4{w.z.x & h0, w.z.y & h1, w.z.z & h2, w.z.w & h3};
}

// ---- rows of 16-bit K and V (the tail, or 32 keys of the block) as operands
struct Rows {
    const uint16_t *k, *v;
    int64_t sk, sv;
    int j0, cnt;      // first row, rows there are
    bool tail;
};
// item x behind the packed groups of (b, h); cnt 0: nothing there
__device__ __forceinline__ Rows rows_of(const AttnArgs &a, const Items &it, int b, int h, int x) {
    Rows r;
    r.tail = it.rem && x == 0;
    if (r.tail) {
        r.k = a.p.kt + (int64_t)b * a.p.s_tb + (int64_t)h * a.p.s_th;
        r.v = a.p.vt + (int64_t)b * a.p.s_tb + (int64_t)h * a.p.s_th;
        r.sk = r.sv = a.p.s_tt;
        r.j0 = 0;
        r.cnt = it.rem;
    } else {
        r.k = (const uint16_t *)a.kc.ptr + (int64_t)b * a.kc.s[0] + (int64_t)h * a.kc.s[1];
        r.v = (const uint16_t *)a.vc.ptr + (int64_t)b * a.vc.s[0] + (int64_t)h * a.vc.s[1];
        r.sk = a.kc.s[2];
        r.sv = a.vc.s[2];
        r.j0 = (x - (it.rem ? 1 : 0)) * PG_GROUP;
        r.cnt = a.kc.ptr ? it.n : 0;
    }
    return r;
}
// the seen ones of lane quarter hh's 8 rows
template <bool MASK>
__device__ __forceinline__ uint32_t rows_live(const AttnArgs &a, const Items &it, const Rows &r, int b, int h, int hh) {
    uint32_t seen = 255u >> min(max(r.j0 + 8 * hh + 8 - r.cnt, 0), 8);
    if (MASK && r.tail) seen &= pg_mask_bits(a.p, b, h, it.len / PG_GROUP * PG_GROUP + 8 * hh);
    return seen;
}
// (rows behind the last are read from the last one, so that no load waits for a branch; their
// scores are masked)
template <int D>
__device__ __forceinline__ void rows_k(const Rows &r, int lane, int mt, uint4 *k) {
    const int n16 = lane & 15, hh = lane >> 4;
    const int j = min(r.j0 + 8 * (n16 >> 2) + 4 * mt + (n16 & 3), r.cnt - 1);
    const uint16_t *src = r.k + (int64_t)j * r.sk + (D / 4) * hh;
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb) k[cb] = pg_load16(src + 8 * cb);
}
// V: 8 tokens x D/16 channels of a lane as they lie (0 where not seen), and one channel of
// them as an operand
template <int D>
__device__ __forceinline__ void rows_v(const Rows &r, int lane, uint32_t seen, uint32_t (&vw)[8][D / 32]) {
    constexpr int NC = D / 16;
    const int n16 = lane & 15, hh = lane >> 4;
#pragma unroll
    for (int y = 0; y < 8; ++y) {
        const int j = min(r.j0 + 8 * hh + y, r.cnt - 1);
        const uint16_t *src = r.v + (int64_t)j * r.sv + NC * n16;
        const uint32_t ok = (seen >> y) & 1u ? 0xffffffffu : 0u;
        if constexpr (NC == 8) {
            const uint4 x = pg_load16(src);
            vw[y][0] = x.x & ok; vw[y][1] = x.y & ok; vw[y][2] = x.z & ok; vw[y][3] = x.w & ok;
        } else {
            const uint2 x = pg_load8(src);
            vw[y][0] = x.x & ok; vw[y][1] = x.y & ok;
        }
    }
}
template <int D>
__device__ __forceinline__ uint4 rows_channel(const uint32_t (&vw)[8][D / 32], int ct) {
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t lo = vw[2 * k][ct / 2], hi = vw[2 * k + 1][ct / 2];
        x[k] = ct & 1 ? (lo >> 16) | (hi & 0xffff0000u) : (lo & 0xffffu) | (hi << 16);
    }
    return uint4{x[0], x[1], x[2], x[3]};
}
// A product takes a weight of 0 times a value that is no number to every query row, also to those
// that do not see it.  So under a causal rule such values of the block are 0 in the products, and are
// added as they are to what was written of the rows that see them (each_odd).
// Bits 15 and 31 of odd_halves: this half of w is none.
template <bool BF16>
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
    return ((w & (BF16 ? 0x7f807f80u : 0x7c007c00u)) + (BF16 ? 0x00800080u : 0x04000400u)) & 0x80008000u;
}
__device__ __forceinline__ uint32_t without(uint32_t w, uint32_t odd) { return w & ~(odd | (odd - (odd >> 15))); }
// how many of the block's keys its position t sees: to the end of its causal block, counted from
// the request's first token (len + t has 32 bits, its sum with a block has not)
__device__ __forceinline__ int keys_seen(const AttnArgs &a, const Items &it, int t) {
    if (a.causal <= 0) return it.n;
    const unsigned in = ((unsigned)it.len + (unsigned)t) % (unsigned)a.causal;    // its place in the block
    return (int)min((unsigned)it.n, (unsigned)t + ((unsigned)a.causal - in));
}
// the tokens of an item behind the packed groups that a row sees which sees `keys` of the block's
__device__ __forceinline__ uint32_t causal_live(const Rows &r, int keys, int hh, uint32_t live) {
    return r.tail ? live : live & (255u >> min(max(r.j0 + 8 * hh + 8 - keys, 0), 8));
}

// a row tile's running softmax and output: lane (n = lane & 15, h = lane >> 4) holds row n,
// channels (D/16)(4 h + r) + ct in acc[ct][r]; the row's reference m and, in every
// component of l, its sum of weights (a product with ones: the sum of what is multiplied)
template <int D>
struct Tile {
    f32x4_t acc[D / 16], l, z;      // z (f16, few rows): the zeros' part of the lane's channels
    float m;
};
template <int D>
__device__ __forceinline__ void clear(Tile<D> &t) {
#pragma unroll
    for (int ct = 0; ct < D / 16; ++ct) t.acc[ct] = f32x4_t{};
    t.l = t.z = f32x4_t{};
    t.m = -P_NEW;
}

// max of three without the quieting that fmaxf puts before each of its arguments
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}
__device__ __forceinline__ float max8(const float (&x)[8]) {
    return max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], x[7]));
}

// scores s (x c -> exponents of 2) of a lane's 8 tokens -> weights; live (where masked): bit i =
// token i is seen.  Moves the row's reference where needed; lo: P_FIRST for the first item, then P_MIN.
template <int D>
__device__ __forceinline__ void softmax8(Tile<D> &t, const f32x4_t &s0, const f32x4_t &s1, float c, float lo, bool masked,
                                         uint32_t live, float (&p)[8]) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf(i < 4 ? s0[i & 3] : s1[i & 3], c, -t.m);
    if (masked) {
        const uint32_t l = (uint32_t)hidden((int)live);   // (its bits are looked at in here only)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (l >> i) & 1u ? x[i] : -INFINITY;
    }
    const float mx = max8(x);
    if (__any((mx > P_MAX) | (mx < lo))) {
        // (what is done to a row depends on its own scores alone)
        const float top = max_rows(mx);
        const bool out = top > P_MAX || -max_rows(-mx) < lo;
        const bool move = out && (top > P_NEW || (top < P_LOW && top > -INFINITY));
        if (__any(move)) {
            const float f = t.l[0] == 0.f ? 0.f : __builtin_amdgcn_exp2f(P_NEW - top);
            const bool fits = move && t.l[0] * f < P_SUM;
            const float g = fits ? f : 1.0f;
#pragma unroll
            for (int ct = 0; ct < D / 16; ++ct) t.acc[ct] *= g;
            t.l *= g;
            t.z *= g;
            t.m = fits ? t.m + (top - P_NEW) : t.m;
            // (what is dead stays at -inf, whatever its score)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = x[i] == -INFINITY ? -INFINITY : __builtin_fmaf(i < 4 ? s0[i & 3] : s1[i & 3], c, -t.m);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(x[i]);
}
// a row that saw nothing says so, when its sums are to be joined with others'
template <int D>
__device__ __forceinline__ void settle(Tile<D> &t) {
    if (t.l[0] == 0.f) t.m = NO_MAX;
}

__device__ __forceinline__ f16x8_t as_f16(const float (&p)[8]) {
    f16x8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (_Float16)p[i];
    return r;
}
__device__ __forceinline__ f16x8_t ones_f16() {
    f16x8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (_Float16)1.0f;
    return r;
}

// weights as a sum of two f16 (22 bits; below 2^-14: the first one's absolute 2^-25)
__device__ __forceinline__ void as_two_f16(const float (&p)[8], f16x8_t &hi, f16x8_t &lo) {
    hi = as_f16(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = (_Float16)(p[i] - (float)hi[i]);
}

// 16-bit rows as they are, with each weight as a sum of two of their type
template <bool BF16>
struct Probs {
    f16x8_t hi, lo;
};
template <>
struct Probs<true> {
    b16x8_t hi, lo;
};
template <int CB, bool BF16>
__device__ __forceinline__ f32x4_t rows_scores(const uint4 *k, const uint4 *q) {
    f32x4_t s{};
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        if constexpr (BF16) s = mfma16(__builtin_bit_cast(b16x8_t, k[cb]), __builtin_bit_cast(b16x8_t, q[cb]), s);
        else s = mfma16(__builtin_bit_cast(f16x8_t, k[cb]), __builtin_bit_cast(f16x8_t, q[cb]), s);
    }
    return s;
}
template <int D, bool BF16>
__device__ __forceinline__ Probs<BF16> rows_probs(Tile<D> &t, const f32x4_t &s0, const f32x4_t &s1, float c, float lo, uint32_t live) {
    Probs<BF16> r;
    float p[8];
    softmax8(t, s0, s1, c, lo, true, live, p);
    if constexpr (BF16) {
        b16x8_t one;
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            r.hi[y] = (__bf16)p[y];
            r.lo[y] = (__bf16)(p[y] - (float)r.hi[y]);
            one[y] = (__bf16)1.0f;
        }
        t.l = mfma16(one, r.lo, mfma16(one, r.hi, t.l));
    } else {
        as_two_f16(p, r.hi, r.lo);
        t.l = mfma16(ones_f16(), r.lo, mfma16(ones_f16(), r.hi, t.l));
    }
    return r;
}
__device__ __forceinline__ f32x4_t rows_values(uint4 v, const Probs<true> &p, f32x4_t acc) {
    const b16x8_t x = __builtin_bit_cast(b16x8_t, v);
    return mfma16(x, p.lo, mfma16(x, p.hi, acc));
}
__device__ __forceinline__ f32x4_t rows_values(uint4 v, const Probs<false> &p, f32x4_t acc) {
    const f16x8_t x = __builtin_bit_cast(f16x8_t, v);
    return mfma16(x, p.lo, mfma16(x, p.hi, acc));
}

// ---- Q of one row tile as B operands: lane (n, h) = row n, channels (D/4) h + 8 cb + (0..7);
// rows behind the request's new tokens are zero
// (WORDS: as they lie there, where such rows are left out later)
// t0: position of the segment's first
template <int D, bool SEL, bool WORDS = false>
__device__ __forceinline__ void load_q(const AttnArgs &a, int b, int h, int t0, int row, int n, int hh, uint4 *q) {
    const int rc = min(row, a.R - 1), g = rc / positions<SEL>(a), t = (SEL ? t0 : 0) + rc - g * positions<SEL>(a);
    const uint32_t ok = WORDS || (row < a.R && t < n) ? 0xffffffffu : 0u;
    const uint16_t *src = (const uint16_t *)a.q.ptr + (int64_t)b * a.q.s[0] + (int64_t)(h * a.G + g) * a.q.s[1] +
                          (int64_t)(SEL ? min(t, a.T - 1) : t) * a.q.s[2] + (D / 4) * hh;
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb) {
        const uint4 x = pg_load16(src + 8 * cb);
        q[cb] = uint4{x.x & ok, x.y & ok, x.z & ok, x.w & ok};
    }
}
// bf16 queries as f16: scaled by a power of two that puts the row's largest in [1, 2), so that
// no query overflows f16 and what underflows is below 2^-24 of it; returns the factor back
template <int D>
__device__ __forceinline__ float q_as_f16(uint4 *q) {
    float mx = 0.f;
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb) {
        const uint32_t w[4] = {q[cb].x, q[cb].y, q[cb].z, q[cb].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
    }
    mx = max_rows(mx);
    const int e = min(max((int)(__float_as_uint(mx) >> 23 & 255u) - 127, -100), 100);
    const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb) {
        uint32_t w[4] = {q[cb].x, q[cb].y, q[cb].z, q[cb].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x2_t v = {(_Float16)(__uint_as_float(w[i] << 16) * down),
                               (_Float16)(__uint_as_float(w[i] & 0xffff0000u) * down)};
            w[i] = __builtin_bit_cast(uint32_t, v);
        }
        q[cb] = uint4{w[0], w[1], w[2], w[3]};
    }
    return up;
}

// ---- the line of items (the host sees to it that its length fits 31 bits)
struct Stretch {
    int w, s, e, chunk;   // this workgroup's place and its items [s, e); items of a stretch
    int pre;              // items (x HR) of the requests before b
    int b;                // the request in which s lies
    Items it;             // ... and what it has
};
struct ScanShared {
    int wsum[16], b, pre, n, len;
};
// this workgroup's stretch of a line of `total` items; stretches are a multiple of `unit`
__device__ __forceinline__ void cut_line(const AttnArgs &a, Stretch &r, int total, int unit) {
    // stretches of one XCD's workgroups lie next to one another: row groups share its L2
    r.w = (int)(blockIdx.x % 8) * (a.W / 8) + (int)(blockIdx.x / 8);
    const int each = (int)((unsigned)(total + a.W - 1) / (unsigned)a.W);
    r.chunk = max((each + unit - 1) / unit, 1) * unit;
    r.s = r.w * r.chunk;
    r.e = min(r.s + r.chunk, total);
}
// Items of all requests, by a scan of the lengths in every workgroup (8 B a request, from L2): of
// up to 64 requests in every wave, without a barrier
template <int THREADS>
__device__ __forceinline__ Stretch find_stretch(const AttnArgs &a, ScanShared &sh, int unit) {
    constexpr int NW = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Stretch r;
    if (a.B <= 64) {
        const Items own = lane < a.B ? items_of(a, lane) : Items{};
        const int inc = (int)ma_wave_prefix_u32((uint32_t)own.items);
        cut_line(a, r, __builtin_amdgcn_readlane(inc, 63) * a.HR, unit);
        const int want = (int)((unsigned)r.s / (unsigned)a.HR);
        // (behind the line's end no lane is found, and nothing is looked at)
        const uint64_t here = __ballot(want >= inc - own.items && want < inc);
        const int l = here ? __ffsll((unsigned long long)here) - 1 : 0;
        r.b = l;
        r.pre = __builtin_amdgcn_readlane(inc - own.items, l);
        r.it = items_from<false>(a, __builtin_amdgcn_readlane(own.n, l), __builtin_amdgcn_readlane(own.len, l));
        return r;
    }
    const int per = (a.B + THREADS - 1) / THREADS, first = tid * per;
    int sum = 0;
    Items own{};   // of this thread's first request
    for (int i = 0; i < per; ++i)
        if (first + i < a.B) {
            const Items it = items_of(a, first + i);
            if (i == 0) own = it;
            sum += it.items;
        }
    const int inc = (int)ma_wave_prefix_u32((uint32_t)sum);
    if (lane == 63) sh.wsum[wave] = inc;
    __syncthreads();
    int before = inc - sum, total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        if (w < wave) before += sh.wsum[w];
        total += sh.wsum[w];
    }
    cut_line(a, r, uniform(total) * a.HR, unit);
    const int want = (int)((unsigned)r.s / (unsigned)a.HR);
    if (want >= before && want < before + sum) {
        int pre = before, b = first;
        while (want >= pre + own.items) {
            pre += own.items;
            own = items_of(a, ++b);
        }
        sh.b = b;
        sh.pre = pre;
        sh.n = own.n;
        sh.len = own.len;
    }
    __syncthreads();
    r.b = uniform(sh.b);
    r.pre = uniform(sh.pre);
    r.it = items_from<false>(a, uniform(sh.n), uniform(sh.len));
    return r;
}

// the part of a segment that lies in a stretch
struct Part {
    int h, rg, hr, i0, i1;   // its items of work [i0, i1); rg: the row group of the head's (SEL: of the run's)
    int run, t0;             // SEL: the run and its first position; else 0
    int entry;               // ... its list's entry of the lane's number, and
    uint16_t touched[4];     // what asked for its 16-bit rows early
    int next;                // where the stretch goes on
    bool first, whole;       // the segment begins here; all of it lies here
    int slot;                // of its partial, where it is not whole: the first or the last of the stretch
};
// items of work before place i of a segment, whose first `start` items are none (one of 16-bit rows lies
// where it begins)
__device__ __forceinline__ int work_before(const AttnArgs &a, const Items &it, int start, int i) {
    const int u = max(i - start, 0), over = u - it.ng - a.rows0;
    return over <= 0 ? min(u, it.ng) : it.ng + ((over + (1 << a.dense) - 1) >> a.dense);
}
__device__ __forceinline__ Part part_of(const AttnArgs &a, const Stretch &st, int pos) {
    Part p;
    const int rel = pos - a.HR * st.pre;
    p.hr = (int)((unsigned)rel / (unsigned)st.it.items);
    const int i0 = rel - p.hr * st.it.items, i1 = min(st.it.items, i0 + (st.e - pos));
    p.h = a.RG == 1 ? p.hr : (int)((unsigned)p.hr / (unsigned)a.RG);
    p.rg = p.hr - p.h * a.RG;
    p.next = pos + i1 - i0;
    p.first = i0 == 0;
    p.whole = i0 == 0 && i1 == st.it.items;
    p.i0 = work_before(a, st.it, START, i0);
    p.i1 = work_before(a, st.it, START, i1);
    p.slot = 2 * st.w + (pos > st.s ? 1 : 0);
    return p;
}
// The segment's first stretch says what the merge needs of it: (first slot, stretches, first
// workgroup), or no stretches where it is whole.
__device__ __forceinline__ void note_segment(const AttnArgs &a, const Stretch &st, const Part &p, int pos) {
    if (!p.first || threadIdx.x != 0) return;
    const int n = p.whole ? 0 : (int)((unsigned)(pos + st.it.items - 1) / (unsigned)st.chunk) - st.w + 1;
    a.desc[(int64_t)st.b * a.HR + p.hr] = int4{p.slot, n, st.w, 0};
}
__device__ __forceinline__ void next_part(const AttnArgs &a, Stretch &st, const Part &p, int &pos) {
    pos = p.next;
    if (pos >= st.e || pos - a.HR * st.pre < a.HR * st.it.items) return;
    st.pre += st.it.items;
    do st.it = items_at(a, ++st.b);
    while (st.it.items == 0);
}

// Over selected blocks every segment holds about as many items as its list, so no line is cut: a segment
// has a.parts workgroups of equal shares, known from the workgroup's number and its request's length.
// (A stretch of one place, or of none where the run lies behind the new tokens.)
template <int D, bool TOUCH>
__device__ __forceinline__ Stretch own_part(const AttnArgs &a, int unit, Part &p) {
    Stretch st{};
    // (workgroups of one XCD next to one another: runs of a head list the same pages)
    const unsigned w = (unsigned)(blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
    const unsigned seg = w / (unsigned)a.parts, part = w - seg * a.parts;
    if (seg >= (unsigned)a.B * a.HR) return st;
    st.b = (int)(seg / (unsigned)a.HR);
    p.hr = (int)(seg - (unsigned)st.b * a.HR);
    p.h = (int)((unsigned)p.hr / (unsigned)a.RG);
    p.rg = p.hr - p.h * a.RG;
    p.run = (int)((unsigned)p.rg / (unsigned)a.RGR);
    p.rg -= p.run * a.RGR;
    p.t0 = p.run * a.run;
    // What needs no length is asked for with it: the list (64 entries, one a lane) and, by one wave of the
    // workgroup that will read them, a word of every line of the tail's and the block's first rows, which
    // come from memory otherwise when nothing is left to do meanwhile.
    const int lane = threadIdx.x & 63;
    p.entry = a.blocks[(((int64_t)st.b * a.H + p.h) * (a.RG / a.RGR) + p.run) * a.count + min(lane, a.count - 1)];
    p.touched[0] = p.touched[1] = p.touched[2] = p.touched[3] = 0;
    if (TOUCH && part == (unsigned)a.parts - 1 && threadIdx.x < 64) {
        const int j = lane >> 1, c = (lane & 1) * (D / 2);
        const int64_t tail = (int64_t)st.b * a.p.s_tb + (int64_t)p.h * a.p.s_th + j * a.p.s_tt + c;
        p.touched[0] = a.p.kt[tail];
        p.touched[1] = a.p.vt[tail];
        if (a.kc.ptr) {
            const int64_t t = min(j, a.T - 1);
            p.touched[2] = ((const uint16_t *)a.kc.ptr)[(int64_t)st.b * a.kc.s[0] + (int64_t)p.h * a.kc.s[1] + t * a.kc.s[2] + c];
            p.touched[3] = ((const uint16_t *)a.vc.ptr)[(int64_t)st.b * a.vc.s[0] + (int64_t)p.h * a.vc.s[1] + t * a.vc.s[2] + c];
        }
    }
    const int n = a.new_lens ? min(max(a.new_lens[st.b], 0), a.T) : a.T, len = min(max(a.p.lengths[st.b], 0), a.max_len);
    if (p.t0 >= n) return st;
    Items it{};
    it.n = n;
    it.len = len;
    st.it = items_from<true>(a, n, len, keys_seen(a, it, min(p.t0 + a.run, n) - 1));
    const int share = max((((st.it.items + a.parts - 1) / a.parts) + unit - 1) / unit, 1) * unit;
    p.first = false;
    p.whole = a.parts == 1;
    p.i0 = work_before(a, st.it, 0, min((int)part * share, st.it.items));
    p.i1 = work_before(a, st.it, 0, min((int)(part + 1) * share, st.it.items));
    p.slot = (int)w;
    st.e = 1;
    return st;
}

// The records of a wave's next 64 packed items, one a lane: items first, first + EVERY, ... below
// last of one (request, head).  Looked up at once, so that no item waits for its table entry
// (a load in the loop also waits for every load before it).  Records are 16-byte aligned: bit 0
// says that the table names no page, and the address is then the pool's first record.
// (SEL: by way of the list's entry, and the group's number, which a mask is looked up by.)
struct Records {
    uint32_t lo, hi;
    int group;
};
template <int D, int EVERY, bool SEL>
__device__ __forceinline__ Records find_records(const AttnArgs &a, const Items &it, int b, int h, int run, int entry,
                                                int first, int last, int lane) {
    const int per = a.p.page_tokens / PG_GROUP;
    int i = first + EVERY * lane;
    uint64_t r = (uint64_t)a.p.pool | 1u;
    bool there = i < last;
    if (SEL) {
        const int e = (int)((unsigned)i / (unsigned)a.m), ng = it.len / PG_GROUP;
        int block = __shfl(entry, min(e, 63));
        if (there && e >= 64) block = a.blocks[(((int64_t)b * a.H + h) * (a.RG / a.RGR) + run) * a.count + e];
        // (a block behind the request's last is none: its first group's number is not computed)
        there = there && block >= 0 && block <= (ng - 1) / a.m;
        i = there ? block * a.m + (i - e * a.m) : 0;
        there = there && i < ng;
    }
    if (there) {
        const int pg = i / per;
        const uint8_t *rec = pg_record(a.p, a.p.table[(int64_t)b * a.p.s_table + pg], i - pg * per, h, 40 * D);
        if (rec) r = (uint64_t)rec;
    }
    return Records{(uint32_t)r, (uint32_t)(r >> 32), i};
}
__device__ __forceinline__ rec_t record_at(const Records &r, int k, bool &dead) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)r.lo, k), hi = (uint32_t)__builtin_amdgcn_readlane((int)r.hi, k);
    dead = lo & 1u;
    return (rec_t)((uint64_t)hi << 32 | (lo & ~1u));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack_out(float x, float y) {
    if constexpr (BF16) return ma_pack_bf16x2(x, y);
    const f16x2_t z = {(_Float16)x, (_Float16)y};
    return __builtin_bit_cast(uint32_t, z);
}
template <bool SEL>
__device__ __forceinline__ uint16_t *out_row(const AttnArgs &a, int b, int h, int t0, int row) {
    const int g = row / positions<SEL>(a), t = (SEL ? t0 : 0) + row - g * positions<SEL>(a);
    return (uint16_t *)a.out.ptr + (int64_t)b * a.out.s[0] + (int64_t)(h * a.G + g) * a.out.s[1] + (int64_t)t * a.out.s[2];
}
// NC channels of a row, to its place in out
template <int NC, bool BF16, bool SEL>
__device__ __forceinline__ void store_out(const AttnArgs &a, int b, int h, int t0, int row, int ch, const float *o) {
    uint16_t *dst = out_row<SEL>(a, b, h, t0, row) + ch;
    uint32_t y[NC / 2];
#pragma unroll
    for (int k = 0; k < NC / 2; ++k) y[k] = pack_out<BF16>(o[2 * k], o[2 * k + 1]);
    if constexpr (NC == 8) pg_store16(dst, uint4{y[0], y[1], y[2], y[3]});
    else pg_store8(dst, uint2{y[0], y[1]});
}

// f(element, value) of every value that is no number, of channels ch + (0 .. n - 1) of the block's rows
// below keys in items [d0, d1).  (Rare: loops that are small beside the code around them.)
template <bool BF16, class F>
__device__ __forceinline__ void each_odd(const AttnArgs &a, const Items &it, int b, int h, int d0, int d1, int keys, int ch,
                                         int n, F f) {
#pragma unroll 1
    for (int i = d0; i < d1; ++i) {
        const Rows r = rows_of(a, it, b, h, i - it.ng);
        const int end = r.tail ? 0 : min(min(r.j0 + PG_GROUP, r.cnt), keys);
#pragma unroll 1
        for (int j = r.j0; j < end; ++j)
#pragma unroll 1
            for (int e = 0; e < n; ++e) {
                const uint16_t v = r.v[(int64_t)j * r.sv + ch + e];
                if (odd_halves<BF16>(v)) f(e, BF16 ? ma_bf16_to_f32(v) : ma_f16_to_f32(v));
            }
    }
}
// ... added to a tile's sums, of a wave's items d0, d0 + NW, ...
template <int D, bool BF16, int NW>
__device__ __forceinline__ void add_odd(const AttnArgs &a, const Items &it, int b, int h, int d0, int d1, int keys, int hh,
                                        Tile<D> &t) {
    constexpr int NC = D / 16;
#pragma unroll 1
    for (int i = d0; i < d1; i += NW) {
        const Rows r = rows_of(a, it, b, h, i - it.ng);
        const int end = r.tail ? 0 : min(r.j0 + PG_GROUP, r.cnt);
#pragma unroll 1
        for (int j = r.j0; j < end; ++j)
#pragma unroll
            for (int e = 0; e < D / 4; ++e) {
                const uint16_t v = r.v[(int64_t)j * r.sv + (D / 4) * hh + e];
                t.acc[e % NC][e / NC] += odd_halves<BF16>(v) && j < keys ? (BF16 ? ma_bf16_to_f32(v) : ma_f16_to_f32(v)) : 0.f;
                if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);     // (few registers: none of this is in a hurry)
            }
    }
}
// ... added to an element of out
template <bool BF16>
__device__ __forceinline__ void add_to(uint16_t &x, float v) {
    x = (uint16_t)pack_out<BF16>((BF16 ? ma_bf16_to_f32(x) : ma_f16_to_f32(x)) + v, 0.f);
}

// ------------------------------------------------------------------ few rows
// NT row tiles of 16; the four waves of a workgroup take a segment's items in turn, each with
// its own reference, sum and output (registers only, no barrier), and are joined in LDS at
// the segment's end.  A wave's next record is asked for as soon as the registers of this one are
// free: keys behind the scores, values behind the second product.
//
// bound: 40 D bytes a group and head, once.  One token of 64 requests of 700 to 16 384 tokens
// (28 query and 4 KV heads, D 128): 208 MB in 52.3 us with the merge, 4.0 TB/s, where a large copy
// reaches 5.1; 2 requests of 90 000 to 131 072 tokens (32 and 8 heads): 66.3 us, 4.7 TB/s.  Some
// 10 us are no traffic: two launches, the scan, the first record's three loads in a row (length,
// table, words), the join and the merge (one token after prompts of up to 700 tokens: 14.0 us in
// all).  Two records under way a wave were no faster (D 128: 55.2 and 69.0 us).
// f16, whose operands are sums of two: the first two 59.0 and 78.6 us (51.5 and 66 with one rounding
// each, and twice the error): bound by the instructions that unpack.
// Registers: for the two workgroups a CU that are launched (for three, the 16-bit rows' path spilled:
// 52.4 -> 80 us).
template <int D, int NT>
struct FewShared {
    static constexpr int OS = D + 4;                 // row stride of a wave's output rows, f32
    float o[WAVES][16 * OS];
    float m[WAVES][16], l[WAVES][16];
    ScanShared scan;
};

template <int D, int NT, bool BF16, bool MASK, bool SEL, int NW>
__global__ __launch_bounds__(64 * NW, 2) void paged_few_kernel(AttnArgs a) {
    constexpr int CB = D / 32, NC = D / 16;
    __shared__ FewShared<D, NT> sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), n16 = lane & 15, hh = lane >> 4;
    Part own;
    Stretch st = SEL ? own_part<D, true>(a, NW, own) : find_stretch<64 * NW>(a, sh.scan, NW);
    int pos = st.s;
    while (pos < st.e) {
        const Items it = st.it;
        const Part pt = SEL ? own : part_of(a, st, pos);
        const int b = st.b, h = pt.h, row0 = pt.rg * NT * 16, t0 = SEL ? pt.t0 : 0;
        uint4 q[NT][CB];
        float c[NT];
        Tile<D> t[NT];
        // (the queries' loads and the table's are under way together, the first record's behind
        // them while the queries are scaled)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) load_q<D, SEL>(a, b, h, t0, row0 + nt * 16 + (hidden(lane) & 15), it.n, hh, q[nt]);
        const int last = min(pt.i1, it.ng);
        int i = pt.i0 + wave, k = 0;
        Records recs = find_records<D, NW, SEL>(a, it, b, h, SEL ? pt.run : 0, SEL ? own.entry : 0, i, last, lane);
        RawK<D> rk;
        RawV<D> rv;
        bool dead = false;
        int group = i;
        if (i < last) {
            if (SEL && MASK) group = __builtin_amdgcn_readlane(recs.group, 0);
            const rec_t rec = record_at(recs, 0, dead);
            load_k(rk, rec, lane);
            load_v(rv, rec, lane);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            c[nt] = (BF16 ? q_as_f16<D>(q[nt]) : 1.f) * a.sl2;
            clear(t[nt]);
        }
        float lo = P_FIRST;
        for (; i < last; i += NW) {
            if (++k == 64) {
                recs = find_records<D, NW, SEL>(a, it, b, h, SEL ? pt.run : 0, SEL ? own.entry : 0, i + NW, last, lane);
                k = 0;
            }
            // (behind the last one the pool's first record is loaded: no branch around the loads)
            bool dead_next;
            const rec_t next = record_at(recs, k, dead_next);
            f32x4_t s0[NT], s1[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s0[nt] = s1[nt] = f32x4_t{};
            if constexpr (BF16) {
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    const f16x8_t k0 = word_values(rk.k[0][cb], rk.s[cb], rk.z[cb]);
                    const f16x8_t k1 = word_values(rk.k[1][cb], rk.s[cb], rk.z[cb]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const f16x8_t qf = __builtin_bit_cast(f16x8_t, q[nt][cb]);
                        s0[nt] = mfma16(k0, qf, s0[nt]);
                        s1[nt] = mfma16(k1, qf, s1[nt]);
                    }
                }
            } else {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {       // (the zeros are those of all 32 tokens)
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb)
                        s0[nt] = mfma16(__builtin_bit_cast(f16x8_t, rk.z[cb]), __builtin_bit_cast(f16x8_t, q[nt][cb]), s0[nt]);
                    s1[nt] = s0[nt];
                }
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    uint4 s_hi, s_lo;
                    split_scale(rk.s[cb], s_hi, s_lo);
                    f16x8_t h0, l0, h1, l1;
                    word_products(rk.k[0][cb], s_hi, s_lo, h0, l0);
                    word_products(rk.k[1][cb], s_hi, s_lo, h1, l1);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const f16x8_t qf = __builtin_bit_cast(f16x8_t, q[nt][cb]);
                        s0[nt] = mfma16(l0, qf, mfma16(h0, qf, s0[nt]));
                        s1[nt] = mfma16(l1, qf, mfma16(h1, qf, s1[nt]));
                    }
                }
            }
            load_k(rk, next, lane);
            const bool masked = MASK || dead;
            uint32_t live = dead ? 0u : 255u;
            if (masked) {
                if (MASK) live &= pg_mask_bits(a.p, b, h, (SEL ? group : i) * PG_GROUP + 8 * (hidden(lane) >> 4));
                clear_dead(rv, live);
            }
            f16x8_t pf[NT], pl[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float p[8];
                softmax8(t[nt], s0[nt], s1[nt], c[nt], lo, masked, live, p);
                if constexpr (BF16) pf[nt] = as_f16(p);
                else as_two_f16(p, pf[nt], pl[nt]);
                t[nt].l = mfma16(ones_f16(), pf[nt], t[nt].l);
                if constexpr (!BF16) t[nt].l = mfma16(ones_f16(), pl[nt], t[nt].l);
            }
            lo = P_MIN;
            if constexpr (BF16) {
#pragma unroll
                for (int ct = 0; ct < NC; ++ct) {
                    const f16x8_t vf = word_values(v_word(rv, ct), rv.s, rv.z);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) t[nt].acc[ct] = mfma16(vf, pf[nt], t[nt].acc[ct]);
                }
            } else {
                const f16x8_t z = __builtin_bit_cast(f16x8_t, rv.z);
                uint4 s_hi, s_lo;
                split_scale(rv.s, s_hi, s_lo);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) t[nt].z = mfma16(z, pl[nt], mfma16(z, pf[nt], t[nt].z));
#pragma unroll
                for (int ct = 0; ct < NC; ++ct) {
                    f16x8_t vh, vl;
                    word_products(v_word(rv, ct), s_hi, s_lo, vh, vl);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        t[nt].acc[ct] = mfma16(vl, pf[nt], mfma16(vh, pl[nt], mfma16(vh, pf[nt], t[nt].acc[ct])));
                }
            }
            load_v(rv, next, lane);
            dead = dead_next;
            if (SEL && MASK) group = __builtin_amdgcn_readlane(recs.group, k);
        }
        if constexpr (!BF16) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int ct = 0; ct < NC; ++ct) t[nt].acc[ct] += t[nt].z;
        }
        // the tail and the block's own keys
        if (SEL) asm volatile("" ::"v"(own.touched[0]), "v"(own.touched[1]), "v"(own.touched[2]), "v"(own.touched[3]));
        bool odd = false;
        const int rows_at = i;
        for (; i < pt.i1; i += NW) {
            const Rows r = rows_of(a, it, b, h, i - it.ng);
            if (r.cnt == 0) continue;
            const int l = hidden(lane), lh = l >> 4;
            const uint32_t seen = rows_live<MASK>(a, it, r, b, h, lh);
            f32x4_t s[2][NT];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                uint4 k[CB];
                rows_k<D>(r, l, mt, k);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    uint4 qr[CB];
                    load_q<D, SEL>(a, b, h, t0, row0 + nt * 16 + (l & 15), it.n, lh, qr);
                    s[mt][nt] = rows_scores<CB, BF16>(k, qr);
                }
            }
            Probs<BF16> p[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                p[nt] = rows_probs<D, BF16>(t[nt], s[0][nt], s[1][nt], a.sl2, lo,
                                            causal_live(r, keys_seen(a, it, t0 + (row0 + nt * 16 + (l & 15)) % positions<SEL>(a)), lh, seen));
            lo = P_MIN;
            // (the values' loads stay behind the scores' registers: ahead of them the main loop spilled)
            __builtin_amdgcn_sched_barrier(0);
            uint32_t vw[8][NC / 2];
            rows_v<D>(r, l, seen, vw);
            if (a.causal > 0 && !r.tail) {
                uint32_t any = 0;
#pragma unroll
                for (int y = 0; y < 8; ++y)
#pragma unroll
                    for (int z = 0; z < NC / 2; ++z) any |= odd_halves<BF16>(vw[y][z]);
                if (__any(any)) {
                    odd = true;
#pragma unroll
                    for (int y = 0; y < 8; ++y)
#pragma unroll
                        for (int z = 0; z < NC / 2; ++z) vw[y][z] = without(vw[y][z], odd_halves<BF16>(vw[y][z]));
                }
            }
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) {
                const uint4 v = rows_channel<D>(vw, ct);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) t[nt].acc[ct] = rows_values(v, p[nt], t[nt].acc[ct]);
            }
        }
        if (odd) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) add_odd<D, BF16, NW>(a, it, b, h, rows_at, pt.i1, keys_seen(a, it, t0 + (row0 + nt * 16 + n16) % positions<SEL>(a)), hh, t[nt]);
        }
        // the waves' parts joined; whole segments written out, cut ones left as a partial
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            settle(t[nt]);
            if constexpr (NW > WAVES) {       // the upper half's into the lower half's first
                __syncthreads();
                if (wave >= WAVES) {
                    if (hh == 0) {
                        sh.m[wave - WAVES][n16] = t[nt].m;
                        sh.l[wave - WAVES][n16] = t[nt].l[0];
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int ct = 0; ct < NC; ct += 4)
                            *(f32x4_t *)&sh.o[wave - WAVES][n16 * FewShared<D, NT>::OS + NC * (4 * hh + r) + ct] =
                                f32x4_t{t[nt].acc[ct][r], t[nt].acc[ct + 1][r], t[nt].acc[ct + 2][r], t[nt].acc[ct + 3][r]};
                }
                __syncthreads();
                if (wave < WAVES) {
                    const float m = fmaxf(t[nt].m, sh.m[wave][n16]);
                    const float f = __builtin_amdgcn_exp2f(t[nt].m - m), g = __builtin_amdgcn_exp2f(sh.m[wave][n16] - m);
                    t[nt].l[0] = t[nt].l[0] * f + sh.l[wave][n16] * g;
                    t[nt].m = m;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int ct = 0; ct < NC; ct += 4) {
                            const f32x4_t v = *(const f32x4_t *)&sh.o[wave][n16 * FewShared<D, NT>::OS + NC * (4 * hh + r) + ct];
#pragma unroll
                            for (int z = 0; z < 4; ++z) t[nt].acc[ct + z][r] = t[nt].acc[ct + z][r] * f + v[z] * g;
                        }
                }
            }
            __syncthreads();
            if (NW > WAVES && wave >= WAVES) {
                __syncthreads();
                continue;
            }
            if (hh == 0) {
                sh.m[wave][n16] = t[nt].m;
                sh.l[wave][n16] = t[nt].l[0];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int ct = 0; ct < NC; ct += 4) {
                    const f32x4_t v = {t[nt].acc[ct][r], t[nt].acc[ct + 1][r], t[nt].acc[ct + 2][r],
                                       t[nt].acc[ct + 3][r]};
                    *(f32x4_t *)&sh.o[wave][n16 * FewShared<D, NT>::OS + NC * (4 * hh + r) + ct] = v;
                }
            __syncthreads();
            const int r = hidden(tid) >> 4, x = tid & 15;      // row, channels NC x + (0 .. NC - 1)
            const int row = row0 + nt * 16 + r;
            if (row < a.R) {
                float m = sh.m[0][r];
#pragma unroll
                for (int v = 1; v < WAVES; ++v) m = fmaxf(m, sh.m[v][r]);
                float lt = 0.f, o[NC];
#pragma unroll
                for (int k = 0; k < NC; ++k) o[k] = 0.f;
#pragma unroll
                for (int v = 0; v < WAVES; ++v) {
                    const float f = __builtin_amdgcn_exp2f(sh.m[v][r] - m);
                    lt += sh.l[v][r] * f;
#pragma unroll
                    for (int k = 0; k < NC; k += 4) {
                        const f32x4_t y = *(const f32x4_t *)&sh.o[v][r * FewShared<D, NT>::OS + NC * x + k];
#pragma unroll
                        for (int z = 0; z < 4; ++z) o[k + z] += y[z] * f;
                    }
                }
                if (pt.whole) {
                    const float inv = lt == 0.f ? 0.f : 1.f / lt;
#pragma unroll
                    for (int k = 0; k < NC; ++k) o[k] *= inv;
                    if (t0 + row % positions<SEL>(a) < it.n) store_out<NC, BF16, SEL>(a, b, h, t0, row, NC * x, o);
                } else {
                    const int64_t at = (int64_t)pt.slot * (NT * 16) + nt * 16 + r;
                    if (x == 0) {
                        a.wm[at] = m;
                        a.wl[at] = lt;
                    }
#pragma unroll
                    for (int k = 0; k < NC; k += 4)
                        *(f32x4_t *)&a.wo[at * D + NC * x + k] = f32x4_t{o[k], o[k + 1], o[k + 2], o[k + 3]};
                }
            }
        }
        if (SEL) break;
        note_segment(a, st, pt, pos);
        next_part(a, st, pt, pos);
    }
}

// ------------------------------------------------------------------ many rows
// 8 waves over 2 RW row tiles of 16: wave w takes row tiles 2 (w % RW) and + 1 and, of a step's
// 4 items, those of w / RW modulo 8 / RW.  A step's K and V become operands in LDS once for all
// rows: wave w unpacks the keys (w even) or values (w odd) of item w / 2 of the next step into
// the other buffer while it computes, one barrier a step.  An item's 16 operands lie as the
// lanes read them (1 KB each, no bank conflicts).
//
// bound: the matrix cores, 4 D operations a row and token.  512 new tokens of 2 requests of 6 000
// to 16 384 tokens (28 query and 4 KV heads, D 128): 205 GFLOP in 222 to 239 us; each 8 192 tokens
// more add 104 us, 1.15 PFLOP/s, where a large library product reaches 1.19.  The rest is start
// and end: partials of 256 rows (128 KB) written and read again, and 16-bit rows, which are not
// pipelined (a step of up to four items is 5 us).  32 new tokens of 8 requests: 53 us, of which
// some 25 are that.  Measured and not kept (chunk, then 251 us): two tiles half an item apart, so
// that one's exponentials lie under the other's products: 268; 4 tiles a wave and one wave a
// SIMD: 368 (operands copied between the two register files); the next 16-bit rows under way in
// registers: 20 % slower, the main loop spilled; a SIMD's two waves unpacking in turn: no gain.
// f16: twice the products and 3 items a step, 32 new tokens of 8 requests 85.6 us (49.8 with one
// rounding each, and twice the error).
// Registers: at D 128 all 256 are in use and 4 to 17 spilled.  What lives across the packed loop
// costs at once: 40 to 60 spilled were 53 -> 61 us (block).
constexpr int MWAVES = 8;
constexpr int step_of(int D, bool BF16) { return D == 128 && !BF16 ? 3 : 4; }      // (what the LDS holds twice)

// place of row rt's channels (D/16) x + (0 .. 3) in a partial: as the tile's wave holds them,
// [tile][channels mod 4][4 channels] of 64 lanes' 16 bytes
template <int D>
__device__ __forceinline__ int partial_at(int rt, int x) {
    return ((rt >> 4) * (D / 16) + (x & 3) * (D / 64)) * 256 + ((x >> 2) * 16 + (rt & 15)) * 4;
}

template <int D, bool BF16>
struct ManyShared {
    // operands of an item: K [2][D/32], V [D/16], and what rounding left of K (f16)
    static constexpr int OPS = 2 * (D / 32) + D / 16 + (BF16 ? 0 : 2 * (D / 32)), STEP = step_of(D, BF16);
    uint4 op[2][STEP][OPS][64];
    uint32_t live[2][STEP];                               // bit j: the item's token j is seen
    uint32_t odd[2][STEP];                                // one of the item's values is no number (causal calls)
    ScanShared scan;
};

template <int D, int RW, bool BF16, bool MASK, bool SEL>
__global__ __launch_bounds__(512, 2) void paged_many_kernel(AttnArgs a) {
    constexpr int CB = D / 32, NC = D / 16, TW = MWAVES / RW, STEP = step_of(D, BF16), LEFT = 2 * CB + NC;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    ManyShared<D, BF16> &sh = *(ManyShared<D, BF16> *)lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), hh = lane >> 4;
    const int rw = wave % RW, tw = wave / RW;
    const int si = wave >> 1;              // the item of a step that this wave unpacks (STEP and more: none)
    const bool sv = wave & 1;              // its values (else its keys)
    Part own;
    Stretch st = SEL ? own_part<D, false>(a, STEP, own) : find_stretch<512>(a, sh.scan, STEP);
    int pos = st.s;
    while (pos < st.e) {
        const Items it = st.it;
        const Part pt = SEL ? own : part_of(a, st, pos);
        const int b = st.b, h = pt.h, row0 = pt.rg * (2 * RW * 16) + rw * 32, t0 = SEL ? pt.t0 : 0;
        const bool busy = row0 < a.R;      // this wave has rows
        uint4 q[2][CB];
        float c[2];
        Tile<D> t[2];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) load_q<D, SEL>(a, b, h, t0, row0 + nt * 16 + (hidden(lane) & 15), it.n, hh, q[nt]);
        // the seen tokens of an item, from its values' wave
        auto note_live = [&](int x, uint32_t live) {
            uint32_t all = 0;
#pragma unroll
            for (int y = 0; y < 4; ++y) all |= (uint32_t)__builtin_amdgcn_readlane((int)live, 16 * y) << (8 * y);
            if (lane == 0) sh.live[x & 1][si] = all;
        };

        // ---- packed groups
        const int last = min(pt.i1, it.ng), steps = max(last - pt.i0 + STEP - 1, 0) / STEP;
        const int poff = sv ? 2 * (32 * (NC * (lane & 15) / 32) + 8 * hh) : (D / 2) * hh;
        RawK<D> raw;
        bool dead = false;
        int group = 0;
        Records recs;
        // the words of step x's item of this wave (behind the last one: of the pool's first record)
        auto fetch = [&](int x) {
            if (si >= STEP) return;
            if (x % 64 == 0) recs = find_records<D, STEP, SEL>(a, it, b, h, SEL ? pt.run : 0, SEL ? own.entry : 0, pt.i0 + x * STEP + si, last, lane);
            if (SEL && MASK) group = __builtin_amdgcn_readlane(recs.group, x % 64);
            const rec_t rec = record_at(recs, x % 64, dead);
            load_either(raw, rec, lane, sv, poff);
        };
        // ... as operands in buffer x & 1
        auto unpack = [&](int x) {
            if (si >= STEP) return;
            uint4(*op)[64] = sh.op[x & 1][si];
            if (!sv) {
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) {
                        if constexpr (BF16) {
                            op[mt * CB + cb][lane] = __builtin_bit_cast(uint4, word_values(raw.k[mt][cb], raw.s[cb], raw.z[cb]));
                        } else {
                            f16x8_t hi, left;
                            word_values2(raw.k[mt][cb], raw.s[cb], raw.z[cb], hi, left);
                            op[mt * CB + cb][lane] = __builtin_bit_cast(uint4, hi);
                            op[LEFT + mt * CB + cb][lane] = __builtin_bit_cast(uint4, left);
                        }
                    }
            } else {
                uint32_t live = dead ? 0u : 255u;
                RawV<D> rv = v_from(raw);
                if (MASK) live &= pg_mask_bits(a.p, b, h, (SEL ? group : pt.i0 + x * STEP + si) * PG_GROUP + 8 * (hidden(lane) >> 4));
                if (MASK || dead) clear_dead(rv, live);
#pragma unroll
                for (int ct = 0; ct < NC; ++ct)
                    op[2 * CB + ct][lane] = __builtin_bit_cast(uint4, word_values(v_word(rv, ct), rv.s, rv.z));
                note_live(x, live);
            }
        };
        if (steps > 0) fetch(0);
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
            c[nt] = (BF16 ? q_as_f16<D>(q[nt]) : 1.f) * a.sl2;
            clear(t[nt]);
        }
        float lo = P_FIRST;
        for (int x = -1; x < steps; ++x) {
            if (x + 1 < steps) {
                unpack(x + 1);
                if (x + 2 < steps) fetch(x + 2);
            }
            const int g1 = busy && x >= 0 ? min(last - pt.i0 - x * STEP, STEP) : 0;
            // the keys' operands of an item come while the one before is multiplied by its values
            f16x8_t kf[2 * CB];
            if (tw < g1) {
#pragma unroll
                for (int y = 0; y < 2 * CB; ++y) kf[y] = __builtin_bit_cast(f16x8_t, sh.op[x & 1][tw][y][lane]);
            }
            for (int g = tw; g < g1; g += TW) {
                const uint4(*op)[64] = sh.op[x & 1][g];
                const uint32_t all = (uint32_t)uniform((int)sh.live[x & 1][g]);
                const uint32_t live = all >> (8 * hh) & 255u;
                f32x4_t s0[2] = {}, s1[2] = {};
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        const f16x8_t qf = __builtin_bit_cast(f16x8_t, q[nt][cb]);
                        s0[nt] = mfma16(kf[cb], qf, s0[nt]);
                        s1[nt] = mfma16(kf[CB + cb], qf, s1[nt]);
                    }
                    if constexpr (!BF16) {
                        const f16x8_t l0 = __builtin_bit_cast(f16x8_t, op[LEFT + cb][lane]);
                        const f16x8_t l1 = __builtin_bit_cast(f16x8_t, op[LEFT + CB + cb][lane]);
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt) {
                            const f16x8_t qf = __builtin_bit_cast(f16x8_t, q[nt][cb]);
                            s0[nt] = mfma16(l0, qf, s0[nt]);
                            s1[nt] = mfma16(l1, qf, s1[nt]);
                        }
                    }
                }
                // the values' operands come while the scores become probabilities
                f16x8_t vf[NC];
#pragma unroll
                for (int ct = 0; ct < NC; ++ct) vf[ct] = __builtin_bit_cast(f16x8_t, op[2 * CB + ct][lane]);
                f16x8_t pf[2], pl[2];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    float p[8];
                    softmax8(t[nt], s0[nt], s1[nt], c[nt], lo, all != 0xffffffffu, live, p);
                    if constexpr (BF16) pf[nt] = as_f16(p);
                    else as_two_f16(p, pf[nt], pl[nt]);
                    t[nt].l = mfma16(ones_f16(), pf[nt], t[nt].l);
                    if constexpr (!BF16) t[nt].l = mfma16(ones_f16(), pl[nt], t[nt].l);
                }
                lo = P_MIN;
                const uint4(*next)[64] = sh.op[x & 1][min(g + TW, STEP - 1)];
#pragma unroll
                for (int y = 0; y < 2 * CB; ++y) kf[y] = __builtin_bit_cast(f16x8_t, next[y][lane]);
#pragma unroll
                for (int ct = 0; ct < NC; ++ct)
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        t[nt].acc[ct] = mfma16(vf[ct], pf[nt], t[nt].acc[ct]);
                        if constexpr (!BF16) t[nt].acc[ct] = mfma16(vf[ct], pl[nt], t[nt].acc[ct]);
                    }
            }
            __syncthreads();
        }

        // ---- the tail and the block's own keys, four items a step too; what no row of the group
        // sees is left out, what none of the wave's sees too
        const int tq = positions<SEL>(a), r1 = min((pt.rg + 1) * (2 * RW * 16), a.R) - 1;
        const int t1 = t0 + (pt.rg * (2 * RW * 16) / tq == r1 / tq ? r1 % tq : tq - 1);
        const int d0 = max(pt.i0, it.ng);
        const int d1 = min(pt.i1, it.ng + (it.rem ? 1 : 0) + (a.kc.ptr ? (keys_seen(a, it, t1) + PG_GROUP - 1) / PG_GROUP : 0));
        int odd = 0;
        if (d0 < d1) {
            const int l = hidden(lane), lh = l >> 4;
            int keys[2];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                const int row = row0 + nt * 16 + (l & 15);
                // (as they are, not as f16; a row that is none is left out when results are stored)
                if (BF16) load_q<D, SEL, true>(a, b, h, t0, row, it.n, lh, q[nt]);
                keys[nt] = keys_seen(a, it, t0 + row % tq);
            }
            for (int i = d0, x = 0; i < d1; i += STEP, ++x) {
                uint32_t any = 0;
                if (si < STEP && i + si < d1) {
                    const Rows r = rows_of(a, it, b, h, i + si - it.ng);
                    uint4(*op)[64] = sh.op[x & 1][si];
                    if (!sv) {
                        uint4 k[2][CB];
#pragma unroll
                        for (int mt = 0; mt < 2; ++mt) rows_k<D>(r, l, mt, k[mt]);
#pragma unroll
                        for (int y = 0; y < 2 * CB; ++y) op[y][l] = k[y / CB][y % CB];
                    } else {
                        const uint32_t live = rows_live<MASK>(a, it, r, b, h, lh);
                        uint32_t w[8][NC / 2];
                        rows_v<D>(r, l, live, w);
#pragma unroll
                        for (int ct = 0; ct < NC; ++ct) {
                            uint4 v = rows_channel<D>(w, ct);
                            if (a.causal > 0 && !r.tail) {
                                const uint32_t o[4] = {odd_halves<BF16>(v.x), odd_halves<BF16>(v.y), odd_halves<BF16>(v.z),
                                                       odd_halves<BF16>(v.w)};
                                any |= o[0] | o[1] | o[2] | o[3];
                                v = uint4{without(v.x, o[0]), without(v.y, o[1]), without(v.z, o[2]), without(v.w, o[3])};
                            }
                            op[2 * CB + ct][l] = v;
                        }
                        note_live(x, live);
                    }
                }
                if (a.causal > 0 && sv && si < STEP) {
                    const bool o = __any(any);
                    if (l == 0) sh.odd[x & 1][si] = o;
                }
                __syncthreads();
                if (a.causal > 0) {
                    uint32_t o = 0;
#pragma unroll
                    for (int y = 0; y < STEP; ++y) o |= sh.odd[x & 1][y];
                    odd |= uniform((int)o);
                }
                const int g1 = busy ? min(d1 - i, STEP) : 0;
                for (int g = tw; g < g1; g += TW) {
                    const Rows r = rows_of(a, it, b, h, i + g - it.ng);
                    const uint4(*op)[64] = sh.op[x & 1][g];
                    const uint32_t all = (uint32_t)uniform((int)sh.live[x & 1][g]) >> (8 * lh) & 255u;
                    const uint32_t see[2] = {causal_live(r, keys[0], lh, all), causal_live(r, keys[1], lh, all)};
                    if (!__any(see[0] | see[1])) continue;
                    f32x4_t s[2][2];
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        uint4 k[CB];
#pragma unroll
                        for (int cb = 0; cb < CB; ++cb) k[cb] = op[mt * CB + cb][l];
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt) s[nt][mt] = rows_scores<CB, BF16>(k, q[nt]);
                    }
                    Probs<BF16> p[2];
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
                        p[nt] = rows_probs<D, BF16>(t[nt], s[nt][0], s[nt][1], a.sl2, lo, see[nt]);
                    lo = P_MIN;
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int ct = 0; ct < NC; ++ct) {
                        const uint4 v = op[2 * CB + ct][l];
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt) t[nt].acc[ct] = rows_values(v, p[nt], t[nt].acc[ct]);
                    }
                }
            }
            __syncthreads();
        }
        settle(t[0]);
        settle(t[1]);
        // waves that share rows joined (lane by lane, through the operands' space), then each row
        // tile written out or left as a partial
        if constexpr (TW > 1) {
            constexpr int NV = NC * 4 + 2;
            float *lw = (float *)sh.op;
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                if (tw > 0) {
                    float *dst = lw + (wave * NV) * 64 + lane;
#pragma unroll
                    for (int ct = 0; ct < NC; ++ct)
#pragma unroll
                        for (int r = 0; r < 4; ++r) dst[(ct * 4 + r) * 64] = t[nt].acc[ct][r];
                    dst[NC * 4 * 64] = t[nt].l[0];
                    dst[(NC * 4 + 1) * 64] = t[nt].m;
                }
                __syncthreads();
                if (tw == 0) {
                    float m = t[nt].m;
#pragma unroll
                    for (int v = 1; v < TW; ++v) m = fmaxf(m, lw[((v * RW + rw) * NV + NC * 4 + 1) * 64 + lane]);
                    const float f0 = __builtin_amdgcn_exp2f(t[nt].m - m);
                    t[nt].l[0] *= f0;
#pragma unroll
                    for (int ct = 0; ct < NC; ++ct) t[nt].acc[ct] *= f0;
#pragma unroll
                    for (int v = 1; v < TW; ++v) {
                        const float *src = lw + ((v * RW + rw) * NV) * 64 + lane;
                        const float f = __builtin_amdgcn_exp2f(src[(NC * 4 + 1) * 64] - m);
                        t[nt].l[0] += src[NC * 4 * 64] * f;
#pragma unroll
                        for (int ct = 0; ct < NC; ++ct)
#pragma unroll
                            for (int r = 0; r < 4; ++r) t[nt].acc[ct][r] += src[(ct * 4 + r) * 64] * f;
                    }
                    t[nt].m = m;
                }
                __syncthreads();
            }
        }
        if (tw == 0 && busy) {
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                const int row = row0 + nt * 16 + (hidden(lane) & 15);
                if (row >= a.R) continue;
                const float l = t[nt].l[0];
                if (pt.whole) {
                    if (t0 + row % tq >= it.n) continue;
                    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float o[NC];
#pragma unroll
                        for (int ct = 0; ct < NC; ++ct) o[ct] = t[nt].acc[ct][r] * inv;
                        store_out<NC, BF16, SEL>(a, b, h, t0, row, NC * (4 * hh + r), o);
                    }
                } else {
                    const int64_t slot = (int64_t)pt.slot * (2 * RW * 16);
                    const int rt = rw * 32 + nt * 16 + (hidden(lane) & 15);
                    if (hh == 0) {
                        a.wm[slot + rt] = t[nt].m;
                        a.wl[slot + rt] = l;
                    }
                    float *dst = a.wo + slot * D + partial_at<D>(rt, 4 * hh);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int ct = 0; ct < NC; ct += 4)
                            *(f32x4_t *)&dst[(r * (NC / 4) + ct / 4) * 256] =
                                f32x4_t{t[nt].acc[ct][r], t[nt].acc[ct + 1][r], t[nt].acc[ct + 2][r], t[nt].acc[ct + 3][r]};
                }
            }
            if (odd) {
                asm volatile("" ::: "memory");      // (what the lane just stored is read again as other types)
#pragma unroll 1
                for (int rt = rw * 32 + (lane & 15); rt < rw * 32 + 32; rt += 16) {
                    const int row = row0 - rw * 32 + rt;
                    if (row >= a.R || (pt.whole && t0 + row % tq >= it.n)) continue;
                    float *dst = a.wo + (int64_t)pt.slot * (2 * RW * 16) * D + partial_at<D>(rt, 4 * hh);
                    each_odd<BF16>(a, it, b, h, d0, d1, keys_seen(a, it, t0 + row % tq), (D / 4) * hh, D / 4, [&](int e, float v) {
                        if (pt.whole) add_to<BF16>(out_row<SEL>(a, b, h, t0, row)[(D / 4) * hh + e], v);
                        else dst[(e / 4) * 256 + e % 4] += v;
                    });
                }
            }
        }
        if (SEL) break;
        note_segment(a, st, pt, pos);
        next_part(a, st, pt, pos);
    }
}

// ------------------------------------------------------------------ merge
// Partials of a cut segment, joined: the first lies in desc.x, the stretch after workgroup w's
// in slot 2 (w + 1), and so on.  A workgroup joins 64 pairs of a row and D/16 channels; each of its
// waves takes every eighth (many rows: fourth) partial, and they are joined in LDS, in a fixed
// order.  Partials of few rows lie row by row (4 rows of 16 pairs), those of many as their waves
// hold them (TILES: 16 rows of a tile's 4 pairs, 256 contiguous bytes a load).
//
// bound: latency (desc, then partials), many rows: their bytes (8 requests' 224 rows of 4 heads, 33
// MB in 8.9 us).  Waves of few rows: one token of 2 long requests, some 30 partials a segment, 66.1
// us with 8, 67.3 with 4, 66.1 with 16; of 64 requests 52.8, 52.3, 53.7.  Of many: 32 tokens of 8
// requests 50.9 us with 4, 51.2 with 2, 51.9 with 8.  Of many over selected blocks, two partials mostly:
// the merge of 128 segments 10.3 us with 4, 8.5 with 2, 7.4 with 1.
constexpr int merge_waves(bool tiles, bool sel) { return tiles ? (sel ? 1 : 4) : 8; }

template <int D, bool BF16, bool TILES, bool SEL>
__global__ __launch_bounds__(64 * merge_waves(TILES, SEL)) void paged_merge_kernel(AttnArgs a, int rows) {
    constexpr int NC = D / 16, GR = merge_waves(TILES, SEL);
    __shared__ float sm[GR][64], sl[GR][64];
    __shared__ f32x4_t so[GR][NC / 4][64];
    const int b = blockIdx.x / a.HR, hr = blockIdx.x - b * a.HR;
    const int n = a.new_lens ? min(max(a.new_lens[b], 0), a.T) : a.T;
    const int h = hr / a.RG, run = SEL ? (hr - h * a.RG) / a.RGR : 0, rg = hr - h * a.RG - (SEL ? run * a.RGR : 0);
    const int t0 = SEL ? run * a.run : 0;
    const int4 d = SEL ? int4{(int)blockIdx.x * a.parts, a.parts, 0, 0} : a.desc[blockIdx.x];
    if ((n <= t0) | (d.y == 0)) return;      // (no new tokens: nobody wrote its segments)
    const int grp = threadIdx.x >> 6, u = threadIdx.x & 63;
    const int x = TILES ? 4 * (blockIdx.y & 3) + (u >> 4) : u & 15;
    const int rt = TILES ? 16 * (blockIdx.y >> 2) + (u & 15) : 4 * blockIdx.y + (u >> 4);
    const int row = rg * rows + rt;
    const int off = TILES ? partial_at<D>(rt, x) : rt * D + NC * x;      // ... of its first 4 channels
    constexpr int next = TILES ? 256 : 4;                                // from 4 channels to the next 4
    float m = NO_MAX, l = 0.f, o[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) o[k] = 0.f;
    if (row < a.R) {
        // two partials a turn, their loads under way together (behind the last one it is loaded again)
        for (int k0 = grp; k0 < d.y; k0 += 2 * GR) {
            float pm[2], pl[2];
            f32x4_t v[2][NC / 4];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int k = min(k0 + z * GR, d.y - 1);
                const int64_t at = (SEL ? (int64_t)d.x + k : k ? 2 * (int64_t)(d.z + k) : (int64_t)d.x) * rows;
                pm[z] = a.wm[at + rt];
                pl[z] = a.wl[at + rt];
#pragma unroll
                for (int y = 0; y < NC / 4; ++y) v[z][y] = *(const f32x4_t *)&a.wo[at * D + off + next * y];
            }
            const bool two = k0 + GR < d.y;
            const float nm = fmaxf(m, two ? fmaxf(pm[0], pm[1]) : pm[0]);
            const float f = __builtin_amdgcn_exp2f(m - nm), g0 = __builtin_amdgcn_exp2f(pm[0] - nm);
            const float g1 = two ? __builtin_amdgcn_exp2f(pm[1] - nm) : 0.f;
            m = nm;
            l = l * f + pl[0] * g0 + pl[1] * g1;
            // (selected, not left out: a branch took the loads with it)
#pragma unroll
            for (int y = 0; y < NC; ++y)
                o[y] = o[y] * f + v[0][y / 4][y % 4] * g0 + (two ? v[1][y / 4][y % 4] : 0.f) * g1;
        }
    }
    sm[grp][u] = m;
    sl[grp][u] = l;
#pragma unroll
    for (int y = 0; y < NC / 4; ++y) so[grp][y][u] = f32x4_t{o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]};
    __syncthreads();
    if (grp != 0) return;
    m = sm[0][u];
#pragma unroll
    for (int v = 1; v < GR; ++v) m = fmaxf(m, sm[v][u]);
    l = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) o[k] = 0.f;
#pragma unroll
    for (int v = 0; v < GR; ++v) {
        const float f = __builtin_amdgcn_exp2f(sm[v][u] - m);
        l += sl[v][u] * f;
#pragma unroll
        for (int k = 0; k < NC; ++k) o[k] += so[v][k / 4][u][k % 4] * f;
    }
    if (row >= a.R || t0 + row % positions<SEL>(a) >= n) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int k = 0; k < NC; ++k) o[k] *= inv;
    store_out<NC, BF16, SEL>(a, b, h, t0, row, NC * x, o);
}

// ------------------------------------------------------------------ host
struct Shape {
    int nt, rw;               // nt > 0: few rows, nt tiles; else many rows, rw waves of 2 tiles
    int rows, RG, W;          // rows of a slot, row groups, workgroups
    int rows0, dense;         // what 16-bit rows are worth (AttnArgs)
};

// Items that a segment's 16-bit rows are worth, beside 1 << dense each.  Few rows (1 each): one token
// of 64 ragged requests 53.2 us with 0 or 4, 52.5 with 8, 54.0 with 12; 8 tokens of 6 requests 19.1, 18.1,
// 18.2, 18.0; of 2 long requests 66.7, 67.2, 67.2, 67.3.  Many (2 each): 32 tokens of 8 requests 57.6 us
// with 0, 54.9 with 4, 54.5 with 8, of 32 requests 150, 143, 147; 512 tokens of 2 requests, 16
// such items a segment: 2 each 224, 1 each 231, 4 each 234.
constexpr int FEW_ROWS0 = 8, MANY_ROWS0 = 4, MANY_DENSE = 1;

// Up to 32 rows go to the waves of the few-rows kernel (1 or 2 tiles each): 28 rows of 64
// requests 70 us there, 114 in the other; of 16 requests 32 and 43; D 64, 32 rows of 48 requests
// 33 and 49, of 6 requests 18 and 19.  More rows go to the many-rows
// kernel in row groups of at most 16 tiles (of at most 8: 32 tokens of 8 requests 54 -> 63 us,
// 512 of 2 requests 220 -> 268), the groups as even as its built 4, 8 and 16 tiles allow.
// Workgroups: two a CU for few rows (three: 54.0 and 71.4 us where two have 52.5 and 67.6; more
// than are resident at once: 62 and 78), one for many (their LDS; two in turn: 54 -> 67 and
// 220 -> 233 us).  D 64, whose registers and LDS would hold more: few rows 34.4 us with two, 33.4
// with three or four where 64 requests are read, 17.2, 17.2 and 18.9 where 5 are; many 42 -> 49 us.
Shape shape_of(int R) {
    const int tiles = (R + 15) / 16, cus = ma_num_cus() / 8 * 8;
    Shape s{};
    if (tiles <= 2) {
        s.nt = tiles;
        s.rows = tiles * 16;
        s.RG = 1;
        s.W = cus * 2;
        s.rows0 = FEW_ROWS0;
        s.dense = 0;
        return s;
    }
    const int groups = (tiles + 15) / 16, per = (tiles + groups - 1) / groups;
    s.rw = per <= 4 ? 2 : per <= 8 ? 4 : 8;
    s.rows = s.rw * 32;
    s.RG = (R + s.rows - 1) / s.rows;
    s.W = cus;
    s.rows0 = MANY_ROWS0;
    s.dense = MANY_DENSE;
    return s;
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

struct Layout {
    int64_t wl, wo, desc, bytes;   // wm at 0
};
Layout layout_of(const Shape &s, int64_t segments, int64_t slots, int D) {
    const int64_t rows = slots * s.rows;
    Layout l;
    l.wl = align256(rows * 4);
    l.wo = l.wl + align256(rows * 4);
    l.desc = l.wo + align256(rows * D * 4);
    l.bytes = l.desc + align256(segments * sizeof(int4));
    return l;
}

// (SEL: a multiple of 8, for the XCDs)
template <bool SEL>
unsigned grid_of(const AttnArgs &a) {
    return SEL ? ((unsigned)a.B * a.HR * a.parts + 7) / 8 * 8 : (unsigned)a.W;
}

template <int D, int RW, bool BF16, bool MASK, bool SEL>
int launch_many(const AttnArgs &a, hipStream_t st) {
    constexpr int LDS = (int)sizeof(ManyShared<D, BF16>);
    static_assert(LDS <= 160 * 1024, "two steps of operands in one CU's LDS");
    if (LDS > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void *)paged_many_kernel<D, RW, BF16, MASK, SEL>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) {
            ma_set_error("ma_paged_attention: %d bytes of LDS refused: %s", LDS, hipGetErrorString(e));
            return MA_EHIP;
        }
    }
    paged_many_kernel<D, RW, BF16, MASK, SEL><<<grid_of<SEL>(a), 512, LDS, st>>>(a);
    return MA_OK;
}

// few rows over selected blocks, 8 waves a workgroup
template <int D, bool BF16, bool MASK>
int launch_wide(const AttnArgs &a, const Shape &s, hipStream_t st) {
    if (s.nt == 1) paged_few_kernel<D, 1, BF16, MASK, true, 2 * WAVES><<<grid_of<true>(a), 512, 0, st>>>(a);
    else paged_few_kernel<D, 2, BF16, MASK, true, 2 * WAVES><<<grid_of<true>(a), 512, 0, st>>>(a);
    return MA_OK;
}

template <int D, bool BF16, bool MASK, bool SEL>
int launch_attn(const AttnArgs &a, const Shape &s, hipStream_t st) {
    if (SEL && s.nt && a.wide) return launch_wide<D, BF16, MASK>(a, s, st);
    if (s.nt == 1) paged_few_kernel<D, 1, BF16, MASK, SEL, WAVES><<<grid_of<SEL>(a), 256, 0, st>>>(a);
    else if (s.nt == 2) paged_few_kernel<D, 2, BF16, MASK, SEL, WAVES><<<grid_of<SEL>(a), 256, 0, st>>>(a);
    else if (s.rw == 2) return launch_many<D, 2, BF16, MASK, SEL>(a, st);
    else if (s.rw == 4) return launch_many<D, 4, BF16, MASK, SEL>(a, st);
    else return launch_many<D, 8, BF16, MASK, SEL>(a, st);
    return MA_OK;
}

template <int D, bool BF16, bool SEL>
int launch(const AttnArgs &a, const Shape &s, hipStream_t st) {
    if (int rc = a.p.mask ? launch_attn<D, BF16, true, SEL>(a, s, st) : launch_attn<D, BF16, false, SEL>(a, s, st)) return rc;
    if (SEL && a.parts == 1) return ma_check_launch("ma_paged_attention_blocks");      // (nothing to join)
    // (a row group of few rows has fewer than its slots hold)
    const int rows = min(s.rows, a.R);
    if (s.nt) paged_merge_kernel<D, BF16, false, SEL><<<dim3(a.B * a.H * a.RG, (rows + 3) / 4), 64 * merge_waves(false, SEL), 0, st>>>(a, s.rows);
    else paged_merge_kernel<D, BF16, true, SEL><<<dim3(a.B * a.H * a.RG, (rows + 15) / 16 * 4), 64 * merge_waves(true, SEL), 0, st>>>(a, s.rows);
    return ma_check_launch(SEL ? "ma_paged_attention_blocks" : "ma_paged_attention");
}

}  // namespace

// What a call over selected blocks is cut into (count 0: over all): positions of a run, runs, row groups of
// all runs, segments, workgroups of a segment.
struct Plan {
    Shape s;
    int run, parts, wide;
    int64_t runs, RG, segments;
    Layout l;
};
// Selected blocks: a segment has as many workgroups as keep the card busy, but each has FEW_SHARE (many
// rows: MANY_SHARE) items at least: 4 096 tokens of 16 segments 14.3 us with 4, 13.5 with 8, 13.3 with 16, 15.4
// with 32; 8 tokens' rows over 32 groups of 24 segments 12.1, 12.8, 15.6, 18.7.  Where a segment of few rows
// would have two, it has one of 8 waves: as many loads under way, and no merge (one token of 64 requests,
// 64 groups of each head, 26.8 -> 22.7 us: 75 MB, 3.3 TB/s, of which 7 us are the launch and the chain of
// loads: length, list, table, record).  8 waves also where it would have more: 13.5 -> 14.2 and 12.8 -> 15.7.
// 12 waves (155 registers, none spilled): 22.2 -> 24.0; 8 that ask two records ahead (211 registers): 23.8.
// Many rows, where it would have two or more and lists of up to HALF_ROWS_ITEMS groups: row groups of 8
// tiles for 16, which unpack every group twice and join half as much: 512 positions in runs of 32 (224
// rows) of 8, 16, 24 groups 47.5 -> 43.8, 51.5 -> 48.8, 56.5 -> 55.1 us; of 32, 40, 48, 64, 128 groups
// 59.0 -> 61.5, 67 -> 68, 72.6 -> 72.8, 81 -> 84, 116 -> 125.
constexpr int FEW_SHARE = 8, MANY_SHARE = 16;
constexpr int HALF_ROWS_ITEMS = 24;

// false: not built
static bool plan_of(int B, int H, int Hq, int T, int D, int query_block, int count, int64_t m, Plan &p) {
    if (B <= 0 || H <= 0 || Hq <= 0 || Hq % H || T <= 0 || (D != 64 && D != 128) || query_block < 0) return false;
    p.run = query_block == 0 || query_block > T ? T : query_block;
    // (a run's rows, and the position behind the last run or 32 keys, have 32 bits)
    if ((int64_t)(Hq / H) * p.run > INT32_MAX / 16 || (int64_t)T + max(p.run, PG_GROUP) > INT32_MAX) return false;
    p.runs = (T + p.run - 1) / p.run;
    p.s = shape_of(Hq / H * p.run);
    if (count && count * m <= HALF_ROWS_ITEMS && p.s.rw == 8 && p.s.RG * p.runs <= p.s.W / 2 / ((int64_t)B * H)) {
        // half as many rows a workgroup where its segment would be cut in two: nothing, or half, to join
        p.s.rw = 4;
        p.s.rows = p.s.rw * 32;
        p.s.RG = (Hq / H * p.run + p.s.rows - 1) / p.s.rows;
    }
    p.RG = p.s.RG * p.runs;
    if (p.RG * H > INT32_MAX || p.RG * H * B > INT32_MAX) return false;
    p.segments = p.RG * H * B;
    p.parts = 1;
    p.wide = 0;
    if (count) {
        const int64_t items = min((int64_t)count * m, (int64_t)INT32_MAX) + p.s.rows0 + ((1 + (T + PG_GROUP - 1) / PG_GROUP) << p.s.dense);
        const int share = p.s.nt ? FEW_SHARE : MANY_SHARE;
        p.parts = (int)max(min(p.s.W / p.segments, (items + share - 1) / share), (int64_t)1);
        if (p.s.nt && p.parts == 2) {         // (as many waves, and nothing to join)
            p.parts = 1;
            p.wide = 1;
        }
        if (p.segments * p.parts > INT32_MAX - 8) return false;
    }
    p.l = layout_of(p.s, count ? 0 : p.segments, !count ? 2LL * p.s.W : p.parts > 1 ? p.segments * p.parts : 0, D);
    return true;
}

extern "C" int64_t ma_paged_workspace_bytes(int B, int H, int Hq, int T, int D) {
    Plan p;
    return plan_of(B, H, Hq, T, D, 0, 0, 0, p) ? p.l.bytes : -1;
}

extern "C" int64_t ma_paged_blocks_workspace_bytes(int B, int H, int Hq, int T, int D, int count, int block_tokens,
                                                   int query_block) {
    Plan p;
    if (count <= 0 || block_tokens <= 0 || block_tokens % PG_GROUP) return -1;
    return plan_of(B, H, Hq, T, D, query_block, count, block_tokens / PG_GROUP, p) ? p.l.bytes : -1;
}

// m: groups of a selected block, 0 where every stored token is read
static int paged_attention(const char *who, const ma_tensor4 &q, int B, int Hq, int T, int D, const ma_pages *p, int H,
                           const ma_tensor4 &kc, const ma_tensor4 &vc, const int32_t *new_lens, int causal_block,
                           float scale, const ma_tensor4 &out, const int32_t *blocks, int count, int m, int query_block,
                           void *workspace, int64_t workspace_bytes, void *stream) {
    if (int rc = pg_check(p, B, H, D, who)) return rc;
    Plan plan;
    const bool built = plan_of(B, H, Hq, T, D, query_block, count, m, plan);
    if (!built || !q.ptr || !out.ptr || causal_block < 0 || (kc.ptr == nullptr) != (vc.ptr == nullptr)) {
        ma_set_error("%s: bad arguments (B=%d H=%d Hq=%d T=%d D=%d causal_block=%d)", who, B, H, Hq, T, D, causal_block);
        return MA_EINVAL;
    }
    if (q.dtype != p->dtype || out.dtype != p->dtype || (kc.ptr && (kc.dtype != p->dtype || vc.dtype != p->dtype))) {
        ma_set_error("%s: queries, the block's keys and values, out and tails must share one dtype", who);
        return MA_EINVAL;
    }
    const int64_t need = plan.l.bytes;
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)) {
        ma_set_error("%s: workspace of %lld bytes (256-byte aligned) needed, got %lld", who, (long long)need,
                     (long long)workspace_bytes);
        return MA_EWORKSPACE;
    }
    const Shape &s = plan.s;
    const Layout &l = plan.l;
    const int64_t RG = plan.RG;
    // the line: every request as long as its table row, with room for what the stretches round up.  (Lists lie
    // on none: a segment holds at most 2^27 groups of its list, twice a table row's, beside its 16-bit rows.)
    const int64_t groups = (int64_t)p->width * p->page_tokens / PG_GROUP;
    const int64_t most = START + s.rows0 + groups + ((1 + (T + PG_GROUP - 1) / PG_GROUP) << s.dense);
    if (!m && most * plan.segments + 64LL * s.W > INT32_MAX) {
        ma_set_error("%s: %d requests of up to %lld tokens and %lld row groups of each head are not built (2^31 items)", who,
                     B, (long long)p->width * p->page_tokens, (long long)RG);
        return MA_EUNSUPPORTED;
    }
    // the merge: a workgroup a segment (and rows), threads of one dimension below 2^32
    if (plan.segments * 64 * merge_waves(s.nt == 0, false) > UINT32_MAX) {
        ma_set_error("%s: %d requests, %d heads and %lld row groups of each are not built (2^%d segments)", who, B, H,
                     (long long)RG, s.nt ? 23 : 24);
        return MA_EUNSUPPORTED;
    }
    if (m && plan.segments * plan.parts * 512 > UINT32_MAX - 8 * 512) {
        ma_set_error("%s: %lld segments are not built (2^32 threads)", who, (long long)plan.segments);
        return MA_EUNSUPPORTED;
    }
    char *ws = (char *)workspace;
    AttnArgs a{};
    a.q = q;
    a.kc = kc;
    a.vc = vc;
    a.out = out;
    a.p = pages_dev(p);
    a.new_lens = new_lens;
    a.B = B;
    a.H = H;
    a.G = Hq / H;
    a.T = T;
    a.R = a.G * plan.run;
    a.RG = (int)RG;
    a.HR = H * a.RG;
    a.max_len = p->width * p->page_tokens;
    a.rows0 = s.rows0;
    a.dense = s.dense;
    a.causal = causal_block;
    a.W = s.W;
    a.sl2 = scale * MA_LOG2E;
    a.wm = (float *)ws;
    a.wl = (float *)(ws + l.wl);
    a.wo = (float *)(ws + l.wo);
    a.desc = (int4 *)(ws + l.desc);
    hipStream_t st = (hipStream_t)stream;
    if (m) {
        a.blocks = blocks;
        a.count = count;
        a.m = m;
        a.run = plan.run;
        a.RGR = s.RG;
        a.parts = plan.parts;
        a.wide = plan.wide;
        if (D == 128) return p->dtype == MA_BF16 ? launch<128, true, true>(a, s, st) : launch<128, false, true>(a, s, st);
        return p->dtype == MA_BF16 ? launch<64, true, true>(a, s, st) : launch<64, false, true>(a, s, st);
    }
    if (D == 128) return p->dtype == MA_BF16 ? launch<128, true, false>(a, s, st) : launch<128, false, false>(a, s, st);
    return p->dtype == MA_BF16 ? launch<64, true, false>(a, s, st) : launch<64, false, false>(a, s, st);
}

extern "C" int ma_paged_attention(ma_tensor4 q, int B, int Hq, int T, int D, const ma_pages *p, int H, ma_tensor4 kc,
                                  ma_tensor4 vc, const int32_t *new_lens, int causal_block, float scale,
                                  ma_tensor4 out, void *workspace, int64_t workspace_bytes, void *stream) {
    return paged_attention("ma_paged_attention", q, B, Hq, T, D, p, H, kc, vc, new_lens, causal_block, scale, out, nullptr, 0,
                           0, 0, workspace, workspace_bytes, stream);
}

extern "C" int ma_paged_attention_blocks(ma_tensor4 q, int B, int Hq, int T, int D, const ma_pages *p, int H, ma_tensor4 kc,
                                         ma_tensor4 vc, const int32_t *new_lens, int causal_block, float scale,
                                         ma_tensor4 out, const int32_t *blocks, int count, int block_tokens,
                                         int query_block, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "ma_paged_attention_blocks";
    if (!blocks || count <= 0 || block_tokens <= 0 || block_tokens % PG_GROUP || query_block < 0) {
        ma_set_error("%s: bad blocks (count=%d block_tokens=%d, a multiple of 32, query_block=%d)", who, count, block_tokens,
                     query_block);
        return MA_EINVAL;
    }
    return paged_attention(who, q, B, Hq, T, D, p, H, kc, vc, new_lens, causal_block, scale, out, blocks, count,
                           block_tokens / PG_GROUP, query_block, workspace, workspace_bytes, stream);
}
