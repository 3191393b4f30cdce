// Pages of 4-bit K/V: the plan (block tables, slot maps, free ring) from request lengths, the
// append that quantizes into pages, and the read-back at 16 or 32 bits.  The store's layout
// is in ma_pages.h.
#include "ma_pages.h"
#include "ma_quant.h"

using namespace ma;

namespace {

// ------------------------------------------------------------------ plan
// pages(x) = ceil(x / P).  Request b grows by max(0, pages(end) - pages(len)) pages, whose ids
// are the ring's entries from head + (growth of the requests before it) on, and gives back
// max(0, pages(len) - pages(end)), which go behind the ring's newest entry.  Reads (the count
// oldest entries) and writes (the places behind them) of the ring never meet, so one launch
// needs no order between its workgroups: each scans all B requests' growth itself (8 B a
// request, from L2 after the first) and writes the slots of its own PLAN_SLOTS (request,
// token) pairs.  The ring's state is written by the workgroup that arrives last, when every
// other has read it.
//
// bound: latency (lengths, page ids, writes: three loads in a row behind a scan).  64 requests of
// one token 6 us, 256 of 2 048 tokens (4 MB of slots) 11, of which the arrivals of 256 workgroups
// at one counter are 2.6; a second launch instead of the counter would cost more.
constexpr int PLAN_THREADS = 256;
constexpr int PLAN_SLOTS = 2048;
constexpr int PLAN_SCAN = 4 * PLAN_THREADS;   // requests per scan step

enum { PLAN_NO_PAGES = 1, PLAN_WIDTH = 2, PLAN_TOKENS = 4, PLAN_LENGTH = 8, PLAN_NEGATIVE = 16 };

struct PlanArgs {
    const int32_t *lengths, *new_lens;
    int32_t *table, *ring, *state, *ends;
    int64_t *slots;
    int64_t s_table, nflat;   // nflat = B * max(T, 1)
    int B, T, page, width, num_pages;
    bool grow;                // no request gives tokens back
};

// a request's step: tokens after it, pages before and after it (`most` + 1 where there are more
// than `most`); all in 32 bits, len + n < 2^32
struct Step {
    uint32_t end, p0, p1;
};
__device__ __forceinline__ Step step_of(int len, int n, uint32_t page, uint32_t most) {
    Step s;
    const int64_t end = max((int64_t)len + n, (int64_t)0);
    s.end = (uint32_t)end;
    s.p0 = ((uint32_t)max(len, 0) + page - 1) / page;
    s.p1 = end > INT32_MAX ? most + 1 : (s.end + page - 1) / page;
    return s;
}

__global__ __launch_bounds__(PLAN_THREADS) void page_plan_kernel(PlanArgs a) {
    __shared__ int grow_off[PLAN_SLOTS], back_off[PLAN_SLOTS];   // of this workgroup's requests
    __shared__ int64_t wsum[2][PLAN_THREADS / 64];
    __shared__ int bad_s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int Tm = max(a.T, 1);
    const int64_t f0 = (int64_t)blockIdx.x * PLAN_SLOTS;
    const int nf = (int)min((int64_t)PLAN_SLOTS, a.nflat - f0);
    const int b0 = (int)(f0 / Tm), b1 = (int)((f0 + nf - 1) / Tm);
    const int r0 = (int)(f0 - (int64_t)b0 * Tm);                  // token of the first pair
    const int head = a.state[0], count = a.state[1];
    if (tid == 0) bad_s = 0;
    __syncthreads();
    int64_t gsum = 0, bsum = 0;   // of the requests before this scan step
    int bad = 0;
    for (int base = 0; base < a.B; base += PLAN_SCAN) {
        int64_t g[4], k[4], gt = 0, kt = 0;
        const int first = base + 4 * tid;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = first + i;
            g[i] = gt;
            k[i] = kt;
            if (b < a.B) {
                const int len = a.lengths[b], n = a.new_lens[b];
                const Step st = step_of(len, n, a.page, a.width);
                if (len < 0) bad |= PLAN_LENGTH;
                if (n > a.T) bad |= PLAN_TOKENS;
                if (a.grow && n < 0) bad |= PLAN_NEGATIVE;
                if (max(st.p0, st.p1) > (uint32_t)a.width) bad |= PLAN_WIDTH;
                gt += st.p1 > st.p0 ? st.p1 - st.p0 : 0;
                kt += st.p0 > st.p1 ? st.p0 - st.p1 : 0;
            }
        }
        const int64_t gi = pg_wave_scan(gt, lane), ki = pg_wave_scan(kt, lane);
        __syncthreads();   // wsum of the step before is read
        if (lane == 63) {
            wsum[0][wave] = gi;
            wsum[1][wave] = ki;
        }
        __syncthreads();
        int64_t go = gsum + gi - gt, ko = bsum + ki - kt;
#pragma unroll
        for (int w = 0; w < PLAN_THREADS / 64; ++w) {
            if (w < wave) {
                go += wsum[0][w];
                ko += wsum[1][w];
            }
            gsum += wsum[0][w];
            bsum += wsum[1][w];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = first + i;
            if (b >= b0 && b <= b1 && b < a.B) {   // (beyond num_pages only where the plan is refused)
                grow_off[b - b0] = (int)min(go + g[i], (int64_t)a.num_pages);
                back_off[b - b0] = (int)min(ko + k[i], (int64_t)a.num_pages);
            }
        }
    }
    if (bad) atomicOr(&bad_s, bad);
    __syncthreads();
    bad = bad_s | (gsum > count ? PLAN_NO_PAGES : 0);
    // head and count are the caller's: a ring outside its own bounds is never indexed
    if (head < 0 || count < 0 || head >= a.num_pages || count > a.num_pages || bsum > a.num_pages - count)
        bad |= PLAN_NO_PAGES;
    // A thread's pairs, in three rounds without branches -- lengths, page ids, writes -- so that
    // each round's loads are under way together (pairs behind the last are the last one again,
    // pairs without a page read the ring's first entry).
    constexpr int PER = PLAN_SLOTS / PLAN_THREADS;
    int bl[PER], tok[PER], len[PER], n[PER], id[PER];
#pragma unroll
    for (int y = 0; y < PER; ++y) {
        const unsigned flat = (unsigned)min(tid + y * PLAN_THREADS, nf - 1) + (unsigned)r0;
        bl[y] = (int)(flat / (unsigned)Tm);
        tok[y] = (int)(flat - (unsigned)bl[y] * (unsigned)Tm);
        len[y] = a.lengths[b0 + bl[y]];
        n[y] = a.new_lens[b0 + bl[y]];
    }
    auto fresh = [&](int y, uint32_t pi) {    // a page that appears (its first token is a new one)
        return pi >= ((uint32_t)len[y] + a.page - 1) / (uint32_t)a.page;
    };
#pragma unroll
    for (int y = 0; y < PER; ++y) {
        const bool has = !bad && tok[y] < n[y];
        const uint32_t pi = (uint32_t)(len[y] + tok[y]) / (uint32_t)a.page;
        const uint32_t p0 = ((uint32_t)len[y] + a.page - 1) / (uint32_t)a.page;
        int at = head + grow_off[bl[y]] + (int)(pi - p0);       // (fresh pages: < 2 num_pages)
        if (at >= a.num_pages) at -= a.num_pages;
        const int32_t *old = a.table + (int64_t)(b0 + bl[y]) * a.s_table + pi;
        const int32_t *src = pi >= p0 ? a.ring + at : old;
        id[y] = *(has ? src : a.ring);
    }
#pragma unroll
    for (int y = 0; y < PER; ++y) {
        if (tid + y * PLAN_THREADS >= nf) continue;
        const int b = b0 + bl[y];
        const uint32_t pos = (uint32_t)(len[y] + tok[y]), pi = pos / (uint32_t)a.page, off = pos - pi * a.page;
        const bool has = !bad && tok[y] < n[y];
        if (tok[y] == 0) a.ends[b] = bad ? len[y] : (int)max((int64_t)len[y] + n[y], (int64_t)0);
        // (an id below 0 is no page, with or without an offset)
        if (tok[y] < a.T) a.slots[(int64_t)b * a.T + tok[y]] = has && id[y] >= 0 ? (int64_t)id[y] * a.page + off : -1;
        if (has && off == 0 && fresh(y, pi)) a.table[(int64_t)b * a.s_table + pi] = id[y];
    }
    // pages that go back: a wave per request that gives some, of the requests whose first pair
    // is this workgroup's
    if (!bad && bsum > 0) {
        const int lo = r0 ? 1 : 0, nb = b1 - b0 + 1;
        for (int s = lo + wave * 64; s < nb; s += PLAN_THREADS) {
            int p0 = 0, p1 = 0;
            if (s + lane < nb) {
                const Step st = step_of(a.lengths[b0 + s + lane], a.new_lens[b0 + s + lane], a.page, a.width);
                p0 = (int)st.p0;
                p1 = (int)st.p1;
            }
            uint64_t todo = __ballot(p0 > p1);
            while (todo) {
                const int l = __ffsll((unsigned long long)todo) - 1;
                todo &= todo - 1;
                const int q0 = __shfl(p0, l), q1 = __shfl(p1, l);
                int32_t *row = a.table + (int64_t)(b0 + s + l) * a.s_table;
                for (int j = lane; j < q0 - q1; j += 64) {
                    int64_t at = (int64_t)head + count + back_off[s + l] + j;   // < 3 num_pages
                    at %= a.num_pages;
                    a.ring[at] = row[q1 + j];
                    row[q1 + j] = -1;
                }
            }
        }
    }
    __syncthreads();   // the workgroup's reads of the state are done
    if (tid == 0 && (gridDim.x == 1 || atomicAdd(&a.state[2], 1) == (int)gridDim.x - 1)) {
        if (!bad) {
            a.state[0] = (int)((head + gsum) % a.num_pages);
            a.state[1] = (int)(count - gsum + bsum);
        }
        a.state[2] = 0;
        if (bad) a.state[3] |= bad;
    }
}

// ------------------------------------------------------------------ append
// One wave = the keys or the values of one group of 32 tokens of one (request, KV head): the
// window of request b is [its tail | its new tokens], group u the window's tokens 32 u ...
// Nothing goes through LDS: the lanes of a values wave hold the 8 tokens x D/16 channels whose
// words they store (1 KB a store instruction), those of a keys wave 4 channels of 16 (D 64: 8)
// tokens, whose minimum and maximum need one (two) lane moves, and two lanes make a word.  The
// waves of group 0 are the only readers of the old tail, so they also write the new one.
//
// bound: 4 D bytes read and 1.25 D written a token and head.  A quotient rounded to a bf16 code
// needs no division: with 8-bit significands a / step is never nearer than 2^-17 (relative) to
// where bf16 rounds the other way, and a * rcp(step) is within 2^-22 of it; a / 15 likewise
// (2^-13).  f16 quotients come as near as 2^-23 and are divided.  8 ragged prompts of up to 8 192
// tokens (8 heads, D 128): 266 MB in 55 to 69 us, 3.9 to 4.8 TB/s (53 without any arithmetic);
// one token of 64 requests 4.3 us.
struct AppendArgs {
    PagesDev p;
    const uint16_t *k, *v;
    int64_t s_kb, s_kh, s_kt, s_vb, s_vh, s_vt;
    const int32_t *new_lens;
    const int64_t *slots;
    int T;
};

template <int DT>
__device__ __forceinline__ void unpack2(uint32_t w, float &a, float &b) {
    if constexpr (DT == MA_BF16) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    } else {
        a = ma_f16_to_f32((uint16_t)w);
        b = ma_f16_to_f32((uint16_t)(w >> 16));
    }
}
// two values rounded to DT, as f32
template <int DT>
__device__ __forceinline__ void round2(float &a, float &b) {
    if constexpr (DT == MA_BF16) unpack2<DT>(ma_pack_bf16x2(a, b), a, b);
    else a = ma_round_f16(a), b = ma_round_f16(b);
}
template <int DT>
__device__ __forceinline__ QuantGroup group_params(float lo, float hi) {
    if constexpr (DT != MA_BF16) return quant_params(lo, hi, DT);
    float step = ma_round_bf16(ma_round_bf16(hi - lo) * (1.0f / 15.0f));
    step = ma_round_bf16(fmaxf(step, 1e-8f));
    return {lo, step, __builtin_amdgcn_rcpf(step)};
}
// the same for a minimum: a signalling NaN as a quiet one, which v_min3 and v_max3 pass over (they
// answer a signalling one with NaN, and the numbers beside it are lost); f16's conversion does so
template <int DT>
__device__ __forceinline__ void unpack2_quiet(uint32_t w, float &a, float &b) {
    unpack2<DT>(w, a, b);
    if constexpr (DT == MA_BF16) a = __builtin_canonicalizef(a), b = __builtin_canonicalizef(b);
}
// minimum / maximum of three quiet values (fminf and fmaxf quiet each argument again)
__device__ __forceinline__ float min3(float x, float y, float z) {
    float r;
    asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}
// The quotients whose nearest whole numbers (half to even) are the codes of two values; NaN's
// code is 0, as quant_code's.  A bf16 quotient is at most 15 (1 + 2^-8); f16's, with a step that
// f16 holds in few bits, may be more.
template <int DT>
__device__ __forceinline__ void codes2(float &a, float &b, const QuantGroup &qa, const QuantGroup &qb) {
    a -= qa.lo;
    b -= qb.lo;
    round2<DT>(a, b);
    if constexpr (DT == MA_BF16) {
        a *= qa.inv;
        b *= qb.inv;
    } else {
        a = quant_div(a, qa, DT);
        b = quant_div(b, qb, DT);
    }
    round2<DT>(a, b);
    if constexpr (DT != MA_BF16) {
        a = __builtin_amdgcn_fmed3f(a, 0.0f, 15.0f);
        b = __builtin_amdgcn_fmed3f(b, 0.0f, 15.0f);
    }
}
// x rounded half to even into one byte of w (v_cvt_pk_u8_f32; NaN: 0)
__device__ __forceinline__ uint32_t put_byte(float x, uint32_t byte, uint32_t w) {
    return __builtin_amdgcn_cvt_pk_u8_f32(x, byte, w);
}
__device__ __forceinline__ uint32_t f16x2_bits(float a, float b) {
    const f16x2_t v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
}

template <int D, int DT>
__global__ __launch_bounds__(256) void page_append_kernel(AppendArgs a) {
    constexpr int NC = D / 16, CL = D / 4, SL = 64 / CL, TPL = PG_GROUP / SL;   // CL lanes a row, SL slices of the tokens
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int u = blockIdx.x * 2 + (wave >> 1), h = blockIdx.y, b = blockIdx.z;
    const bool val = wave & 1;
    // (looked at together, so that their loads are under way together)
    const int n = min(a.new_lens[b], a.T), len = pg_length(a.p, b), r = len & (PG_GROUP - 1);
    const int64_t slot0 = a.slots[(int64_t)b * a.T];
    if ((n <= 0) | (slot0 < 0)) return;
    const int whole = (r + n) / PG_GROUP;
    if (u >= max(whole, 1)) return;
    const uint16_t *fresh = val ? a.v + (int64_t)b * a.s_vb + (int64_t)h * a.s_vh
                                : a.k + (int64_t)b * a.s_kb + (int64_t)h * a.s_kh;
    const int64_t st = val ? a.s_vt : a.s_kt;
    uint16_t *tail = (val ? a.p.vt : a.p.kt) + (int64_t)b * a.p.s_tb + (int64_t)h * a.p.s_th;
    if (u < whole) {
        const int j0 = u * PG_GROUP - r;    // the new token that is the group's token 0 (below 0: a row of the tail)
        // rows first, first + 1, ... of the group at a lane's channel ch: read(i, pointer to row first + i)
        auto rows = [&](int first, int count, int ch, auto read) {
            if (j0 >= 0) {      // new tokens alone: one pointer a lane, moved on by a scalar
                const uint16_t *p = fresh + (int64_t)(j0 + first) * st + ch;
#pragma unroll
                for (int i = 0; i < count; ++i, p += st) read(i, p);
            } else {
#pragma unroll
                for (int i = 0; i < count; ++i) {
                    const int t = first + i;
                    read(i, (j0 + t < 0 ? tail + (int64_t)t * a.p.s_tt : fresh + (int64_t)(j0 + t) * st) + ch);
                }
            }
        };
        // the group's record: its last token is a new one, and a group lies in one page
        const int64_t slot = a.slots[(int64_t)b * a.T + j0 + PG_GROUP - 1];
        const int64_t page = slot >= 0 ? slot / a.p.page_tokens : -1;
        uint8_t *rec = nullptr;
        if (page >= 0 && page < a.p.num_pages)
            rec = a.p.pool + page * a.p.s_page + (int64_t)h * a.p.s_head +
                  (slot - page * a.p.page_tokens) / PG_GROUP * (int64_t)(40 * D);
        if (!val) {
            const int c4 = lane % CL, sl = lane / CL, odd = c4 & 1;
            uint2 x[TPL];
            rows(sl * TPL, TPL, 4 * c4, [&](int i, const uint16_t *src) { x[i] = pg_load8(src); });
            float lo[4], hi[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) lo[c] = INFINITY, hi[c] = -INFINITY;
#pragma unroll
            for (int i = 0; i < TPL; i += 2) {
                float v[2][4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    unpack2_quiet<DT>(x[i + e].x, v[e][0], v[e][1]);
                    unpack2_quiet<DT>(x[i + e].y, v[e][2], v[e][3]);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    lo[c] = min3(lo[c], v[0][c], v[1][c]);
                    hi[c] = max3(hi[c], v[0][c], v[1][c]);
                }
            }
            QuantGroup q[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                lo[c] = -ma_max_xor32(-lo[c]);
                hi[c] = ma_max_xor32(hi[c]);
                if constexpr (SL == 4) {
                    lo[c] = fminf(lo[c], __shfl_xor(lo[c], 16));
                    hi[c] = fmaxf(hi[c], __shfl_xor(hi[c], 16));
                }
                q[c] = group_params<DT>(lo[c], hi[c]);
            }
            if (!rec) goto tail_rows;
            if (sl == 0) {
                *(uint2 *)(rec + 32 * D + 8 * c4) = uint2{f16x2_bits(q[0].step, q[1].step), f16x2_bits(q[2].step, q[3].step)};
                *(uint2 *)(rec + 34 * D + 8 * c4) = uint2{f16x2_bits(q[0].lo, q[1].lo), f16x2_bits(q[2].lo, q[3].lo)};
            }
            // a lane's bytes of a token's word: elements 0..3 (even lanes) or 4..7 of the octet
            const int o = c4 >> 1, hh = o / (D / 32), cb = o % (D / 32);
#pragma unroll
            for (int i = 0; i < TPL; i += 2) {
                uint32_t w[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float v[4];
                    unpack2<DT>(x[i + e].x, v[0], v[1]);
                    unpack2<DT>(x[i + e].y, v[2], v[3]);
                    codes2<DT>(v[0], v[1], q[0], q[1]);
                    codes2<DT>(v[2], v[3], q[2], q[3]);
                    const uint32_t lo4 = put_byte(v[1], 2 + odd, put_byte(v[0], odd, 0));
                    const uint32_t hi4 = put_byte(v[3], 2 + odd, put_byte(v[2], odd, 0));
                    const uint32_t mine = lo4 | hi4 << 4;
                    w[e] = mine | ma_dpp<0xB1>(mine);      // with the other lane's, lane ^ 1
                }
                // even lanes store the word of token i, odd lanes that of token i + 1
                const int t = sl * TPL + i, mt = (t >> 2) & 1, m = 4 * (t >> 3) + (t & 3) + odd;
                *(uint32_t *)(rec + ((mt * 4 + hh) * 16 + m) * (D / 8) + 4 * cb) = odd ? w[1] : w[0];
            }
        } else {
            const int m = lane & 15, hh = lane >> 4;
            uint32_t x[8][NC / 2];
            rows(8 * hh, 8, NC * m, [&](int i, const uint16_t *src) {
                if constexpr (NC == 8) {
                    const uint4 y = pg_load16(src);
                    x[i][0] = y.x; x[i][1] = y.y; x[i][2] = y.z; x[i][3] = y.w;
                } else {
                    const uint2 y = pg_load8(src);
                    x[i][0] = y.x; x[i][1] = y.y;
                }
            });
            QuantGroup q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float lo = INFINITY, hi = -INFINITY;
#pragma unroll
                for (int c = 0; c < NC / 2; ++c) {
                    float v0, v1;
                    unpack2_quiet<DT>(x[i][c], v0, v1);
                    lo = min3(lo, v0, v1);
                    hi = max3(hi, v0, v1);
                }
                lo = fminf(lo, ma_quad<0xB1>(lo));
                hi = fmaxf(hi, ma_quad<0xB1>(hi));
                lo = fminf(lo, ma_quad<0x4E>(lo));
                hi = fmaxf(hi, ma_quad<0x4E>(hi));
                if constexpr (NC == 4) {                   // 8 lanes a channel group
                    lo = fminf(lo, ma_quad<0x141>(lo));
                    hi = fmaxf(hi, ma_quad<0x141>(hi));
                }
                q[i] = group_params<DT>(lo, hi);
            }
            if (!rec) goto tail_rows;
            if (m % (32 / NC) == 0) {
                uint8_t *par = rec + 36 * D + 2 * (32 * (NC * m / 32) + 8 * hh);
                *(uint4 *)par = uint4{f16x2_bits(q[0].step, q[1].step), f16x2_bits(q[2].step, q[3].step),
                                      f16x2_bits(q[4].step, q[5].step), f16x2_bits(q[6].step, q[7].step)};
                *(uint4 *)(par + 2 * D) = uint4{f16x2_bits(q[0].lo, q[1].lo), f16x2_bits(q[2].lo, q[3].lo),
                                                f16x2_bits(q[4].lo, q[5].lo), f16x2_bits(q[6].lo, q[7].lo)};
            }
            uint32_t w[NC];
#pragma unroll
            for (int c = 0; c < NC / 2; ++c) {
                // tokens 0 4 1 5 in the low nibbles of the bytes, 2 6 3 7 in the high ones
                uint32_t lo0 = 0, lo1 = 0, hi0 = 0, hi1 = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float v0, v1;
                    unpack2<DT>(x[i][c], v0, v1);
                    codes2<DT>(v0, v1, q[i], q[i]);
                    const uint32_t byte = (i >> 2) + 2 * (i & 1);
                    if (i & 2) hi0 = put_byte(v0, byte, hi0), hi1 = put_byte(v1, byte, hi1);
                    else lo0 = put_byte(v0, byte, lo0), lo1 = put_byte(v1, byte, lo1);
                }
                w[2 * c] = lo0 | hi0 << 4;
                w[2 * c + 1] = lo1 | hi1 << 4;
            }
#pragma unroll
            for (int half = 0; half < D / 64; ++half)
                *(uint4 *)(rec + 16 * D + 1024 * half + 16 * lane) = uint4{w[4 * half], w[4 * half + 1], w[4 * half + 2],
                                                                           w[4 * half + 3]};
        }
    }
tail_rows:
    if (u != 0) return;
    // the tail: new tokens behind the last whole group (in front of them, where none was
    // completed, the tail's own rows stay); its old rows were read above, by this wave alone
    const int first = whole ? 0 : r, j0 = whole ? whole * PG_GROUP - r : 0, cnt = n - j0;
    constexpr int CH = D / 8;           // 16-byte chunks of a row
    for (int x = lane; x < cnt * CH; x += 64) {
        const int rw = x / CH, c = x % CH;
        pg_store16(tail + (int64_t)(first + rw) * a.p.s_tt + 8 * c, pg_load16(fresh + (int64_t)(j0 + rw) * st + 8 * c));
    }
}

// ------------------------------------------------------------------ read-back
// One wave = one group of 32 tokens of one (request, KV head), K by code words of 8 channels
// (a lane keeps one octet of channels, so its parameters, for every token), V by lanes of
// D / 16 channels x 8 tokens; every store instruction writes whole rows.
//
// bound: 1.25 D bytes read and 4 D (f32: 8 D) written a token and head.  2 requests' 65 536 tokens
// (8 heads, D 128, bf16): 697 MB in 143 us, 4.9 TB/s, a large copy's 5.1.
struct DequantArgs {
    PagesDev p;
    const int32_t *starts;
    void *ko, *vo;
    int64_t s_kb, s_kh, s_kt, s_vb, s_vh, s_vt;
    int n, groups;
};

// elements 2k, 2k+1 of a code word
__device__ __forceinline__ void unpack_word(uint32_t w, uint32_t (&c)[8]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        c[2 * k] = (w >> (4 * k)) & 15u;
        c[2 * k + 1] = (w >> (16 + 4 * k)) & 15u;
    }
}

template <int OT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (OT == MA_BF16) return ma_pack_bf16x2(a, b);
    const f16x2_t v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
}

// N (4 or 8) values at element offset off
template <int OT, int N>
__device__ __forceinline__ void store_n(void *base, int64_t off, const float *x) {
    if constexpr (OT == MA_F32) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            pg_store16((float *)base + off + i, uint4{__float_as_uint(x[i]), __float_as_uint(x[i + 1]),
                                                      __float_as_uint(x[i + 2]), __float_as_uint(x[i + 3])});
    } else if constexpr (N == 8) {
        pg_store16((uint16_t *)base + off, uint4{pack2<OT>(x[0], x[1]), pack2<OT>(x[2], x[3]), pack2<OT>(x[4], x[5]),
                                                 pack2<OT>(x[6], x[7])});
    } else {
        pg_store8((uint16_t *)base + off, uint2{pack2<OT>(x[0], x[1]), pack2<OT>(x[2], x[3])});
    }
}

__device__ __forceinline__ float half_of(uint32_t w, int hi) { return ma_f16_to_f32((uint16_t)(hi ? w >> 16 : w)); }

template <int D, int OT>
__global__ __launch_bounds__(256) void page_dequant_kernel(DequantArgs a, int dtype) {
    constexpr int NO = D / 8, TPI = 64 / NO;   // octets of a row, tokens a wave takes at once
    constexpr int NC = D / 16;
    const int lane = threadIdx.x & 63;
    const int gx = blockIdx.x * 4 + (threadIdx.x >> 6), h = blockIdx.y, b = blockIdx.z;
    if (gx >= a.groups) return;
    const int start = a.starts ? max(a.starts[b], 0) : 0;
    const int len = pg_length(a.p, b);
    const int64_t grp = start / PG_GROUP + (int64_t)gx;
    const int64_t t0 = grp * PG_GROUP - start;                 // output row of the group's token 0
    if (t0 >= a.n) return;
    const int live = (int)min(max((int64_t)len - grp * PG_GROUP, (int64_t)0), (int64_t)PG_GROUP);   // its tokens
    const int64_t kb = (int64_t)b * a.s_kb + (int64_t)h * a.s_kh, vb = (int64_t)b * a.s_vb + (int64_t)h * a.s_vh;
    const int oct = lane % NO, tk = lane / NO;
    if (live < PG_GROUP) {   // the tail, and what lies behind it
        const int64_t tb = (int64_t)b * a.p.s_tb + (int64_t)h * a.p.s_th;
        for (int t = tk; t < PG_GROUP; t += TPI) {
            const int64_t row = t0 + t;
            if (row < 0 || row >= a.n) continue;
            float k[8] = {}, v[8] = {};
            if (t < live) {
                const uint4 kw = pg_load16(a.p.kt + tb + t * a.p.s_tt + 8 * oct);
                const uint4 vw = pg_load16(a.p.vt + tb + t * a.p.s_tt + 8 * oct);
                const uint32_t kx[4] = {kw.x, kw.y, kw.z, kw.w}, vx[4] = {vw.x, vw.y, vw.z, vw.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint16_t ke = (uint16_t)(kx[i / 2] >> (16 * (i & 1)));
                    const uint16_t ve = (uint16_t)(vx[i / 2] >> (16 * (i & 1)));
                    k[i] = dtype == MA_BF16 ? ma_bf16_to_f32(ke) : ma_f16_to_f32(ke);
                    v[i] = dtype == MA_BF16 ? ma_bf16_to_f32(ve) : ma_f16_to_f32(ve);
                }
            }
            store_n<OT, 8>(a.ko, kb + row * a.s_kt + 8 * oct, k);
            store_n<OT, 8>(a.vo, vb + row * a.s_vt + 8 * oct, v);
        }
        return;
    }
    const int per = a.p.page_tokens / PG_GROUP;
    const int64_t pg = grp / per;
    const uint8_t *rec = pg_record(a.p, a.p.table[(int64_t)b * a.p.s_table + pg], (int)(grp - pg * per), h, 40 * D);
    {
        const int hh = oct / (D / 32), cb = oct % (D / 32);
        uint4 s4{}, z4{};
        if (rec) {
            s4 = *(const uint4 *)(rec + 32 * D + 16 * oct);
            z4 = *(const uint4 *)(rec + 34 * D + 16 * oct);
        }
        const uint32_t sw[4] = {s4.x, s4.y, s4.z, s4.w}, zw[4] = {z4.x, z4.y, z4.z, z4.w};
        uint32_t w[PG_GROUP / TPI];
#pragma unroll
        for (int i = 0; i < PG_GROUP / TPI; ++i) {
            const int t = tk + i * TPI, mt = (t >> 2) & 1, m = 4 * (t >> 3) + (t & 3);
            w[i] = rec ? *(const uint32_t *)(rec + 4 * (((mt * 4 + hh) * 16 + m) * (D / 32) + cb)) : 0u;
        }
#pragma unroll
        for (int i = 0; i < PG_GROUP / TPI; ++i) {
            const int64_t row = t0 + tk + i * TPI;
            uint32_t c[8];
            unpack_word(w[i], c);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = ma_dq(c[e], half_of(sw[e / 2], e & 1), half_of(zw[e / 2], e & 1));
            if (row >= 0 && row < a.n) store_n<OT, 8>(a.ko, kb + row * a.s_kt + 8 * oct, x);
        }
    }
    {
        const int m = lane & 15, hh = lane >> 4;
        uint4 s4{}, z4{};
        uint32_t w[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) w[i] = 0u;
        if (rec) {
            const int cg = NC * m / 32;
            s4 = *(const uint4 *)(rec + 36 * D + 2 * (32 * cg + 8 * hh));
            z4 = *(const uint4 *)(rec + 38 * D + 2 * (32 * cg + 8 * hh));
#pragma unroll
            for (int half = 0; half < D / 64; ++half) {
                const uint4 c = *(const uint4 *)(rec + 16 * D + 16 * (half * 64 + lane));
                w[4 * half] = c.x;
                w[4 * half + 1] = c.y;
                w[4 * half + 2] = c.z;
                w[4 * half + 3] = c.w;
            }
        }
        const uint32_t sw[4] = {s4.x, s4.y, s4.z, s4.w}, zw[4] = {z4.x, z4.y, z4.z, z4.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t row = t0 + 8 * hh + i;
            const float s = half_of(sw[i / 2], i & 1), z = half_of(zw[i / 2], i & 1);
            float x[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) x[c] = ma_dq((w[c] >> ((i & 1) * 16 + (i / 2) * 4)) & 15u, s, z);
            if (row >= 0 && row < a.n) store_n<OT, NC>(a.vo, vb + row * a.s_vt + NC * m, x);
        }
    }
}

bool no_data(const ma_tensor4 &t) { return t.ptr == nullptr; }

}  // namespace

int ma::pg_check(const ma_pages *p, int B, int H, int D, const char *who) {
    if (!p || B <= 0 || H <= 0) {
        ma_set_error("%s: bad geometry (B=%d H=%d)", who, B, H);
        return MA_EINVAL;
    }
    if (D != 64 && D != 128) {
        ma_set_error("%s: head_dim %d is not built (64, 128)", who, D);
        return MA_EUNSUPPORTED;
    }
    if (p->dtype != MA_BF16 && p->dtype != MA_F16) {
        ma_set_error("%s: tails must be bf16 or f16", who);
        return MA_EUNSUPPORTED;
    }
    if (!p->pool || !p->k_tail || !p->v_tail || !p->table || !p->lengths) {
        ma_set_error("%s: NULL page store", who);
        return MA_EINVAL;
    }
    if (p->num_pages <= 0 || p->width <= 0 || p->page_tokens <= 0 || p->page_tokens % PG_GROUP ||
        (p->mask && p->mask_tokens < 0)) {
        ma_set_error("%s: bad page store (num_pages=%d width=%d page_tokens=%d, a multiple of 32)", who, p->num_pages,
                     p->width, p->page_tokens);
        return MA_EINVAL;
    }
    if (((uintptr_t)p->pool | (uintptr_t)p->s_pool[0] | (uintptr_t)p->s_pool[1]) % 16) {
        ma_set_error("%s: pool and its strides must be 16-byte aligned", who);
        return MA_EINVAL;
    }
    if ((int64_t)p->width * p->page_tokens > INT32_MAX) {
        ma_set_error("%s: a request of more than 2^31 - 1 tokens is not built", who);
        return MA_EUNSUPPORTED;
    }
    return MA_OK;
}

static int page_plan(const char *who, bool grow, const int32_t *lengths, const int32_t *new_lens, int B, int T,
                     int page_tokens, int32_t *table, int64_t s_table, int width, int32_t *ring, int num_pages,
                     int32_t *state, int64_t *slots, int32_t *ends, void *stream) {
    if (B <= 0 || T < 0 || page_tokens <= 0 || page_tokens % PG_GROUP || width <= 0 || num_pages <= 0) {
        ma_set_error("%s: bad arguments (B=%d T=%d page_tokens=%d, a multiple of 32, width=%d num_pages=%d)", who, B, T,
                     page_tokens, width, num_pages);
        return MA_EINVAL;
    }
    if (!lengths || !new_lens || !table || !ring || !state || !ends || (T > 0 && !slots)) {
        ma_set_error("%s: NULL argument", who);
        return MA_EINVAL;
    }
    const int64_t nflat = (int64_t)B * (T > 0 ? T : 1), wgs = (nflat + PLAN_SLOTS - 1) / PLAN_SLOTS;
    if ((int64_t)width * page_tokens > INT32_MAX || wgs > INT32_MAX || num_pages > INT32_MAX / 4) {
        ma_set_error("%s: more than 2^31 - 1 tokens of a request, 2^29 pages or 2^42 slots are not built", who);
        return MA_EUNSUPPORTED;
    }
    // every workgroup reads all lengths, and one writes its requests' ends and table rows
    const uintptr_t e = (uintptr_t)ends, span = (uintptr_t)B * sizeof(int32_t);
    for (const uintptr_t x : {(uintptr_t)lengths, (uintptr_t)new_lens})
        if (e < x + span && x < e + span) {
            ma_set_error("%s: ends overlaps lengths or new_lens", who);
            return MA_EINVAL;
        }
    if (B > 1 && s_table < width) {
        ma_set_error("%s: the requests' table rows overlap (stride %lld, width %d)", who, (long long)s_table, width);
        return MA_EINVAL;
    }
    PlanArgs a{lengths, new_lens, table, ring, state, ends, slots, s_table, nflat, B, T, page_tokens, width, num_pages,
               grow};
    page_plan_kernel<<<dim3((unsigned)wgs), PLAN_THREADS, 0, (hipStream_t)stream>>>(a);
    return ma_check_launch(who);
}

extern "C" int ma_page_plan(const int32_t *lengths, const int32_t *new_lens, int B, int T, int page_tokens,
                            int32_t *table, int64_t s_table, int width, int32_t *ring, int num_pages, int32_t *state,
                            int64_t *slots, int32_t *ends, void *stream) {
    return page_plan("ma_page_plan", false, lengths, new_lens, B, T, page_tokens, table, s_table, width, ring, num_pages,
                     state, slots, ends, stream);
}

extern "C" int ma_page_plan_append(const int32_t *lengths, const int32_t *new_lens, int B, int T, int page_tokens,
                                   int32_t *table, int64_t s_table, int width, int32_t *ring, int num_pages,
                                   int32_t *state, int64_t *slots, int32_t *ends, void *stream) {
    return page_plan("ma_page_plan_append", true, lengths, new_lens, B, T, page_tokens, table, s_table, width, ring,
                     num_pages, state, slots, ends, stream);
}

extern "C" int ma_page_append(const ma_pages *p, ma_tensor4 k, ma_tensor4 v, int B, int H, int T, int D,
                              const int32_t *new_lens, const int64_t *slots, void *stream) {
    const char *who = "ma_page_append";
    if (int rc = pg_check(p, B, H, D, who)) return rc;
    if (T <= 0 || no_data(k) || no_data(v) || !new_lens || !slots) {
        ma_set_error("%s: bad arguments (T=%d, or a NULL tensor)", who, T);
        return MA_EINVAL;
    }
    if (k.dtype != p->dtype || v.dtype != p->dtype) {
        ma_set_error("%s: new tokens and tails must share one dtype", who);
        return MA_EINVAL;
    }
    const int64_t units = ((int64_t)T + PG_GROUP - 1) / PG_GROUP;
    if (B > 65535 || H > 65535) {
        ma_set_error("%s: more than 65535 requests or heads are not built", who);
        return MA_EUNSUPPORTED;
    }
    AppendArgs a{pages_dev(p), (const uint16_t *)k.ptr, (const uint16_t *)v.ptr, k.s[0], k.s[1], k.s[2], v.s[0],
                 v.s[1], v.s[2], new_lens, slots, T};
    // (31 + T) / 32 groups can become whole, one at least writes the tail; two groups a workgroup
    const dim3 grid((unsigned)((units + 1) / 2), H, B);
    hipStream_t st = (hipStream_t)stream;
    if (D == 128 && p->dtype == MA_BF16) page_append_kernel<128, MA_BF16><<<grid, 256, 0, st>>>(a);
    else if (D == 128) page_append_kernel<128, MA_F16><<<grid, 256, 0, st>>>(a);
    else if (p->dtype == MA_BF16) page_append_kernel<64, MA_BF16><<<grid, 256, 0, st>>>(a);
    else page_append_kernel<64, MA_F16><<<grid, 256, 0, st>>>(a);
    return ma_check_launch(who);
}

extern "C" int ma_page_dequant(const ma_pages *p, int B, int H, int D, const int32_t *starts, int n, ma_tensor4 k_out,
                               ma_tensor4 v_out, void *stream) {
    const char *who = "ma_page_dequant";
    if (int rc = pg_check(p, B, H, D, who)) return rc;
    if (n < 0 || (n > 0 && (no_data(k_out) || no_data(v_out)))) {
        ma_set_error("%s: bad arguments (n=%d, or a NULL output)", who, n);
        return MA_EINVAL;
    }
    if (k_out.dtype != v_out.dtype || k_out.dtype < MA_F32 || k_out.dtype > MA_BF16) {
        ma_set_error("%s: outputs must share one dtype of bf16, f16, f32", who);
        return MA_EINVAL;
    }
    if (B > 65535 || H > 65535) {
        ma_set_error("%s: more than 65535 requests or heads are not built", who);
        return MA_EUNSUPPORTED;
    }
    if (n == 0) return MA_OK;
    // a range that begins inside a group touches one more
    const int groups = (int)(((int64_t)n + PG_GROUP - 1) / PG_GROUP) + (starts ? 1 : 0);
    DequantArgs a{pages_dev(p), starts, k_out.ptr, v_out.ptr, k_out.s[0], k_out.s[1], k_out.s[2], v_out.s[0],
                  v_out.s[1], v_out.s[2], n, groups};
    const dim3 grid((unsigned)((groups + 3) / 4), H, B);
    hipStream_t st = (hipStream_t)stream;
#define MA_DQ(d, o) page_dequant_kernel<d, o><<<grid, 256, 0, st>>>(a, p->dtype)
    if (D == 128) {
        if (k_out.dtype == MA_BF16) MA_DQ(128, MA_BF16);
        else if (k_out.dtype == MA_F16) MA_DQ(128, MA_F16);
        else MA_DQ(128, MA_F32);
    } else {
        if (k_out.dtype == MA_BF16) MA_DQ(64, MA_BF16);
        else if (k_out.dtype == MA_F16) MA_DQ(64, MA_F16);
        else MA_DQ(64, MA_F32);
    }
#undef MA_DQ
    return ma_check_launch(who);
}
