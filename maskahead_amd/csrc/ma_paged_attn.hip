// Attention of a block of queries of every request over [its pages of 4-bit K/V | its 16-bit
// tail | the block's own keys], for ragged requests whose lengths lie on the device.
//
// The work is a line of items: a group of 32 packed tokens, the tail, or 32 keys of the
// block, of one segment = (request, KV head, row group of up to 16 NT query rows).  Every
// workgroup takes an equal stretch of the line, whatever segments it crosses, so ragged
// lengths need no plan and no read-back: it finds its first request by a scan of the lengths.
// Its four waves take the stretch's items of a segment in turn, each with its own running
// maximum, sum and output (registers only, no barrier), and join them in LDS at the segment's
// end.  A segment that lies in one stretch is written out; one cut between workgroups leaves
// partials, which page_merge_kernel joins.
//
// Per item and wave: S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32, K and V as A
// operands.  A lane of S^T holds 8 tokens of one query row, which is the B operand that P^T
// needs: nothing moves between lanes.  Codes become f16 in place (mask into the mantissa of
// 1024 or 64, subtract, one fused multiply-add by scale and zero: one rounding of 2^-12
// relative, where a bf16 copy of the cache has 2^-9); scores, maxima, sums and outputs are
// f32; probabilities are rounded to f16 (2^-12) for the second product, their sum is not.
// The tail and the block's keys are read as they are: f16 like the above, bf16 in bf16
// products with the probability as a sum of two bf16 (2^-17).
#include "ma_pages.h"

using namespace ma;

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 b16x8_t;

constexpr int WAVES = 4;
// a row's reference maximum is raised only when a score exceeds it by 2^8: most items leave
// the accumulators alone, and p <= 2^8 keeps f16's full precision
constexpr float LAZY = 8.0f;
constexpr float NO_MAX = -1e30f;

struct AttnArgs {
    ma_tensor4 q, kc, vc, out;
    PagesDev p;
    const int32_t *new_lens;
    int B, H, G, T, R, RG, causal, W;
    float sl2;                // scale * log2(e)
    float *wm, *wl, *wo;      // partials of slots [2 W]: per row maximum and sum, unnormalised rows
    int4 *desc;               // [W]: the segment whose first stretch is this workgroup's (see merge)
};

// values that every lane holds alike, as scalars
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
    return (int64_t)(uint32_t)uniform((int)(uint32_t)x) | ((int64_t)uniform((int)(x >> 32)) << 32);
}

struct Items {
    int n, len, ng, rem, items;   // the request's new tokens, stored tokens, whole groups, tail, items
};

__device__ __forceinline__ Items items_of(const AttnArgs &a, int b) {
    Items r;
    r.n = a.new_lens ? min(max(a.new_lens[b], 0), a.T) : a.T;
    r.len = pg_length(a.p, b);
    r.ng = r.len / PG_GROUP;
    r.rem = r.len % PG_GROUP;
    const int cur = a.kc.ptr ? (r.n + PG_GROUP - 1) / PG_GROUP : 0;
    r.items = r.n ? max(r.ng + (r.rem ? 1 : 0) + cur, 1) : 0;
    return r;
}

// pairs of codes as f16 (exact), the k-th pair of a code word
__device__ __forceinline__ f16x2_t code_pair(uint32_t w, int k) {
    const uint32_t x = k & 2 ? w >> 8 : w;
    if (k & 1) {
        const uint32_t y = (x & 0x00f000f0u) | 0x54005400u;   // 64 + code
        return __builtin_bit_cast(f16x2_t, y) - (f16x2_t){(_Float16)64.0f, (_Float16)64.0f};
    }
    const uint32_t y = (x & 0x000f000fu) | 0x64006400u;       // 1024 + code
    return __builtin_bit_cast(f16x2_t, y) - (f16x2_t){(_Float16)1024.0f, (_Float16)1024.0f};
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

// one record's words of a wave
template <int D>
struct Raw {
    uint4 ks[D / 32], kz[D / 32], vs, vz, v[D / 64];
    uint32_t k[2][D / 32];
};

template <int D>
__device__ __forceinline__ void load_k(Raw<D> &w, const uint8_t *rec, int lane) {
    const int h = lane >> 4;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        if constexpr (D == 128) {
            const uint4 c = *(const uint4 *)(rec + mt * 1024 + lane * 16);
            w.k[mt][0] = c.x; w.k[mt][1] = c.y; w.k[mt][2] = c.z; w.k[mt][3] = c.w;
        } else {
            const uint2 c = *(const uint2 *)(rec + mt * 512 + lane * 8);
            w.k[mt][0] = c.x; w.k[mt][1] = c.y;
        }
    }
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb) {
        w.ks[cb] = *(const uint4 *)(rec + 32 * D + 2 * (D / 4) * h + 16 * cb);
        w.kz[cb] = *(const uint4 *)(rec + 34 * D + 2 * (D / 4) * h + 16 * cb);
    }
}
template <int D>
__device__ __forceinline__ void load_v(Raw<D> &w, const uint8_t *rec, int lane) {
    const int h = lane >> 4, m = lane & 15, cg = (D / 16) * m / 32;
#pragma unroll
    for (int half = 0; half < D / 64; ++half) w.v[half] = *(const uint4 *)(rec + 16 * D + 16 * (64 * half + lane));
    w.vs = *(const uint4 *)(rec + 36 * D + 2 * (32 * cg + 8 * h));
    w.vz = *(const uint4 *)(rec + 38 * D + 2 * (32 * cg + 8 * h));
}

// a row tile's running softmax and output: lane (n = lane & 15, h = lane >> 4) holds row n,
// channels (D/16)(4 h + r) + ct in acc[ct][r]; m and l of row n, l over the lane's own tokens
template <int D>
struct Tile {
    f32x4_t acc[D / 16];
    float m, l;
};

// scores s (x sl2 -> exponents of 2) of a lane's 8 tokens -> probabilities; live: bit i =
// token i is seen.  Raises the row's maximum where needed.
template <int D>
__device__ __forceinline__ void softmax8(Tile<D> &t, const f32x4_t &s0, const f32x4_t &s1, float c, bool masked,
                                         uint32_t live, float (&p)[8]) {
    float x[8];
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = __builtin_fmaf(i < 4 ? s0[i & 3] : s1[i & 3], c, -t.m);
        if (masked) x[i] = (live >> i) & 1u ? x[i] : -INFINITY;
        mx = fmaxf(mx, x[i]);
    }
    if (__any(mx > LAZY)) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = (i < 4 ? s0[i & 3] : s1[i & 3]) * c;
            if (masked) x[i] = (live >> i) & 1u ? x[i] : -INFINITY;
            top = fmaxf(top, x[i]);
        }
        const float m = fmaxf(t.m, max_rows(top));
        const float f = __builtin_amdgcn_exp2f(t.m - m);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] -= m;
#pragma unroll
        for (int ct = 0; ct < D / 16; ++ct) t.acc[ct] *= f;
        t.l *= f;
        t.m = m;
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(x[i]);
        sum += p[i];
    }
    t.l += sum;
}

__device__ __forceinline__ uint32_t halves_of(uint32_t bits) {   // bit 0 -> low half, bit 1 -> high half
    return (bits & 1u ? 0xffffu : 0u) | (bits & 2u ? 0xffff0000u : 0u);
}

// the seen ones of a lane's 8 tokens from position pos on
__device__ __forceinline__ uint32_t mask_bits(const PagesDev &p, int b, int h, int64_t pos) {
    const uint8_t *m = p.mask + (int64_t)b * p.s_mb + (int64_t)h * p.s_mh + pos;
    uint32_t bits = 0;
    if (pos + 8 <= p.mask_tokens) {
        const pg_b8 v = *(const pg_b8 *)m;
#pragma unroll
        for (int i = 0; i < 8; ++i) bits |= ((i < 4 ? v.x : v.y) >> (8 * (i & 3)) & 255u) ? 1u << i : 0u;
    } else {
        for (int i = 0; i < 8; ++i)
            if (pos + i < p.mask_tokens && m[i]) bits |= 1u << i;
    }
    return bits;
}

// Q of one row tile as B operands: lane (n, h) = row n, channels (D/4) h + 8 cb + (0..7)
template <int D>
__device__ __forceinline__ const uint16_t *q_row(const AttnArgs &a, int b, int h, int row, int n, bool &ok) {
    const int g = row / a.T, t = row - g * a.T;
    ok = row < a.R && t < n;
    return (const uint16_t *)a.q.ptr + (int64_t)b * a.q.s[0] + (int64_t)(h * a.G + g) * a.q.s[1] +
           (int64_t)t * a.q.s[2];
}
template <int D>
__device__ __forceinline__ void load_q_raw(const AttnArgs &a, int b, int h, int row, int n, int hh, uint4 *q) {
    bool ok;
    const uint16_t *src = q_row<D>(a, b, h, row, n, ok);
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb) q[cb] = ok ? pg_load16(src + (D / 4) * hh + 8 * cb) : uint4{0, 0, 0, 0};
}
// bf16 queries as f16: scaled by a power of two that puts the row's largest in [1, 2), so that
// no query overflows f16 and what underflows is below 2^-24 of it; the factor goes into c
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

template <int D, int NT>
struct Shared {
    static constexpr int OS = D + 4;                 // row stride of a wave's output rows, f32
    float o[WAVES][16 * OS];
    float m[WAVES][16], l[WAVES][16];
    uint4 q[NT > 2 ? NT * (D / 32) * 64 : 1];        // Q operands of many row tiles
    float qc[NT > 2 ? NT * 16 : 1];
    int64_t wsum[WAVES];
    int64_t found_pre;
    int found_b;
};

// items of all requests; the request in which the line's position s (of HR lines of every
// request's items, in a row) lies and the items before it
template <class S>
__device__ __forceinline__ int64_t scan_items(const AttnArgs &a, S &sh, int64_t &total_out, int64_t HR, int min_items,
                                              int64_t &chunk) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (a.B + 255) / 256, first = tid * per;
    int64_t sum = 0;
    for (int i = 0; i < per; ++i)
        if (first + i < a.B) sum += items_of(a, first + i).items;
    int64_t inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(inc, o);
        if (lane >= o) inc += y;
    }
    if (lane == 63) sh.wsum[wave] = inc;
    __syncthreads();
    int64_t before = inc - sum, total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) before += sh.wsum[w];
        total += sh.wsum[w];
    }
    total = uniform(total) * HR;
    const int64_t most = (total + min_items - 1) / min_items;
    const int64_t weff = most < a.W ? most : (int64_t)a.W;
    chunk = weff > 0 ? (total + weff - 1) / weff : 1;
    // stretches of one XCD's workgroups lie next to one another: row groups share its L2
    const int w8 = a.W / 8;
    const int64_t w = (int64_t)(blockIdx.x % 8) * w8 + blockIdx.x / 8;
    const int64_t s = w * chunk;
    if (s < total) {
        const int64_t want = s / HR;
        if (want >= before && want < before + sum) {
            int64_t pre = before;
            int b = first;
            for (;; ++b) {
                const int n = items_of(a, b).items;
                if (want < pre + n) break;
                pre += n;
            }
            sh.found_b = b;
            sh.found_pre = pre;
        }
    }
    __syncthreads();
    total_out = total;
    return w;
}

template <int D, int NT, bool BF16>
__global__ __launch_bounds__(256, NT == 1 ? 2 : 1) void paged_attn_kernel(AttnArgs a, int min_items) {
    constexpr int CB = D / 32, NC = D / 16;
    constexpr bool QLDS = NT > 2;
    __shared__ Shared<D, NT> sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), n16 = lane & 15, hh = lane >> 4;
    const int HR = a.H * a.RG;
    int64_t total, chunk;
    const int64_t w = scan_items(a, sh, total, HR, min_items, chunk);
    const int64_t s = w * chunk;
    int4 desc{-1, 0, 0, 0};
    const int64_t e = min(s + chunk, total);
    int b = uniform(sh.found_b);
    int64_t pre = uniform(sh.found_pre), pos = s;
    Items it = pos < e ? items_of(a, b) : Items{};
    while (pos < e) {
        const int64_t rel = pos - HR * pre;
        const int hr = (int)(rel / it.items), i0 = (int)(rel - (int64_t)hr * it.items);
        const int i1 = (int)min((int64_t)it.items, i0 + (e - pos));
        const int h = hr / a.RG, rg = hr - h * a.RG;
        const int row0 = rg * NT * 16;

        // ---- Q
        uint4 q[QLDS ? 1 : NT][CB];
        float c[NT];
        if constexpr (QLDS) {
            __syncthreads();   // the segment before is done with sh.q
            for (int nt = wave; nt < NT; nt += WAVES) {
                uint4 t[CB];
                load_q_raw<D>(a, b, h, row0 + nt * 16 + n16, it.n, hh, t);
                const float up = BF16 ? q_as_f16<D>(t) : 1.f;
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) sh.q[(nt * CB + cb) * 64 + lane] = t[cb];
                if (hh == 0) sh.qc[nt * 16 + n16] = up * a.sl2;
            }
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) c[nt] = sh.qc[nt * 16 + n16];
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                load_q_raw<D>(a, b, h, row0 + nt * 16 + n16, it.n, hh, q[nt]);
                c[nt] = (BF16 ? q_as_f16<D>(q[nt]) : 1.f) * a.sl2;
            }
        }
        Tile<D> t[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) t[nt].acc[ct] = f32x4_t{};
            t[nt].m = NO_MAX;
            t[nt].l = 0.f;
        }

        // ---- packed groups: this wave's items i0 + wave, + 4, ...
        const int per = a.p.page_tokens / PG_GROUP;
        const int32_t *trow = a.p.table + (int64_t)b * a.p.s_table;
        auto record = [&](int i) -> const uint8_t * {
            const int pg = i / per;
            return pg_record(a.p, trow[pg], i - pg * per, h, 40 * D);
        };
        const int last = min(i1, it.ng);
        Raw<D> w4;
        int i = i0 + wave;
        const uint8_t *rec = nullptr;
        if (i < last) {
            rec = record(i);
            if (rec) {
                load_k(w4, rec, lane);
                load_v(w4, rec, lane);
            }
        }
        for (; i < last; i += WAVES) {
            const uint8_t *next = i + WAVES < last ? record(i + WAVES) : nullptr;
            const bool dead = rec == nullptr;
            f16x8_t kf[2][CB], vf[NC];
            if (!dead) {
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) kf[mt][cb] = word_values(w4.k[mt][cb], w4.ks[cb], w4.kz[cb]);
            }
            if (next) load_k(w4, next, lane);
            bool masked = false;
            uint32_t live = 255u;
            if (!dead) {
                if (a.p.mask) {
                    masked = true;
                    live = mask_bits(a.p, b, h, (int64_t)i * PG_GROUP + 8 * hh);
                    // a dead token's value is 0 whatever its parameters say
                    const uint32_t h0 = halves_of(live), h1 = halves_of(live >> 2), h2 = halves_of(live >> 4),
                                   h3 = halves_of(live >> 6);
                    w4.vs = uint4{w4.vs.x & h0, w4.vs.y & h1, w4.vs.z & h2, w4.vs.w & h3};
                    w4.vz = uint4{w4.vz.x & h0, w4.vz.y & h1, w4.vz.z & h2, w4.vz.w & h3};
                }
#pragma unroll
                for (int ct = 0; ct < NC; ++ct) {
                    const uint4 x = w4.v[ct / 4];
                    const uint32_t word = (ct & 3) == 0 ? x.x : (ct & 3) == 1 ? x.y : (ct & 3) == 2 ? x.z : x.w;
                    vf[ct] = word_values(word, w4.vs, w4.vz);
                }
            }
            if (next) load_v(w4, next, lane);
            rec = next;
            if (dead) continue;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                f32x4_t s0{}, s1{};
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) {
                    const uint4 qw = QLDS ? sh.q[(nt * CB + cb) * 64 + lane] : q[QLDS ? 0 : nt][cb];
                    const f16x8_t qf = __builtin_bit_cast(f16x8_t, qw);
                    s0 = mfma16(kf[0][cb], qf, s0);
                    s1 = mfma16(kf[1][cb], qf, s1);
                }
                float p[8];
                softmax8(t[nt], s0, s1, c[nt], masked, live, p);
                f16x8_t pf;
#pragma unroll
                for (int x = 0; x < 8; ++x) pf[x] = (_Float16)p[x];
#pragma unroll
                for (int ct = 0; ct < NC; ++ct) t[nt].acc[ct] = mfma16(vf[ct], pf, t[nt].acc[ct]);
            }
        }

        // ---- the tail and the block's own keys
        for (; i < i1; i += WAVES) {
            const int x = i - it.ng;
            const bool tail = it.rem && x == 0;
            const int j0 = tail ? 0 : (x - (it.rem ? 1 : 0)) * PG_GROUP;      // first row
            const int cnt = tail ? it.rem : it.n;                              // rows there are
            if (!tail && !a.kc.ptr) continue;                                  // (a request with nothing to see)
            const uint16_t *kb, *vb;
            int64_t sk, sv;
            if (tail) {
                kb = a.p.kt + (int64_t)b * a.p.s_tb + (int64_t)h * a.p.s_th;
                vb = a.p.vt + (int64_t)b * a.p.s_tb + (int64_t)h * a.p.s_th;
                sk = sv = a.p.s_tt;
            } else {
                kb = (const uint16_t *)a.kc.ptr + (int64_t)b * a.kc.s[0] + (int64_t)h * a.kc.s[1];
                vb = (const uint16_t *)a.vc.ptr + (int64_t)b * a.vc.s[0] + (int64_t)h * a.vc.s[1];
                sk = a.kc.s[2];
                sv = a.vc.s[2];
            }
            uint32_t seen = 0;
#pragma unroll
            for (int y = 0; y < 8; ++y) seen |= j0 + 8 * hh + y < cnt ? 1u << y : 0u;
            if (tail && a.p.mask) seen &= mask_bits(a.p, b, h, (int64_t)it.ng * PG_GROUP + 8 * hh);
            uint4 kw[2][CB];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const int j = j0 + 8 * (n16 >> 2) + 4 * mt + (n16 & 3);
#pragma unroll
                for (int cb = 0; cb < CB; ++cb)
                    kw[mt][cb] = j < cnt ? pg_load16(kb + (int64_t)j * sk + (D / 4) * hh + 8 * cb) : uint4{0, 0, 0, 0};
            }
            // V: 8 tokens x NC channels of a lane, turned so that a register pair holds tokens
            uint32_t vw[8][NC / 2];
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                const bool ok = (seen >> y) & 1u;
                const uint16_t *src = vb + (int64_t)(j0 + 8 * hh + y) * sv + NC * n16;
                if constexpr (NC == 8) {
                    const uint4 r = ok ? pg_load16(src) : uint4{0, 0, 0, 0};
                    vw[y][0] = r.x; vw[y][1] = r.y; vw[y][2] = r.z; vw[y][3] = r.w;
                } else {
                    const uint2 r = ok ? pg_load8(src) : uint2{0, 0};
                    vw[y][0] = r.x; vw[y][1] = r.y;
                }
            }
            uint4 vt[NC];
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) {
                uint32_t r[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t lo = vw[2 * k][ct / 2], hi = vw[2 * k + 1][ct / 2];
                    r[k] = ct & 1 ? (lo >> 16) | (hi & 0xffff0000u) : (lo & 0xffffu) | (hi << 16);
                }
                vt[ct] = uint4{r[0], r[1], r[2], r[3]};
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int row = row0 + nt * 16 + n16;
                uint4 qw[CB];
                load_q_raw<D>(a, b, h, row, it.n, hh, qw);
                uint32_t live = seen;
                if (!tail && a.causal > 0) {
                    const int tq = row % a.T;
                    const int64_t lim = ((int64_t)it.len + tq) / a.causal * a.causal + a.causal - it.len;
                    uint32_t ok = 0;
#pragma unroll
                    for (int y = 0; y < 8; ++y) ok |= j0 + 8 * hh + y < lim ? 1u << y : 0u;
                    live &= ok;
                }
                f32x4_t s0{}, s1{};
                float p[8];
                if constexpr (BF16) {
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) {
                        const b16x8_t qf = __builtin_bit_cast(b16x8_t, qw[cb]);
                        s0 = mfma16(__builtin_bit_cast(b16x8_t, kw[0][cb]), qf, s0);
                        s1 = mfma16(__builtin_bit_cast(b16x8_t, kw[1][cb]), qf, s1);
                    }
                    softmax8(t[nt], s0, s1, a.sl2, true, live, p);
                    b16x8_t hi, lo;
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        hi[y] = (__bf16)p[y];
                        lo[y] = (__bf16)(p[y] - (float)hi[y]);
                    }
#pragma unroll
                    for (int ct = 0; ct < NC; ++ct) {
                        const b16x8_t vf = __builtin_bit_cast(b16x8_t, vt[ct]);
                        t[nt].acc[ct] = mfma16(vf, lo, mfma16(vf, hi, t[nt].acc[ct]));
                    }
                } else {
#pragma unroll
                    for (int cb = 0; cb < CB; ++cb) {
                        const f16x8_t qf = __builtin_bit_cast(f16x8_t, qw[cb]);
                        s0 = mfma16(__builtin_bit_cast(f16x8_t, kw[0][cb]), qf, s0);
                        s1 = mfma16(__builtin_bit_cast(f16x8_t, kw[1][cb]), qf, s1);
                    }
                    softmax8(t[nt], s0, s1, a.sl2, true, live, p);
                    f16x8_t pf;
#pragma unroll
                    for (int y = 0; y < 8; ++y) pf[y] = (_Float16)p[y];
#pragma unroll
                    for (int ct = 0; ct < NC; ++ct)
                        t[nt].acc[ct] = mfma16(__builtin_bit_cast(f16x8_t, vt[ct]), pf, t[nt].acc[ct]);
                }
            }
        }

        // ---- the waves' parts joined; whole segments written out, cut ones left as a partial
        const bool whole = i0 == 0 && i1 == it.items;
        const int64_t slot = 2 * w + (pos > s ? 1 : 0);   // cut: the first or the last of the stretch
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float l = sum_rows(t[nt].l);
            __syncthreads();
            if (hh == 0) {
                sh.m[wave][n16] = t[nt].m;
                sh.l[wave][n16] = l;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int ct = 0; ct < NC; ct += 4) {
                    const f32x4_t v = {t[nt].acc[ct][r], t[nt].acc[ct + 1][r], t[nt].acc[ct + 2][r],
                                       t[nt].acc[ct + 3][r]};
                    *(f32x4_t *)&sh.o[wave][n16 * Shared<D, NT>::OS + NC * (4 * hh + r) + ct] = v;
                }
            __syncthreads();
            const int r = tid >> 4, x = tid & 15;      // row, channels NC x + (0 .. NC - 1)
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
                        const f32x4_t y = *(const f32x4_t *)&sh.o[v][r * Shared<D, NT>::OS + NC * x + k];
#pragma unroll
                        for (int z = 0; z < 4; ++z) o[k + z] += y[z] * f;
                    }
                }
                if (whole) {
                    const int g = row / a.T, tq = row - g * a.T;
                    if (tq < it.n) {
                        const float inv = lt == 0.f ? 0.f : 1.f / lt;
                        uint16_t *dst = (uint16_t *)a.out.ptr + (int64_t)b * a.out.s[0] +
                                        (int64_t)(h * a.G + g) * a.out.s[1] + (int64_t)tq * a.out.s[2] + NC * x;
                        uint32_t y[NC / 2];
#pragma unroll
                        for (int k = 0; k < NC / 2; ++k) {
                            if constexpr (BF16) {
                                y[k] = ma_pack_bf16x2(o[2 * k] * inv, o[2 * k + 1] * inv);
                            } else {
                                const f16x2_t z = {(_Float16)(o[2 * k] * inv), (_Float16)(o[2 * k + 1] * inv)};
                                y[k] = __builtin_bit_cast(uint32_t, z);
                            }
                        }
                        if constexpr (NC == 8) pg_store16(dst, uint4{y[0], y[1], y[2], y[3]});
                        else pg_store8(dst, uint2{y[0], y[1]});
                    }
                } else {
                    const int64_t at = slot * (NT * 16) + nt * 16 + r;
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
        // the first stretch of a cut segment names it to the merge: (request, (head, row group),
        // first slot, stretches)
        if (!whole && i0 == 0) {
            const int64_t seg_end = pos + it.items;
            desc = int4{b, hr, (int)slot, (int)((seg_end - 1) / chunk - w + 1)};
        }
        pos += i1 - i0;
        if (i1 == it.items && hr == HR - 1 && pos < e) {
            pre += it.items;
            do it = items_of(a, ++b);
            while (it.items == 0);
        }
    }
    if (tid == 0) a.desc[w] = desc;
}

// Partials of a cut segment, joined: its first partial lies in slot desc.z, the stretch after
// workgroup w's in slot 2 (w + 1), and so on.  A workgroup takes 4 rows; 4 groups of 16 threads
// a row take every fourth partial and are joined in LDS, in a fixed order.
template <int D, int NT, bool BF16>
__global__ __launch_bounds__(256) void page_merge_kernel(AttnArgs a) {
    constexpr int NC = D / 16;
    __shared__ float sm[4][4], sl[4][4];
    __shared__ float so[4][4][D];
    const int w = blockIdx.x;
    const int4 d = a.desc[w];
    if (d.x < 0) return;
    const int r = threadIdx.x >> 6, grp = (threadIdx.x >> 4) & 3, x = threadIdx.x & 15;
    const int h = d.y / a.RG, rg = d.y - h * a.RG;
    const int rt = blockIdx.y * 4 + r, row = rg * NT * 16 + rt;
    const int n = a.new_lens ? min(max(a.new_lens[d.x], 0), a.T) : a.T;
    float m = NO_MAX, l = 0.f, o[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) o[k] = 0.f;
    if (row < a.R) {
        for (int k = grp; k < d.w; k += 4) {
            const int64_t at = (k ? 2 * (int64_t)(w + k) : (int64_t)d.z) * (NT * 16) + rt;
            const float pm = a.wm[at], pl = a.wl[at];
            const float nm = fmaxf(m, pm);
            const float f = __builtin_amdgcn_exp2f(m - nm), g = __builtin_amdgcn_exp2f(pm - nm);
            m = nm;
            l = l * f + pl * g;
#pragma unroll
            for (int y = 0; y < NC; y += 4) {
                const f32x4_t v = *(const f32x4_t *)&a.wo[at * D + NC * x + y];
#pragma unroll
                for (int z = 0; z < 4; ++z) o[y + z] = o[y + z] * f + v[z] * g;
            }
        }
    }
    if (x == 0) {
        sm[r][grp] = m;
        sl[r][grp] = l;
    }
#pragma unroll
    for (int y = 0; y < NC; ++y) so[r][grp][NC * x + y] = o[y];
    __syncthreads();
    if (grp != 0 || row >= a.R) return;
    const int g = row / a.T, t = row - g * a.T;
    if (t >= n) return;
    m = fmaxf(fmaxf(sm[r][0], sm[r][1]), fmaxf(sm[r][2], sm[r][3]));
    l = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) o[k] = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const float f = __builtin_amdgcn_exp2f(sm[r][v] - m);
        l += sl[r][v] * f;
#pragma unroll
        for (int k = 0; k < NC; ++k) o[k] += so[r][v][NC * x + k] * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t *dst = (uint16_t *)a.out.ptr + (int64_t)d.x * a.out.s[0] + (int64_t)(h * a.G + g) * a.out.s[1] +
                    (int64_t)t * a.out.s[2] + NC * x;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        if constexpr (BF16) dst[k] = ma_f32_to_bf16(o[k] * inv);
        else dst[k] = __builtin_bit_cast(uint16_t, (_Float16)(o[k] * inv));
    }
}

// ------------------------------------------------------------------ host
struct Shape {
    int NT, RG, W;
};

// Row tiles of 16 a wave holds, and row groups.  An item costs a wave about 100 (unpacking K
// and V) + 65 a row tile (both products and the softmax), so more tiles a wave are better until
// registers end; of the built numbers the cheapest split of ceil(R / 16) tiles is taken.
Shape shape_of(int R) {
    const int tiles = (R + 15) / 16;
    const int built[] = {1, 2, 4, 7};
    Shape best{1, tiles, 0};
    int64_t cost = INT64_MAX;
    for (int nt : built) {
        const int rg = (tiles + nt - 1) / nt;
        const int64_t c = (int64_t)rg * (100 + 65 * nt);
        if (c < cost) {
            cost = c;
            best = Shape{nt, rg, 0};
        }
    }
    // as many workgroups as are resident at once
    best.W = ma_num_cus() / 8 * 8 * (best.NT == 1 ? 2 : 1);
    return best;
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

struct Layout {
    int64_t wl, wo, desc, bytes;   // wm at 0
};
Layout layout_of(const Shape &s, int D) {
    const int64_t rows = 2LL * s.W * s.NT * 16;
    Layout l;
    l.wl = align256(rows * 4);
    l.wo = l.wl + align256(rows * 4);
    l.desc = l.wo + align256(rows * D * 4);
    l.bytes = l.desc + align256((int64_t)s.W * sizeof(int4));
    return l;
}

template <int D, int NT, bool BF16>
int launch(const AttnArgs &a, hipStream_t st) {
    paged_attn_kernel<D, NT, BF16><<<a.W, 256, 0, st>>>(a, WAVES);
    page_merge_kernel<D, NT, BF16><<<dim3(a.W, NT * 4), 256, 0, st>>>(a);
    return ma_check_launch("ma_paged_attention");
}
template <int D, bool BF16>
int launch_nt(const AttnArgs &a, int nt, hipStream_t st) {
    if (nt == 1) return launch<D, 1, BF16>(a, st);
    if (nt == 2) return launch<D, 2, BF16>(a, st);
    if (nt == 4) return launch<D, 4, BF16>(a, st);
    return launch<D, 7, BF16>(a, st);
}

}  // namespace

extern "C" int64_t ma_paged_workspace_bytes(int B, int H, int Hq, int T, int D) {
    if (B <= 0 || H <= 0 || Hq <= 0 || Hq % H || T <= 0 || (D != 64 && D != 128)) return -1;
    if ((int64_t)(Hq / H) * T > INT32_MAX / 16) return -1;
    return layout_of(shape_of(Hq / H * T), D).bytes;
}

extern "C" int ma_paged_attention(ma_tensor4 q, int B, int Hq, int T, int D, const ma_pages *p, int H, ma_tensor4 kc,
                                  ma_tensor4 vc, const int32_t *new_lens, int causal_block, float scale,
                                  ma_tensor4 out, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "ma_paged_attention";
    if (int rc = pg_check(p, B, H, D, who)) return rc;
    const int64_t need = ma_paged_workspace_bytes(B, H, Hq, T, D);
    if (need < 0 || !q.ptr || !out.ptr || causal_block < 0 || (kc.ptr == nullptr) != (vc.ptr == nullptr)) {
        ma_set_error("%s: bad arguments (B=%d H=%d Hq=%d T=%d D=%d causal_block=%d)", who, B, H, Hq, T, D, causal_block);
        return MA_EINVAL;
    }
    if (q.dtype != p->dtype || out.dtype != p->dtype || (kc.ptr && (kc.dtype != p->dtype || vc.dtype != p->dtype))) {
        ma_set_error("%s: queries, the block's keys and values, out and tails must share one dtype", who);
        return MA_EINVAL;
    }
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256) {
        ma_set_error("%s: workspace of %lld bytes (256-byte aligned) needed, got %lld", who, (long long)need,
                     (long long)workspace_bytes);
        return MA_EWORKSPACE;
    }
    const Shape s = shape_of(Hq / H * T);
    const Layout l = layout_of(s, D);
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
    a.R = a.G * T;
    a.RG = s.RG;
    a.causal = causal_block;
    a.W = s.W;
    a.sl2 = scale * MA_LOG2E;
    a.wm = (float *)ws;
    a.wl = (float *)(ws + l.wl);
    a.wo = (float *)(ws + l.wo);
    a.desc = (int4 *)(ws + l.desc);
    hipStream_t st = (hipStream_t)stream;
    if (D == 128) return p->dtype == MA_BF16 ? launch_nt<128, true>(a, s.NT, st) : launch_nt<128, false>(a, s.NT, st);
    return p->dtype == MA_BF16 ? launch_nt<64, true>(a, s.NT, st) : launch_nt<64, false>(a, s.NT, st);
}
