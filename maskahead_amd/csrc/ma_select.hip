// Blocks of stored tokens for a run of query positions, by a score that reads a tenth of the cache.
//
// A packed key is z_c + s_c j with a code j of 0 .. 15, and its record holds z and s of every channel
// c for its 32 tokens.  So no token of the group scores a query row more than
//     sum over c of max(q_c z_c, q_c (z_c + 15 s_c)) = sum of q_c z_c + max(q_c, 0) 15 s_c
// (s not negative): one matrix product with [z | 15 s], 4 D of a record's 40 D bytes.
//
// Which blocks are read must not hang on the order of a sum, so the products are of whole numbers:
// q_c times 2^(13 - e), rounded, where 2^e is the power of two at or below the row's largest (e at
// least -100), and z_c and 15 s_c times 2^(13 - f) with the group's largest alike (f at least -24).
// A code of at most 2^14 is two digits, 256 hi + lo with lo of -128 .. 127, so the product of 8-bit
// integers computes it: four of digits, each at most 2^22 over 2 D channels.  The score, a whole number
// below 2^37 times 2^(e + f - 26), is rounded once, to f32.
#include "ma_pages.h"

using namespace ma;

namespace {

constexpr float LEAST = -3.4028234663852886e38f;

struct SelectArgs {
    ma_tensor4 q;
    PagesDev p;
    const int32_t *new_lens;
    float *group;               // [B, H, runs, ngcap] scores of groups
    float *scores;              // [B, H, runs, nbcap] of blocks, or NULL
    int32_t *blocks;            // [B, H, runs, count]
    int64_t ngcap, nbcap;
    int B, H, G, T, run, runs, m, count, first, last;
    int units;                  // workgroups' worth of groups in a batch of requests as long as their table rows
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int new_of(const SelectArgs &a, int b) {
    return a.new_lens ? min(max(a.new_lens[b], 0), a.T) : a.T;
}

template <int DT>
__device__ __forceinline__ void unpack8(uint4 w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == MA_BF16) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else {
            x[2 * i] = ma_f16_to_f32((uint16_t)u[i]);
            x[2 * i + 1] = ma_f16_to_f32((uint16_t)(u[i] >> 16));
        }
    }
}

typedef __attribute__((ext_vector_type(4))) int i32x4_t;
// Codes, rounded half to even, and their digits (2.25 instructions a value): the sum with 1.5 2^23 + 128
// leaves code + 128 in the lowest 16 bits, whose upper byte is hi, and whose lower is lo + 128.  Two codes
// + 128 in a word:
__device__ __forceinline__ uint32_t code_pair(float x, float y, float scale) {
    const uint32_t a = __float_as_uint(__builtin_fmaf(x, scale, 12583040.0f));
    const uint32_t b = __float_as_uint(__builtin_fmaf(y, scale, 12583040.0f));
    return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
// ... into word i of the digits; ... and 0 for a negative code
__device__ __forceinline__ void put_digits(uint32_t x, uint32_t y, int i, i32x4_t &hi, i32x4_t &lo) {
    lo[i] = (int)(__builtin_amdgcn_perm(y, x, 0x06040200u) ^ 0x80808080u);
    hi[i] = (int)__builtin_amdgcn_perm(y, x, 0x07050301u);
}
typedef __attribute__((ext_vector_type(2))) int16_t s16x2_t;
__device__ __forceinline__ uint32_t positive(uint32_t x) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(s16x2_t, x), (s16x2_t){128, 128}));
}
// 16 channels: f(i, pairs of channels 4 i .. 4 i + 3)
template <int DT, class F>
__device__ __forceinline__ void each_pair(const uint4 (&w)[2], float scale, F f) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        float v[8];
        unpack8<DT>(w[y], v);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            f(2 * y + i, code_pair(v[4 * i], v[4 * i + 1], scale), code_pair(v[4 * i + 2], v[4 * i + 3], scale));
    }
}
__device__ __forceinline__ void group_digits(const uint4 (&w)[2], float scale, i32x4_t &hi, i32x4_t &lo) {
    each_pair<MA_F16>(w, scale, [&](int i, uint32_t x, uint32_t y) { put_digits(x, y, i, hi, lo); });
}
__device__ __forceinline__ i32x4_t mfma_i8(i32x4_t a, i32x4_t b, i32x4_t c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// maximum over the four lanes of a row (lane ^ 16, lane ^ 32)
__device__ __forceinline__ float max_rows(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return ma_max_xor32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
// Largest magnitude of 16-bit floats, as bits of one: without its sign a float is ordered like a whole
// number, infinities and NaN above all.
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2_t;
__device__ __forceinline__ void most_of(uint4 w, u16x2_t &most) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, u[i] & 0x7fff7fffu));
}
// ... over the four lanes of a row, as f32; not finite: infinite
template <int DT>
__device__ __forceinline__ float most_float(u16x2_t most) {
    const float x = max_rows((float)max(most[0], most[1]));         // (16 bits: a whole number of f32)
    const uint16_t h = (uint16_t)x;
    if constexpr (DT == MA_BF16) return h >= 0x7f80 ? INFINITY : ma_bf16_to_f32(h);
    return h >= 0x7c00 ? INFINITY : ma_f16_to_f32(h);
}

// a workgroup's work: spans of its groups, runs of positions, heads, requests (fastest to slowest: runs,
// heads, spans, so that what is under way together reads the same pages)
struct Unit {
    int b, len, n;       // request, its stored tokens and new positions; b < 0: behind the last
    int run, h, span;
};
__device__ __forceinline__ Unit find_unit(const SelectArgs &a, int u, int span, int lane) {
    Unit r{-1, 0, 0, 0, 0, 0};
    unsigned pre = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {       // 64 requests at a time, the units of those before
        int len = 0, n = 0;
        unsigned units = 0;
        if (b0 + lane < a.B) {
            len = pg_length(a.p, b0 + lane);
            n = new_of(a, b0 + lane);
            units = (unsigned)((len / PG_GROUP + span - 1) / span) * a.H * ((unsigned)(n + a.run - 1) / (unsigned)a.run);
        }
        const unsigned inc = pre + ma_wave_prefix_u32(units);
        const uint64_t here = __ballot((unsigned)u >= inc - units && (unsigned)u < inc);
        if (here) {
            const int l = __ffsll((unsigned long long)here) - 1;
            r.b = b0 + l;
            r.len = __builtin_amdgcn_readlane(len, l);
            r.n = __builtin_amdgcn_readlane(n, l);
            const unsigned rel = (unsigned)u - (unsigned)__builtin_amdgcn_readlane((int)(inc - units), l);
            const unsigned runs = (unsigned)(r.n + a.run - 1) / (unsigned)a.run, rest = rel / runs;
            r.run = (int)(rel - rest * runs);
            r.span = (int)(rest / (unsigned)a.H);
            r.h = (int)(rest - (unsigned)r.span * (unsigned)a.H);
            break;
        }
        pre = (unsigned)__builtin_amdgcn_readlane((int)inc, 63);
    }
    return r;
}

// ------------------------------------------------------------------ scores of groups
// A workgroup of NW waves: 16 NW groups of one (request, head) and the rows of one run; a wave holds the
// digits of its 16 groups' parameters and passes all rows by them, whose digits lie in LDS, a tile of 16
// rows from every wave at a time.
//
// bound: few rows: latency (lengths, table and rows, parameters: three loads in a row) and 4 D bytes a
// group and head.  One token of 64 requests of 700 to 16 384 tokens (28 query and 4 KV heads, D 128): 20 MB
// in 9.7 us; of 2 requests of 90 000 to 131 072 (32 and 8 heads): 29 MB in 10.5.  A workgroup for every unit
// that a table row can name, which need not look for its request, was slower where most rows are shorter
// (the first with its top 16.3 -> 19.7).  Many rows: the instructions around the products.  224 rows of 16
// runs over 350 and 512 groups: 22.1 us, of which the matrix cores 5 and the other instructions 10 (1 640 a
// wave: the running maximum 340, digits of rows 350 and of parameters 250), at 14 waves a CU; waves of 32
// groups 24.9.  Digits of f16 and their products, which take twice the time and registers: 12.3, 13.4 and
// 44.5 us.
struct RowScale {
    double by, add;      // a row's power of two and 0; no row: 0 and -inf; one that is not finite: 0 and inf
};
template <int D, int DT, int NW>
__global__ __launch_bounds__(64 * NW, 4) void select_score_kernel(SelectArgs a) {
    constexpr int KB = D / 64, SPAN = 16 * NW;
    __shared__ i32x4_t dig[NW][4][KB][64];         // hi, lo, and those of the positive codes
    __shared__ RowScale scales[NW][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), n16 = lane & 15, hh = lane >> 4;
    const int R = a.G * a.run, tiles = (R + 15) / 16, per = a.p.page_tokens / PG_GROUP;
    for (int u = blockIdx.x; u < a.units; u += gridDim.x) {
        const Unit x = find_unit(a, u, SPAN, lane);
        if (x.b < 0) return;         // (all waves alike)
        const int b = x.b, h = x.h, n = x.n, ng = x.len / PG_GROUP;
        // the lane's group (behind the last: the last, which is not stored again)
        const int g = x.span * SPAN + 16 * wave + n16, gc = min(g, ng - 1), pg = gc / per;
        const int page = a.p.table[(int64_t)b * a.p.s_table + pg];
        // the rows of tile t (this wave's), or of the only one
        uint4 w[KB][2];
        int pos_of_row = 0;
        auto load_rows = [&](int t) {
            const int rc = min(16 * t + n16, R - 1), qh = rc / a.run;
            pos_of_row = x.run * a.run + rc - qh * a.run;
            const uint16_t *src = (const uint16_t *)a.q.ptr + (int64_t)b * a.q.s[0] + (int64_t)(h * a.G + qh) * a.q.s[1] +
                                  (int64_t)min(pos_of_row, a.T - 1) * a.q.s[2] + 16 * hh;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int y = 0; y < 2; ++y) w[kb][y] = pg_load16(src + 64 * kb + 8 * y);
        };
        load_rows(tiles == 1 ? 0 : wave);       // (behind the last tile: the last row)
        const uint8_t *rec = pg_record(a.p, page, gc - pg * per, h, 40 * D);
        bool live = rec != nullptr;
        if (!rec) rec = a.p.pool;
        uint4 sw[KB][2], zw[KB][2];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                sw[kb][z] = *(const uint4 *)(rec + 32 * D + 2 * (64 * kb + 16 * hh + 8 * z));
                zw[kb][z] = *(const uint4 *)(rec + 34 * D + 2 * (64 * kb + 16 * hh + 8 * z));
            }
        if (a.p.mask) {
            const bool any = pg_mask_bits(a.p, b, h, gc * PG_GROUP + 8 * hh) != 0;
            live = live && max_rows(any ? 1.f : 0.f) != 0.f;
        }
        // the rows' digits into LDS: a tile a wave, or 64 channels of the only one
        auto put_rows = [&](int t0) {
            const int t = tiles == 1 ? 0 : wave;
            if (t0 + t >= tiles || (tiles == 1 && wave >= KB)) return;
            u16x2_t most{};
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) most_of(w[kb][0], most), most_of(w[kb][1], most);
            const float mx = most_float<DT>(most);
            const bool odd = mx == INFINITY;
            const int e = max((int)(__float_as_uint(mx) >> 23) - 127, -100);
            const float scale = odd ? 0.f : pow2(13 - e);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                if (tiles == 1 && kb != wave) continue;
                i32x4_t hi, lo, rh, rl;
                each_pair<DT>(w[kb], scale, [&](int i, uint32_t v0, uint32_t v1) {
                    put_digits(v0, v1, i, hi, lo);
                    put_digits(positive(v0), positive(v1), i, rh, rl);
                });
                dig[t][0][kb][lane] = hi;
                dig[t][1][kb][lane] = lo;
                dig[t][2][kb][lane] = rh;
                dig[t][3][kb][lane] = rl;
            }
            const bool none = 16 * (t0 + t) + n16 >= R || pos_of_row >= n;
            if (hh == 0) scales[t][n16] = RowScale{none || odd ? 0.0 : (double)pow2(e), none ? -INFINITY : odd ? INFINITY : 0.0};
        };
        __syncthreads();         // the unit's before is read
        put_rows(0);
        u16x2_t ms{}, mz{};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int z = 0; z < 2; ++z) most_of(sw[kb][z], ms), most_of(zw[kb][z], mz);
        const float top = fmaxf(15.0f * most_float<MA_F16>(ms), most_float<MA_F16>(mz));
        const bool odd = top == INFINITY;
        const int f = max((int)(__float_as_uint(top) >> 23) - 127, -24);
        const float scale = odd ? 0.f : pow2(13 - f);
        i32x4_t zh[KB], zl[KB], sh[KB], sl[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            group_digits(zw[kb], scale, zh[kb], zl[kb]);
            group_digits(sw[kb], 15.0f * scale, sh[kb], sl[kb]);
        }
        double best = -INFINITY;         // the rows' largest exact score, before the group's power of two
        for (int t0 = 0; t0 < tiles; t0 += NW) {
            if (t0) {
                __syncthreads();          // the rows before are read
                put_rows(t0);
            }
            __syncthreads();
            if (t0 + NW < tiles) load_rows(t0 + NW + wave);
            for (int t = 0; t < min(NW, tiles - t0); ++t) {
                i32x4_t c2{}, c1{}, c0{};
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const i32x4_t qh = dig[t][0][kb][lane], ql = dig[t][1][kb][lane];
                    const i32x4_t rh = dig[t][2][kb][lane], rl = dig[t][3][kb][lane];
                    c1 = mfma_i8(qh, zl[kb], c1);
                    c2 = mfma_i8(qh, zh[kb], c2);
                    c0 = mfma_i8(ql, zl[kb], c0);
                    c1 = mfma_i8(ql, zh[kb], c1);
                    c2 = mfma_i8(rh, sh[kb], c2);
                    c1 = mfma_i8(rh, sl[kb], c1);
                    c0 = mfma_i8(rl, sl[kb], c0);
                    c1 = mfma_i8(rl, sh[kb], c1);
                }
                // lane (n, h): rows 4 h + r by group n (256 c1 + c0 is below 2^31)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const RowScale e = scales[t][4 * hh + r];
                    const double s = __builtin_fma((double)c2[r], 65536.0, (double)(c1[r] * 256 + c0[r]));
                    best = __builtin_fmax(best, __builtin_fma(s, e.by, e.add));
                }
            }
        }
        float v = best == -INFINITY ? -INFINITY : fmaxf((float)__builtin_ldexp(best, f - 26), LEAST);
        v = max_rows(odd && v > -INFINITY ? INFINITY : v);
        if (hh == 0 && g < ng) a.group[(((int64_t)b * a.H + h) * a.runs + x.run) * a.ngcap + g] = live ? v : -INFINITY;
    }
}

// ------------------------------------------------------------------ selection
// One workgroup a (request, head, run): the count largest block scores, ties to the lowest index, in
// ascending order.  A key is the score's place in the order of floats, 0 for no block; blocks that are
// always taken stand outside the search.  The search counts keys in equal ranges between the
// smallest and the largest, four a thread, then within the range that the last one lies in, and so on:
// three turns (1 024 ranges: four) at most, mostly one, as a range that is taken whole ends it; and scores
// alike do not meet in one counter as they would by their leading bits.
constexpr uint32_t KEY_TAKEN = 0xffffffffu;

template <int THREADS>
struct TopShared {
    static constexpr int WAVES = THREADS / 64, BINS = 4 * THREADS;
    uint32_t bin[BINS], red[4][WAVES], sum[WAVES], pick[2][WAVES];
    uint32_t at, above, in;
};
// the waves' values of one array, one a lane (0 behind the last)
template <int WAVES>
__device__ __forceinline__ uint32_t of_waves(const uint32_t (&x)[WAVES], int lane) {
    const uint32_t v = x[min(lane, WAVES - 1)];
    return lane < WAVES ? v : 0;
}
// what the waves before this one have, and all
__device__ __forceinline__ void wave_offsets(uint32_t v, int wave, uint32_t &before, uint32_t &all) {
    const uint32_t inc = ma_wave_prefix_u32(v);
    before = wave ? (uint32_t)__builtin_amdgcn_readlane((int)inc, wave - 1) : 0;
    all = (uint32_t)__builtin_amdgcn_readlane((int)inc, 63);
}

// PER > 0: a thread keeps its keys, at most PER, of at most THREADS * PER blocks; 0: they are read again in
// every turn.  Scores are read a wave's width at a time and handed over in LDS (dynamic, THREADS * PER keys)
// to the threads that hold PER neighbours; the first are asked for before the request's length is known.
//
// bound: latency (loads, then five barriers).  256 rows of up to 512 blocks 5.5 us, 16 of up to 2 048 (of two
// groups) 8.0, of which some 3 are the launch.  256 threads hold up to 1 024 blocks (1 024 threads: 6.5 us where
// they take 5.9), 1 024 threads more (256: 14.3 us where they take 8.9).
template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void select_top_kernel(SelectArgs a) {
    using Shared = TopShared<THREADS>;
    constexpr int BINS = Shared::BINS, BPT = BINS / THREADS, BIN_BITS = THREADS == 256 ? 10 : 12;
    static_assert(BINS == 1 << BIN_BITS, "ranges are told apart by a shift");
    __shared__ Shared sh;
    extern __shared__ uint32_t all_keys[];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int64_t row = blockIdx.x;
    const float *group = a.group + row * a.ngcap;
    constexpr int U = PER < 8 ? PER : 8;             // blocks of a thread whose loads are under way together
    float v[U ? U : 1][2];
    // groups j and j + 1 of blocks y0 THREADS + tid + ..., below `blocks` and `groups` (a last one twice)
    auto load = [&](int y0, int j, int blocks, int groups) {
#pragma unroll
        for (int y = 0; y < U; ++y)
#pragma unroll
            for (int z = 0; z < 2; ++z)
                v[y][z] = group[min(min(tid + (y0 + y) * THREADS, blocks - 1) * a.m + min(j + z, a.m - 1), groups - 1)];
    };
    if constexpr (PER > 0) load(0, 0, (int)a.nbcap, (int)a.ngcap);
    const int run = (int)((unsigned)blockIdx.x % (unsigned)a.runs), b = (int)((unsigned)blockIdx.x / (unsigned)a.runs / (unsigned)a.H);
    const int n = new_of(a, b), len = pg_length(a.p, b), ng = run * a.run < n ? len / PG_GROUP : 0;
    const int nb = (int)((unsigned)(ng + a.m - 1) / (unsigned)a.m);
#pragma unroll
    for (int y = 0; y < BPT; ++y) sh.bin[tid + y * THREADS] = 0;
    // this thread's blocks [i0, i1)
    const int each = (nb + THREADS - 1) / THREADS, i0 = min(tid * each, nb), i1 = min(i0 + each, nb);
    auto key_of = [&](int i, float s) -> uint32_t {
        if (s == -INFINITY) return 0;
        return i < a.first || i >= nb - a.last ? KEY_TAKEN : ma_order_key(s);
    };
    uint32_t key[PER ? PER : 1];
    uint32_t lo = 0xffffffffu, hi = 0, some = 0, taken = 0;
    auto note = [&](uint32_t k) {
        if (k == 0) return;
        ++some;
        if (k == KEY_TAKEN) ++taken;
        else lo = min(lo, k), hi = max(hi, k);
    };
    auto score_of = [&](int i) {
        float s = -INFINITY;
        for (int y = i * a.m; y < min((i + 1) * a.m, ng); ++y) s = fmaxf(s, group[y]);
        return s;
    };
    if constexpr (PER > 0) {
#pragma unroll
        for (int y0 = 0; y0 < PER; y0 += U) {
            if (y0 * THREADS >= nb) break;
            float s[U];
#pragma unroll
            for (int y = 0; y < U; ++y) s[y] = -INFINITY;
            for (int j = 0; j < min(a.m, ng); j += 2) {
                if (y0 + j > 0) load(y0, j, nb, ng);
#pragma unroll
                for (int y = 0; y < U; ++y)
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        // (what was asked for early may lie behind the length)
                        const int i = tid + (y0 + y) * THREADS;
                        if (i < nb && i * a.m + min(j + z, a.m - 1) < ng) s[y] = fmaxf(s[y], v[y][z]);
                    }
            }
#pragma unroll
            for (int y = 0; y < U; ++y) {
                const int i = tid + (y0 + y) * THREADS;
                const uint32_t k = i < nb ? key_of(i, s[y]) : 0;
                all_keys[i] = k;
                note(k);
                if (a.scores && a.scores != a.group && i < nb) a.scores[row * a.nbcap + i] = s[y];
            }
        }
    } else {
        for (int i = i0; i < i1; ++i) {
            const float s = score_of(i);
            note(key_of(i, s));
            if (a.scores && a.scores != a.group) a.scores[row * a.nbcap + i] = s;
        }
    }
    some = ma_wave_sum_u32(some);
    taken = ma_wave_sum_u32(taken);
    lo = ma_wave_max_u32(~lo);
    hi = ma_wave_max_u32(hi);
    if (lane == 0) sh.red[0][wave] = some, sh.red[1][wave] = taken, sh.red[2][wave] = lo, sh.red[3][wave] = hi;
    __syncthreads();
    if constexpr (PER > 0) {
#pragma unroll
        for (int y = 0; y < PER; ++y) key[y] = i0 + y < i1 ? all_keys[i0 + y] : 0;
    }
    auto each_key = [&](auto f) {
        if constexpr (PER > 0) {
#pragma unroll
            for (int y = 0; y < PER; ++y) f(i0 + y, key[y]);
        } else {
            for (int i = i0; i < i1; ++i) f(i, key_of(i, score_of(i)));
        }
    };
    const uint32_t all = ma_wave_sum_u32(of_waves(sh.red[0], lane)), forced = ma_wave_sum_u32(of_waves(sh.red[1], lane));
    lo = ~ma_wave_max_u32(of_waves(sh.red[2], lane));
    hi = ma_wave_max_u32(of_waves(sh.red[3], lane));
    // what is taken: keys above cut, and the first `ties` of those equal to it
    uint32_t cut = 0, ties = 0;
    const uint32_t want = min((uint32_t)a.count, all);
    if (want < all) {
        uint32_t need = want - min(forced, want);
        if (need == 0) cut = KEY_TAKEN - 1;
        for (bool again = false; need; again = true) {
            if (again) {
#pragma unroll
                for (int y = 0; y < BPT; ++y) sh.bin[tid + y * THREADS] = 0;
                __syncthreads();
            }
            const uint32_t range = hi - lo;
            const int bits = range ? 32 - __builtin_clz(range) : 0, s = max(bits - BIN_BITS, 0);
            each_key([&](int, uint32_t k) {
                if (k >= lo && k <= hi && k != 0) atomicAdd(&sh.bin[(k - lo) >> s], 1u);
            });
            __syncthreads();
            // ranges from the top, BPT a thread: the one in which the need-th lies
            uint32_t c[BPT], sum = 0;
#pragma unroll
            for (int y = 0; y < BPT; ++y) {
                c[y] = sh.bin[BINS - 1 - (tid * BPT + y)];
                sum += c[y];
            }
            const uint32_t inc = ma_wave_prefix_u32(sum);
            if (lane == 63) sh.sum[wave] = inc;
            __syncthreads();
            uint32_t above, total;
            wave_offsets(of_waves(sh.sum, lane), wave, above, total);
            above += inc - sum;
#pragma unroll
            for (int y = 0; y < BPT; ++y) {
                if (above < need && need <= above + c[y]) {
                    sh.at = BINS - 1 - (tid * BPT + y);
                    sh.above = above;
                    sh.in = c[y];
                }
                above += c[y];
            }
            __syncthreads();
            lo += sh.at << s;
            hi = min(hi, lo + (s ? (1u << s) - 1 : 0));
            need -= sh.above;
            if (need == sh.in) {         // all of the range
                cut = lo - 1;
                break;
            }
            if (s == 0) {
                cut = lo;
                ties = need;
                break;
            }
        }
    }
    uint32_t over = 0, equal = 0;
    each_key([&](int, uint32_t k) {
        if (k > cut) ++over;
        else if (k == cut && k != 0) ++equal;
    });
    const uint32_t oi = ma_wave_prefix_u32(over), ei = ma_wave_prefix_u32(equal);
    if (lane == 63) sh.pick[0][wave] = oi, sh.pick[1][wave] = ei;
    __syncthreads();
    uint32_t ob, eb, unused;
    wave_offsets(of_waves(sh.pick[0], lane), wave, ob, unused);
    wave_offsets(of_waves(sh.pick[1], lane), wave, eb, unused);
    ob += oi - over;
    eb += ei - equal;
    int32_t *out = a.blocks + row * a.count;
    each_key([&](int i, uint32_t k) {
        if (k > cut) {
            out[ob + min(eb, ties)] = i;
            ++ob;
        } else if (k == cut && k != 0) {
            if (eb < ties) out[ob + eb] = i;
            ++eb;
        }
    });
    for (int i = (int)want + tid; i < a.count; i += THREADS) out[i] = -1;
    if (a.scores)
        for (int64_t i = nb + tid; i < a.nbcap; i += THREADS) a.scores[row * a.nbcap + i] = -INFINITY;
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

// Waves of a workgroup: 8 share the rows' digits among twice the groups, which pays where those take several
// turns of 4 tiles and the workgroups keep every SIMD busy; else 4, which wait for less.  With their tops:
// 512 positions of 2 requests in runs of 32 (224 rows) 28.4 us with 8, 31.8 with 4; 32 tokens of 32 requests
// 20.6 and 22.2, of 64 29.9 and 28.6, of 16 19.3 and 17.4, of 8 18.9 and 17.1; 8 tokens (56 rows) of 64
// requests 19.2 and 17.8; one token of 64 17.3 and 15.3.
int waves_of(int rows, int64_t selections, int64_t groups) {
    return rows > 64 && selections * ((groups + 127) / 128) >= 2LL * ma_num_cus() ? 8 : 4;
}
template <int D, int DT>
void launch_score(const SelectArgs &a, int waves, unsigned grid, hipStream_t st) {
    if (waves == 4) select_score_kernel<D, DT, 4><<<grid, 256, 0, st>>>(a);
    else select_score_kernel<D, DT, 8><<<grid, 512, 0, st>>>(a);
}
template <int THREADS, int PER>
int launch_top(const SelectArgs &a, unsigned rows, hipStream_t st) {
    constexpr int LDS = THREADS * PER * 4;
    if (LDS > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void *)select_top_kernel<THREADS, PER>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (e != hipSuccess) {
            ma_set_error("ma_select_blocks: %d bytes of LDS refused: %s", LDS, hipGetErrorString(e));
            return MA_EHIP;
        }
    }
    select_top_kernel<THREADS, PER><<<rows, THREADS, LDS, st>>>(a);
    return MA_OK;
}

}  // namespace

extern "C" int64_t ma_select_workspace_bytes(int B, int H, int runs, int64_t tokens) {
    if (B <= 0 || H <= 0 || runs <= 0 || tokens <= 0 || tokens > INT32_MAX) return -1;
    const int64_t rows = (int64_t)B * H * runs, groups = (tokens + PG_GROUP - 1) / PG_GROUP;
    return rows > INT32_MAX ? -1 : align256(rows * groups * 4);
}

extern "C" int ma_select_blocks(ma_tensor4 q, int B, int Hq, int T, int D, const ma_pages *p, int H,
                                const int32_t *new_lens, int query_block, int block_tokens, int count, int keep_first,
                                int keep_last, int32_t *blocks, float *scores, void *workspace, int64_t workspace_bytes,
                                void *stream) {
    const char *who = "ma_select_blocks";
    if (int rc = pg_check(p, B, H, D, who)) return rc;
    if (Hq <= 0 || Hq % H || T <= 0 || query_block < 0 || block_tokens <= 0 || block_tokens % PG_GROUP || count <= 0 ||
        keep_first < 0 || keep_last < 0 || (int64_t)keep_first + keep_last > count || !q.ptr || !blocks) {
        ma_set_error("%s: bad arguments (Hq=%d H=%d T=%d query_block=%d block_tokens=%d, a multiple of 32, count=%d "
                     "keep_first=%d keep_last=%d, together at most count)", who, Hq, H, T, query_block, block_tokens, count,
                     keep_first, keep_last);
        return MA_EINVAL;
    }
    if (q.dtype != p->dtype) {
        ma_set_error("%s: queries and tails must share one dtype", who);
        return MA_EINVAL;
    }
    const int run = query_block == 0 || query_block > T ? T : query_block;
    if ((int64_t)T + run > INT32_MAX) {         // (the position behind the last run has 32 bits)
        ma_set_error("%s: %d positions in runs of %d are not built (2^31 together)", who, T, run);
        return MA_EUNSUPPORTED;
    }
    const int runs = (T + run - 1) / run;
    const int64_t tokens = (int64_t)p->width * p->page_tokens, need = ma_select_workspace_bytes(B, H, runs, tokens);
    if (need < 0 || (int64_t)(Hq / H) * run > INT32_MAX / 16) {
        ma_set_error("%s: %d rows of %d heads, or 2^31 selections, are not built", who, run, Hq / H);
        return MA_EUNSUPPORTED;
    }
    // blocks of one group: the groups' scores are the blocks', where they are asked for
    const bool same = scores && block_tokens == PG_GROUP;
    if (!same && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)) {
        ma_set_error("%s: workspace of %lld bytes (256-byte aligned) needed, got %lld", who, (long long)need,
                     (long long)workspace_bytes);
        return MA_EWORKSPACE;
    }
    SelectArgs a{};
    a.q = q;
    a.p = pages_dev(p);
    a.new_lens = new_lens;
    a.group = same ? scores : (float *)workspace;
    a.scores = scores;
    a.blocks = blocks;
    a.ngcap = tokens / PG_GROUP;
    a.m = block_tokens / PG_GROUP;
    a.nbcap = (a.ngcap + a.m - 1) / a.m;
    a.B = B;
    a.H = H;
    a.G = Hq / H;
    a.T = T;
    a.run = run;
    a.runs = runs;
    a.count = count;
    a.first = keep_first;
    a.last = keep_last;
    const int64_t rows = (int64_t)B * H * runs;
    const int waves = waves_of(a.G * run, rows, a.ngcap), span = 16 * waves;
    const int64_t units = rows * ((a.ngcap + span - 1) / span);
    // (threads of a launch's one dimension: below 2^32)
    if (units > INT32_MAX / 2 || rows > UINT32_MAX / 1024) {
        ma_set_error("%s: %lld selections over %lld tokens are not built (2^22, and 2^30 times %d groups)", who,
                     (long long)rows, (long long)tokens, span);
        return MA_EUNSUPPORTED;
    }
    a.units = (int)units;
    const unsigned grid = (unsigned)min(units, (int64_t)ma_num_cus() * 4);
    hipStream_t st = (hipStream_t)stream;
    if (D == 128) p->dtype == MA_BF16 ? launch_score<128, MA_BF16>(a, waves, grid, st) : launch_score<128, MA_F16>(a, waves, grid, st);
    else p->dtype == MA_BF16 ? launch_score<64, MA_BF16>(a, waves, grid, st) : launch_score<64, MA_F16>(a, waves, grid, st);
    if (int rc = ma_check_launch(who)) return rc;
    int rc;
    if (a.nbcap <= 1024) rc = launch_top<256, 4>(a, (unsigned)rows, st);
    else if (a.nbcap <= 4096) rc = launch_top<1024, 4>(a, (unsigned)rows, st);
    else if (a.nbcap <= 32768) rc = launch_top<1024, 32>(a, (unsigned)rows, st);
    else rc = launch_top<1024, 0>(a, (unsigned)rows, st);
    return rc ? rc : ma_check_launch(who);
}
