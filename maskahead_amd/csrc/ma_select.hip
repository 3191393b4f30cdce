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
// Codes of at most 2^14 are two digits of 7 bits (sign with both), which f16 holds; each of the
// four products of digits sums to at most 2^22 over 2 D channels, which f32 accumulates without
// rounding whatever the order (two share an accumulator).  The score, a whole number below 2^37
// times 2^(e + f - 26), is rounded once, to f32.
#include "ma_pages.h"

using namespace ma;

namespace {

constexpr int SEL_WAVES = 4, SEL_TILES = 4;             // 16 groups a wave; row tiles in LDS at once
constexpr int SEL_SPAN = 16 * SEL_WAVES;                // groups of a workgroup
constexpr int ROW_ABSENT = INT32_MIN, ROW_ODD = INT32_MAX;
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
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int new_of(const SelectArgs &a, int b) {
    return a.new_lens ? min(max(a.new_lens[b], 0), a.T) : a.T;
}

typedef __attribute__((ext_vector_type(2))) __fp16 fp16x2_t;
__device__ __forceinline__ f16x2_t pk(float a, float b) {      // (whole numbers below 2^11: exact)
    return __builtin_bit_cast(f16x2_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}
// 8 values times scale, rounded to whole numbers, as two digits: code = 128 hi + lo, both of its sign
__device__ __forceinline__ void digits8(const float (&x)[8], float scale, f16x8_t &hi, f16x8_t &lo) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float h[2], l[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float c = rintf(x[i + k] * scale);
            h[k] = truncf(c * 0.0078125f);
            l[k] = __builtin_fmaf(h[k], -128.0f, c);
        }
        const f16x2_t hv = pk(h[0], h[1]), lv = pk(l[0], l[1]);
        hi[i] = hv[0], hi[i + 1] = hv[1];
        lo[i] = lv[0], lo[i + 1] = lv[1];
    }
}
__device__ __forceinline__ f16x8_t relu(f16x8_t x) { return __builtin_elementwise_max(x, (f16x8_t)(_Float16)0.0f); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// maximum over the four lanes of a row (lane ^ 16, lane ^ 32)
__device__ __forceinline__ float max_rows(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return ma_max_xor32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
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

// ------------------------------------------------------------------ scores of groups
// A workgroup: 64 groups of one (request, head) and the rows of one run; a wave holds the digits of
// its 16 groups' parameters and passes all rows by them, whose digits lie in LDS, 64 rows at a time.
template <int D, int DT>
__global__ __launch_bounds__(64 * SEL_WAVES, 2) void select_score_kernel(SelectArgs a) {
    constexpr int KB = D / 32;
    __shared__ f16x8_t dig[SEL_TILES][2][KB][64];
    __shared__ int expo[SEL_TILES][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), n16 = lane & 15, hh = lane >> 4;
    const int R = a.G * a.run, tiles = (R + 15) / 16, per = a.p.page_tokens / PG_GROUP;
    for (int64_t u = blockIdx.x;; u += gridDim.x) {
        // the unit's request: units of those before it, 64 requests at a time
        int64_t pre = 0;
        int b = -1, len = 0, n = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            int own_len = 0, own_n = 0;
            int64_t units = 0;
            if (b0 + lane < a.B) {
                own_len = pg_length(a.p, b0 + lane);
                own_n = new_of(a, b0 + lane);
                units = (int64_t)((own_len / PG_GROUP + SEL_SPAN - 1) / SEL_SPAN) * a.H * ((own_n + a.run - 1) / a.run);
            }
            const int64_t inc = pre + pg_wave_scan(units, lane);
            const uint64_t here = __ballot(u >= inc - units && u < inc);
            if (here) {
                const int l = __ffsll((unsigned long long)here) - 1;
                b = b0 + l;
                len = __builtin_amdgcn_readlane(own_len, l);
                n = __builtin_amdgcn_readlane(own_n, l);
                const int64_t before = inc - units;
                pre = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(before >> 32), l) << 32 |
                                (uint32_t)__builtin_amdgcn_readlane((int)before, l));
                break;
            }
            pre = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(inc >> 32), 63) << 32 |
                            (uint32_t)__builtin_amdgcn_readlane((int)inc, 63));
        }
        if (b < 0) return;       // behind the last unit (all waves alike)
        const int ng = len / PG_GROUP, runs = (n + a.run - 1) / a.run;
        const int64_t rel = u - pre;
        const int run = (int)(rel % runs), h = (int)(rel / runs % a.H), span = (int)(rel / runs / a.H);
        // the wave's groups
        const int g = span * SEL_SPAN + 16 * wave + n16, gc = min(g, ng - 1), pg = gc / per;
        const uint8_t *rec = pg_record(a.p, a.p.table[(int64_t)b * a.p.s_table + pg], gc - pg * per, h, 40 * D);
        const bool there = rec != nullptr;
        if (!there) rec = a.p.pool;
        uint4 sw[KB], zw[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            sw[kb] = *(const uint4 *)(rec + 32 * D + 2 * (32 * kb + 8 * hh));
            zw[kb] = *(const uint4 *)(rec + 34 * D + 2 * (32 * kb + 8 * hh));
        }
        float top = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            float s[8], z[8];
            unpack8<MA_F16>(sw[kb], s);
            unpack8<MA_F16>(zw[kb], z);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // (a NaN becomes infinite, so that the maximum shows it)
                const float x = fmaxf(fabsf(15.0f * s[i]), fabsf(z[i]));
                top = s[i] != s[i] || z[i] != z[i] ? INFINITY : fmaxf(top, x);
            }
        }
        top = max_rows(top);
        const bool odd = top == INFINITY;
        const int f = max((int)(__float_as_uint(top) >> 23) - 127, -24);
        const float scale = odd ? 0.f : pow2(13 - f);
        f16x8_t zh[KB], zl[KB], sh[KB], sl[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            float x[8];
            unpack8<MA_F16>(zw[kb], x);
            digits8(x, scale, zh[kb], zl[kb]);
            unpack8<MA_F16>(sw[kb], x);
            digits8(x, 15.0f * scale, sh[kb], sl[kb]);
        }
        bool live = there;
        if (a.p.mask) {
            const bool any = pg_mask_bits(a.p, b, h, gc * PG_GROUP + 8 * hh) != 0;
            live = live && max_rows(any ? 1.f : 0.f) != 0.f;
        }
        float best = -INFINITY;
        for (int t0 = 0; t0 < tiles; t0 += SEL_TILES) {
            __syncthreads();          // the rows before are read
            for (int t = wave; t < min(SEL_TILES, tiles - t0); t += SEL_WAVES) {
                const int row = 16 * (t0 + t) + n16, rc = min(row, R - 1), qh = rc / a.run, pos = run * a.run + rc - qh * a.run;
                const uint16_t *src = (const uint16_t *)a.q.ptr + (int64_t)b * a.q.s[0] + (int64_t)(h * a.G + qh) * a.q.s[1] +
                                      (int64_t)min(pos, a.T - 1) * a.q.s[2] + 8 * hh;
                uint4 w[KB];
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) w[kb] = pg_load16(src + 32 * kb);
                float mx = 0.f;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    float x[8];
                    unpack8<DT>(w[kb], x);
#pragma unroll
                    for (int i = 0; i < 8; ++i) mx = x[i] != x[i] ? INFINITY : fmaxf(mx, fabsf(x[i]));
                }
                mx = max_rows(mx);
                const bool odd_row = mx == INFINITY;
                const int e = max((int)(__float_as_uint(mx) >> 23) - 127, -100);
                const float qs = odd_row ? 0.f : pow2(13 - e);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    float x[8];
                    f16x8_t hi, lo;
                    unpack8<DT>(w[kb], x);
                    digits8(x, qs, hi, lo);
                    dig[t][0][kb][lane] = hi;
                    dig[t][1][kb][lane] = lo;
                }
                if (hh == 0) expo[t][n16] = row >= R || pos >= n ? ROW_ABSENT : odd_row ? ROW_ODD : e;
            }
            __syncthreads();
            for (int t = 0; t < min(SEL_TILES, tiles - t0); ++t) {
                f32x4_t c2{}, c1{}, c0{};
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    const f16x8_t qh = dig[t][0][kb][lane], ql = dig[t][1][kb][lane], rh = relu(qh), rl = relu(ql);
                    c2 = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh, zh[kb], c2, 0, 0, 0);
                    c1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh, zl[kb], c1, 0, 0, 0);
                    c1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(ql, zh[kb], c1, 0, 0, 0);
                    c0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(ql, zl[kb], c0, 0, 0, 0);
                    c2 = __builtin_amdgcn_mfma_f32_16x16x32_f16(rh, sh[kb], c2, 0, 0, 0);
                    c1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(rh, sl[kb], c1, 0, 0, 0);
                    c1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(rl, sh[kb], c1, 0, 0, 0);
                    c0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(rl, sl[kb], c0, 0, 0, 0);
                }
                // lane (n, h): rows 4 h + r by group n
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int e = expo[t][4 * hh + r];
                    const double s = (double)c2[r] * 16384.0 + ((double)c1[r] * 128.0 + (double)c0[r]);
                    float v = fmaxf((float)__builtin_ldexp(s, (e == ROW_ODD || e == ROW_ABSENT ? 0 : e) + f - 26), LEAST);
                    if (odd || e == ROW_ODD) v = INFINITY;
                    if (e != ROW_ABSENT) best = fmaxf(best, v);
                }
            }
        }
        best = max_rows(best);
        if (hh == 0 && g < ng)
            a.group[(((int64_t)b * a.H + h) * a.runs + run) * a.ngcap + g] = live ? best : -INFINITY;
    }
}

// ------------------------------------------------------------------ selection
// One workgroup a (request, head, run): the count largest block scores, ties to the lowest index, in
// ascending order.  A key is the score's place in the order of floats, 0 for no block; blocks that are
// always taken stand outside the search.  The search counts keys in 1 024 equal ranges between the
// smallest and the largest, then within the range that the last one lies in, and so on: three
// turns at most, and scores alike do not meet in one counter as they would by their leading bits.
constexpr int SEL_BINS = 1024;
constexpr uint32_t KEY_TAKEN = 0xffffffffu;

template <int THREADS>
struct TopShared {
    uint32_t bin[SEL_BINS], wsum[2][THREADS / 64], red[2][THREADS / 64];
    uint32_t at, above, in;
};

// sum of the threads before this one, and of all; both of two counts
template <int THREADS>
__device__ __forceinline__ void block_scan(TopShared<THREADS> &sh, uint32_t x, uint32_t y, uint32_t &bx, uint32_t &by,
                                           uint32_t &tx, uint32_t &ty) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t ix = ma_wave_prefix_u32(x), iy = ma_wave_prefix_u32(y);
    __syncthreads();
    if (lane == 63) sh.wsum[0][wave] = ix, sh.wsum[1][wave] = iy;
    __syncthreads();
    bx = ix - x, by = iy - y, tx = ty = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) bx += sh.wsum[0][w], by += sh.wsum[1][w];
        tx += sh.wsum[0][w];
        ty += sh.wsum[1][w];
    }
}

// PER > 0: a thread keeps its keys, at most PER; 0: they are read again in every turn
template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void select_top_kernel(SelectArgs a) {
    __shared__ TopShared<THREADS> sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const int run = (int)(row % a.runs), b = (int)(row / a.runs / a.H);
    const int n = new_of(a, b), ng = run * a.run < n ? pg_length(a.p, b) / PG_GROUP : 0, nb = (ng + a.m - 1) / a.m;
    const float *group = a.group + row * a.ngcap;
    // this thread's blocks [i0, i1)
    const int each = (nb + THREADS - 1) / THREADS, i0 = min(tid * each, nb), i1 = min(i0 + each, nb);
    auto score_of = [&](int i) {
        float s = -INFINITY;
        for (int y = i * a.m; y < min((i + 1) * a.m, ng); ++y) s = fmaxf(s, group[y]);
        return s;
    };
    auto key_of = [&](int i, float s) -> uint32_t {
        if (s == -INFINITY) return 0;
        return i < a.first || i >= nb - a.last ? KEY_TAKEN : ma_order_key(s);
    };
    uint32_t key[PER ? PER : 1];
    uint32_t lo = 0xffffffffu, hi = 0, some = 0, taken = 0;
    auto note = [&](int i, uint32_t k) {
        if (k == 0) return;
        ++some;
        if (k == KEY_TAKEN) ++taken;
        else lo = min(lo, k), hi = max(hi, k);
    };
    if constexpr (PER > 0) {
        float s[PER];
#pragma unroll
        for (int y = 0; y < PER; ++y) s[y] = i0 + y < i1 ? score_of(i0 + y) : -INFINITY;
#pragma unroll
        for (int y = 0; y < PER; ++y) {
            key[y] = i0 + y < i1 ? key_of(i0 + y, s[y]) : 0;
            note(i0 + y, key[y]);
            if (a.scores && i0 + y < i1) a.scores[row * a.nbcap + i0 + y] = s[y];
        }
    } else {
        for (int i = i0; i < i1; ++i) {
            const float s = score_of(i);
            note(i, key_of(i, s));
            if (a.scores) a.scores[row * a.nbcap + i] = s;
        }
    }
    if (a.scores)
        for (int64_t i = nb + tid; i < a.nbcap; i += THREADS) a.scores[row * a.nbcap + i] = -INFINITY;
    auto each_key = [&](auto f) {
        if constexpr (PER > 0) {
#pragma unroll
            for (int y = 0; y < PER; ++y) f(i0 + y, key[y]);
        } else {
            for (int i = i0; i < i1; ++i) f(i, key_of(i, score_of(i)));
        }
    };
    uint32_t before, before2, all, forced;
    block_scan<THREADS>(sh, some, taken, before, before2, all, forced);
    const uint32_t wlo = ~ma_wave_max_u32(~lo), whi = ma_wave_max_u32(hi);
    if (lane == 0) sh.red[0][wave] = wlo, sh.red[1][wave] = whi;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) lo = min(lo, sh.red[0][w]), hi = max(hi, sh.red[1][w]);
    // what is taken: keys above cut, and the first `ties` of those equal to it
    uint32_t cut = 0, ties = 0;
    const uint32_t want = min((uint32_t)a.count, all);
    if (want < all) {
        uint32_t need = want - min(forced, want);
        if (need == 0) cut = KEY_TAKEN - 1;
        while (need) {
            const uint32_t range = hi - lo;
            const int bits = range ? 32 - __builtin_clz(range) : 0, s = max(bits - 10, 0);
            for (int i = tid; i < SEL_BINS; i += THREADS) sh.bin[i] = 0;
            __syncthreads();
            each_key([&](int, uint32_t k) {
                if (k >= lo && k <= hi && k != 0) atomicAdd(&sh.bin[(k - lo) >> s], 1u);
            });
            __syncthreads();
            // bins from the top, BPT a thread: the one in which the need-th lies
            constexpr int BPT = SEL_BINS / THREADS;
            uint32_t c[BPT], sum = 0;
#pragma unroll
            for (int y = 0; y < BPT; ++y) {
                c[y] = sh.bin[SEL_BINS - 1 - (tid * BPT + y)];
                sum += c[y];
            }
            uint32_t above, unused, total, unused2;
            block_scan<THREADS>(sh, sum, 0, above, unused, total, unused2);
#pragma unroll
            for (int y = 0; y < BPT; ++y) {
                if (above < need && need <= above + c[y]) {
                    sh.at = SEL_BINS - 1 - (tid * BPT + y);
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
            __syncthreads();             // at, above and in are read
        }
    }
    uint32_t over = 0, equal = 0;
    each_key([&](int, uint32_t k) {
        if (k > cut) ++over;
        else if (k == cut && k != 0) ++equal;
    });
    uint32_t ob, eb, ot, et;
    block_scan<THREADS>(sh, over, equal, ob, eb, ot, et);
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
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

template <int D, int DT>
void launch_score(const SelectArgs &a, unsigned grid, hipStream_t st) {
    select_score_kernel<D, DT><<<grid, 64 * SEL_WAVES, 0, st>>>(a);
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
    const int run = query_block == 0 || query_block > T ? T : query_block, runs = (T + run - 1) / run;
    const int64_t tokens = (int64_t)p->width * p->page_tokens, need = ma_select_workspace_bytes(B, H, runs, tokens);
    if (need < 0 || (int64_t)(Hq / H) * run > INT32_MAX / 16) {
        ma_set_error("%s: %d rows of %d heads, or 2^31 selections, are not built", who, run, Hq / H);
        return MA_EUNSUPPORTED;
    }
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256) {
        ma_set_error("%s: workspace of %lld bytes (256-byte aligned) needed, got %lld", who, (long long)need,
                     (long long)workspace_bytes);
        return MA_EWORKSPACE;
    }
    SelectArgs a{};
    a.q = q;
    a.p = pages_dev(p);
    a.new_lens = new_lens;
    a.group = (float *)workspace;
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
    const int64_t rows = (int64_t)B * H * runs, units = rows * ((a.ngcap + SEL_SPAN - 1) / SEL_SPAN);
    const unsigned grid = (unsigned)min(units, (int64_t)ma_num_cus() * 4);
    hipStream_t st = (hipStream_t)stream;
    if (D == 128) p->dtype == MA_BF16 ? launch_score<128, MA_BF16>(a, grid, st) : launch_score<128, MA_F16>(a, grid, st);
    else p->dtype == MA_BF16 ? launch_score<64, MA_BF16>(a, grid, st) : launch_score<64, MA_F16>(a, grid, st);
    if (int rc = ma_check_launch(who)) return rc;
    if (a.nbcap <= 256 * 4) select_top_kernel<256, 4><<<(unsigned)rows, 256, 0, st>>>(a);
    else if (a.nbcap <= 256 * 16) select_top_kernel<256, 16><<<(unsigned)rows, 256, 0, st>>>(a);
    else select_top_kernel<1024, 0><<<(unsigned)rows, 1024, 0, st>>>(a);
    return ma_check_launch(who);
}
