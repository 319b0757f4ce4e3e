// The loss that query adapters are trained with, and the clipping of their gradients (C ABI: include/hvs.h).
#include <algorithm>
#include <climits>
#include <new>
#include <utility>
#include <vector>

#include "hvs_learn.h"

// ---------------------------------------------------------------------------------------------------------------
// preference loss
// ---------------------------------------------------------------------------------------------------------------
// With c^ = c / |c| etc., e_p = c^ - r^ and s_p = y^ . e_p (the difference of the cosines):  d s / d y = (e - s y^) / |y|, so the
// gradient of a query is
//     (sum_p g_p e_p  -  (sum_p g_p s_p) y^) / |y|,   g_p = w_p beta (eps sigma(h_p) - (1 - eps) sigma(-h_p)):
// one vector and one number are kept over the pairs of a query, and every row is read once.  The margin, the small difference
// of two such differences, is summed as (y^ - y0^) . e_p: both differences are taken element by element, before the sum.
struct PreferenceParams {
    const void *y, *ref;
    int64_t ld_y, ld_ref;
    const int64_t *offsets, *chosen, *rejected;
    const float *weights;
    float *loss, *margin;
    void *grad;
    int64_t ld_grad;
    int64_t n_pairs, n_queries, first_query;  // first_query: of this launch
    const void *rows;
    int64_t ld_rows, n_rows;
    int dim;
    float beta, smoothing, default_weight;
    float *part_vec;  // [n_queries][shares][dim] sums of queries that several blocks work on
    float *part_num;  // [n_queries][shares]
    float *part_inv;  // [n_queries] 1 / |y|
    int per_block;    // pairs a block takes before a second one joins in
};

// eight consecutive elements of a row as they lie in memory, zeros past its end, and as fp32
template <int DT> struct Raw8 {
    f32x4 c[8 / Elem<DT>::EPC];
};
template <int DT, bool ALIGNED> __device__ __forceinline__ void load8(const void *base, int64_t row, int64_t ld, int k, int dim, Raw8<DT> &out) {
    typedef typename Elem<DT>::type E;
    constexpr int EPC = Elem<DT>::EPC;
    const E *p = reinterpret_cast<const E *>(base) + row * ld;
#pragma unroll
    for (int i = 0; i < 8 / EPC; i++) out.c[i] = load_chunk<DT, ALIGNED>(p, k + i * EPC, dim);
}
template <int DT> __device__ __forceinline__ void raw8_to_float(const Raw8<DT> &r, float *out) {
    constexpr int EPC = Elem<DT>::EPC;
#pragma unroll
    for (int i = 0; i < 8 / EPC; i++) chunk_to_float<DT>(r.c[i], out + i * EPC);
}

// 16-bit rows are converted again for every use rather than kept twice as wide across the sums
template <int DT, int CH> __device__ __forceinline__ void keep_raw(Raw8<DT> (&a)[CH], Raw8<DT> (&b)[CH]) {
    if (DT == HVS_F32) return;
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
        for (int k = 0; k < 8 / Elem<DT>::EPC; k++) asm volatile("" : "+v"(a[c].c[k]), "+v"(b[c].c[k]));
}

__device__ __forceinline__ float softplus(float z) { return fmaxf(z, 0.0f) + log1pf(expf(-fabsf(z))); }
__device__ __forceinline__ float inverse_norm(float sum_of_squares) { return sum_of_squares == 0.0f ? 0.0f : 1.0f / sqrtf(sum_of_squares); }

// Rows of fp32 and bf16 may be longer than 2^64 or shorter than 2^-50: their squares leave fp32, or its normal numbers.  Only the
// direction of a row counts, so the elements of such a row are multiplied by the power of two that brings the largest to
// [0.5, 1): exact, but for those that are then below 2^-126 and do not matter beside it.
__device__ __forceinline__ bool plain_square_sum(float v) { return v >= 0x1p-100f && v < __builtin_inff(); }
// use(element) -> what becomes of it, for the elements of a row's part, four bytes at a time: what this seldom path holds in
// registers the usual one pays for
template <int DT, int CH, class USE> __device__ __forceinline__ void for_each_element(Raw8<DT> (&r)[CH], float &state, USE use) {
    static_assert(DT == HVS_F32 || DT == HVS_BF16, "no such rows of fp16");
    constexpr int EPC = Elem<DT>::EPC;
#pragma unroll
    for (int i = 0; i < CH * 32 / EPC; i++) {
        f32x4 &four = r[i / (32 / EPC)].c[i / 4 % (8 / EPC)];
        float word = four[i % 4];
        asm volatile("" : "+v"(word), "+v"(state));  // one word after the other
        if (DT == HVS_F32) four[i % 4] = use(word);
        else {
            const uint32_t low = __float_as_uint(use(__uint_as_float(__float_as_uint(word) << 16)));
            const uint32_t high = __float_as_uint(use(__uint_as_float(__float_as_uint(word) & 0xFFFF0000u)));
            four[i % 4] = __uint_as_float((high & 0xFFFF0000u) | (low >> 16));
        }
    }
}
template <int DT, int CH> __device__ __forceinline__ float row_largest(Raw8<DT> (&r)[CH]) {
    float largest = 0.0f;
    for_each_element<DT, CH>(r, largest, [&](float v) {
        largest = fmaxf(largest, fabsf(v));
        return v;
    });
    return largest;
}
// scales the row (not if there is nothing but zeros, or an infinite element) and returns its sum of squares
template <int DT, int CH> __device__ __forceinline__ float row_scale(Raw8<DT> (&r)[CH], float largest) {
    const int exponent = __builtin_amdgcn_readfirstlane(-__builtin_amdgcn_frexp_expf(largest));  // the same in every lane
    float sum = 0.0f;
    for_each_element<DT, CH>(r, sum, [&](float v) {
        v = ldexpf(v, exponent);
        sum = fmaf(v, v, sum);
        return v;
    });
    return sum;
}

// how the pairs [b0, b1) of a query are shared out; the same on every side that asks
__device__ __forceinline__ void pair_share(const PreferenceParams &p, int64_t q, int shares, int64_t &b0, int64_t &b1, int64_t &per, int &used) {
    b0 = p.offsets[q];
    b1 = p.offsets[q + 1];
    b0 = b0 < 0 ? 0 : (b0 > p.n_pairs ? p.n_pairs : b0);
    b1 = b1 < b0 ? b0 : (b1 > p.n_pairs ? p.n_pairs : b1);
    const int64_t len = b1 - b0;
    per = (len + shares - 1) / shares;
    per = per < p.per_block ? p.per_block : per;
    used = len > 0 ? (int)((len + per - 1) / per) : 1;
}

// A team of TW waves holds the rows of a pair, CH x 8 elements a lane, as they lie in memory, and the gradient sum in fp32;
// the rows of the team's next pair are on their way meanwhile.  Teams of one wave read the query and the reference query
// from LDS (registers then allow four waves per SIMD), larger teams hold their part.  The block's teams take the pairs of
// its share in turn and are added up in team order.  Bound by reading the rows.
// (513 - 1024 columns: registers for five waves a SIMD; with four, 4096 queries x 8 pairs of 1024 bf16 columns take 49.7 instead of 45.6 us)
template <int QDT, int RDT, int CH, int TW, int WAVES, bool ALIGNED>
__global__ __launch_bounds__(64 * WAVES, TW == 1 && CH == 2 && WAVES == 4 ? 5 : 1) void preference_kernel(PreferenceParams p) {
    typedef typename Elem<QDT>::type Q;
    constexpr int TEAMS = WAVES / TW, SPAN = CH * TW * 512;  // SPAN: dim rounded up to what a team covers
    extern __shared__ __attribute__((aligned(16))) float smem[];  // TW 1: [2][SPAN] the queries, then [TEAMS][SPAN]; else [dim]
    __shared__ float sums[WAVES][2];
    __shared__ double sums_query[WAVES][2];
    static_assert(TW == 1 ? CH <= WAVES : TW == WAVES, "a piece of the query for every wave, or one team");
    __shared__ float num[TEAMS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int team = wave / TW, tl = (wave % TW) * 64 + lane;
    const int64_t q = p.first_query + blockIdx.x;
    const int z = blockIdx.y, shares = gridDim.y;
    int64_t b0, b1, per;
    int used;
    pair_share(p, q, shares, b0, b1, per, used);
    if (z >= used) return;
    const int64_t lo = b0 + z * per, hi = lo + per < b1 ? lo + per : b1;

    // two sums over a team's elements, the same in every lane
    auto team_sum = [&](float &a, float &b) {
        learn_wave_sum2(a, b);
        if (TW > 1) {
            __syncthreads();
            if (lane == 0) sums[wave][0] = a, sums[wave][1] = b;
            __syncthreads();
            a = b = 0.0f;
#pragma unroll
            for (int w = 0; w < TW; w++) a += sums[team * TW + w][0], b += sums[team * TW + w][1];
        }
    };
    auto team_max = [&](float &a, float &b) {
        learn_wave_max2(a, b);
        if (TW > 1) {
            __syncthreads();
            if (lane == 0) sums[wave][0] = a, sums[wave][1] = b;
            __syncthreads();
            a = b = 0.0f;
#pragma unroll
            for (int w = 0; w < TW; w++) a = fmaxf(a, sums[team * TW + w][0]), b = fmaxf(b, sums[team * TW + w][1]);
        }
    };
    auto left_out = [&](int64_t a, int64_t b) { return a < 0 || b < 0 || a >= p.n_rows || b >= p.n_rows; };

    // the first pair's positions and rows
    int64_t i = lo + team, a = -1, b = -1, a_next = -1, b_next = -1;
    if (i < hi) a = p.chosen[i], b = p.rejected[i];
    if (i + TEAMS < hi) a_next = p.chosen[i + TEAMS], b_next = p.rejected[i + TEAMS];
    Raw8<RDT> ra[CH], rb[CH];
    auto fetch = [&](int64_t ka, int64_t kb) {
        if (left_out(ka, kb)) return;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int k = (c * TW * 64 + tl) * 8;
            load8<RDT, ALIGNED>(p.rows, ka, p.ld_rows, k, p.dim, ra[c]);
            load8<RDT, ALIGNED>(p.rows, kb, p.ld_rows, k, p.dim, rb[c]);
        }
    };
    fetch(a, b);

    // y^ and y^ - y0^ (without a reference: y^), which the sums over a pair are taken with.  After a few steps of training y is close
    // to y0: an error of 2^-24 in either norm, or in the smaller product, would be many steps of the difference.  So the norms are
    // held in double precision, their inverses as two floats, and the product y0 / |y0| keeps what its rounding cuts off
    // (difference 1e-2 of the queries, 16 pairs: margins off by 1e-7 instead of 5e-6 of their size).
    float y_own[TW > 1 ? CH * 8 : 1], d_own[TW > 1 ? CH * 8 : 1], g[CH * 8];
    float inv_y;
#pragma unroll
    for (int k = 0; k < CH * 8; k++) g[k] = 0.0f;
    {
        // teams of one wave share the work: wave c takes piece c (there are at least as many waves)
        constexpr int PIECES = TW > 1 ? CH : 1;
        const bool has = TW > 1 || team < CH;
        Raw8<QDT> ry[PIECES], rf[PIECES];
        double yy = 0.0, ff = 0.0;
#pragma unroll
        for (int c = 0; c < PIECES; c++) {
            const int k = ((TW > 1 ? c : team) * TW * 64 + tl) * 8;
            float v[8];
            if (!has) continue;
            load8<QDT, ALIGNED>(p.y, q, p.ld_y, k, p.dim, ry[c]);
            if (p.ref) load8<QDT, ALIGNED>(p.ref, q, p.ld_ref, k, p.dim, rf[c]);
            raw8_to_float<QDT>(ry[c], v);
#pragma unroll
            for (int e = 0; e < 8; e++) yy = fma((double)v[e], (double)v[e], yy);
            if (!p.ref) continue;
            raw8_to_float<QDT>(rf[c], v);
#pragma unroll
            for (int e = 0; e < 8; e++) ff = fma((double)v[e], (double)v[e], ff);
        }
        if (has) {
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) {
                yy += __shfl_xor(yy, o);
                ff += __shfl_xor(ff, o);
            }
            if (lane == 0) sums_query[wave][0] = yy, sums_query[wave][1] = ff;
        }
        __syncthreads();
        yy = ff = 0.0;
#pragma unroll
        for (int w = 0; w < (TW > 1 ? WAVES : CH); w++) yy += sums_query[w][0], ff += sums_query[w][1];
        yy = yy < 1e-76 ? 0.0 : 1.0 / sqrt(yy);  // below 1e-38 the inverse is no fp32 number: such a norm counts as 0
        ff = ff < 1e-76 ? 0.0 : 1.0 / sqrt(ff);
        inv_y = (float)yy;
        const float inv_f = (float)ff, rest_y = (float)(yy - (double)inv_y), rest_f = (float)(ff - (double)inv_f);
#pragma unroll
        for (int c = 0; c < PIECES; c++) {
            float yv[8], dv[8];
            if (!has) continue;
            raw8_to_float<QDT>(ry[c], yv);
            if (p.ref) raw8_to_float<QDT>(rf[c], dv);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (p.ref) {
                    const float f = dv[e] * inv_f, cut = fmaf(dv[e], inv_f, -f);
                    dv[e] = fmaf(yv[e], inv_y, -f) + (fmaf(yv[e], rest_y, -cut) - dv[e] * rest_f);
                } else dv[e] = yv[e] * inv_y;
                yv[e] *= inv_y;
                if (TW > 1) y_own[c * 8 + e] = yv[e], d_own[c * 8 + e] = dv[e];
            }
            if (TW == 1) {
                const int k = (team * 64 + tl) * 8;
                f32x4 *yl = reinterpret_cast<f32x4 *>(smem + k), *dl = reinterpret_cast<f32x4 *>(smem + SPAN + k);
                yl[0] = f32x4{yv[0], yv[1], yv[2], yv[3]}, yl[1] = f32x4{yv[4], yv[5], yv[6], yv[7]};
                dl[0] = f32x4{dv[0], dv[1], dv[2], dv[3]}, dl[1] = f32x4{dv[4], dv[5], dv[6], dv[7]};
            }
        }
    }
    if (TW == 1) __syncthreads();
    auto query8 = [&](int which, int c, float *out) {  // this lane's piece c of y^ (0) or of the difference (1)
        if (TW > 1) {
#pragma unroll
            for (int e = 0; e < 8; e++) out[e] = which ? d_own[c * 8 + e] : y_own[c * 8 + e];
        } else {
            const f32x4 *l = reinterpret_cast<const f32x4 *>(smem + which * SPAN + (c * 64 + tl) * 8);
            const f32x4 v0 = l[0], v1 = l[1];
#pragma unroll
            for (int e = 0; e < 4; e++) out[e] = v0[e], out[4 + e] = v1[e];
        }
    };

    float total = 0.0f;  // sum of g_p s_p
    for (; i < hi; i += TEAMS) {
        if (left_out(a, b)) {
            const float v = a < 0 || b < 0 ? 0.0f : __builtin_nanf("");
            if (tl == 0) p.loss[i] = p.margin[i] = v;
            total += v;
        } else {
            float ia = 0.0f, ib = 0.0f, cos = 0.0f, m = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; c++) {
                float av[8], bv[8];
                raw8_to_float<RDT>(ra[c], av);
                raw8_to_float<RDT>(rb[c], bv);
#pragma unroll
                for (int e = 0; e < 8; e++) ia = fmaf(av[e], av[e], ia), ib = fmaf(bv[e], bv[e], ib);
            }
            team_sum(ia, ib);
            if constexpr (RDT != HVS_F16) {  // (squares of fp16 stay well inside)
                if (!(plain_square_sum(ia) && plain_square_sum(ib))) {
                    float ma = row_largest<RDT, CH>(ra), mb = row_largest<RDT, CH>(rb);
                    team_max(ma, mb);
                    ia = row_scale<RDT, CH>(ra, ma);
                    ib = row_scale<RDT, CH>(rb, mb);
                    team_sum(ia, ib);
                }
            }
            // a row against itself is no preference: exactly 0, whatever the roundings below
            ia = a == b ? 0.0f : inverse_norm(ia);
            ib = a == b ? 0.0f : inverse_norm(ib);
            keep_raw(ra, rb);
#pragma unroll
            for (int c = 0; c < CH; c++) {
                float av[8], bv[8], yv[8], dv[8];
                raw8_to_float<RDT>(ra[c], av);
                raw8_to_float<RDT>(rb[c], bv);
                query8(0, c, yv);
                query8(1, c, dv);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float d = fmaf(av[e], ia, -(bv[e] * ib));
                    cos = fmaf(yv[e], d, cos);
                    m = fmaf(dv[e], d, m);
                }
            }
            team_sum(cos, m);
            const float h = p.beta * m, e = p.smoothing;
            const float up = 1.0f / (1.0f + expf(-h)), down = 1.0f / (1.0f + expf(h));  // sigma(h), sigma(-h): each without cancellation
            if (tl == 0) {
                p.loss[i] = (1.0f - e) * softplus(-h) + e * softplus(h);
                p.margin[i] = m;
            }
            const float w = (p.weights ? p.weights[i] : p.default_weight) * p.beta * (e * up - (1.0f - e) * down);
            total = fmaf(w, cos, total);
            const float wa = w * ia, wb = w * ib;
            keep_raw(ra, rb);
#pragma unroll
            for (int c = 0; c < CH; c++) {
                float av[8], bv[8];
                raw8_to_float<RDT>(ra[c], av);
                raw8_to_float<RDT>(rb[c], bv);
#pragma unroll
                for (int k = 0; k < 8; k++) g[c * 8 + k] = fmaf(wa, av[k], fmaf(-wb, bv[k], g[c * 8 + k]));
            }
        }
        a = a_next, b = b_next;
        fetch(a, b);
        a_next = b_next = -1;
        if (i + 2 * TEAMS < hi) a_next = p.chosen[i + 2 * TEAMS], b_next = p.rejected[i + 2 * TEAMS];
    }

    // the teams that had pairs, in team order
    const int busy = TEAMS == 1 ? 1 : (hi - lo < TEAMS ? (hi - lo > 0 ? (int)(hi - lo) : 1) : TEAMS);
    float *vec = smem + (TW == 1 ? 2 * SPAN : 0);
    if (tl == 0) num[team] = total;
    if (team < busy) {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int k = (c * TW * 64 + tl) * 8;
            if (TW == 1) {
                f32x4 *l = reinterpret_cast<f32x4 *>(vec + team * SPAN + k);
                l[0] = f32x4{g[c * 8], g[c * 8 + 1], g[c * 8 + 2], g[c * 8 + 3]};
                l[1] = f32x4{g[c * 8 + 4], g[c * 8 + 5], g[c * 8 + 6], g[c * 8 + 7]};
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (k + e < p.dim) vec[k + e] = g[c * 8 + e];
            }
        }
    }
    __syncthreads();
    float sum = 0.0f;
    for (int t = 0; t < busy; t++) sum += num[t];
    const Q *yr = reinterpret_cast<const Q *>(p.y) + q * p.ld_y;
    Q *out = reinterpret_cast<Q *>(p.grad) + q * p.ld_grad;
    float *pv = used == 1 ? nullptr : p.part_vec + (q * shares + z) * p.dim;
    for (int k = tid; k < p.dim; k += 64 * WAVES) {
        float v = vec[k];
        for (int t = 1; t < busy; t++) v += vec[t * SPAN + k];
        if (used == 1) out[k] = learn_from_float<Q>(inv_y * (v - sum * (TW == 1 ? smem[k] : inv_y * learn_to_float(yr[k]))));
        else pv[k] = v;
    }
    // pairs before the first query's and after the last one's are left out like those with a negative position
    if (z == 0) {
        if (q == 0)
            for (int64_t k = tid; k < b0; k += 64 * WAVES) p.loss[k] = p.margin[k] = 0.0f;
        if (q == p.n_queries - 1)
            for (int64_t k = b1 + tid; k < p.n_pairs; k += 64 * WAVES) p.loss[k] = p.margin[k] = 0.0f;
    }
    if (used > 1 && tid == 0) {
        p.part_num[q * shares + z] = sum;
        if (z == 0) p.part_inv[q] = inv_y;
    }
}

// Queries whose pairs several blocks shared: their sums, a block per query and 64 columns.  Each of the waves adds its part of the
// shares in order, then the waves are added in order.
#define JOIN_WAVES 8
template <int QDT> __global__ __launch_bounds__(64 * JOIN_WAVES) void preference_join_kernel(PreferenceParams p, int shares) {
    typedef typename Elem<QDT>::type Q;
    __shared__ float part[JOIN_WAVES][64];
    const int64_t q = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = blockIdx.y * 64 + lane;
    int64_t b0, b1, per;
    int used;
    pair_share(p, q, shares, b0, b1, per, used);
    if (used == 1) return;
    const float *vec = p.part_vec + q * shares * p.dim + k, *num = p.part_num + q * shares;
    float v = 0.0f, sum = 0.0f;
    if (k < p.dim) {
#pragma unroll 8
        for (int z = wave; z < used; z += JOIN_WAVES) v += vec[(int64_t)z * p.dim];
    }
    part[wave][lane] = v;
    __syncthreads();
    if (wave) return;
    for (int z = lane; z < used; z += 64) sum += num[z];
    sum = learn_wave_sum(sum);
    if (k >= p.dim) return;
    v = part[0][lane];
#pragma unroll
    for (int w = 1; w < JOIN_WAVES; w++) v += part[w][lane];
    const float inv_y = p.part_inv[q], y = learn_to_float(reinterpret_cast<const Q *>(p.y)[q * p.ld_y + k]);
    reinterpret_cast<Q *>(p.grad)[q * p.ld_grad + k] = learn_from_float<Q>(inv_y * (v - sum * (inv_y * y)));
}

// Columns up to which a wave takes a pair by itself; beyond, 4 waves take it together (past 8192 columns 8).  2000 queries x 8 pairs of fp16:
// 2048 columns 40 us; 2560, 4096, 8192, 16 384 columns 65, 74, 165, 367 us (with 16 waves on a pair 199, 207, 250, 631)
#define PREF_WAVE_DIM 2048

// How the pairs are spread over the chip, by counts alone (the host does not see the offsets); 1536 columns, fp16 rows.
struct PreferencePlan {
    int shares;     // blocks a query's pairs may be shared by
    int per_block;  // pairs a block takes before another one joins in
    bool wide;      // 16 waves a block instead of 4
};
static PreferencePlan preference_plan(const hvs_preference *p, int dim) {
    const int64_t nq = p->n_queries, pairs = p->n_pairs;
    const bool one = dim > PREF_WAVE_DIM;  // the waves of a block take one pair together
    // queries enough for the chip: a block each
    if (nq < 1 || nq > 512) return {1, INT_MAX, false};
    // Few pairs each: a block each saves the join, which reads a vector per block (a block each / shared: 16 x 16 10.6 / 9.9 us,
    // 64 x 64 22.9 / 15.0; 100 x 16 10.5 / 13.0, 100 x 64 23.3 / 22.1, 400 x 32 27.5 / 36).  16 waves where there is a CU for each
    // block and more than one pair for a wave (4 waves / 16: 100 x 4 7.1 / 7.3, 250 x 8 9.1 / 8.7, 250 x 16 13.2 / 11.2, 400 x 16 17.4 / 22.8).
    // With a pair at a time (4096 columns, alone / shared): 1 x 4 12.7 / 9.5, 16 x 16 31 / 11; 100 x 4 13.3 / 20.7, 100 x 16 34 / 27; 400 x 8 28.5 / 61.
    const int64_t alone = one ? (nq <= 64 ? 2 : nq <= 128 ? 8 : 64) : (nq <= 64 ? 16 : 64);
    if (pairs <= alone * nq) return {1, INT_MAX, nq <= 256 && pairs > 4 * nq};
    // more: blocks of a pair at a time, or one for each of 4 waves, until they are 512; then more pairs each
    // (4, 8, 16, 32 pairs a block: 1 x 64 10.9, 12.2, 15.8, 22.6 us; 64 x 64 16.9, 15.0, 16.5, 23.2)
    const int64_t even = (pairs + 511) / 512, per = one ? even : even < 4 ? 4 : (even + 3) / 4 * 4, most = 1024 / nq, shares = (pairs + per - 1) / per;
    return {(int)(shares < most ? shares : most), (int)(per < INT_MAX ? per : INT_MAX), false};
}

static int check_preference(const char *who, const hvs_preference *p, int dim) {
    HVS_REQUIRE(p != nullptr, "%s: NULL argument", who);
    HVS_REQUIRE(learn_dtype_ok(p->query_dtype), "%s: unknown query dtype %d", who, p->query_dtype);
    HVS_REQUIRE(dim >= 1 && dim <= 16384, "%s: dim %d not in [1, 16384]", who, dim);
    HVS_REQUIRE(p->n_queries >= 0 && p->n_pairs >= 0, "%s: negative count", who);
    HVS_REQUIRE(p->n_queries <= 0x7FFFFFFF, "%s: %lld queries, at most 2^31 - 1", who, (long long)p->n_queries);
    HVS_REQUIRE(p->beta > 0.0f && std::isfinite(p->beta), "%s: beta %g must be positive and finite", who, (double)p->beta);
    HVS_REQUIRE(p->label_smoothing >= 0.0f && p->label_smoothing <= 0.5f, "%s: label_smoothing %g not in [0, 0.5]", who, (double)p->label_smoothing);
    return 0;
}

extern "C" int hvs_preference_workspace(const hvs_preference *p, int dim, uint64_t *out_bytes) {
    HVS_TRY(check_preference("hvs_preference_workspace", p, dim));
    HVS_REQUIRE(out_bytes != nullptr, "hvs_preference_workspace: NULL argument");
    const int shares = preference_plan(p, dim).shares;
    WorkspaceCut w(nullptr);
    if (shares > 1) {
        w.take<float>((uint64_t)p->n_queries * shares * dim * 4);
        w.take<float>((uint64_t)p->n_queries * shares * 4);
        w.take<float>((uint64_t)p->n_queries * 4);
    }
    *out_bytes = w.used;
    return 0;
}

// Queries of one launch: a grid dimension ends below 2^32 threads, 2^23 blocks of 512.
#define PREF_LAUNCH_QUERIES (1ll << 22)
template <int QDT, int RDT, int CH, int TW, int WAVES>
static int launch_preference(hipStream_t st, PreferenceParams p, int64_t nq, int shares, bool aligned) {
    const size_t lds = (TW == 1 ? (size_t)(2 + WAVES) * CH * 512 : (size_t)p.dim) * 4;
    if (aligned) HVS_TRY((learn_allow_lds<preference_kernel<QDT, RDT, CH, TW, WAVES, true>>((int)lds)));
    else HVS_TRY((learn_allow_lds<preference_kernel<QDT, RDT, CH, TW, WAVES, false>>((int)lds)));
    for (p.first_query = 0; p.first_query < nq; p.first_query += PREF_LAUNCH_QUERIES) {
        const int64_t left = nq - p.first_query;
        const dim3 grid((unsigned)(left < PREF_LAUNCH_QUERIES ? left : PREF_LAUNCH_QUERIES), shares);
        if (aligned) preference_kernel<QDT, RDT, CH, TW, WAVES, true><<<grid, 64 * WAVES, lds, st>>>(p);
        else preference_kernel<QDT, RDT, CH, TW, WAVES, false><<<grid, 64 * WAVES, lds, st>>>(p);
        HVS_HIP(hipGetLastError());
    }
    return 0;
}

template <int QDT, int RDT> static int run_preference(hipStream_t st, const PreferenceParams &p, int64_t nq, int shares, bool wide) {
    const int qs = hvs_elem_size(QDT), rs = hvs_elem_size(RDT);
    const bool al = p.dim % 8 == 0 && learn_aligned(p.y, p.ld_y * qs, 0) && (!p.ref || learn_aligned(p.ref, p.ld_ref * qs, 0)) &&
                    learn_aligned(p.rows, p.ld_rows * rs, 0);
    if (p.dim > 8192) HVS_TRY((launch_preference<QDT, RDT, 4, 8, 8>(st, p, nq, shares, al)));
    else if (p.dim > 4096) HVS_TRY((launch_preference<QDT, RDT, 4, 4, 4>(st, p, nq, shares, al)));
    else if (p.dim > PREF_WAVE_DIM) HVS_TRY((launch_preference<QDT, RDT, 2, 4, 4>(st, p, nq, shares, al)));
    else {
        const int ch = (p.dim + 511) / 512;
#define PREF(CH_) (wide ? launch_preference<QDT, RDT, CH_, 1, 16>(st, p, nq, shares, al) : launch_preference<QDT, RDT, CH_, 1, 4>(st, p, nq, shares, al))
        if (ch == 1) HVS_TRY(PREF(1));
        else if (ch == 2) HVS_TRY(PREF(2));
        else if (ch == 3) HVS_TRY(PREF(3));
        else HVS_TRY(PREF(4));
#undef PREF
    }
    if (shares > 1) {
        preference_join_kernel<QDT><<<dim3((unsigned)nq, (p.dim + 63) / 64), 64 * JOIN_WAVES, 0, st>>>(p, shares);
        HVS_HIP(hipGetLastError());
    }
    return 0;
}

static int check_preference_buffers(const char *who, const hvs_preference *p, const void *rows, int rows_dtype, int dim, int64_t ld_rows, int64_t n_rows,
                                    const void *workspace, uint64_t workspace_bytes) {
    const int qs = hvs_elem_size(p->query_dtype);
    HVS_REQUIRE(p->queries && p->grad && p->offsets, "%s: queries, grad or offsets is NULL", who);
    HVS_REQUIRE(p->n_pairs == 0 || (p->chosen && p->rejected && p->loss && p->margin), "%s: chosen, rejected, loss or margin is NULL", who);
    HVS_REQUIRE(n_rows >= 0 && (n_rows == 0 || rows), "%s: rows is NULL or n_rows negative", who);
    HVS_REQUIRE(p->ld_queries >= dim && p->ld_grad >= dim && ld_rows >= dim && (!p->reference || p->ld_reference >= dim), "%s: a row pitch is below dim %d", who, dim);
    HVS_REQUIRE((uintptr_t)p->queries % qs == 0 && (uintptr_t)p->reference % qs == 0 && (uintptr_t)p->grad % qs == 0 &&
                    (uintptr_t)rows % hvs_elem_size(rows_dtype) == 0,
                "%s: a tensor is not aligned to its elements", who);
    HVS_REQUIRE(((uintptr_t)p->offsets | (uintptr_t)p->chosen | (uintptr_t)p->rejected) % 8 == 0 &&
                    ((uintptr_t)p->weights | (uintptr_t)p->loss | (uintptr_t)p->margin) % 4 == 0,
                "%s: a list is not aligned to its elements", who);
    HVS_REQUIRE(!learn_overlap(p->queries, p->n_queries, p->ld_queries * qs, (int64_t)dim * qs, p->grad, p->n_queries, p->ld_grad * qs, (int64_t)dim * qs) &&
                    !(p->reference && learn_overlap(p->reference, p->n_queries, p->ld_reference * qs, (int64_t)dim * qs, p->grad, p->n_queries, p->ld_grad * qs,
                                                    (int64_t)dim * qs)),
                "%s: grad overlaps an input", who);
    uint64_t need = 0;
    HVS_TRY(hvs_preference_workspace(p, dim, &need));
    HVS_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= need),
                "%s: workspace of %llu bytes at %p, needs %llu aligned to 256", who, (unsigned long long)workspace_bytes, workspace, (unsigned long long)need);
    return 0;
}

static int preference_core(hipStream_t st, const hvs_preference *p, const void *rows, int rows_dtype, int dim, int64_t ld_rows, int64_t n_rows, void *workspace) {
    const PreferencePlan plan = preference_plan(p, dim);
    const int shares = plan.shares;
    PreferenceParams k = {};
    k.y = p->queries, k.ref = p->reference, k.ld_y = p->ld_queries, k.ld_ref = p->ld_reference;
    k.offsets = p->offsets, k.chosen = p->chosen, k.rejected = p->rejected, k.weights = p->weights;
    k.loss = p->loss, k.margin = p->margin, k.grad = p->grad, k.ld_grad = p->ld_grad, k.n_pairs = p->n_pairs, k.n_queries = p->n_queries;
    k.rows = rows, k.ld_rows = ld_rows, k.n_rows = n_rows, k.dim = dim;
    k.beta = p->beta, k.smoothing = p->label_smoothing, k.default_weight = p->n_pairs > 0 ? (float)(1.0 / (double)p->n_pairs) : 0.0f;
    k.per_block = plan.per_block;
    if (shares > 1) {
        WorkspaceCut w(workspace);
        k.part_vec = w.take<float>((uint64_t)p->n_queries * shares * dim * 4);
        k.part_num = w.take<float>((uint64_t)p->n_queries * shares * 4);
        k.part_inv = w.take<float>((uint64_t)p->n_queries * 4);
    }
#define ROWS(Q_)                                                                                     \
    (rows_dtype == HVS_F32 ? run_preference<Q_, HVS_F32>(st, k, p->n_queries, shares, plan.wide)        \
                           : rows_dtype == HVS_F16 ? run_preference<Q_, HVS_F16>(st, k, p->n_queries, shares, plan.wide) \
                                                   : run_preference<Q_, HVS_BF16>(st, k, p->n_queries, shares, plan.wide))
    if (p->query_dtype == HVS_F32) return ROWS(HVS_F32);
    if (p->query_dtype == HVS_F16) return ROWS(HVS_F16);
    return ROWS(HVS_BF16);
#undef ROWS
}

extern "C" int hvs_preference_loss(int device_id, void *stream, const hvs_preference *p, const void *rows, int rows_dtype, int dim, int64_t ld_rows,
                                   int64_t n_rows, void *workspace, uint64_t workspace_bytes) {
    const char *who = "hvs_preference_loss";
    HVS_TRY(check_preference(who, p, dim));
    HVS_REQUIRE(learn_dtype_ok(rows_dtype), "%s: unknown row dtype %d", who, rows_dtype);
    if (p->n_queries == 0) {
        HVS_REQUIRE(p->n_pairs == 0, "%s: %lld pairs but no query", who, (long long)p->n_pairs);
        return 0;
    }
    HVS_TRY(check_preference_buffers(who, p, rows, rows_dtype, dim, ld_rows, n_rows, workspace, workspace_bytes));
    DeviceGuard guard(device_id);
    HVS_HIP(guard.status);
    return preference_core((hipStream_t)stream, p, rows, rows_dtype, dim, ld_rows, n_rows, workspace);
}

extern "C" int hvs_index_preference_loss(hvs_index *idx, void *stream, const hvs_preference *p, void *workspace, uint64_t workspace_bytes) {
    const char *who = "hvs_index_preference_loss";
    HVS_REQUIRE(idx != nullptr, "%s: idx is NULL", who);
    HVS_TRY(check_preference(who, p, idx->dim));
    if (p->n_queries == 0) {
        HVS_REQUIRE(p->n_pairs == 0, "%s: %lld pairs but no query", who, (long long)p->n_pairs);
        return 0;
    }
    HVS_TRY(check_preference_buffers(who, p, idx->rows, idx->dtype, idx->dim, idx->ld, idx->n, workspace, workspace_bytes));
    DeviceGuard guard(idx->device);
    HVS_HIP(guard.status);
    hipStream_t st = (hipStream_t)stream;
    for (hipStream_t own : {st, idx->stream}) {
        hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
        if (own != nullptr) HVS_HIP(hipStreamIsCapturing(own, &capturing));
        HVS_REQUIRE(capturing == hipStreamCaptureStatusNone, "%s: the %s is being captured; a graph would keep the address of rows the table may move", who,
                    own == st ? "stream" : "table's stream");
    }
    if (st == idx->stream) return preference_core(st, p, idx->rows, idx->dtype, idx->dim, idx->ld, idx->n, workspace);
    for (hipEvent_t *ev : {&idx->ev_table, &idx->ev_reader})
        if (*ev == nullptr) HVS_HIP(hipEventCreateWithFlags(ev, hipEventDisableTiming | hipEventDisableSystemFence));
    // after the work the table's stream holds; mostly it holds none, and then there is nothing to wait for
    const hipError_t idle = hipStreamQuery(idx->stream);
    if (idle == hipErrorNotReady) {
        (void)hipGetLastError();  // an answer, not an error to be found by the next launch
        HVS_HIP(hipEventRecord(idx->ev_table, idx->stream));
        HVS_HIP(hipStreamWaitEvent(st, idx->ev_table, 0));
    } else HVS_HIP(idle);
    // ev_reader is about to stand for this read: the table's stream waits now for an earlier one on another stream
    if (idx->reader_pending && idx->reader_stream != st) HVS_TRY(hvs_index_enter(idx));
    const int failed = preference_core(st, p, idx->rows, idx->dtype, idx->dim, idx->ld, idx->n, workspace);
    const hipError_t recorded = hipEventRecord(idx->ev_reader, st);
    if (failed || recorded != hipSuccess) (void)hipStreamSynchronize(st);  // a read that no event stands for must not be left behind
    HVS_TRY(failed);
    HVS_HIP(recorded);
    idx->reader_stream = st;
    idx->reader_pending = true;
    return 0;
}

// ---------------------------------------------------------------------------------------------------------------
// global norm and clipping
// ---------------------------------------------------------------------------------------------------------------
#define CLIP_BATCH 64      // tensors per launch: their table travels in the kernel's arguments
#define CLIP_CHUNK 8192    // most elements a block takes at a time,
#define CLIP_CHUNK_MIN 1024  // ... and fewest: small sets are spread over as many blocks as that gives (1024 / 8192 alone: 100 000 elements 6.0 / 8.0 us)
// Up to so many elements in so few tensors one block does it all.  One launch / two, 2 tensors of 24 576 fp32 elements: 9.2 / 6.1 us
// on the GPU (16 000 elements in all: 5.7 / 6.1), 12.0 / 15.4 us on the host, which is what an eager call waits for; 30 tensors
// one after the other would take 33 us.
#define CLIP_ONCE 65536
#define CLIP_ONCE_TENSORS 4
#define CLIP_BLOCKS 2048   // blocks of a norm launch, one partial sum each

struct ClipTable {
    const void *data[CLIP_BATCH];
    void *out[CLIP_BATCH];
    int64_t numel[CLIP_BATCH];
    uint32_t first_chunk[CLIP_BATCH + 1];
    int32_t dtype[CLIP_BATCH];
    int n, chunk;  // chunk: elements a block takes at a time
};

// two partial results of a norm: sums of squares add up, largest values do not, a NaN stays
__device__ __forceinline__ double norm_join(double a, double b, bool inf_norm) {
    if (!inf_norm) return a + b;
    return a != a || b != b ? __builtin_nan("") : (a > b ? a : b);
}
template <int THREADS> __device__ __forceinline__ double block_join(double v, bool inf_norm, double *lds) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = norm_join(v, __shfl_xor(v, o), inf_norm);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; w++) v = norm_join(v, lds[w], inf_norm);
    return v;
}
__device__ __forceinline__ float clip_factor(float norm, double max_norm) {
    if (norm != norm) return norm;
    return max_norm < __builtin_inf() ? (float)fmin(max_norm / ((double)norm + 1e-6), 1.0) : 1.0f;
}

__device__ __forceinline__ int clip_tensor_of(const ClipTable &t, uint32_t chunk) {
    int lo = 0, hi = t.n;  // the last tensor whose first chunk is not past this one
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first_chunk[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <int DT, int THREADS> __device__ __forceinline__ double chunk_norm(const void *data, int64_t begin, int64_t end, bool inf_norm) {
    typedef typename Elem<DT>::type E;
    constexpr int EPC = Elem<DT>::EPC;
    const E *p = reinterpret_cast<const E *>(data);
    double acc = 0.0;
    auto add = [&](float v) { acc = inf_norm ? norm_join(acc, (double)fabsf(v), true) : fma((double)v, (double)v, acc); };
    int64_t i = begin;
    if (((uintptr_t)data & 15) == 0) {
        const int64_t whole = begin + ((end - begin) / EPC) * EPC;
        i = begin + threadIdx.x * EPC;
        for (; i + 3 * THREADS * EPC < whole; i += 4 * THREADS * EPC) {  // four loads in flight (118 -> 100 us)
            f32x4 c[4];
#pragma unroll
            for (int k = 0; k < 4; k++) c[k] = *reinterpret_cast<const f32x4 *>(p + i + k * THREADS * EPC);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float v[EPC];
                chunk_to_float<DT>(c[k], v);
#pragma unroll
                for (int e = 0; e < EPC; e++) add(v[e]);
            }
        }
        for (; i < whole; i += THREADS * EPC) {
            float v[EPC];
            chunk_to_float<DT>(*reinterpret_cast<const f32x4 *>(p + i), v);
#pragma unroll
            for (int e = 0; e < EPC; e++) add(v[e]);
        }
        i = whole;
    }
    for (i += threadIdx.x; i < end; i += THREADS) add(learn_to_float(p[i]));
    return acc;
}

template <int DT, int THREADS> __device__ __forceinline__ void chunk_scale(const void *data, void *out, int64_t begin, int64_t end, float f) {
    typedef typename Elem<DT>::type E;
    constexpr int EPC = Elem<DT>::EPC;
    typedef E vec __attribute__((ext_vector_type(EPC)));
    const E *p = reinterpret_cast<const E *>(data);
    E *o = reinterpret_cast<E *>(out);
    int64_t i = begin;
    if (((uintptr_t)data & 15) == 0 && ((uintptr_t)out & 15) == 0) {
        const int64_t whole = begin + ((end - begin) / EPC) * EPC;
        // what is written is not read again here: kept out of the caches, it leaves them to what the next norm pass reads
        // (565 MB of gradients: norm pass 139 -> 118 us).  Four loads in flight, as the norm pass has them, cost 10 us here.
        for (i = begin + threadIdx.x * EPC; i < whole; i += THREADS * EPC) {
            float v[EPC];
            chunk_to_float<DT>(*reinterpret_cast<const f32x4 *>(p + i), v);
            vec r;
#pragma unroll
            for (int e = 0; e < EPC; e++) r[e] = learn_from_float<E>(v[e] * f);
            __builtin_nontemporal_store(r, reinterpret_cast<vec *>(o + i));
        }
        i = whole;
    }
    for (i += threadIdx.x; i < end; i += THREADS) o[i] = learn_from_float<E>(learn_to_float(p[i]) * f);
}

// the same for an element range of a tensor of any type
template <int THREADS> __device__ __forceinline__ double range_norm(const ClipTable &t, int k, int64_t begin, int64_t end, bool inf_norm) {
    return t.dtype[k] == HVS_F32   ? chunk_norm<HVS_F32, THREADS>(t.data[k], begin, end, inf_norm)
           : t.dtype[k] == HVS_F16 ? chunk_norm<HVS_F16, THREADS>(t.data[k], begin, end, inf_norm)
                                   : chunk_norm<HVS_BF16, THREADS>(t.data[k], begin, end, inf_norm);
}
template <int THREADS> __device__ __forceinline__ void range_scale(const ClipTable &t, int k, int64_t begin, int64_t end, float f) {
    if (f == 1.0f && t.out[k] == t.data[k]) return;  // in place and nothing to clip: the tensor is its own result
    if (t.dtype[k] == HVS_F32) chunk_scale<HVS_F32, THREADS>(t.data[k], t.out[k], begin, end, f);
    else if (t.dtype[k] == HVS_F16) chunk_scale<HVS_F16, THREADS>(t.data[k], t.out[k], begin, end, f);
    else chunk_scale<HVS_BF16, THREADS>(t.data[k], t.out[k], begin, end, f);
}

__global__ __launch_bounds__(256) void clip_norm_kernel(ClipTable t, int inf_norm, double *__restrict__ partial) {
    __shared__ double lds[4];
    double acc = 0.0;
    for (uint32_t c = blockIdx.x; c < t.first_chunk[t.n]; c += gridDim.x) {
        const int k = clip_tensor_of(t, c);
        const int64_t begin = (int64_t)(c - t.first_chunk[k]) * t.chunk;
        const int64_t end = begin + t.chunk < t.numel[k] ? begin + t.chunk : t.numel[k];
        acc = norm_join(acc, range_norm<256>(t, k, begin, end, inf_norm), inf_norm);
    }
    acc = block_join<256>(acc, inf_norm, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// Every block adds up the partial sums itself (the same order everywhere), then scales its chunks, the last ones first: they
// are what the norm pass has left in the caches.
__global__ __launch_bounds__(256) void clip_scale_kernel(ClipTable t, int inf_norm, const double *__restrict__ partial, int n_partial, double max_norm,
                                                         float *__restrict__ norm_out, int write_norm) {
    __shared__ double lds[4];
    double acc = 0.0;
    for (int i = threadIdx.x; i < n_partial; i += 256) acc = norm_join(acc, partial[i], inf_norm);
    acc = block_join<256>(acc, inf_norm, lds);
    const float norm = (float)(inf_norm ? acc : sqrt(acc));
    if (write_norm && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    const float f = clip_factor(norm, max_norm);
    const uint32_t chunks = t.first_chunk[t.n];
    for (uint32_t i = blockIdx.x; i < chunks; i += gridDim.x) {
        const uint32_t c = chunks - 1 - i;
        const int k = clip_tensor_of(t, c);
        const int64_t begin = (int64_t)(c - t.first_chunk[k]) * t.chunk;
        const int64_t end = begin + t.chunk < t.numel[k] ? begin + t.chunk : t.numel[k];
        range_scale<256>(t, k, begin, end, f);
    }
}

// A few tensors of a few elements (CLIP_ONCE): one block does both passes, and a launch is saved.
__global__ __launch_bounds__(1024) void clip_once_kernel(ClipTable t, int inf_norm, double max_norm, float *__restrict__ norm_out) {
    __shared__ double lds[16];
    double acc = 0.0;
    for (int k = 0; k < t.n; k++) acc = norm_join(acc, range_norm<1024>(t, k, 0, t.numel[k], inf_norm), inf_norm);
    acc = block_join<1024>(acc, inf_norm, lds);
    const float norm = (float)(inf_norm ? acc : sqrt(acc));
    if (threadIdx.x == 0) *norm_out = norm;
    const float f = clip_factor(norm, max_norm);
    for (int k = 0; k < t.n; k++) range_scale<1024>(t, k, 0, t.numel[k], f);
}

static int check_tensors(const char *who, const hvs_tensor *t, int n) {
    HVS_REQUIRE(n >= 0 && (n == 0 || t), "%s: negative tensor count or NULL argument", who);
    for (int i = 0; i < n; i++) {
        HVS_REQUIRE(learn_dtype_ok(t[i].dtype), "%s: tensor %d: unknown dtype %d", who, i, t[i].dtype);
        HVS_REQUIRE(t[i].numel >= 0 && t[i].numel <= (int64_t)1 << 40, "%s: tensor %d: %lld elements, must be in [0, 2^40]", who, i, (long long)t[i].numel);
        if (t[i].numel == 0) continue;
        const int es = hvs_elem_size(t[i].dtype);
        HVS_REQUIRE(t[i].data && t[i].out, "%s: tensor %d is NULL", who, i);
        HVS_REQUIRE((uintptr_t)t[i].data % es == 0 && (uintptr_t)t[i].out % es == 0, "%s: tensor %d is not aligned to its elements", who, i);
        HVS_REQUIRE(t[i].data == t[i].out || !learn_overlap(t[i].data, 1, 0, t[i].numel * es, t[i].out, 1, 0, t[i].numel * es),
                    "%s: tensor %d: out overlaps data without being data", who, i);
    }
    return 0;
}

// No tensor may be written while another one is read or written: a tensor named twice would be scaled twice.
struct ClipRange {
    uintptr_t begin, end;
    bool written;
};
static int check_apart(const char *who, const hvs_tensor *t, int n) {
    std::vector<ClipRange> r;
    try {
        r.reserve(2 * (size_t)n);
    } catch (const std::bad_alloc &) {
        hvs_set_error("%s: out of host memory", who);
        return 1;
    }
    for (int i = 0; i < n; i++) {
        const uintptr_t bytes = (uintptr_t)t[i].numel * hvs_elem_size(t[i].dtype);
        if (bytes == 0) continue;
        r.push_back({(uintptr_t)t[i].out, (uintptr_t)t[i].out + bytes, true});
        if (t[i].data != t[i].out) r.push_back({(uintptr_t)t[i].data, (uintptr_t)t[i].data + bytes, false});
    }
    std::sort(r.begin(), r.end(), [](const ClipRange &a, const ClipRange &b) { return a.begin < b.begin; });
    uintptr_t any_end = 0, written_end = 0;  // how far the ranges so far reach
    for (const ClipRange &c : r) {
        HVS_REQUIRE(c.begin >= (c.written ? any_end : written_end), "%s: two tensors share memory", who);
        any_end = any_end > c.end ? any_end : c.end;
        if (c.written) written_end = written_end > c.end ? written_end : c.end;
    }
    return 0;
}

// elements a block takes at a time: about 2048 chunks in all, within the limits
static int clip_chunk(const hvs_tensor *t, int n) {
    int64_t total = 0;
    for (int i = 0; i < n && total < (int64_t)CLIP_CHUNK << 11; i++) total += t[i].numel;
    int chunk = CLIP_CHUNK_MIN;
    while (chunk < CLIP_CHUNK && (int64_t)chunk << 11 < total) chunk *= 2;
    return chunk;
}
// The tensors of one launch, from number `at` on; returns the number of the first one left over.  2^40 elements are at most
// 2^30 chunks, so at least one tensor always fits.
static int fill_table(const hvs_tensor *t, int n, int at, int chunk, ClipTable *tab) {
    tab->n = 0;
    tab->chunk = chunk;
    tab->first_chunk[0] = 0;
    while (at < n && tab->n < CLIP_BATCH) {
        const uint64_t chunks = ((uint64_t)t[at].numel + chunk - 1) / chunk;
        const uint64_t end = tab->first_chunk[tab->n] + chunks;
        if (end > 0x7FFFFFFFull) break;
        tab->data[tab->n] = t[at].data, tab->out[tab->n] = t[at].out, tab->numel[tab->n] = t[at].numel, tab->dtype[tab->n] = t[at].dtype;
        tab->first_chunk[++tab->n] = (uint32_t)end;
        at++;
    }
    return at;
}

extern "C" int hvs_clip_workspace(const hvs_tensor *tensors, int n_tensors, uint64_t *out_bytes) {
    HVS_TRY(check_tensors("hvs_clip_workspace", tensors, n_tensors));
    HVS_REQUIRE(out_bytes != nullptr, "hvs_clip_workspace: NULL argument");
    ClipTable tab;
    const int chunk = clip_chunk(tensors, n_tensors);
    uint64_t partials = 0;
    for (int at = 0; at < n_tensors;) {
        at = fill_table(tensors, n_tensors, at, chunk, &tab);
        partials += tab.first_chunk[tab.n] < CLIP_BLOCKS ? tab.first_chunk[tab.n] : CLIP_BLOCKS;
    }
    *out_bytes = (partials ? partials : 1) * sizeof(double);
    return 0;
}

extern "C" int hvs_clip_grad_norm(int device_id, void *stream, const hvs_tensor *tensors, int n_tensors, double max_norm, int infinity_norm, float *norm,
                                  void *workspace, uint64_t workspace_bytes) {
    const char *who = "hvs_clip_grad_norm";
    uint64_t need = 0;
    HVS_TRY(hvs_clip_workspace(tensors, n_tensors, &need));
    HVS_TRY(check_apart(who, tensors, n_tensors));
    HVS_REQUIRE(norm != nullptr, "%s: norm is NULL", who);
    HVS_REQUIRE(max_norm >= 0.0, "%s: max_norm %g must not be negative or NaN", who, max_norm);
    HVS_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= need, "%s: workspace of %llu bytes at %p, needs %llu aligned to 256", who,
                (unsigned long long)workspace_bytes, workspace, (unsigned long long)need);
    DeviceGuard guard(device_id);
    HVS_HIP(guard.status);
    hipStream_t st = (hipStream_t)stream;
    double *partial = (double *)workspace;
    ClipTable tab;
    const int chunk = clip_chunk(tensors, n_tensors);
    int64_t total = 0;
    for (int i = 0; i < n_tensors && total <= CLIP_ONCE; i++) total += tensors[i].numel;
    if (n_tensors <= CLIP_ONCE_TENSORS && total <= CLIP_ONCE) {
        fill_table(tensors, n_tensors, 0, chunk, &tab);
        clip_once_kernel<<<1, 1024, 0, st>>>(tab, infinity_norm != 0, max_norm, norm);
        HVS_HIP(hipGetLastError());
        return 0;
    }
    int n_partial = 0;
    for (int at = 0; at < n_tensors;) {
        at = fill_table(tensors, n_tensors, at, chunk, &tab);
        const int blocks = (int)(tab.first_chunk[tab.n] < CLIP_BLOCKS ? tab.first_chunk[tab.n] : CLIP_BLOCKS);
        if (blocks == 0) continue;
        clip_norm_kernel<<<blocks, 256, 0, st>>>(tab, infinity_norm != 0, partial + n_partial);
        HVS_HIP(hipGetLastError());
        n_partial += blocks;
    }
    bool first = true;
    for (int at = 0; at < n_tensors || first; first = false) {
        at = fill_table(tensors, n_tensors, at, chunk, &tab);
        const uint32_t chunks = tab.first_chunk[tab.n];
        if (chunks == 0 && !first) continue;
        clip_scale_kernel<<<(int)(chunks < 1 ? 1 : (chunks < 2048 ? chunks : 2048)), 256, 0, st>>>(tab, infinity_norm != 0, partial, n_partial, max_norm, norm, first);
        HVS_HIP(hipGetLastError());
    }
    return 0;
}
