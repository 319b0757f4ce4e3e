// Low-rank adapters of many tenants beside one shared projection (C ABI: include/hvs.h).
//
//     y_i = W x_i + s_c B_c (A_c x_i),  c = code of row i            (forward)
//     v_i = s_c B_c^T g_i,  dx_i = W^T g_i + A_c^T v_i,  dA_c = sum v_i x_i^T,  dB_c = s_c sum g_i u_i^T   (backward)
//
// Two routes.  Few rows (few_rows): blocks of 16 x 16 to 32 x 32 outputs, rows in arrival order; bound by the latency of
// reading W, from some hundred rows on by what 32 x 32 blocks read out of the L2: 777 x 1001 -> 770 in fp32 reads 155 MB in
// 34 us (4.5 TB/s; 2.27 million requests, 89 % hits), with the matrix pipe busy 38 % of the time.  Many rows: rows are
// ordered by code (a stable counting sort), so that a tile of rows meets few adapters; W x comes from the matrix-pipe loop
// the searches use, the low-rank term is added in its accumulators, and y is rounded and written once.
//
// u = A_c x is held in fp32.  For 16-bit weights the product with B runs on the 16-bit pipe: u is divided by a power of
// two that brings its largest element to [0.5, 1) (no overflow in fp16 whatever the inputs), split into two 16-bit parts
// hi + lo (relative error 2^-16 for bf16, 2^-22 for fp16: far below the output's own rounding), and the product is
// multiplied by that power and by s_c as it is added to W x.
#include "hvs_learn.h"

// rows up to which one launch does all.  One launch / two, rows of as many tenants, 1536 x 1536, rank 16, us: fp32 1 row 8.3 / 12.3,
// 2 rows 11.7 / 13.5, 4 rows 18.8 / 13.5; bf16 4.5 / 7.9, 6.1 / 7.9, 9.4 / 7.9
#define ONCE_ROWS 2
// Rows, and outputs (rows times columns), up to which blocks of few outputs take the rows in arrival order.  That costs by outputs
// times K, the grouped tiles by K alone until they fill the chip.  A call of 32 adapters of rank 16, this route / the tiles, us:
// fp32 1536 x 1536 1024 rows (1.6 million outputs) 94 / 108; 4096 x 4096 400 rows (1.6) 222 / 265, 600 rows (2.5) 316 / 268, 1024 rows 515 / 271
// bf16 1536 x 1536 600 rows (0.9) 25 / 29, 768 rows (1.2) 29 / 30; 4096 x 4096 256 rows (1.05) 43 / 56, 400 rows (1.6) 72 / 56, 768 rows 135 / 60
#define FEW_ROWS 1024
#define FEW_OUTPUTS_F32 1900000
#define FEW_OUTPUTS_16 1100000
#define GROUP_CHUNK 1024  // rows per block of the grouping kernels
#define MAX_CHUNK_ROWS 65536
// rows from which u = A x is taken 32 rows a wave instead of 16 a block.  A call with 64-column outputs, wide / narrow, us: 8192 rows of
// 16 adapters 25.7 / 21.9, 16 384 29.0 / 28.6, 32 768 33.3 / 38.3, 65 536 42.3 / 58.5; 256 adapters 32.6 / 24.8, 40.4 / 41.0, 43.7 / 51.5, 53.8 / 72.5
#define SHRINK_WIDE_ROWS 16384
#define SHRINK_WAVES 8
#define SHRINK_SHARES 4  // blocks that share the adapters among 16 rows in code order (1, 2, 4, 8: 11.2, 9.5, 8.9, 9.6 us, mean of three sizes)
#define OUTER_ROWS 512       // rows whose numbers a block of the stack gradients holds at a time
#define OUTER_PARTIAL_BYTES (128ll << 20)  // what their partial sums may take

// ---------------------------------------------------------------------------------------------------------------
// grouping: rows ordered by adapter, equal codes in row order
// ---------------------------------------------------------------------------------------------------------------
// bin 0: no adapter, bin c + 1: adapter c, bin S + 1: codes past the last adapter
__device__ __forceinline__ int group_bin(int32_t code, int S) { return code < 0 ? 0 : (code >= S ? S + 1 : code + 1); }

// The rows of every adapter cut into pieces of `rows` rows (one piece, an empty one, for an adapter without rows): what a
// block of the stack gradients works on.
struct Piece {
    int32_t adapter;
    uint32_t begin, end;  // rows, in code order
    int32_t slot;         // place of its partial sums, -1 when it is all of its adapter's rows
};
struct PieceTable {
    Piece *piece;     // [S + n / rows]; NULL: no table wanted
    uint32_t *slot;   // [S] first slot of an adapter of several pieces
    uint32_t *count;  // [1]
    int rows;
};

__global__ __launch_bounds__(GROUP_CHUNK) void group_count_kernel(const int32_t *__restrict__ codes, int n, int S, uint32_t *__restrict__ counts) {
    extern __shared__ uint32_t hist[];  // [S + 2]
    const int nb = S + 2;
    for (int b = threadIdx.x; b < nb; b += GROUP_CHUNK) hist[b] = 0;
    __syncthreads();
    const int i = blockIdx.x * GROUP_CHUNK + threadIdx.x;
    if (i < n) atomicAdd(&hist[group_bin(codes[i], S)], 1u);  // whole numbers: the order does not matter
    __syncthreads();
    for (int b = threadIdx.x; b < nb; b += GROUP_CHUNK) counts[(size_t)blockIdx.x * nb + b] = hist[b];
}

// Every block finds the first place of each bin and how many of the bin's rows lie before its own, and places its rows; nothing
// depends on timing.  Up to GROUP_SELF chunks it counts all rows itself; beyond, it adds up the counts of group_count_kernel, a
// wave per bin with a lane per chunk (a call with 64-column outputs, counting itself / adding up: 4096 rows 16 adapters 17.8 /
// 19.5 us, 256 adapters 20 / 34; 16 384 rows 31.3 / 29, 33 / 41; 32 768 rows 40 / 33, 41 / 44; 65 536 rows 59 / 42, 61 / 54).
// FEW_BINS: the waves' counts per bin lie side by side in LDS and one barrier ranks the rows of the block; with more bins the
// 16 waves take turns.  Inside a wave lanes of one bin find each other with one ballot per bit of the bin.
#define GROUP_SELF 16
#define GROUP_FEW_BINS 512  // (16 adapters with / without the waves' counts side by side: 2048 rows 16.5 / 17.3 us a call, 65 536 42.4 / 53.1)
struct GroupParams {
    const int32_t *codes;
    int n, S, bits, chunks;  // bits: of a bin's number
    uint32_t *counts;        // [chunks][S + 2] of group_count_kernel
    uint32_t *order;
    int32_t *scodes;
    uint32_t *seg_begin;
    PieceTable pieces;
};
// next: LDS, [S + 2] next free place of every bin, then [S + 2] its rows before this block's
template <bool FEW_BINS> __device__ __forceinline__ void group_place(const GroupParams &p, uint32_t *next) {
    constexpr int WAVES = GROUP_CHUNK / 64;
    const int32_t *__restrict__ codes = p.codes;
    const uint32_t *__restrict__ counts = p.counts;
    uint32_t *__restrict__ order = p.order, *__restrict__ seg_begin = p.seg_begin;
    int32_t *__restrict__ scodes = p.scodes;
    const PieceTable &pieces = p.pieces;
    const int n = p.n, S = p.S, bits = p.bits, chunks = p.chunks;
    __shared__ uint32_t wave_sum[WAVES];
    __shared__ uint16_t by_wave[FEW_BINS ? WAVES : 1][FEW_BINS ? GROUP_FEW_BINS : 1];
    const int nb = S + 2, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, me = blockIdx.x;
    uint32_t *before = next + nb;
    const int i = me * GROUP_CHUNK + tid;
    const int32_t code = i < n ? codes[i] : 0;
    const uint32_t bin = i < n ? group_bin(code, S) : 0;
    if (chunks <= GROUP_SELF) {
        for (int b = tid; b < 2 * nb; b += GROUP_CHUNK) next[b] = 0;
        __syncthreads();
        for (int k = 0; k < chunks; k++) {
            const int at = k * GROUP_CHUNK + tid;
            if (at < n) {
                const uint32_t q = k == me ? bin : group_bin(codes[at], S);
                atomicAdd(&next[q], 1u);  // whole numbers: the order does not matter
                if (k < me) atomicAdd(&before[q], 1u);
            }
        }
    } else if (FEW_BINS) {
        for (int b = wave; b < nb; b += WAVES) {
            const uint32_t v = lane < chunks ? counts[(size_t)lane * nb + b] : 0;  // at most 64 chunks
            uint32_t all = v, mine = lane < me ? v : 0;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) {
                all += __shfl_xor(all, o);
                mine += __shfl_xor(mine, o);
            }
            if (lane == 0) next[b] = all, before[b] = mine;
        }
    } else {
        for (int b = tid; b < nb; b += GROUP_CHUNK) {
            uint32_t all = 0, mine = 0;
            for (int k = 0; k < chunks; k++) {
                const uint32_t v = counts[(size_t)k * nb + b];
                all += v;
                mine += k < me ? v : 0u;
            }
            next[b] = all, before[b] = mine;
        }
    }
    if (FEW_BINS)
        for (int b = tid; b < WAVES * GROUP_FEW_BINS; b += GROUP_CHUNK) (&by_wave[0][0])[b] = 0;
    __syncthreads();
    // exclusive sum over the bins of a round of 1024, on top of what came before
    auto block_scan = [&](uint32_t v, uint32_t &carry) {
        uint32_t inc = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t u = __shfl_up(inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 63) wave_sum[wave] = inc;
        __syncthreads();
        uint32_t base = carry, all = 0;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            if (w < wave) base += wave_sum[w];
            all += wave_sum[w];
        }
        carry += all;
        __syncthreads();
        return base + inc - v;
    };
    uint32_t carry = 0, cut_carry = 0;
    for (int b0 = 0; b0 < nb; b0 += GROUP_CHUNK) {
        const int b = b0 + tid;
        const uint32_t total = b < nb ? next[b] : 0;
        const uint32_t start = block_scan(total, carry);
        if (b < nb) {
            next[b] = start + before[b];
            if (me == 0 && b >= 1) seg_begin[b - 1] = start;  // seg_begin[S] = end of the last adapter's rows
        }
        if (me == 0 && pieces.piece) {
            // pieces in the low half, slots for partial sums in the high half: fewer than 2^16 of each
            const bool is_adapter = b >= 1 && b <= S;
            const uint32_t np = is_adapter ? (total > 0 ? (total + pieces.rows - 1) / pieces.rows : 1) : 0;
            const uint32_t at = block_scan(np + (np > 1 ? np << 16 : 0), cut_carry);
            if (is_adapter) {
                pieces.slot[b - 1] = at >> 16;
                for (uint32_t k = 0; k < np; k++) {
                    const uint32_t lo = k * pieces.rows, hi = lo + pieces.rows < total ? lo + pieces.rows : total;
                    pieces.piece[(at & 0xFFFFu) + k] = Piece{b - 1, start + lo, start + hi, np > 1 ? (int32_t)((at >> 16) + k) : -1};
                }
            }
        }
    }
    if (me == 0 && tid == 0 && pieces.piece) *pieces.count = cut_carry & 0xFFFFu;
    uint64_t peers = __ballot(i < n);
    for (int bit = 0; bit < bits; bit++) {
        const bool one = (bin >> bit) & 1u;
        const uint64_t m = __ballot(one);
        peers &= one ? m : ~m;
    }
    const uint32_t rank = (uint32_t)__popcll(peers & ((1ull << lane) - 1ull)), here = (uint32_t)__popcll(peers);
    const bool highest = i < n && (peers >> lane) == 1ull;
    if (FEW_BINS) {
        if (highest) by_wave[wave][bin] = (uint16_t)here;
        __syncthreads();
        if (i < n) {
            uint32_t place = next[bin] + rank;
            for (int w = 0; w < wave; w++) place += by_wave[w][bin];
            order[place] = (uint32_t)i;
            scodes[place] = code;
        }
    } else {
        __syncthreads();  // the first places of the last round of bins are down
        for (int w = 0; w < WAVES; w++) {
            if (w == wave && i < n) {
                const uint32_t place = next[bin] + rank;
                order[place] = (uint32_t)i;
                scodes[place] = code;
            }
            __syncthreads();
            if (w == wave && highest) next[bin] += here;
            __syncthreads();
        }
    }
}

template <bool FEW_BINS> __global__ __launch_bounds__(GROUP_CHUNK) void group_place_kernel(GroupParams p) {
    extern __shared__ uint32_t lds[];
    group_place<FEW_BINS>(p, lds);
}

// ---------------------------------------------------------------------------------------------------------------
// u = A_c x
// ---------------------------------------------------------------------------------------------------------------
struct ShrinkParams {
    const void *x;
    int64_t ld_x;
    const void *a;  // [S][r] rows of K elements, pitch lda
    int64_t lda;
    const int32_t *codes;   // in the order of `order` when that is given, else by row
    const uint32_t *order;  // row numbers ordered by code, or NULL
    int n, K, r, rp, S;     // rp: r rounded up to 16
    float *hidden;          // [n][r] by row, or NULL
    void *u_hi, *u_lo;      // [n][rp] in the order of `order` (fp32: u_hi alone), or NULL
    float *factor;          // [n] likewise: what the tile product multiplies the low-rank sums by (0 without adapter)
    const float *scale;
};

// what the sums u of one row, spread over the lanes that hold them, become: the caller's fp32 copy, and the two 16-bit parts
// (fp32 weights: u itself) with the factor of their product.  `largest` = max |u| of the row; 4 ranks j .. j + 3 per call
template <int DT> __device__ __forceinline__ void shrink_store(const ShrinkParams &p, int64_t at, int j, const float *u, float largest, int32_t c) {
    typedef typename Elem<DT>::type E;
    const bool known = c >= 0 && c < p.S;
    if (p.hidden) {
        float *out = p.hidden + (p.order ? (int64_t)p.order[at] : at) * p.r;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (j + e < p.r) out[j + e] = c < p.S ? u[e] : __builtin_nanf("");
    }
    if (!p.u_hi || j >= p.rp) return;
    typedef E vec __attribute__((ext_vector_type(4)));
    // (within 64: the power times the scale must stay a number, and beyond 2^64 bf16 holds u as it is, fp16 has none)
    const int e2 = largest > 0.0f && largest < __builtin_inff() ? min(max(ilogbf(largest) + 1, -64), 64) : 0;
    vec hi, lo;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        // ranks past r: A's rows there are zeros, but zeros times an infinite element of x are NaN
        const float v = known && j + e < p.r ? (DT == HVS_F32 ? u[e] : ldexpf(u[e], -e2)) : 0.0f;
        hi[e] = learn_from_float<E>(v);
        const float rest = v - learn_to_float((E)hi[e]);
        lo[e] = learn_from_float<E>(largest < __builtin_inff() ? rest : 0.0f);  // inf - inf: the first part says it all
    }
    *reinterpret_cast<vec *>(reinterpret_cast<E *>(p.u_hi) + at * p.rp + j) = hi;
    if (DT != HVS_F32) *reinterpret_cast<vec *>(reinterpret_cast<E *>(p.u_lo) + at * p.rp + j) = lo;
    if (j == 0) p.factor[at] = known ? (DT == HVS_F32 ? p.scale[c] : ldexpf(p.scale[c], e2)) : 0.0f;
}

// One block per 16 rows (and per share blockIdx.y of the adapters among them): D[rank][row] on 16x16 matrix tiles, the
// block's waves split K and add up through LDS.  4096 rows of 1536 bf16, 256 adapters: 10 us for 25 MB, bound by the latency of
// two rounds of loads (waves wait 87 % of their time, the matrix pipe is busy 2 %); the other round's loads ahead, or both at
// once, cost registers and were slower (11.4 us).
template <int DT, int RT, bool ALIGNED>
__global__ __launch_bounds__(64 * SHRINK_WAVES) void shrink_kernel(ShrinkParams p) {
    typedef typename Elem<DT>::type E;
    constexpr int EPC = Elem<DT>::EPC, STEP = 4 * EPC;
    constexpr int UNROLL = RT == 1 ? 3 : (RT == 2 ? 2 : 1);
    __shared__ float part[SHRINK_WAVES][16][RT * 16 + 4];  // [wave][row][rank]
    __shared__ __attribute__((aligned(16))) char turn[SHRINK_WAVES][(1 + RT) * 1024];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m = lane & 15, g = lane >> 4;
    const bool valid = blockIdx.x * 16 + m < p.n;
    const int32_t code = valid ? p.codes[blockIdx.x * 16 + m] : -1;
    const int at = blockIdx.x * 16 + turn_row(lane), kx = at < p.n ? p.K : 0;
    const int row = at < p.n ? (p.order ? (int)p.order[at] : at) : 0;
    const E *x = reinterpret_cast<const E *>(p.x) + (int64_t)row * p.ld_x;
    uint32_t todo = (uint32_t)__ballot(valid) & 0xFFFFu;
    for (int ordinal = 0; todo; ordinal++) {
        const int32_t c = __builtin_amdgcn_readlane(code, __builtin_ctz(todo));
        const uint32_t members = (uint32_t)__ballot(valid && code == c) & 0xFFFFu;
        todo &= ~members;
        if (ordinal % (int)gridDim.y != (int)blockIdx.y) continue;
        f32x4 acc[RT];
#pragma unroll
        for (int q = 0; q < RT; q++) acc[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (c >= 0 && c < p.S) {
            const E *a = reinterpret_cast<const E *>(p.a) + (int64_t)c * p.r * p.lda;
            for (int k0 = wave * STEP; k0 < p.K; k0 += SHRINK_WAVES * STEP * UNROLL) {
                f32x4 fx[UNROLL], fa[UNROLL][RT];
#pragma unroll
                for (int s = 0; s < UNROLL; s++) {
                    const int k = k0 + s * SHRINK_WAVES * STEP + turn_k<DT>(lane);
                    fx[s] = load_chunk<DT, ALIGNED>(x, k, kx);
#pragma unroll
                    for (int q = 0; q < RT; q++) {
                        const int j = q * 16 + turn_row(lane);
                        fa[s][q] = load_chunk<DT, ALIGNED>(a + (int64_t)(j < p.r ? j : 0) * p.lda, k, j < p.r ? p.K : 0);
                    }
                }
#pragma unroll
                for (int s = 0; s < UNROLL; s++) {
                    turn_put(turn[wave], fx[s], lane);
#pragma unroll
                    for (int q = 0; q < RT; q++) turn_put(turn[wave] + (1 + q) * 1024, fa[s][q], lane);
                    const f32x4 bx = turn_get(turn[wave], lane);
#pragma unroll
                    for (int q = 0; q < RT; q++) acc[q] = mfma_chunk<DT>(turn_get(turn[wave] + (1 + q) * 1024, lane), bx, acc[q]);
                }
            }
        }
#pragma unroll
        for (int q = 0; q < RT; q++)
#pragma unroll
            for (int e = 0; e < 4; e++) part[wave][m][q * 16 + 4 * g + e] = acc[q][e];
        __syncthreads();
        // 4 RT lanes of one wave per row, 4 ranks each: the waves' sums in wave order
        if (tid < 64 * RT) {
            const int mm = tid / (4 * RT), j = tid % (4 * RT) * 4;
            float u[4] = {0.0f, 0.0f, 0.0f, 0.0f}, mx = 0.0f;
#pragma unroll
            for (int w = 0; w < SHRINK_WAVES; w++)
#pragma unroll
                for (int e = 0; e < 4; e++) u[e] += part[w][mm][j + e];
#pragma unroll
            for (int e = 0; e < 4; e++) mx = fmaxf(mx, fabsf(u[e]));
#pragma unroll
            for (int o = 2 * RT; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
            if (members >> mm & 1) shrink_store<DT>(p, (int64_t)blockIdx.x * 16 + mm, j, u, mx, c);
        }
        __syncthreads();
    }
}

// Many rows: a wave takes 32 rows and all of K, so that nothing is added up across waves and an adapter is read once per 32
// rows of it.  Bound by reading x.
template <int DT, int RT, bool ALIGNED> __global__ __launch_bounds__(256) void shrink_wide_kernel(ShrinkParams p) {
    typedef typename Elem<DT>::type E;
    constexpr int EPC = Elem<DT>::EPC, STEP = 4 * EPC;
    __shared__ __attribute__((aligned(16))) char turns[4][(2 + RT) * 1024];
    char *turn = turns[threadIdx.x >> 6];
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int row0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 32;
    const bool valid = lane < 32 && row0 + lane < p.n;
    const int32_t code = valid ? p.codes[row0 + lane] : -1;
    const E *x[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int at = row0 + t * 16 + turn_row(lane);
        x[t] = reinterpret_cast<const E *>(p.x) + (int64_t)p.order[at < p.n ? at : p.n - 1] * p.ld_x;
    }
    uint32_t todo = (uint32_t)__ballot(valid);
    while (todo) {
        const int32_t c = __builtin_amdgcn_readlane(code, __builtin_ctz(todo));
        const uint32_t members = (uint32_t)__ballot(valid && code == c);
        todo &= ~members;
        f32x4 acc[2][RT];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int q = 0; q < RT; q++) acc[t][q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (c >= 0 && c < p.S) {
            const E *a = reinterpret_cast<const E *>(p.a) + (int64_t)c * p.r * p.lda;
            constexpr int UNROLL = RT == 1 ? 6 : (RT == 2 ? 4 : (RT == 4 ? 2 : 1));
            for (int k0 = 0; k0 < p.K; k0 += STEP * UNROLL) {
                f32x4 fx[UNROLL][2], fa[UNROLL][RT];
#pragma unroll
                for (int s = 0; s < UNROLL; s++) {
                    const int k = k0 + s * STEP + turn_k<DT>(lane);
#pragma unroll
                    for (int q = 0; q < RT; q++) {
                        const int j = q * 16 + turn_row(lane);
                        fa[s][q] = load_chunk<DT, ALIGNED>(a + (int64_t)(j < p.r ? j : 0) * p.lda, k, j < p.r ? p.K : 0);
                    }
#pragma unroll
                    for (int t = 0; t < 2; t++) fx[s][t] = load_chunk<DT, ALIGNED>(x[t], k, members >> (16 * t) & 0xFFFFu ? p.K : 0);
                }
#pragma unroll
                for (int s = 0; s < UNROLL; s++) {
#pragma unroll
                    for (int t = 0; t < 2; t++) turn_put(turn + t * 1024, fx[s][t], lane);
#pragma unroll
                    for (int q = 0; q < RT; q++) turn_put(turn + (2 + q) * 1024, fa[s][q], lane);
                    const f32x4 b0 = turn_get(turn, lane), b1 = turn_get(turn + 1024, lane);
#pragma unroll
                    for (int q = 0; q < RT; q++) {
                        const f32x4 aq = turn_get(turn + (2 + q) * 1024, lane);
                        acc[0][q] = mfma_chunk<DT>(aq, b0, acc[0][q]);
                        acc[1][q] = mfma_chunk<DT>(aq, b1, acc[1][q]);
                    }
                }
            }
        }
        // lane (m, g): ranks q 16 + 4 g .. + 3 of row m
#pragma unroll
        for (int t = 0; t < 2; t++) {
            float mx = 0.0f;
#pragma unroll
            for (int q = 0; q < RT; q++)
#pragma unroll
                for (int e = 0; e < 4; e++) mx = fmaxf(mx, fabsf(acc[t][q][e]));
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            if (members >> (16 * t + m) & 1) {
#pragma unroll
                for (int q = 0; q < RT; q++) {
                    const float u[4] = {acc[t][q][0], acc[t][q][1], acc[t][q][2], acc[t][q][3]};
                    shrink_store<DT>(p, row0 + t * 16 + m, q * 16 + 4 * g, u, mx, c);
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------
// few rows: y = W x + s B u
// ---------------------------------------------------------------------------------------------------------------
struct ProjectParams {
    const void *x;
    int64_t ld_x;
    const void *w;  // [N] rows of K elements, pitch ldw
    int64_t ldw;
    const void *b;  // [S][N] rows of r elements, pitch ldb
    int64_t ldb;
    const float *scale;
    const int32_t *codes;   // few rows: by row; many rows: in the order of `order`
    const uint32_t *order;
    const float *hidden;    // few rows: [n][r]
    const void *u_hi, *u_lo;
    const float *factor;
    void *out;
    int64_t ld_out;
    int n, K, N, r, rp, S;
    int b_aligned;   // rows of b start on 16 bytes and r is a whole number of chunks
    int out_vec;     // rows of out start on 16 bytes
};

// One block per 16 MT columns and 16 NT rows of y: the block's waves split K, W and x fragments go straight from memory to
// registers, the partial sums meet in LDS, and every thread adds the low-rank term of its outputs.  The loads of the first
// round are on their way while the low-rank terms are worked out; with 16 waves that round is all of K at 1536 columns.
template <int DT, int MT, int NT, int WAVES, bool ALIGNED>
__global__ __launch_bounds__(64 * WAVES, 4) void project_few_kernel(ProjectParams p) {
    typedef typename Elem<DT>::type E;
    constexpr int EPC = Elem<DT>::EPC, STEP = 4 * EPC, UNROLL = MT + NT <= 2 ? 6 : (MT + NT <= 4 ? 4 : 3), THREADS = 64 * WAVES;
    constexpr int OUTS = (MT * NT * 256 + THREADS - 1) / THREADS;
    // [wave][row][column] partial sums at the end; before, the waves' room to turn fragments
    constexpr int PART = WAVES * NT * 16 * (MT * 16 + 1) * 4, TURN = WAVES * (MT + NT) * 1024;
    __shared__ __attribute__((aligned(16))) char room[PART > TURN ? PART : TURN];
    float (*part)[NT * 16][MT * 16 + 1] = reinterpret_cast<float (*)[NT * 16][MT * 16 + 1]>(room);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m = lane & 15, g = lane >> 4;
    // blocks of one XCD (dispatched round robin) take neighbouring columns for all rows: its L2 holds their rows of W and sees
    // x once per few columns.  In launch order every XCD would stream all of W for every 16 NT rows
    const int row_blocks = (p.n + 16 * NT - 1) / (16 * NT), blocks = gridDim.x, xcd = blockIdx.x & 7, q8 = blocks >> 3, rem = blocks & 7;
    const int at = xcd * q8 + (xcd < rem ? xcd : rem) + (blockIdx.x >> 3);
    const int col0 = at / row_blocks * (16 * MT), row0 = at % row_blocks * (16 * NT);
    const E *w[MT], *x[NT];
    int kw[MT], kx[NT];  // K, or 0 for rows that are not there
#pragma unroll
    for (int t = 0; t < MT; t++) {
        const int col = col0 + t * 16 + turn_row(lane);
        kw[t] = col < p.N ? p.K : 0;
        w[t] = reinterpret_cast<const E *>(p.w) + (int64_t)(col < p.N ? col : 0) * p.ldw;
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int row = row0 + t * 16 + turn_row(lane);
        kx[t] = row < p.n ? p.K : 0;
        x[t] = reinterpret_cast<const E *>(p.x) + (int64_t)(row < p.n ? row : 0) * p.ld_x;
    }
    f32x4 acc[MT][NT], fw[UNROLL][MT], fx[UNROLL][NT];
#pragma unroll
    for (int a = 0; a < MT; a++)
#pragma unroll
        for (int t = 0; t < NT; t++) acc[a][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto load = [&](int k0) {
#pragma unroll
        for (int s = 0; s < UNROLL; s++) {
            const int k = k0 + s * WAVES * STEP + turn_k<DT>(lane);
#pragma unroll
            for (int t = 0; t < MT; t++) fw[s][t] = load_chunk<DT, ALIGNED>(w[t], k, kw[t]);
#pragma unroll
            for (int t = 0; t < NT; t++) fx[s][t] = load_chunk<DT, ALIGNED>(x[t], k, kx[t]);
        }
    };
    load(wave * STEP);
    float low[OUTS];
#pragma unroll
    for (int o = 0; o < OUTS; o++) {
        const int q = tid + o * THREADS, row = row0 + q / (16 * MT), col = col0 + q % (16 * MT);
        low[o] = 0.0f;
        if (q >= MT * NT * 256 || row >= p.n || col >= p.N) continue;
        const int32_t c = p.codes[row];
        if (c >= p.S) low[o] = __builtin_nanf("");
        else if (c >= 0) {
            const E *b = reinterpret_cast<const E *>(p.b) + ((int64_t)c * p.N + col) * p.ldb;
            const float *u = p.hidden + (int64_t)row * p.r;
            float sum = 0.0f;
            for (int j0 = 0; j0 < p.r; j0 += 16) {  // 16 ranks: their loads go out together
                f32x4 fb[16 / EPC], fu[4];
#pragma unroll
                for (int i = 0; i < 16 / EPC; i++) fb[i] = load_chunk<DT, false>(b, j0 + i * EPC, p.r);
#pragma unroll
                for (int i = 0; i < 4; i++) fu[i] = load_chunk<HVS_F32, false>(u, j0 + 4 * i, p.r);
#pragma unroll
                for (int i = 0; i < 16 / EPC; i++) {
                    float v[EPC];
                    chunk_to_float<DT>(fb[i], v);
#pragma unroll
                    for (int e = 0; e < EPC; e++) sum = fmaf(v[e], fu[(i * EPC + e) / 4][(i * EPC + e) % 4], sum);
                }
            }
            low[o] = p.scale[c] * sum;
        }
    }
    char *turn = room + wave * (MT + NT) * 1024;
    for (int k0 = wave * STEP;;) {
#pragma unroll
        for (int s = 0; s < UNROLL; s++) {
#pragma unroll
            for (int t = 0; t < MT; t++) turn_put(turn + t * 1024, fw[s][t], lane);
#pragma unroll
            for (int t = 0; t < NT; t++) turn_put(turn + (MT + t) * 1024, fx[s][t], lane);
            f32x4 aw[MT], bx[NT];
#pragma unroll
            for (int a = 0; a < MT; a++) aw[a] = turn_get(turn + a * 1024, lane);
#pragma unroll
            for (int t = 0; t < NT; t++) bx[t] = turn_get(turn + (MT + t) * 1024, lane);
            if (DT == HVS_F32) {  // the sums take turns: a product does not wait for the one before it
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int a = 0; a < MT; a++)
#pragma unroll
                        for (int t = 0; t < NT; t++) acc[a][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(aw[a][j], bx[t][j], acc[a][t], 0, 0, 0);
            } else {
#pragma unroll
                for (int a = 0; a < MT; a++)
#pragma unroll
                    for (int t = 0; t < NT; t++) acc[a][t] = mfma_chunk<DT>(aw[a], bx[t], acc[a][t]);
            }
        }
        k0 += WAVES * STEP * UNROLL;
        if (k0 >= p.K) break;
        load(k0);
    }
    __syncthreads();  // every wave is done turning
#pragma unroll
    for (int a = 0; a < MT; a++)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) part[wave][t * 16 + m][a * 16 + 4 * g + e] = acc[a][t][e];
    __syncthreads();
#pragma unroll
    for (int o = 0; o < OUTS; o++) {
        const int q = tid + o * THREADS, r = q / (16 * MT), row = row0 + r, col = col0 + q % (16 * MT);
        if (q >= MT * NT * 256 || row >= p.n || col >= p.N) continue;
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < WAVES; k++) s += part[k][r][q % (16 * MT)];
        reinterpret_cast<E *>(p.out)[(int64_t)row * p.ld_out + col] = learn_from_float<E>(s + low[o]);
    }
}

// A handful of rows in one launch: every block works out u = A x itself, beside its 16 columns of W x.  Rows of one tenant
// (the variants of one question) read one adapter: 16 more rows next to a block's 16 rows of W, against a second launch that
// costs more.  The 16 waves split K (8 in the launch of u alone: other sums, so the last bits may differ from it) and join
// through LDS, first u, then y.  1536 columns are one round of loads in 16 bits, two in fp32; they start when the codes, which
// name the adapter, have arrived.  One row of 1536 in fp32: 8.3 us for 9.65 MB, a chain of those latencies on the 96 CUs that
// have a block (waves wait 85 % of their time, the matrix pipe is busy 34 %).
template <int DT, int RT, bool ALIGNED>
__global__ __launch_bounds__(1024) void project_once_kernel(ProjectParams p, float *__restrict__ hidden, const void *a_stack, int64_t lda) {
    typedef typename Elem<DT>::type E;
    constexpr int EPC = Elem<DT>::EPC, STEP = 4 * EPC, WAVES = 16, UNROLL = RT == 1 ? 3 : (RT == 2 ? 2 : 1);
    __shared__ float part[WAVES][ONCE_ROWS][17];
    __shared__ float part_u[WAVES][ONCE_ROWS][RT * 16 + 4];
    __shared__ float u_all[ONCE_ROWS][RT * 16];
    __shared__ __attribute__((aligned(16))) char turns[WAVES][(2 + RT) * 1024];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m = lane & 15, g = lane >> 4;
    const int col0 = blockIdx.x * 16;
    const int tr = turn_row(lane), kw = col0 + tr < p.N ? p.K : 0, kx = tr < p.n ? p.K : 0;
    const E *w = reinterpret_cast<const E *>(p.w) + (int64_t)(kw ? col0 + tr : 0) * p.ldw;
    const E *x = reinterpret_cast<const E *>(p.x) + (int64_t)(kx ? tr : 0) * p.ld_x;
    char *turn = turns[wave];
    const int32_t code = lane < p.n ? p.codes[lane] : -1;
    // this thread's output, and its row of B as far as the first ranks go
    const int out_row = tid >> 4, out_col = col0 + (tid & 15);
    const bool out_ok = out_row < p.n && out_col < p.N;
    const int32_t out_code = out_ok ? p.codes[out_row] : -1;
    const bool out_known = out_code >= 0 && out_code < p.S;
    const E *b = reinterpret_cast<const E *>(p.b) + ((int64_t)(out_known ? out_code : 0) * p.N + (out_known ? out_col : 0)) * p.ldb;
    f32x4 fb[RT * 16 / EPC];
#pragma unroll
    for (int i = 0; i < RT * 16 / EPC; i++) fb[i] = load_chunk<DT, false>(b, i * EPC, out_known ? p.r : 0);
    const float out_scale = out_known ? p.scale[out_code] : 0.0f;

    uint32_t todo = (uint32_t)__ballot(code >= 0 && code < p.S);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (bool first = true; first || todo; first = false) {
        const int32_t c = todo ? __builtin_amdgcn_readlane(code, __builtin_ctz(todo)) : 0;
        const uint32_t members = todo ? (uint32_t)__ballot(code == c) : 0;
        todo &= ~members;
        const E *a = reinterpret_cast<const E *>(a_stack) + (int64_t)c * p.r * lda;
        const int ka = members ? p.K : 0;
        f32x4 acc_u[RT];
#pragma unroll
        for (int q = 0; q < RT; q++) acc_u[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int k0 = wave * STEP; k0 < p.K; k0 += WAVES * STEP * UNROLL) {
            f32x4 fw[UNROLL], fx[UNROLL], fa[UNROLL][RT];
#pragma unroll
            for (int s = 0; s < UNROLL; s++) {
                const int k = k0 + s * WAVES * STEP + turn_k<DT>(lane);
                fw[s] = load_chunk<DT, ALIGNED>(w, k, first ? kw : 0);
                fx[s] = load_chunk<DT, ALIGNED>(x, k, kx);
#pragma unroll
                for (int q = 0; q < RT; q++) {
                    const int j = q * 16 + tr;
                    fa[s][q] = load_chunk<DT, ALIGNED>(a + (int64_t)(j < p.r ? j : 0) * lda, k, j < p.r ? ka : 0);
                }
            }
#pragma unroll
            for (int s = 0; s < UNROLL; s++) {
                turn_put(turn, fx[s], lane);
                if (first) turn_put(turn + 1024, fw[s], lane);
#pragma unroll
                for (int q = 0; q < RT; q++) turn_put(turn + (2 + q) * 1024, fa[s][q], lane);
                const f32x4 bx = turn_get(turn, lane);
                if (first) acc = mfma_chunk<DT>(turn_get(turn + 1024, lane), bx, acc);
#pragma unroll
                for (int q = 0; q < RT; q++) acc_u[q] = mfma_chunk<DT>(turn_get(turn + (2 + q) * 1024, lane), bx, acc_u[q]);
            }
        }
        if (m < ONCE_ROWS) {
            if (first)
#pragma unroll
                for (int e = 0; e < 4; e++) part[wave][m][4 * g + e] = acc[e];
#pragma unroll
            for (int q = 0; q < RT; q++)
#pragma unroll
                for (int e = 0; e < 4; e++) part_u[wave][m][q * 16 + 4 * g + e] = acc_u[q][e];
        }
        __syncthreads();
        if (tid < ONCE_ROWS * RT * 16) {
            const int row = tid / (RT * 16), j = tid % (RT * 16);
            if (members >> row & 1) {
                float s = 0.0f;
#pragma unroll
                for (int k = 0; k < WAVES; k++) s += part_u[k][row][j];
                u_all[row][j] = j < p.r ? s : 0.0f;  // ranks past r: 0 times an infinite element of x is NaN
                if (hidden && blockIdx.x == 0 && j < p.r) hidden[(int64_t)row * p.r + j] = s;
            }
        }
        __syncthreads();
    }
    if (hidden && blockIdx.x == 0 && tid < p.n * p.r) {  // rows without an adapter, and codes past the last one
        const int32_t c = p.codes[tid / p.r];
        if (c < 0 || c >= p.S) hidden[tid] = c < 0 ? 0.0f : __builtin_nanf("");
    }
    if (!out_ok) return;
    float low = 0.0f;
    if (out_known) {
#pragma unroll
        for (int i = 0; i < RT * 16 / EPC; i++) {
            float v[EPC];
            chunk_to_float<DT>(fb[i], v);
#pragma unroll
            for (int e = 0; e < EPC; e++) low = fmaf(v[e], u_all[out_row][i * EPC + e], low);
        }
        low *= out_scale;
    }
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < WAVES; k++) s += part[k][out_row][tid & 15];
    s = out_code >= p.S ? __builtin_nanf("") : s + low;
    reinterpret_cast<E *>(p.out)[(int64_t)out_row * p.ld_out + out_col] = learn_from_float<E>(s);
}

// ---------------------------------------------------------------------------------------------------------------
// many rows: the tile product
// ---------------------------------------------------------------------------------------------------------------
// Offsets of a tile's 16-byte chunks for the LDS-DMA: tile row t is row rows[t] of the matrix (order == NULL: row0 + t).
// Tile rows past the end re-read the last one.  `base` must be wave-uniform and every offset below 2^31.
template <class T>
__device__ __forceinline__ void adapter_src_init(TileSrcT<T::DMA_N> &t, const void *base, const uint32_t *order, int row0, int n_rows, int64_t pitch_bytes,
                                                 int64_t num_bytes, int tid) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)base);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)base >> 32));
    const int bytes = __builtin_amdgcn_readfirstlane((int)num_bytes);
    t.rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)(((uintptr_t)hi << 32) | lo), 0, bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < T::DMA_N; i++) {
        const int P = T::GT * i + tid;
        const int slot = P >> 3, kc = (P & 7) ^ lds_swz(slot);
        int row = row0 + slot;
        row = row < n_rows ? row : n_rows - 1;
        if (order) row = (int)order[row];
        t.voff[i] = (int)(row * pitch_bytes) + kc * 16;
    }
}
// The last k-step of rows that end inside its 128 bytes: chunks past the row's end are sent past the buffer's end, where
// loads return 0 (they would otherwise read the next row).
template <class T> __device__ __forceinline__ void adapter_src_tail(TileSrcT<T::DMA_N> &t, int chunks_left, int tid) {
#pragma unroll
    for (int i = 0; i < T::DMA_N; i++) {
        const int P = T::GT * i + tid;
        const int kc = (P & 7) ^ lds_swz(P >> 3);
        if (kc >= chunks_left) t.voff[i] = 0x7FFFFFFF - 15;
    }
}

// swaps the upper half of a with the lower half of b: a keeps its lower lanes and gets b's lower lanes above them, b gets a's
// upper lanes below its own
__device__ __forceinline__ void swap_halves(uint32_t &a, uint32_t &b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

// A block walks a range of tiles, columns first, and fetches the first k-step of the next tile while it finishes the last
// one, so that only the block's first tile waits for memory before it can start.
template <int DT, class T>
__global__ __launch_bounds__(T::GT, 2) void project_tile_kernel(ProjectParams p) {
#if defined(__HIP_DEVICE_COMPILE__)  // device-only types (buffer descriptors) inside
    typedef typename Elem<DT>::type E;
    constexpr int EPC = Elem<DT>::EPC, MT = T::MT, NT = T::NT;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / T::WN, wn = wave % T::WN;
    const int l32 = lane & 31, h = lane >> 5;
    // blocks of one XCD (dispatched round robin) take consecutive ranges: they share rows of x and all of W
    const int CT = (p.N + T::BM - 1) / T::BM, tiles = CT * ((p.n + T::BN - 1) / T::BN);
    const int blocks = gridDim.x, xcd = blockIdx.x & 7, q8 = blocks >> 3, rem = blocks & 7;
    const int at = xcd * q8 + (xcd < rem ? xcd : rem) + (blockIdx.x >> 3);
    const int tile_lo = (int)((int64_t)tiles * at / blocks), tile_hi = (int)((int64_t)tiles * (at + 1) / blocks);
    if (tile_lo >= tile_hi) return;

    TileSrcT<T::DMA_N> srcA, srcB;
    const int k_bytes = p.K * (int)sizeof(E);
    const int nks = (k_bytes + KB - 1) / KB, tail = (k_bytes % KB) / 16;
    auto init_src = [&](int tile) {
        const int rt = tile / CT, col0 = (tile - rt * CT) * T::BM;
        const int cols = p.N - col0, last = cols < T::BM ? cols : T::BM;
        const char *wbase = reinterpret_cast<const char *>(p.w) + (int64_t)col0 * p.ldw * sizeof(E);
        adapter_src_init<T>(srcA, wbase, nullptr, 0, last, p.ldw * sizeof(E), (int64_t)(last - 1) * p.ldw * sizeof(E) + k_bytes, tid);
        adapter_src_init<T>(srcB, p.x, p.order, rt * T::BN, p.n, p.ld_x * sizeof(E), (int64_t)(p.n - 1) * p.ld_x * sizeof(E) + k_bytes, tid);
    };
    auto before_step = [&](int ks) {  // the sources of step ks are about to be used
        if (tail && ks == nks - 1) {
            adapter_src_tail<T>(srcA, tail, tid);
            adapter_src_tail<T>(srcB, tail, tid);
        }
    };
    init_src(tile_lo);
    before_step(0);
    dma_tiles<T>(srcA, srcB, smem, koff_plain(0), wave);
    __syncthreads();

    int cur = 0;
    for (int tile = tile_lo; tile < tile_hi; tile++) {
        const int rt = tile / CT;
        const int wcol = (tile - rt * CT) * T::BM + wm * (MT * 32), wrow = rt * T::BN + wn * (NT * 32);
        int32_t codes[NT];
        float factor[NT];
        uint32_t out_row[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {  // wanted after the product: on their way during it
            const int j = wrow + nt * 32 + l32;
            codes[nt] = j < p.n ? p.codes[j] : -1;
            factor[nt] = j < p.n ? p.factor[j] : 0.0f;
            out_row[nt] = j < p.n ? p.order[j] : 0;
        }
        f32x16 acc[MT][NT];
        zero_acc(acc);
        for (int ks = 0; ks + 1 < nks; ks++) {
            before_step(ks + 1);
            compute_step<DT, T>(acc, smem + cur * T::STAGE_BYTES, wm, wn, lane, srcA, srcB, smem + (cur ^ 1) * T::STAGE_BYTES, koff_plain(ks + 1), wave);
            __syncthreads();
            cur ^= 1;
        }
        // the last step fetches the next tile's first one (after the last tile: its own again, which nothing reads)
        init_src(tile + 1 < tile_hi ? tile + 1 : tile);
        before_step(0);
        compute_step<DT, T>(acc, smem + cur * T::STAGE_BYTES, wm, wn, lane, srcA, srcB, smem + (cur ^ 1) * T::STAGE_BYTES, koff_plain(0), wave);
        cur ^= 1;

        // low-rank term, adapter by adapter, in sums of its own that only the rows of the adapter take over: a weight that is
        // not finite stays with its tenant.  KC matrix steps of ranks at a time, GROUPS row groups together: their u fragments
        // serve every adapter among the rows, an adapter's fragments of b serve all its rows, and with registers to spare
        // the next adapter's are on their way meanwhile
        constexpr int KC = 2, GROUPS = MT <= 2 ? NT : 1;
#pragma unroll
        for (int n0 = 0; n0 < NT; n0 += GROUPS)
            for (int k0 = 0; k0 < p.rp; k0 += KC * 2 * EPC) {
                f32x4 ub[GROUPS][KC], ul[GROUPS][KC];
                uint32_t todo[GROUPS];
#pragma unroll
                for (int t = 0; t < GROUPS; t++) {
                    const int32_t code = codes[n0 + t];
                    const bool use = code >= 0 && code < p.S;
                    todo[t] = (uint32_t)__ballot(use);
                    const int64_t u_row = (int64_t)(wrow + (n0 + t) * 32 + l32) * p.rp;
#pragma unroll
                    for (int s = 0; s < KC; s++) {
                        const int k = k0 + s * 2 * EPC + h * EPC;
                        ub[t][s] = ul[t][s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                        if (use && k < p.rp) {
                            ub[t][s] = *reinterpret_cast<const f32x4 *>(reinterpret_cast<const E *>(p.u_hi) + u_row + k);
                            if (DT != HVS_F32) ul[t][s] = *reinterpret_cast<const f32x4 *>(reinterpret_cast<const E *>(p.u_lo) + u_row + k);
                        }
                    }
                }
                auto take = [&]() {  // the next adapter among the rows, -1 when there is none
                    int32_t c = -1;
#pragma unroll
                    for (int t = GROUPS - 1; t >= 0; t--)
                        if (todo[t]) c = __builtin_amdgcn_readlane(codes[n0 + t], __builtin_ctz(todo[t]));
#pragma unroll
                    for (int t = 0; t < GROUPS; t++)
                        if (c >= 0) todo[t] &= ~(uint32_t)__ballot(codes[n0 + t] == c);
                    return c;
                };
                auto fetch = [&](int32_t c, f32x4 (&fb)[MT][KC]) {
                    const E *b = reinterpret_cast<const E *>(p.b) + (int64_t)c * p.N * p.ldb;
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        const int col = wcol + mt * 32 + l32;
                        const E *brow = b + (int64_t)(col < p.N ? col : 0) * p.ldb;
#pragma unroll
                        for (int s = 0; s < KC; s++) {
                            const int k = k0 + s * 2 * EPC + h * EPC, r_here = col < p.N ? p.r : 0;
                            fb[mt][s] = p.b_aligned ? load_chunk<DT, true>(brow, k, r_here) : load_chunk<DT, false>(brow, k, r_here);
                        }
                    }
                };
                f32x4 fb[MT][KC], fb_next[GROUPS > 1 ? MT : 1][KC];
                int32_t c = take();
                if (c >= 0) fetch(c, fb);
                while (c >= 0) {
                    const int32_t next = take();
                    if constexpr (GROUPS > 1)
                        if (next >= 0) fetch(next, fb_next);
#pragma unroll
                    for (int t = 0; t < GROUPS; t++) {
                        const bool mine = codes[n0 + t] == c;
                        if (!__ballot(mine)) continue;
                        const float f = factor[n0 + t];
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            f32x16 low;
#pragma unroll
                            for (int e = 0; e < 16; e++) low[e] = 0.0f;
#pragma unroll
                            for (int s = 0; s < KC; s++) {
                                if (DT == HVS_F32) {
#pragma unroll
                                    for (int e = 0; e < 4; e++) low = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[mt][s][e], ub[t][s][e], low, 0, 0, 0);
                                } else {
                                    low = mfma16<DT>(fb[mt][s], ub[t][s], low);
                                    low = mfma16<DT>(fb[mt][s], ul[t][s], low);
                                }
                            }
#pragma unroll
                            for (int e = 0; e < 16; e++) acc[mt][n0 + t][e] = mine ? fmaf(f, low[e], acc[mt][n0 + t][e]) : acc[mt][n0 + t][e];
                        }
                    }
                    c = next;
                    if constexpr (GROUPS > 1) {
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
#pragma unroll
                            for (int s = 0; s < KC; s++) fb[mt][s] = fb_next[mt][s];
                    } else if (c >= 0) fetch(c, fb);
                }
            }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int j = wrow + nt * 32 + l32;
            const bool valid = j < p.n;
            const int32_t code = codes[nt];
            const bool lost = valid && code >= p.S;  // a code past the last adapter
            E *out = reinterpret_cast<E *>(p.out) + (int64_t)out_row[nt] * p.ld_out;
            // accumulator element e of lane (l32, h): column 8 (e / 4) + 4 h + e % 4 of its 32, row l32
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                E v[16];
#pragma unroll
                for (int e = 0; e < 16; e++) v[e] = learn_from_float<E>(lost ? __builtin_nanf("") : acc[mt][nt][e]);
                if (DT != HVS_F32 && p.out_vec && wcol + mt * 32 + 32 <= p.N) {
                    // the two halves trade quarters, so that a lane holds 8 columns in a row: 16-byte stores
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) w[i] = __builtin_bit_cast(uint32_t, *reinterpret_cast<uint32_t *>(v + 2 * i));
#pragma unroll
                    for (int i = 0; i < 8; i += 4) {
                        swap_halves(w[i], w[i + 2]);
                        swap_halves(w[i + 1], w[i + 3]);
                        typedef uint32_t vec __attribute__((ext_vector_type(4)));
                        if (valid) *reinterpret_cast<vec *>(out + wcol + mt * 32 + i * 4 + h * 8) = vec{w[i], w[i + 1], w[i + 2], w[i + 3]};
                    }
                } else {
#pragma unroll
                    for (int e4 = 0; e4 < 4; e4++) {
                        const int col = wcol + mt * 32 + 8 * e4 + 4 * h;
                        typedef E vec __attribute__((ext_vector_type(4)));
                        if (valid && p.out_vec && col + 3 < p.N) *reinterpret_cast<vec *>(out + col) = vec{v[4 * e4], v[4 * e4 + 1], v[4 * e4 + 2], v[4 * e4 + 3]};
                        else if (valid) {
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (col + e < p.N) out[col + e] = v[4 * e4 + e];
                        }
                    }
                }
            }
        }
        __syncthreads();  // the next tile's first step has landed for every wave
    }
#endif
}

// ---------------------------------------------------------------------------------------------------------------
// layout: rows brought to 16-byte pitch, transposed weights for the backward pass
// ---------------------------------------------------------------------------------------------------------------
template <typename E>
__global__ __launch_bounds__(256) void pack_rows_kernel(const E *__restrict__ src, int64_t ld, int n, int K, int Kp, E *__restrict__ dst) {
    const int64_t total = (int64_t)n * Kp;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / Kp;
        const int k = (int)(i - r * Kp);
        dst[i] = k < K ? src[r * ld + k] : (E)0.0f;
    }
}

// dst[z][c][r] = src[z][r][c] for `count` matrices of R x C; dst rows have pitch ld (>= R), filled with zeros past R
// tiles of 2^12, 2^13, 2^14 elements: 96 rows of fp32 weights 768 x 768 5.2, 6.1, 7.8 us; 8192 rows, bf16 1536 x 1536 14.9, 12.0, 12.6
#define TILE_LOG 13
#define TILE_LOG_NARROW 4
struct TransposeJob {
    const void *src;
    void *dst;
    int R, C, ld, tiles_c, tiles_r, log_c;  // tiles of 2^TILE_LOG elements, 2^log_c columns wide: narrow matrices get narrow tiles
    int64_t blocks;                         // tiles_c tiles_r count
};
struct TransposeJobs {
    TransposeJob job[3];
};
// All transposed weights of a backward pass in one launch, a block per tile, jobs one after the other; the first group_blocks
// blocks group the rows meanwhile, where they count them by themselves (a launch of its own took 4 us more at 96 rows).
// first: the launch's first tile (a grid dimension ends below 2^32 threads: LAYOUT_TILES tiles a launch, 2^31 elements).
#define LAYOUT_TILES (1ll << 18)
template <typename E> __global__ __launch_bounds__(GROUP_CHUNK) void layout_kernel(TransposeJobs jobs, int64_t first, GroupParams group, int group_blocks) {
    extern __shared__ uint32_t lds[];
    if ((int)blockIdx.x < group_blocks) {
        group_place<true>(group, lds);
        return;
    }
    E *tile = reinterpret_cast<E *>(lds);  // rows of 2^log_c + 1 elements
    constexpr int PER = (1 << TILE_LOG) / GROUP_CHUNK;
    int64_t at = first + blockIdx.x - group_blocks;
    int which = 0;
    while (which < 2 && at >= jobs.job[which].blocks) at -= jobs.job[which++].blocks;
    const TransposeJob &t = jobs.job[which];
    const int64_t z = at / (t.tiles_c * t.tiles_r);
    const int rest = (int)(at - z * (t.tiles_c * t.tiles_r));
    const int log_c = t.log_c, log_r = TILE_LOG - log_c, pitch = (1 << log_c) + 1;
    const E *s = reinterpret_cast<const E *>(t.src) + z * (int64_t)t.R * t.C;
    E *d = reinterpret_cast<E *>(t.dst) + z * (int64_t)t.C * t.ld;
    const int r0 = rest / t.tiles_c << log_r, c0 = rest % t.tiles_c << log_c;
    E v[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int i = threadIdx.x + GROUP_CHUNK * k, r = r0 + (i >> log_c), c = c0 + (i & ((1 << log_c) - 1));
        v[k] = r < t.R && c < t.C ? s[(int64_t)r * t.C + c] : (E)0.0f;
    }
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int i = threadIdx.x + GROUP_CHUNK * k;
        tile[(i >> log_c) * pitch + (i & ((1 << log_c) - 1))] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int i = threadIdx.x + GROUP_CHUNK * k, c = i >> log_r, r = i & ((1 << log_r) - 1);
        if (c0 + c < t.C && r0 + r < t.ld) d[(int64_t)(c0 + c) * t.ld + r0 + r] = tile[r * pitch + c];
    }
}

// ---------------------------------------------------------------------------------------------------------------
// gradients of the stacks: G_c[j][col] = s_c sum over the rows of adapter c of q[row][j] X[row][col]
// ---------------------------------------------------------------------------------------------------------------
struct OuterProblem {
    const float *q;  // [n][r] by row
    const void *x;   // [n][d], pitch ld_x
    int64_t ld_x;
    float *out;      // [S][r][d], or [S][d][r] when transposed
    float *partial;  // [slots][r d], each laid out as out
    int d, transposed, cols;  // cols: blocks over d
};
struct OuterParams {
    OuterProblem problem[2];  // grad_a: q = v, X = x;  grad_b: q = hidden, X = grad
    const uint32_t *order;
    const uint32_t *seg_begin;  // [S + 1]
    PieceTable pieces;
    const float *scale;
    int r, S, accumulate;
};

// A block takes one piece of an adapter's rows, 16 ranks and 16 chunks of columns (more ranks a block read X less often and held fewer
// blocks a CU: 4096 rows, rank 128, 64 ranks a block / 16: bf16 223 / 148 us a call, fp32 209 / 198); fp32 matrix products (16x16x4: lane = (rank or column
// chunk, row), so q needs no rounding and X no transposition).  An adapter of one piece is written out, zeros where it has no
// rows; one of several leaves its sums in `partial`, and outer_join_kernel adds them in order.  A block per adapter and
// piece keeps the blocks alike whether there are few adapters or hundreds (96 rows, 256 adapters: cutting the rows alone, so
// that a block met many adapters one after the other, took twice as long).
template <int DT, bool ALIGNED> __global__ __launch_bounds__(256, 5) void outer_kernel(OuterParams p) {
    typedef typename Elem<DT>::type E;
    constexpr int EPC = Elem<DT>::EPC, CC = 16 * EPC, COPIES = 2;
    __shared__ float red[COPIES][16][CC + 4];  // column m EPC + e of a row lies at 16 e + m: the 64 lanes of a sum hit 64 banks
    __shared__ uint32_t rows[OUTER_ROWS];
    const Piece piece = p.pieces.piece[blockIdx.x];
    if (blockIdx.x >= *p.pieces.count) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m = lane & 15, g = lane >> 4;
    const bool second = (int)blockIdx.y >= p.problem[0].cols;
    const OuterProblem &o = p.problem[second ? 1 : 0];
    const int c0 = ((int)blockIdx.y - (second ? p.problem[0].cols : 0)) * CC, j0 = blockIdx.z * 16;
    const int32_t c = piece.adapter;
    const int lo = (int)piece.begin, hi = (int)piece.end;
    const bool whole = piece.slot < 0;
    if (lo >= hi && p.accumulate) return;
    const float s = p.scale[c];
    f32x4 acc[EPC];
#pragma unroll
    for (int e = 0; e < EPC; e++) acc[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int base = lo; base < hi; base += OUTER_ROWS) {
        const int end = base + OUTER_ROWS < hi ? base + OUTER_ROWS : hi;
        for (int i = base + tid; i < end; i += 256) rows[i - base] = p.order[i];
        __syncthreads();
        constexpr int UNROLL = 4;
        for (int b = base + 4 * wave; b < end; b += 16 * UNROLL) {
            f32x4 fx[UNROLL];
            float fq[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const int at = b + 16 * u + g;
                const bool ok = at < end;
                const int64_t row = rows[ok ? at - base : 0];
                fx[u] = load_chunk<DT, ALIGNED>(reinterpret_cast<const E *>(o.x) + row * o.ld_x, c0 + m * EPC, ok ? o.d : 0);
                fq[u] = ok && j0 + m < p.r ? o.q[row * p.r + j0 + m] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                float v[EPC];
                chunk_to_float<DT>(fx[u], v);
#pragma unroll
                for (int e = 0; e < EPC; e++) acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(fq[u], v[e], acc[e], 0, 0, 0);
            }
        }
        __syncthreads();
    }
    // the four waves' sums, in a fixed order: the upper two put theirs down, the lower two add to them
    auto put = [&](int copy, bool add) {
#pragma unroll
        for (int e = 0; e < EPC; e++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float *cell = &red[copy][4 * g + k][16 * e + m];
                *cell = add ? *cell + acc[e][k] : acc[e][k];
            }
    };
    if (wave >= 2) put(wave - 2, false);
    __syncthreads();
    if (wave < 2) put(wave, true);
    __syncthreads();
    const int64_t size = (int64_t)p.r * o.d;
    float *out = whole ? o.out + (int64_t)c * size : o.partial + (int64_t)piece.slot * size;
    const int rn = p.r - j0 < 16 ? p.r - j0 : 16, cn = o.d - c0 < CC ? o.d - c0 : CC;
    for (int k = tid; k < 16 * CC; k += 256) {
        const int j = o.transposed ? k % 16 : k / CC, col = o.transposed ? k / 16 : k % CC;
        if (j >= rn || col >= cn) continue;
        const float v = red[0][j][col % EPC * 16 + col / EPC] + red[1][j][col % EPC * 16 + col / EPC];
        float *cell = out + (o.transposed ? (int64_t)(c0 + col) * p.r + j0 + j : (int64_t)(j0 + j) * o.d + c0 + col);
        *cell = !whole ? v : (lo < hi ? s * v : 0.0f) + (p.accumulate ? *cell : 0.0f);  // no rows: 0, whatever s is
    }
}

// adapters of several pieces: their partial sums in order
template <int VEC> __global__ __launch_bounds__(256) void outer_join_kernel(OuterParams p) {
    typedef float vec __attribute__((ext_vector_type(VEC)));
    const int c = blockIdx.x, n = (int)(p.seg_begin[c + 1] - p.seg_begin[c]);
    if (n <= p.pieces.rows) return;
    const int np = (n + p.pieces.rows - 1) / p.pieces.rows;
    const OuterProblem &o = p.problem[blockIdx.z];
    const int64_t size = (int64_t)p.r * o.d / VEC;
    vec *out = reinterpret_cast<vec *>(o.out) + (int64_t)c * size;
    const vec *part = reinterpret_cast<const vec *>(o.partial) + (int64_t)p.pieces.slot[c] * size;
    const float s = p.scale[c];
    for (int64_t k = blockIdx.y * 256ll + threadIdx.x; k < size; k += gridDim.y * 256ll) {
        vec v = part[k];
#pragma unroll 4
        for (int t = 1; t < np; t++) v += part[t * size + k];
        out[k] = p.accumulate ? s * v + out[k] : s * v;
    }
}

__global__ __launch_bounds__(256) void fill_zero_kernel(float *dst, int64_t n) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) dst[i] = 0.0f;
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
static int check_adapters(const char *who, const hvs_adapters *ad) {
    HVS_REQUIRE(ad != nullptr, "%s: adapters is NULL", who);
    HVS_REQUIRE(learn_dtype_ok(ad->dtype), "%s: unknown dtype %d", who, ad->dtype);
    HVS_REQUIRE(ad->d_in >= 1 && ad->d_in <= HVS_MAX_ADAPTER_DIM && ad->d_out >= 1 && ad->d_out <= HVS_MAX_ADAPTER_DIM,
                "%s: projection %d x %d, both sides must be in [1, %d]", who, ad->d_out, ad->d_in, HVS_MAX_ADAPTER_DIM);
    HVS_REQUIRE(ad->rank >= 1 && ad->rank <= HVS_MAX_ADAPTER_RANK, "%s: rank %d not in [1, %d]", who, ad->rank, HVS_MAX_ADAPTER_RANK);
    HVS_REQUIRE(ad->n_adapters >= 1 && ad->n_adapters <= HVS_MAX_ADAPTERS, "%s: %d adapters, must be in [1, %d]", who, ad->n_adapters, HVS_MAX_ADAPTERS);
    return 0;
}
static bool once(int64_t n, int rank) { return n <= ONCE_ROWS && rank <= 64; }
static bool few_rows(int dtype, int64_t n, int N) { return n <= FEW_ROWS && n * N <= (dtype == HVS_F32 ? FEW_OUTPUTS_F32 : FEW_OUTPUTS_16); }
static int round_up(int v, int to) { return (v + to - 1) / to * to; }
static int elems_per_chunk(int dtype) { return dtype == HVS_F32 ? 4 : 8; }

// rows handled at once: the grouping's counters and the 31-bit offsets of the tile loads set the limit
static int64_t chunk_rows(int64_t n, int64_t max_ld, int es) {
    int64_t by_offset = ((int64_t)0x7FFFFFFF - 65536) / ((max_ld + 8) * es);  // + 8: the pitch of rows that are brought to whole chunks
    int64_t c = by_offset < MAX_CHUNK_ROWS ? by_offset : MAX_CHUNK_ROWS;
    if (c < 1) c = 1;
    return n < c ? n : c;
}

// what one chunk of rows needs; every pass of a direction shares it
struct AdapterWs {
    uint32_t *order, *seg_begin, *counts;
    int32_t *scodes;
    float *factor, *hidden, *partial_a, *partial_b;
    char *u_hi, *u_lo, *packed_w, *packed_x, *w_t, *a_t, *b_t;
    PieceTable pieces;
};

// Rows in a piece of the stack gradients, for passes of up to n rows: 128, in large passes 256, more where the partial sums would
// take too much (8192 rows of 64 adapters, 128 / 256 / 512 / 1024 rows: 34, 38, 42, 52 us with the join).  Adapters of several pieces have at most 2 n / rows of them.
static int piece_rows(int64_t n, const hvs_adapters *ad) {
    int64_t rows = n <= 16384 ? 128 : 256;
    while (rows < MAX_CHUNK_ROWS && 2 * ((n + rows - 1) / rows) * ad->rank * (ad->d_in + ad->d_out) * 4 > OUTER_PARTIAL_BYTES) rows *= 2;
    return (int)rows;
}
static int outer_cols(int d, int dtype) { return (d + 16 * elems_per_chunk(dtype) - 1) / (16 * elems_per_chunk(dtype)); }

static uint64_t cut_workspace(const hvs_adapters *ad, int64_t nc, int backward, void *base, AdapterWs *ws) {
    *ws = {};
    WorkspaceCut w(base);
    const int es = hvs_elem_size(ad->dtype), epc = elems_per_chunk(ad->dtype), rp = round_up(ad->rank, 16);
    const int64_t chunks = (nc + GROUP_CHUNK - 1) / GROUP_CHUNK;
    const int wide = ad->d_in > ad->d_out ? ad->d_in : ad->d_out;
    const bool few = few_rows(ad->dtype, nc, backward ? ad->d_in : ad->d_out);
    ws->hidden = w.take<float>(nc * ad->rank * 4);
    ws->order = w.take<uint32_t>(nc * 4);
    ws->scodes = w.take<int32_t>(nc * 4);
    ws->seg_begin = w.take<uint32_t>(((uint64_t)ad->n_adapters + 1) * 4);
    ws->counts = w.take<uint32_t>(chunks > GROUP_SELF ? (uint64_t)chunks * (ad->n_adapters + 2) * 4 : 0);
    ws->factor = w.take<float>(nc * 4);
    ws->u_hi = w.take<char>(nc * rp * es);
    ws->u_lo = w.take<char>(ad->dtype == HVS_F32 ? 0 : nc * rp * es);
    ws->packed_w = w.take<char>(!few ? (uint64_t)wide * round_up(wide, epc) * es : 0);
    ws->packed_x = w.take<char>(!few ? (uint64_t)nc * round_up(wide, epc) * es : 0);
    if (backward) {
        ws->w_t = w.take<char>((uint64_t)ad->d_in * round_up(ad->d_out, epc) * es);
        ws->b_t = w.take<char>((uint64_t)ad->n_adapters * ad->rank * round_up(ad->d_out, epc) * es);
        ws->a_t = w.take<char>((uint64_t)ad->n_adapters * ad->d_in * rp * es);
        ws->pieces.rows = piece_rows(nc, ad);
        const uint64_t several = (nc + ws->pieces.rows - 1) / ws->pieces.rows, slots = nc > ws->pieces.rows ? 2 * several * ad->rank : 0;
        ws->pieces.piece = w.take<Piece>(((uint64_t)ad->n_adapters + several) * sizeof(Piece));
        ws->pieces.slot = w.take<uint32_t>((uint64_t)ad->n_adapters * 4);
        ws->pieces.count = w.take<uint32_t>(4);
        ws->partial_a = w.take<float>(slots * ad->d_in * 4);
        ws->partial_b = w.take<float>(slots * ad->d_out * 4);
    }
    return w.used;
}

extern "C" int hvs_adapters_workspace(const hvs_adapters *ad, int64_t n, int64_t max_ld, int backward, uint64_t *out_bytes) {
    HVS_TRY(check_adapters("hvs_adapters_workspace", ad));
    HVS_REQUIRE(n >= 0 && out_bytes, "hvs_adapters_workspace: negative row count or NULL argument");
    HVS_REQUIRE(max_ld <= 0x7FFFFFFF, "hvs_adapters_workspace: row pitch %lld is 2 GB or more", (long long)max_ld);
    const int64_t nc = chunk_rows(n, max_ld > 0 ? max_ld : 1, hvs_elem_size(ad->dtype));
    AdapterWs ws;
    *out_bytes = n == 0 || (!backward && once(n, ad->rank)) ? 0 : cut_workspace(ad, nc, backward, nullptr, &ws);
    return 0;
}

static GroupParams group_params(const int32_t *codes, int n, int S, const AdapterWs &ws) {
    int bits = 1;
    while ((1 << bits) < S + 2) bits++;
    return {codes, n, S, bits, (n + GROUP_CHUNK - 1) / GROUP_CHUNK, ws.counts, ws.order, ws.scodes, ws.seg_begin, ws.pieces};
}
static bool group_alone(const GroupParams &g) { return g.chunks <= GROUP_SELF && g.S + 2 <= GROUP_FEW_BINS; }  // by one launch, in little LDS

static int launch_group(hipStream_t st, const GroupParams &g) {
    const size_t lds = (size_t)(g.S + 2) * 4;
    if (g.chunks > GROUP_SELF) {
        HVS_TRY((learn_allow_lds<group_count_kernel>((int)lds)));
        group_count_kernel<<<g.chunks, GROUP_CHUNK, lds, st>>>(g.codes, g.n, g.S, g.counts);
    }
    if (g.S + 2 <= GROUP_FEW_BINS) {
        group_place_kernel<true><<<g.chunks, GROUP_CHUNK, 2 * lds, st>>>(g);
    } else {
        HVS_TRY((learn_allow_lds<group_place_kernel<false>>((int)(2 * lds))));
        group_place_kernel<false><<<g.chunks, GROUP_CHUNK, 2 * lds, st>>>(g);
    }
    HVS_HIP(hipGetLastError());
    return 0;
}

template <int DT> static int launch_shrink(hipStream_t st, const ShrinkParams &p, int shares) {
    const int es = hvs_elem_size(DT);
    const bool al = learn_aligned(p.x, p.ld_x * es, (int64_t)p.K * es) && learn_aligned(p.a, p.lda * es, (int64_t)p.K * es);
    const bool wide = p.order && p.n >= SHRINK_WIDE_ROWS;
    const dim3 grid((p.n + 15) / 16, shares), wgrid((p.n + 127) / 128);
#define SHRINK(RT_)                                                                                          \
    do {                                                                                                     \
        if (wide && al) shrink_wide_kernel<DT, RT_, true><<<wgrid, 256, 0, st>>>(p);                         \
        else if (wide) shrink_wide_kernel<DT, RT_, false><<<wgrid, 256, 0, st>>>(p);                         \
        else if (al) shrink_kernel<DT, RT_, true><<<grid, 64 * SHRINK_WAVES, 0, st>>>(p);                    \
        else shrink_kernel<DT, RT_, false><<<grid, 64 * SHRINK_WAVES, 0, st>>>(p);                           \
    } while (0)
    if (p.r <= 16) SHRINK(1);
    else if (p.r <= 32) SHRINK(2);
    else if (p.r <= 64) SHRINK(4);
    else SHRINK(8);
#undef SHRINK
    HVS_HIP(hipGetLastError());
    return 0;
}

template <int DT> static int launch_few(hipStream_t st, const ProjectParams &p) {
    const int es = hvs_elem_size(DT);
    const bool al = learn_aligned(p.x, p.ld_x * es, (int64_t)p.K * es) && learn_aligned(p.w, p.ldw * es, (int64_t)p.K * es);
#define FEW(MT_, NT_, WAVES_)                                                                                                     \
    do {                                                                                                                          \
        const int grid = (p.N + 16 * MT_ - 1) / (16 * MT_) * ((p.n + 16 * NT_ - 1) / (16 * NT_));                                 \
        if (al) project_few_kernel<DT, MT_, NT_, WAVES_, true><<<grid, 64 * WAVES_, 0, st>>>(p);                                  \
        else project_few_kernel<DT, MT_, NT_, WAVES_, false><<<grid, 64 * WAVES_, 0, st>>>(p);                                    \
    } while (0)
    // The smallest blocks while every CU has at most one (fp32, whose products take longer than their loads: two), then twice the rows,
    // then 32 x 32, which read half as much.  A call with 1536 x 1536 weights, rank 16, blocks of 16 x 16 / 16 x 32 / 32 x 32, us: bf16
    // 32 rows 8.9 / 9.9 / 11.3, 64 rows 12.2 / 9.9 / 11.5, 128 rows 15.1 / 13.9 / 11.9; fp32 32 rows 12.5 / 16.1 / 20.2, 64 rows 16.5 / 16.9 / 20.2,
    // 128 rows 23.1 / 26.5 / 22.7, 512 rows 67 / 63 / 49
    auto blocks = [&](int rows) { return (int64_t)((p.N + 15) / 16) * ((p.n + rows - 1) / rows); };
    if (blocks(16) <= (DT == HVS_F32 ? 512 : 256)) FEW(1, 1, 16);
    else if constexpr (DT == HVS_F32) FEW(2, 2, 8);
    else if (blocks(32) <= 256) FEW(1, 2, 16);
    else FEW(2, 2, 8);
#undef FEW
    HVS_HIP(hipGetLastError());
    return 0;
}

template <int DT> static int launch_once(hipStream_t st, const ProjectParams &p, float *hidden, const void *a, int64_t lda) {
    const int es = hvs_elem_size(DT), grid = (p.N + 15) / 16;
    const int64_t row = (int64_t)p.K * es;
    const bool al = learn_aligned(p.x, p.ld_x * es, row) && learn_aligned(p.w, p.ldw * es, row) && learn_aligned(a, lda * es, row);
#define ONCE(RT_)                                                                                      \
    do {                                                                                               \
        if (al) project_once_kernel<DT, RT_, true><<<grid, 1024, 0, st>>>(p, hidden, a, lda);          \
        else project_once_kernel<DT, RT_, false><<<grid, 1024, 0, st>>>(p, hidden, a, lda);            \
    } while (0)
    if (p.r <= 16) ONCE(1);
    else if (p.r <= 32) ONCE(2);
    else ONCE(4);
#undef ONCE
    HVS_HIP(hipGetLastError());
    return 0;
}

template <int DT, class T> static int launch_tile(hipStream_t st, const ProjectParams &p) {
    const int tiles = ((p.N + T::BM - 1) / T::BM) * ((p.n + T::BN - 1) / T::BN);
    const size_t lds = 2 * T::STAGE_BYTES;
    HVS_TRY((learn_allow_lds<project_tile_kernel<DT, T>>((int)lds)));
    const int resident = 256 * (512 / T::GT);  // blocks the chip holds at once
    project_tile_kernel<DT, T><<<tiles < resident ? tiles : resident, T::GT, lds, st>>>(p);
    HVS_HIP(hipGetLastError());
    return 0;
}

template <int DT> static int launch_pack(hipStream_t st, const void *src, int64_t ld, int n, int K, int Kp, void *dst) {
    typedef typename Elem<DT>::type E;
    const int64_t blocks = ((int64_t)n * Kp + 255) / 256;
    pack_rows_kernel<E><<<(int)(blocks < 4096 ? blocks : 4096), 256, 0, st>>>((const E *)src, ld, n, K, Kp, (E *)dst);
    HVS_HIP(hipGetLastError());
    return 0;
}

static TransposeJob transpose_job(const void *src, int64_t count, int R, int C, int ld, void *dst) {
    TransposeJob t = {};
    t.src = src, t.dst = dst, t.R = R, t.C = C, t.ld = ld;
    t.log_c = C <= 32 ? TILE_LOG_NARROW : (ld <= 32 ? TILE_LOG - TILE_LOG_NARROW : TILE_LOG / 2);
    const int tc = 1 << t.log_c, tr = (1 << TILE_LOG) >> t.log_c;
    t.tiles_c = (C + tc - 1) / tc, t.tiles_r = (ld + tr - 1) / tr;  // the row tiles cover the pitch, so that the padding is written
    t.blocks = count * t.tiles_c * t.tiles_r;
    return t;
}

// One direction for one chunk of rows: u = A x into hidden, y = W x + s B u into out.  A: [S][r] rows of K, pitch lda;
// W: [N] rows of K, pitch ldw; B: [S][N] rows of r, pitch ldb.
struct Direction {
    const void *x, *a, *w, *b;
    int64_t ld_x, lda, ldw, ldb;
    int K, N;
    bool b_padded;  // rows of b are zero from r to their pitch
    void *out;  // NULL: u alone
    int64_t ld_out;
};

template <int DT>
static int run_direction(hipStream_t st, const hvs_adapters *ad, const Direction &d, const int32_t *codes, int n, float *hidden, AdapterWs &ws, bool grouped) {
    const int es = hvs_elem_size(DT), epc = Elem<DT>::EPC;
    const bool few = few_rows(DT, n, d.N);
    Direction dd = d;
    if (!few && d.out) {
        // the tile loads take whole 16-byte chunks: rows that do not offer them are brought to that pitch first
        const int Kp = round_up(d.K, epc);
        if (!learn_aligned(d.x, d.ld_x * es, (int64_t)d.K * es)) {
            HVS_TRY(launch_pack<DT>(st, d.x, d.ld_x, n, d.K, Kp, ws.packed_x));
            dd.x = ws.packed_x;
            dd.ld_x = Kp;
        }
        if (!learn_aligned(d.w, d.ldw * es, (int64_t)d.K * es)) {
            HVS_TRY(launch_pack<DT>(st, d.w, d.ldw, d.N, d.K, Kp, ws.packed_w));
            dd.w = ws.packed_w;
            dd.ldw = Kp;
        }
    }
    ShrinkParams s = {};
    s.x = d.x, s.ld_x = d.ld_x, s.a = d.a, s.lda = d.lda;
    s.n = n, s.K = d.K, s.r = ad->rank, s.rp = round_up(ad->rank, 16), s.S = ad->n_adapters, s.scale = ad->scale;
    s.hidden = hidden;
    ProjectParams p = {};
    p.x = dd.x, p.ld_x = dd.ld_x, p.w = dd.w, p.ldw = dd.ldw, p.b = d.b, p.ldb = d.ldb, p.scale = ad->scale;
    p.out = d.out, p.ld_out = d.ld_out, p.n = n, p.K = d.K, p.N = d.N, p.r = s.r, p.rp = s.rp, p.S = s.S;
    if (few) {
        if (d.out && once(n, p.r)) {
            p.codes = codes;
            return launch_once<DT>(st, p, hidden, d.a, d.lda);
        }
        if (!hidden) s.hidden = ws.hidden;
        s.codes = codes;
        HVS_TRY(launch_shrink<DT>(st, s, n < 16 ? n : 16));
        if (!d.out) return 0;
        p.codes = codes;
        p.hidden = s.hidden;
        return launch_few<DT>(st, p);
    }
    if (!grouped) HVS_TRY(launch_group(st, group_params(codes, n, s.S, ws)));
    s.codes = ws.scodes, s.order = ws.order;
    if (d.out) s.u_hi = ws.u_hi, s.u_lo = ws.u_lo, s.factor = ws.factor;
    HVS_TRY(launch_shrink<DT>(st, s, SHRINK_SHARES));
    if (!d.out) return 0;
    p.K = round_up(d.K, epc);  // whole chunks: K itself where rows were taken as they are, their padded width where they were packed
    p.codes = ws.scodes, p.order = ws.order, p.u_hi = ws.u_hi, p.u_lo = ws.u_lo, p.factor = ws.factor;
    p.b_aligned = learn_aligned(d.b, d.ldb * es, 0) && (d.b_padded || s.r % epc == 0);
    p.out_vec = learn_aligned(d.out, d.ld_out * es, 0);
    // The tile whose rounds over the chip take least time, in units of a round of two 128-tiles per CU.  Four 64-tiles per CU
    // take 0.55 of that (fp32 0.48) when they are all there is and 0.7 round after round, a single 128-tile per CU 0.7 (fp32
    // 0.5), a 256-tile per CU 1.75 for four times the work.  With 1536 x 1536 bf16 weights, us a call: 2048 rows 64 / 128 33 / 39,
    // 4096 rows 59 / 48; 8192 rows 64 / 128 / 256 83 / 77 / 68; 16 384 rows 128 / 256 120 / 135.
    auto rounds = [&](int t, int slots) { return (((int64_t)(p.N + t - 1) / t) * ((n + t - 1) / t) + slots - 1) / slots; };
    const bool f32 = DT == HVS_F32;
    const double c64 = rounds(64, 1024) == 1 ? (f32 ? 0.48 : 0.55) : 0.7 * (double)rounds(64, 1024);
    const double c128 = rounds(128, 256) == 1 ? (f32 ? 0.5 : 0.7) : (double)rounds(128, 512);
    if constexpr (DT != HVS_F32) {
        const double c256 = 1.75 * (double)rounds(256, 256);
        if (c256 <= c128 && c256 <= c64) return launch_tile<DT, Tile256>(st, p);
    }
    if (c128 <= c64) return launch_tile<DT, Tile128>(st, p);
    return launch_tile<DT, Tile64>(st, p);
}

static int dispatch_direction(hipStream_t st, const hvs_adapters *ad, const Direction &d, const int32_t *codes, int n, float *hidden, AdapterWs &ws, bool grouped) {
    if (ad->dtype == HVS_F32) return run_direction<HVS_F32>(st, ad, d, codes, n, hidden, ws, grouped);
    if (ad->dtype == HVS_F16) return run_direction<HVS_F16>(st, ad, d, codes, n, hidden, ws, grouped);
    return run_direction<HVS_BF16>(st, ad, d, codes, n, hidden, ws, grouped);
}

static int check_rows(const char *who, const char *what, const void *p, int64_t ld, int width, int es) {
    HVS_REQUIRE(p != nullptr, "%s: %s is NULL", who, what);
    HVS_REQUIRE(ld >= width, "%s: row pitch %lld of %s is below its %d columns", who, (long long)ld, what, width);
    HVS_REQUIRE((uintptr_t)p % es == 0, "%s: %s is not aligned to its elements", who, what);
    HVS_REQUIRE(ld <= ((int64_t)0x7FFFFFFF - 65536) / es - 8, "%s: row pitch %lld of %s is 2 GB or more", who, (long long)ld, what);
    return 0;
}
static int check_workspace(const char *who, const hvs_adapters *ad, int64_t n, int64_t max_ld, int backward, const void *ws, uint64_t bytes) {
    uint64_t need = 0;
    HVS_TRY(hvs_adapters_workspace(ad, n, max_ld, backward, &need));
    HVS_REQUIRE(need == 0 || (ws != nullptr && ((uintptr_t)ws & 255) == 0 && bytes >= need), "%s: workspace of %llu bytes at %p, needs %llu aligned to 256", who,
                (unsigned long long)bytes, ws, (unsigned long long)need);
    return 0;
}
static int check_weights(const char *who, const hvs_adapters *ad) {
    const int es = hvs_elem_size(ad->dtype);
    HVS_REQUIRE(ad->projection && ad->a && ad->b && ad->scale, "%s: a weight is NULL", who);
    HVS_REQUIRE((uintptr_t)ad->projection % es == 0 && (uintptr_t)ad->a % es == 0 && (uintptr_t)ad->b % es == 0 && (uintptr_t)ad->scale % 4 == 0,
                "%s: a weight is not aligned to its elements", who);
    return 0;
}

// what is written (rows of `width` elements) is no part of the weights that are read meanwhile
static int check_apart_from_weights(const char *who, const char *what, const hvs_adapters *ad, const void *p, int64_t rows, int64_t ld, int width) {
    const int64_t es = hvs_elem_size(ad->dtype), ranks = (int64_t)ad->n_adapters * ad->rank;
    const struct {
        const void *p;
        int64_t bytes;
    } weights[] = {{ad->projection, (int64_t)ad->d_out * ad->d_in * es}, {ad->a, ranks * ad->d_in * es}, {ad->b, ranks * ad->d_out * es}, {ad->scale, (int64_t)ad->n_adapters * 4}};
    for (const auto &w : weights) HVS_REQUIRE(!learn_overlap(p, rows, ld * es, width * es, w.p, 1, 0, w.bytes), "%s: %s overlaps the weights", who, what);
    return 0;
}

extern "C" int hvs_adapters_apply(int device_id, void *stream, const hvs_adapters *ad, const void *x, int64_t ld_x, const int32_t *codes, int64_t n,
                                  void *out, int64_t ld_out, float *hidden, void *workspace, uint64_t workspace_bytes) {
    const char *who = "hvs_adapters_apply";
    HVS_TRY(check_adapters(who, ad));
    HVS_REQUIRE(n >= 0, "%s: negative row count", who);
    if (n == 0) return 0;
    const int es = hvs_elem_size(ad->dtype);
    HVS_TRY(check_weights(who, ad));
    HVS_TRY(check_rows(who, "x", x, ld_x, ad->d_in, es));
    HVS_TRY(check_rows(who, "out", out, ld_out, ad->d_out, es));
    HVS_REQUIRE(codes != nullptr, "%s: codes is NULL", who);
    HVS_REQUIRE(((uintptr_t)codes | (uintptr_t)hidden) % 4 == 0, "%s: codes or hidden is not aligned to its elements", who);
    HVS_REQUIRE(!learn_overlap(x, n, ld_x * es, (int64_t)ad->d_in * es, out, n, ld_out * es, (int64_t)ad->d_out * es), "%s: out overlaps x", who);
    const int64_t max_ld = ld_x > ld_out ? ld_x : ld_out;
    HVS_TRY(check_apart_from_weights(who, "out", ad, out, n, ld_out, ad->d_out));
    HVS_TRY(check_workspace(who, ad, n, max_ld, 0, workspace, workspace_bytes));
    DeviceGuard guard(device_id);
    HVS_HIP(guard.status);
    const int64_t nc = chunk_rows(n, max_ld, es);
    AdapterWs ws;
    cut_workspace(ad, nc, 0, workspace, &ws);
    for (int64_t r0 = 0; r0 < n; r0 += nc) {
        const int rows = (int)(n - r0 < nc ? n - r0 : nc);
        Direction d = {};
        d.x = (const char *)x + r0 * ld_x * es, d.ld_x = ld_x;
        d.a = ad->a, d.lda = ad->d_in, d.w = ad->projection, d.ldw = ad->d_in, d.b = ad->b, d.ldb = ad->rank;
        d.K = ad->d_in, d.N = ad->d_out;
        d.out = (char *)out + r0 * ld_out * es, d.ld_out = ld_out;
        HVS_TRY(dispatch_direction((hipStream_t)stream, ad, d, codes + r0, rows, hidden ? hidden + r0 * ad->rank : nullptr, ws, false));
    }
    return 0;
}

template <int DT> static int launch_outer(hipStream_t st, const OuterParams &p, int64_t n) {
    const int es = hvs_elem_size(DT);
    bool al = true, vec = true;
    for (const OuterProblem &o : p.problem) {
        al = al && learn_aligned(o.x, o.ld_x * es, (int64_t)o.d * es);
        vec = vec && (int64_t)p.r * o.d % 4 == 0 && (uintptr_t)o.out % 16 == 0;
    }
    // (the table says how many pieces there are; the launch has room for the most there can be)
    const int64_t most = p.S + (n + p.pieces.rows - 1) / p.pieces.rows;
    const int cols = p.problem[0].cols + p.problem[1].cols;
    const dim3 grid((unsigned)most, cols, (p.r + 15) / 16);
    if (al) outer_kernel<DT, true><<<grid, 256, 0, st>>>(p);
    else outer_kernel<DT, false><<<grid, 256, 0, st>>>(p);
    HVS_HIP(hipGetLastError());
    if (n <= p.pieces.rows) return 0;
    const int wide = p.problem[0].d > p.problem[1].d ? p.problem[0].d : p.problem[1].d;
    const int64_t by = (int64_t)p.r * wide / 1024;
    const dim3 join_grid(p.S, (unsigned)(by < 1 ? 1 : (by > 64 ? 64 : by)), 2);
    if (vec) outer_join_kernel<4><<<join_grid, 256, 0, st>>>(p);
    else outer_join_kernel<1><<<join_grid, 256, 0, st>>>(p);
    HVS_HIP(hipGetLastError());
    return 0;
}

template <int DT>
static int run_backward(hipStream_t st, const hvs_adapters *ad, const void *grad, int64_t ld_grad, const void *x, int64_t ld_x, const int32_t *codes,
                        const float *hidden, int64_t n, void *grad_x, int64_t ld_gx, float *grad_a, float *grad_b, int64_t nc, AdapterWs &ws) {
    const int es = hvs_elem_size(DT), epc = Elem<DT>::EPC, rp = round_up(ad->rank, 16);
    const int dop = round_up(ad->d_out, epc);
    // the weights of the transposed product; frozen W too is laid out by every call, so that nothing can be out of date
    TransposeJobs jobs = {};
    int k = 0;
    jobs.job[k++] = transpose_job(ad->b, ad->n_adapters, ad->d_out, ad->rank, dop, ws.b_t);
    if (grad_x) {
        jobs.job[k++] = transpose_job(ad->projection, 1, ad->d_out, ad->d_in, dop, ws.w_t);
        jobs.job[k++] = transpose_job(ad->a, ad->n_adapters, ad->rank, ad->d_in, rp, ws.a_t);
    }
    const int64_t blocks = jobs.job[0].blocks + jobs.job[1].blocks + jobs.job[2].blocks;
    const GroupParams first = group_params(codes, (int)(n < nc ? n : nc), ad->n_adapters, ws);
    const int beside = group_alone(first) ? first.chunks : 0;
    const size_t tile_lds = ((1 << TILE_LOG) + (1 << (TILE_LOG - TILE_LOG_NARROW))) * sizeof(typename Elem<DT>::type), group_lds = (size_t)(ad->n_adapters + 2) * 8;
    const size_t lds = beside && group_lds > tile_lds ? group_lds : tile_lds;
    HVS_TRY((learn_allow_lds<layout_kernel<typename Elem<DT>::type>>((int)lds)));
    for (int64_t at = 0; at < blocks; at += LAYOUT_TILES) {
        const int64_t tiles = blocks - at < LAYOUT_TILES ? blocks - at : LAYOUT_TILES;
        const int grouping = at == 0 ? beside : 0;
        layout_kernel<typename Elem<DT>::type><<<(unsigned)(tiles + grouping), GROUP_CHUNK, lds, st>>>(jobs, at, first, grouping);
        HVS_HIP(hipGetLastError());
    }
    for (int64_t r0 = 0; r0 < n; r0 += nc) {
        const int rows = (int)(n - r0 < nc ? n - r0 : nc);
        if (r0 > 0 || !beside) HVS_TRY(launch_group(st, group_params(codes + r0, rows, ad->n_adapters, ws)));
        Direction d = {};
        d.x = (const char *)grad + r0 * ld_grad * es, d.ld_x = ld_grad;
        d.a = ws.b_t, d.lda = dop, d.w = ws.w_t, d.ldw = dop, d.b = ws.a_t, d.ldb = rp, d.b_padded = true;
        d.K = ad->d_out, d.N = ad->d_in;
        d.out = grad_x ? (char *)grad_x + r0 * ld_gx * es : nullptr, d.ld_out = ld_gx;
        HVS_TRY(run_direction<DT>(st, ad, d, codes + r0, rows, ws.hidden, ws, true));
        OuterParams o = {};
        o.order = ws.order, o.seg_begin = ws.seg_begin, o.pieces = ws.pieces, o.scale = ad->scale;
        o.r = ad->rank, o.S = ad->n_adapters, o.accumulate = r0 > 0;
        const char *xr = (const char *)x + r0 * ld_x * es;
        o.problem[0] = {ws.hidden, xr, ld_x, grad_a, ws.partial_a, ad->d_in, 0, outer_cols(ad->d_in, DT)};
        o.problem[1] = {hidden + r0 * ad->rank, d.x, ld_grad, grad_b, ws.partial_b, ad->d_out, 1, outer_cols(ad->d_out, DT)};
        HVS_TRY(launch_outer<DT>(st, o, rows));
    }
    return 0;
}

extern "C" int hvs_adapters_backward(int device_id, void *stream, const hvs_adapters *ad, const void *grad, int64_t ld_grad, const void *x, int64_t ld_x,
                                     const int32_t *codes, const float *hidden, int64_t n, void *grad_x, int64_t ld_gx, float *grad_a, float *grad_b,
                                     void *workspace, uint64_t workspace_bytes) {
    const char *who = "hvs_adapters_backward";
    HVS_TRY(check_adapters(who, ad));
    HVS_REQUIRE(n >= 0, "%s: negative row count", who);
    HVS_REQUIRE(grad_a && grad_b, "%s: grad_a or grad_b is NULL", who);
    HVS_REQUIRE((uintptr_t)grad_a % 4 == 0 && (uintptr_t)grad_b % 4 == 0, "%s: grad_a or grad_b is not aligned to its elements", who);
    hipStream_t st = (hipStream_t)stream;
    const int64_t size_a = (int64_t)ad->n_adapters * ad->rank * ad->d_in, size_b = (int64_t)ad->n_adapters * ad->rank * ad->d_out;
    if (n == 0) {
        DeviceGuard guard(device_id);
        HVS_HIP(guard.status);
        fill_zero_kernel<<<1024, 256, 0, st>>>(grad_a, size_a);
        fill_zero_kernel<<<1024, 256, 0, st>>>(grad_b, size_b);
        HVS_HIP(hipGetLastError());
        return 0;
    }
    const int es = hvs_elem_size(ad->dtype);
    HVS_TRY(check_weights(who, ad));
    HVS_TRY(check_rows(who, "grad", grad, ld_grad, ad->d_out, es));
    HVS_TRY(check_rows(who, "x", x, ld_x, ad->d_in, es));
    HVS_REQUIRE(codes && hidden, "%s: codes or hidden is NULL", who);
    HVS_REQUIRE(((uintptr_t)codes | (uintptr_t)hidden) % 4 == 0, "%s: codes or hidden is not aligned to its elements", who);
    int64_t max_ld = ld_grad > ld_x ? ld_grad : ld_x;
    if (grad_x) {
        HVS_TRY(check_rows(who, "grad_x", grad_x, ld_gx, ad->d_in, es));
        HVS_REQUIRE(!learn_overlap(grad, n, ld_grad * es, (int64_t)ad->d_out * es, grad_x, n, ld_gx * es, (int64_t)ad->d_in * es) &&
                        !learn_overlap(x, n, ld_x * es, (int64_t)ad->d_in * es, grad_x, n, ld_gx * es, (int64_t)ad->d_in * es),
                    "%s: grad_x overlaps an input", who);
        HVS_TRY(check_apart_from_weights(who, "grad_x", ad, grad_x, n, ld_gx, ad->d_in));
        max_ld = max_ld > ld_gx ? max_ld : ld_gx;
    }
    HVS_TRY(check_workspace(who, ad, n, max_ld, 1, workspace, workspace_bytes));
    DeviceGuard guard(device_id);
    HVS_HIP(guard.status);
    const int64_t nc = chunk_rows(n, max_ld, es);
    AdapterWs ws;
    cut_workspace(ad, nc, 1, workspace, &ws);
    if (ad->dtype == HVS_F32) return run_backward<HVS_F32>(st, ad, grad, ld_grad, x, ld_x, codes, hidden, n, grad_x, ld_gx, grad_a, grad_b, nc, ws);
    if (ad->dtype == HVS_F16) return run_backward<HVS_F16>(st, ad, grad, ld_grad, x, ld_x, codes, hidden, n, grad_x, ld_gx, grad_a, grad_b, nc, ws);
    return run_backward<HVS_BF16>(st, ad, grad, ld_grad, x, ld_x, codes, hidden, n, grad_x, ld_gx, grad_a, grad_b, nc, ws);
}
