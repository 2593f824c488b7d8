// Attention of one new token per sequence over a paged key-value cache:
//   s_j = scale q k_j + w[bucket(len - 1 - j)],  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j.
// Four operations per byte of cache and query head: bound by reading the cache once.
#include <math.h>

#include "attn_mma.cuh"
#include "paged.cuh"
#include "relbias.cuh"
#include "sm100_prims.cuh"

namespace rgd {
namespace paged {

int append_status_fetch();

__device__ int g_attn_status = 0;

using attn::LOG2E;
constexpr float LN2 = 0.6931471805599453f;

struct AttnParams {
    PagedView view;
    const int32_t *lengths;
    const void *q, *k, *v;
    int64_t q_sb, q_sh, k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;
    void *o;
    int64_t o_sb, o_sh;
    float *lse;                             // null: not wanted
    int B, Hq, Hkv, G, d;                   // G: query heads of a cache head
    int groups, units;                      // units of a cache head, of a sequence
    FastDiv by_units, by_groups;
    int direct;                             // a CTA per unit, nothing to join
    char *work;
    float scale_log2;
    const void *w;                          // null: no position bias
    int64_t w_sk, w_sh;
    int w_dtype;
    relbias::Borders borders;
};

// Tokens of a sequence that the kernels look at.
__device__ __forceinline__ int live_length(const AttnParams &p, int b, bool report) {
    const int64_t n = p.lengths[b], most = capacity(p.view);
    if (report && (n < 0 || n > most)) g_attn_status = 1;
    return (int)(n < 0 ? 0 : n > most ? most : n);
}

// ---------------------------------------------------------------------------------------------------------------
// Work.  A unit is a sequence, a cache head and up to 16 of the query heads that share it (one or two column tiles of 8);
// its keys come in tiles.  The tiles of all units, one after the other, are dealt out to the warps of the grid in runs
// of equal cost, whatever the lengths are; a CTA finds its warps' runs from the lengths, which are on the device.  A unit
// that one warp has whole is finished there; of a unit that several have, each leaves its part (row maximum, row sum,
// unnormalised output) in the workspace, and join_kernel adds the parts in order.
//
// A warp does everything for its tiles: it streams the keys and values through a ring of cp.async stages of its own,
// which goes on across units, keeps the running maximum, sum and output in registers, and waits for no other warp.
// Two forms in which the four warps of a CTA shared a unit were slower: with the maxima and weights of a tile exchanged
// and the channels split, three barriers a tile held the loop (120 us for one sequence of 131 thousand keys, 93 us
// without); with 16 keys of a tile each, added up at the unit's end, short sequences paid for that (103 us for 64 of 16
// to 8192 keys, 72 us without).
//
// One B200, cold L2: 64 sequences of 16 to 8192 keys, 32 / 8 heads of 128 (366 MB) 65 us, one of 131 thousand (537 MB)
// 90 us (some GPUs take 7 % longer).  6 us go by before the rings are full (lengths, table entries and first tiles are reads
// that wait for one another) and the join takes 3-4 us; in between the keys arrive at the copy rate.
//
// With two warps on a scheduler the chain of a tile's instructions counts next to the reads.  So a tile without gaps is
// loaded and scored without a check per key (95 us for the long one with them), and the products are taken transposed:
// up to eight query heads of a cache head are one column tile, where as rows they would leave half of a row tile's
// scores, weights and sums empty (70 us for the 64, 9.8 instead of 8.5 for one sequence of 300).  Nine and more take two
// (16 sequences of 8000 keys, 2 cache heads with 16 heads of 128 each: 45 us, 43 with heads as rows).
//
// Weights are split into two numbers of the cache's type (hi + lo): rounded to one, they would cost as much accuracy
// as the output's own rounding, and the matrix pipe idles anyway.  Two bf16 numbers hold a weight to 2^-18 of itself,
// which is noise: it averages out over the keys.  fp16 ends at 2^-24, where it would drop all weights below 2^-25 of the
// largest while the row sum counts them: 30 thousand keys 17 nats below one other came out 44 % off.  So fp16 weights
// are multiplied by 2^15 first, and the output by 2^-15 when it leaves the registers (both exact): they are held to 2^-22
// of themselves and 2^-40 of the largest.
//
// The matrix unit cuts off what its sums have past 24 bits, always towards zero: an output kept in it along a run, with two
// additions for 16 keys, came out 0.06 % low after 131 thousand keys (half a step of fp16 is 0.05 %).  So the products of 16
// keys are summed from zero and added with a rounding, which errs to either side: no such drift is left, at the same time
// (66.6 us for the 64 sequences, 90.1 for the long one, each within 0.5 % of before; 16 sequences of 8000 keys with 16 heads
// to a cache head, one call after another, 40.6 for 39.2).
// ---------------------------------------------------------------------------------------------------------------
constexpr int WARPS = 4, THREADS = WARPS * 32, ROWS = 16, STAGES = 3, CTAS_PER_SM = 2;
// In tiles: what a unit's queries and output cost, and the least run of a warp.  us for 64 sequences of 16 to 8192 keys
// with 8 cache heads / 48 of up to 2500 with 24 / 16 of up to 1500 with 16: 65.3 / 32.3 / 13.4 like this, 65.4 / 32.0 / 13.8
// at 1 and 2, 65.7 / 32.8 / 13.3 at 3 and 4.
constexpr int UNIT_COST = 2, MIN_COST = 3;
static_assert(MIN_COST > UNIT_COST, "a run that begins a unit has its first tile");

__host__ __device__ constexpr int tile_keys(int D) { return D > 64 ? 16 : 32; }      // 8 KB of keys and values

template <typename T> struct WeightScale { static constexpr float UP = 1.f, DOWN = 1.f; };
template <> struct WeightScale<__half> { static constexpr float UP = 32768.f, DOWN = 1.f / UP; };      // a weight is at most 1, 65504 the largest fp16

constexpr int NEAR = 256;               // distances whose bucket is looked up

template <typename T, int D>
struct Smem {
    static constexpr int KEYS = tile_keys(D);
    // rows of D channels; the 16-byte chunks of row r change places by r mod 8, so that the rows of an ldmatrix lie in
    // different banks
    struct alignas(16) Stage {
        T k[KEYS * D], v[KEYS * D];
    };
    Stage ring[WARPS][STAGES];
    struct alignas(16) Row {
        const T *k, *v;                                 // null: none
    };
    Row row[WARPS][2][KEYS];                            // of the tiles to load next
    int upto[THREADS], filled[THREADS];                 // costs and sequences with a token, of a warp's threads up to each
    int unit, tile;                                     // where the CTA's runs begin
    int borders[relbias::MAX_SIDE];                     // with a position bias
    uint8_t bucket[NEAR];                               // of the distances below NEAR
    static_assert(relbias::MAX_SIDE <= 256, "a bucket in a byte");
};

__device__ __forceinline__ void cp16(void *dst, const void *src, bool valid) {
    // not valid: nothing is read, 16 zero bytes are written
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(valid ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Workspace: per warp of the grid a header and two parts, [0] of a unit that began in another warp's run, [1] of one
// that ends in another's.
struct Header {
    int last;                   // the unit of part [1] ends in this warp's run; -1: there is none
    int merged;                 // part [1] holds what the four warps of the CTA have
    int b, hk, row0;
};
// A CTA whose runs lie inside one unit that ends behind them leaves one part, its first warp's.  So of a unit that ends
// in another CTA, every CTA in between has one part, the last one a part per warp, the first one either.
__host__ __device__ constexpr int64_t part_floats(int D) { return ROWS * (D + 2); }
static_assert(WARPS * sizeof(Header) % 16 == 0, "parts lie behind the headers, on 16 bytes");
__host__ __device__ __forceinline__ int64_t workspace_bytes(int ctas, int D) {
    return (int64_t)ctas * WARPS * ((int64_t)sizeof(Header) + 2 * part_floats(D) * (int64_t)sizeof(float));
}
__device__ __forceinline__ float *part_of(const AttnParams &p, int warps, int D, int warp, int which) {
    return reinterpret_cast<float *>(p.work + (int64_t)warps * sizeof(Header)) + (warp * 2 + which) * part_floats(D);
}

// The costs [0, total) dealt out to the warps: equal shares, the first ones with one more.
struct Runs {
    int total = 0, busy = 0, share = 0, more = 0;       // busy: warps with a share
    Runs() = default;
    __device__ __forceinline__ Runs(int total, int warps) : total(total) {
        busy = total == 0 ? 0 : max(1, min(warps, total / MIN_COST));       // a share is at least MIN_COST: a tile
        share = busy > 0 ? (int)((unsigned)total / (unsigned)busy) : 0;
        more = total - share * busy;
    }
    __device__ __forceinline__ int begin(int w) const { return w >= busy ? total : w * share + min(w, more); }
    __device__ __forceinline__ int owner(int pos) const {
        const int longer = more * (share + 1);
        return pos < longer ? pos / (share + 1) : more + (pos - longer) / share;
    }
};

// Where a warp stands in the tiles of all units.
struct Cursor {
    int b, hk, group, tile, tiles, len;
};

// The transpose of an 8 x 8 matrix of 16-bit elements in a warp's registers.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// HT: column tiles of 8 query heads.  VEC: rows of 16-byte words; without it every element is a guarded 2-byte load that the
// warp waits for (16 sequences of 4000 keys, 32 / 8 heads of 128: 49 us, one element off 575, heads of 100 channels 430).
template <typename T, int D, bool VEC, bool BIAS, int HT>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) attn_kernel(const __grid_constant__ AttnParams p) {
    using S = Smem<T, D>;
    constexpr int KEYS = S::KEYS, CPR = D / 8, RPP = 32 / CPR, PASSES = KEYS / RPP;      // 16-byte chunks of a row, rows a warp copies at once
    constexpr int MT = D / 16, KT = KEYS / 16;              // row tiles of the output, of the scores
    extern __shared__ __align__(16) unsigned char raw[];
    S &sm = *reinterpret_cast<S *>(raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
    const int warps = gridDim.x * WARPS, me = blockIdx.x * WARPS + warp;
    sm100::grid_trigger();
    if (BIAS) {
        for (int k = tid; k < p.borders.side - 1; k += THREADS) sm.borders[k] = p.borders.at[k];
        __syncthreads();
        for (int n = tid; n < NEAR; n += THREADS) sm.bucket[n] = (uint8_t)relbias::bucket_of_distance(sm.borders, p.borders.side, n);
        __syncthreads();
    }
    sm100::grid_wait();         // the launch may overlap the end of what ran before; nothing of that has been read so far
    auto tiles_of = [](int len) { return (len + KEYS - 1) / KEYS; };
    auto cost_of = [&](int tiles) { return tiles > 0 ? tiles + UNIT_COST : 0; };

    Cursor at{}, to{};          // of the tile that is computed, of the tile whose table entries are fetched next
    Runs runs{};
    int n;
    bool merge;                 // the warps' parts are added up in the CTA
    if (p.direct) {
        // one CTA's unit; its warps take every fourth tile
        at.b = (int)fdiv(blockIdx.x, p.by_units);
        const int unit = (int)blockIdx.x - at.b * p.units;
        at.len = live_length(p, at.b, unit == 0);
        at.tiles = tiles_of(at.len);
        at.hk = (int)fdiv((uint32_t)unit, p.by_groups);
        at.group = unit - at.hk * p.groups;
        at.tile = warp;
        n = at.tiles > warp ? (at.tiles - warp + WARPS - 1) / WARPS : 0;
        merge = true;
    } else {
        // cost of a head's units before each sequence: every thread sums a run of sequences, then the runs are added up
        const int chunk = (p.B + THREADS - 1) / THREADS, b0 = min(tid * chunk, p.B), b1 = min(b0 + chunk, p.B);
        int upto = 0, filled = 0;                               // cost; sequences with a token
        for (int b = b0; b < b1; ++b) {
            const int tiles = tiles_of(live_length(p, b, blockIdx.x == 0));
            upto += cost_of(tiles);
            filled += tiles > 0;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o), y = __shfl_up_sync(0xffffffffu, filled, o);
            if (lane >= o) {
                upto += x;
                filled += y;
            }
        }
        sm.upto[tid] = upto;
        sm.filled[tid] = filled;
        __syncthreads();
        int all = 0, all_filled = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            all += sm.upto[w * 32 + 31];
            all_filled += sm.filled[w * 32 + 31];
        }
        runs = Runs(all * p.units, warps);
        // Where the CTA's runs begin and end, a lane per boundary, every warp for itself: the thread whose sequences hold
        // the boundary by bisection, then the sequence.  A unit's cost comes before its tiles.
        const int pos = runs.begin((int)blockIdx.x * WARPS + min(lane, WARPS));
        int tiles_before = (all - all_filled * UNIT_COST) * p.units;    // of all units
        int b_at = p.B, unit_at = 0, tile_at = 0, len_at = 0;
        if (pos < runs.total) {
            const int cost_at = (int)((unsigned)pos / (unsigned)p.units);
            int t = 0, before = 0, filled_before = 0;
#pragma unroll
            for (int w = 0; w < WARPS - 1; ++w)
                if (t == w * 32 && cost_at >= before + sm.upto[w * 32 + 31]) {
                    before += sm.upto[w * 32 + 31];
                    filled_before += sm.filled[w * 32 + 31];
                    t += 32;
                }
            int in_warp = 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
                if (cost_at >= before + sm.upto[t + in_warp + o - 1]) in_warp += o;
            if (in_warp > 0) {
                before += sm.upto[t + in_warp - 1];
                filled_before += sm.filled[t + in_warp - 1];
            }
            t += in_warp;
            for (int b = t * chunk; b < min((t + 1) * chunk, p.B); ++b) {
                const int len = live_length(p, b, false), tiles = tiles_of(len), cost = cost_of(tiles);
                if (cost_at < before + cost) {
                    const int in = pos - before * p.units;
                    b_at = b;
                    len_at = len;
                    unit_at = (int)((unsigned)in / (unsigned)cost);
                    tile_at = max(in - unit_at * cost - UNIT_COST, 0);
                    tiles_before = (before - filled_before * UNIT_COST) * p.units + unit_at * tiles + tile_at;
                    break;
                }
                before += cost;
                filled_before += tiles > 0;
            }
        }
        auto of = [](int x, int boundary) { return __shfl_sync(0xffffffffu, x, boundary); };
        merge = of(b_at, 0) < p.B && of(b_at, 0) == of(b_at, WARPS) && of(unit_at, 0) == of(unit_at, WARPS);
        n = of(tiles_before, warp + 1) - of(tiles_before, warp);
        if (tid == 0) {
            sm.unit = unit_at;
            sm.tile = tile_at;
        }
        if (lane == 0) reinterpret_cast<Header *>(p.work)[me].last = -1;
        at.b = of(b_at, warp);
        at.len = of(len_at, warp);
        at.tile = of(tile_at, warp);
        at.tiles = tiles_of(at.len);
        const int unit = of(unit_at, warp);
        at.hk = (int)fdiv((uint32_t)unit, p.by_groups);
        at.group = unit - at.hk * p.groups;
    }
    to = at;
    auto advance = [&](Cursor &c) {
        c.tile += p.direct ? WARPS : 1;
        if (p.direct || c.tile < c.tiles) return;
        c.tile = 0;
        if (++c.group < p.groups) return;
        c.group = 0;
        if (++c.hk < p.Hkv) return;
        c.hk = 0;
        for (++c.b; c.b < p.B; ++c.b) {
            c.len = live_length(p, c.b, false);
            c.tiles = tiles_of(c.len);
            if (c.tiles > 0) return;
        }
    };

    // Loading a tile takes three steps, a tile apart: a lane fetches the table entry of one key, works out where its row
    // (of keys and of values; of one of them where there are 16 keys) lies and leaves that in shared memory, and then
    // all lanes copy the rows, 16 bytes each.
    const int my_key = lane % KEYS;
    struct Fetched {
        int entry, slot, hk;        // slot -1: past the sequence
    };
    uint32_t live[STAGES + 1] = {};             // which of the keys of tile i, i + 1, ... there are
    auto fetch = [&]() {
        Fetched f{-1, -1, to.hk};
        const int key = to.tile * KEYS + my_key;
        if (key < to.len) {
            int index;
            split_position(p.view, (uint32_t)key, index, f.slot);
            f.entry = p.view.table[(int64_t)to.b * p.view.table_stride + index];
        }
        advance(to);
        return f;
    };
    auto find = [&](const Fetched &f, int i) {
        const bool ok = f.slot >= 0 && page_ok(p.view, f.entry);
        if (f.slot >= 0 && !ok) g_attn_status = 1;
        typename S::Row &row = sm.row[warp][i & 1][my_key];
        if (KEYS == 32 || lane < KEYS)
            row.k = ok ? reinterpret_cast<const T *>(p.k) + (f.entry * p.k_sp + f.slot * p.k_ss + f.hk * p.k_sh) : nullptr;
        if (KEYS == 32 || lane >= KEYS)
            row.v = ok ? reinterpret_cast<const T *>(p.v) + (f.entry * p.v_sp + f.slot * p.v_ss + f.hk * p.v_sh) : nullptr;
        return __ballot_sync(0xffffffffu, ok);
    };
    constexpr uint32_t ALL = 0xffffffffu;       // the keys of a whole tile (those of 16 are there twice)
    auto load = [&](int i, uint32_t there) {
        typename S::Stage &st = sm.ring[warp][i % STAGES];
        const int part = lane % CPR, c = part * 8;
        const typename S::Row *row = sm.row[warp][i & 1] + lane / CPR;
        auto to = [&](int j) { return (j * RPP + lane / CPR) * D + (part ^ ((j * RPP + lane / CPR) & 7)) * 8; };
        if (VEC && there == ALL && p.d == D) {
#pragma unroll
            for (int j = 0; j < PASSES; ++j) {
                const typename S::Row from = row[j * RPP];
                cp16(st.k + to(j), from.k + c);
                cp16(st.v + to(j), from.v + c);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < PASSES; ++j) {
            const typename S::Row from = row[j * RPP];
            T *kd = st.k + to(j), *vd = st.v + to(j);
            if constexpr (VEC) {
                const bool in = from.k && c < p.d;
                cp16(kd, in ? from.k + c : p.k, in);
                cp16(vd, in ? from.v + c : p.v, in);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool in = from.k && c + e < p.d;
                    kd[e] = in ? from.k[c + e] : from_f32<T>(0.f);
                    vd[e] = in ? from.v[c + e] : from_f32<T>(0.f);
                }
            }
        }
    };
    // Keys are the rows of the scores and channels the rows of the output, heads the columns of both: few heads leave no
    // rows empty.  A lane has the heads 8 h + 2 tq and the next one.
    uint32_t bq[D / 16][HT][2];         // the unit's queries as B fragments, heads past the group and channels past d as zeros
    float o[MT][HT][4];
    float m_ref[HT][2], l_sum[HT][2];
    auto clear = [&]() {
#pragma unroll
        for (int h = 0; h < HT; ++h) {
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][h][e] = 0.f;
            m_ref[h][0] = m_ref[h][1] = -INFINITY;
            l_sum[h][0] = l_sum[h][1] = 0.f;
        }
    };
    clear();                            // a warp without a tile has its part in a unit's end too
    bool whole = false;                 // the unit's first tile was in this run
    const int mi = lane >> 3, mr = lane & 7;

    auto read_queries = [&]() {
        const int row0 = at.group * ROWS, rows = min(ROWS, p.G - row0);
        const T *qg = reinterpret_cast<const T *>(p.q) + (int64_t)at.b * p.q_sb + (int64_t)(at.hk * p.G + row0) * p.q_sh;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = h * 8 + gq, c = kk * 16 + e * 8 + tq * 2;
                    uint32_t x = 0u;
                    if constexpr (VEC) {
                        if (r < rows && c < p.d) x = *reinterpret_cast<const uint32_t *>(qg + (int64_t)r * p.q_sh + c);
                    } else if (r < rows) {
                        const T *qr = qg + (int64_t)r * p.q_sh + c;
                        x = attn::Mma<T>::pack(c < p.d ? to_f32<T>(qr[0]) : 0.f, c + 1 < p.d ? to_f32<T>(qr[1]) : 0.f);
                    }
                    bq[kk][h][e] = x;
                }
    };

    // A unit's end: the lanes' sums are added up, its numbers written as a part.
    auto add_lanes = [&]() {
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int x = 4; x < 32; x *= 2) l_sum[h][e] += __shfl_xor_sync(0xffffffffu, l_sum[h][e], x);
    };
    auto store_part = [&](float *to_o, float *to_m, int rows) {
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = h * 8 + tq * 2 + e;
                if (row >= rows) continue;
                if (gq == 0) {
                    to_m[row] = m_ref[h][e];
                    to_m[ROWS + row] = l_sum[h][e];
                }
#pragma unroll
                for (int j = 0; j < MT; ++j)
#pragma unroll
                    for (int r = 0; r < 2; ++r) to_o[row * D + j * 16 + r * 8 + gq] = o[j][h][r * 2 + e] * WeightScale<T>::DOWN;
            }
    };

    static_assert(STAGES == 3, "the steps below are three tiles long");
    Fetched next{-1, -1, 0};            // of tile i + STAGES once tile i is computed
    if (n > 0) {
        Fetched f[STAGES];              // the first tiles' entries together: one wait
#pragma unroll
        for (int i = 0; i < STAGES; ++i)
            if (i < n) f[i] = fetch();
        if (STAGES < n) next = fetch();
        read_queries();
#pragma unroll
        for (int i = 0; i < STAGES; ++i) {
            if (i < n) {
                live[i] = find(f[i], i);
                __syncwarp();
                if (i < STAGES - 1) load(i, live[i]);
                __syncwarp();           // the third tile's rows go where the first one's were
            }
            if (i < STAGES - 1) asm volatile("cp.async.commit_group;" ::: "memory");
        }
    }

    const int last_border = BIAS && p.borders.side > 1 ? p.borders.at[p.borders.side - 2] : 0;
    for (int i = 0; i < n; ++i) {
        const int row0 = at.group * ROWS, rows = min(ROWS, p.G - row0);
        const int h0 = at.hk * p.G + row0;              // query head of row 0
        if (i == 0 || at.tile == 0) {
            whole = at.tile == 0;
            if (i > 0) {
                read_queries();
                clear();
            }
        }
        // The position bias, read while the tile is on its way and converted when it is used: a conversion behind each
        // read would make the reads wait for one another (1.0 us of 16 sequences of up to 1500 tokens; the buckets of
        // near distances are looked up, to search for them would cost 1.2 us).
        uint32_t add[BIAS ? KT : 1][HT][4];
        if constexpr (BIAS) {
            const int far = max(at.len - 1 - (at.tile * KEYS + my_key), 0);
            const int bucket = far < NEAR ? sm.bucket[far] : far >= last_border ? p.borders.side - 1
                                                                 : relbias::bucket_of_distance(sm.borders, p.borders.side, far);
            auto read_bias = [&](auto *w) {
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int64_t w_at = __shfl_sync(0xffffffffu, bucket, t * 16 + r * 8 + gq) * p.w_sk + (h0 + tq * 2) * p.w_sh;
#pragma unroll
                        for (int h = 0; h < HT; ++h)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                add[t][h][r * 2 + e] = h * 8 + tq * 2 + e < rows ? w[w_at + (h * 8 + e) * p.w_sh] : 0u;
                    }
            };
            if (p.w_dtype == RGD_F32) read_bias(reinterpret_cast<const uint32_t *>(p.w));
            else read_bias(reinterpret_cast<const uint16_t *>(p.w));
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();                   // this tile has landed; all lanes are done with the tile before it
        if (i + STAGES - 1 < n) load(i + STAGES - 1, live[STAGES - 1]);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (i + STAGES < n) {
            live[STAGES] = find(next, i + STAGES);
            if (i + STAGES + 1 < n) next = fetch();
        }
        const typename S::Stage &st = sm.ring[warp][i % STAGES];

        float s[KT][HT][4], s2[KT][HT][4];      // two sums, of every other 16 channels: shorter chains
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][h][e] = s2[t][h][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                uint32_t a[4];
                attn::ldmatrix_x4(a, st.k + (t * 16 + (mi & 1) * 8 + mr) * D + ((kk * 2 + (mi >> 1)) ^ mr) * 8);
#pragma unroll
                for (int h = 0; h < HT; ++h) attn::Mma<T>::mma(kk % 2 ? s2[t][h] : s[t][h], a, bq[kk][h][0], bq[kk][h][1]);
            }
        if constexpr (BIAS) {
            if (p.w_dtype != RGD_F32)
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int h = 0; h < HT; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            add[t][h][e] = p.w_dtype == RGD_BF16 ? add[t][h][e] << 16
                                                                 : __float_as_uint(__half2float(__ushort_as_half((uint16_t)add[t][h][e])));
        }
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[t][h][e] = (s[t][h][e] + s2[t][h][e]) * p.scale_log2;
                    if constexpr (BIAS) s[t][h][e] += attn::bias_log2<float>(__uint_as_float(add[t][h][e]));
                }
        if (live[0] != ALL)
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!(live[0] >> (t * 16 + (e >> 1) * 8 + gq) & 1))
#pragma unroll
                        for (int h = 0; h < HT; ++h) s[t][h][e] = -INFINITY;
        float mx[HT][2];
        bool more = false;
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mx[h][e] = fmaxf(s[0][h][e], s[0][h][2 + e]);
#pragma unroll
                for (int t = 1; t < KT; ++t) mx[h][e] = fmaxf(mx[h][e], fmaxf(s[t][h][e], s[t][h][2 + e]));
                more |= mx[h][e] > m_ref[h][e];
            }
        // the reference follows the maximum: a new one gets rare along the keys
        if (__any_sync(0xffffffffu, more)) {
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) mx[h][e] = fmaxf(mx[h][e], __shfl_xor_sync(0xffffffffu, mx[h][e], x));
                    const bool higher = mx[h][e] > m_ref[h][e];
                    const float alpha = !higher ? 1.f : m_ref[h][e] == -INFINITY ? 0.f : ex2(m_ref[h][e] - mx[h][e]);
                    if (higher) m_ref[h][e] = mx[h][e];
                    l_sum[h][e] *= alpha;
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        o[j][h][e] *= alpha;
                        o[j][h][2 + e] *= alpha;
                    }
                }
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            uint32_t hi[HT][2], lo[HT][2];
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float pr[2], rest[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        pr[e] = ex2(s[t][h][r * 2 + e] - (m_ref[h][e] == -INFINITY ? 0.f : m_ref[h][e]));
                        l_sum[h][e] += pr[e];
                        pr[e] *= WeightScale<T>::UP;
                        rest[e] = pr[e] - round_to<T>(pr[e]);
                    }
                    hi[h][r] = transposed(attn::Mma<T>::pack(pr[0], pr[1]));
                    lo[h][r] = transposed(attn::Mma<T>::pack(rest[0], rest[1]));
                }
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                uint32_t a[4];
                attn::ldmatrix_x4_trans(a, st.v + (t * 16 + (mi >> 1) * 8 + mr) * D + ((j * 2 + (mi & 1)) ^ mr) * 8);
#pragma unroll
                for (int h = 0; h < HT; ++h) {
                    // 16 keys from zero on, then added: the matrix unit cuts its sums off (see above)
                    float y[4] = {0.f, 0.f, 0.f, 0.f};
                    attn::Mma<T>::mma(y, a, hi[h][0], hi[h][1]);
                    attn::Mma<T>::mma(y, a, lo[h][0], lo[h][1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][h][e] += y[e];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < STAGES; ++j) live[j] = live[j + 1];

        const bool done = at.tile == at.tiles - 1;
        if (!p.direct && (done || i == n - 1)) {
            add_lanes();
            if (done && whole) {
#pragma unroll
                for (int h = 0; h < HT; ++h) {
                    float inv[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int row = h * 8 + tq * 2 + e;
                        inv[e] = l_sum[h][e] == 0.f ? 0.f : WeightScale<T>::DOWN / l_sum[h][e];
                        if (p.lse && gq == 0 && row < rows)
                            p.lse[(int64_t)at.b * p.Hq + h0 + row] = l_sum[h][e] == 0.f ? -INFINITY : (m_ref[h][e] + log2f(l_sum[h][e])) * LN2;
                    }
                    // a head's two neighbouring channels, for one store; all lanes take part in the transposes
                    uint32_t y[MT][2];
#pragma unroll
                    for (int j = 0; j < MT; ++j)
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                            y[j][r] = transposed(attn::Mma<T>::pack(o[j][h][r * 2] * inv[0], o[j][h][r * 2 + 1] * inv[1]));
                    __syncwarp();
                    if (h * 8 + gq < rows) {
                        T *out = reinterpret_cast<T *>(p.o) + (int64_t)at.b * p.o_sb + (int64_t)(h0 + h * 8 + gq) * p.o_sh;
#pragma unroll
                        for (int j = 0; j < MT; ++j)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const int c = j * 16 + r * 8 + tq * 2;
                                if constexpr (VEC) {
                                    if (c < p.d) *reinterpret_cast<uint32_t *>(out + c) = y[j][r];
                                } else {
                                    const uint16_t y0 = (uint16_t)y[j][r], y1 = (uint16_t)(y[j][r] >> 16);
                                    if (c < p.d) reinterpret_cast<uint16_t *>(out)[c] = y0;
                                    if (c + 1 < p.d) reinterpret_cast<uint16_t *>(out)[c + 1] = y1;
                                }
                            }
                    }
                    __syncwarp();
                }
            } else if (!merge) {
                float *part = part_of(p, warps, D, me, whole ? 1 : 0);
                store_part(part + 2 * ROWS, part, rows);
            }
            if (!done && whole && lane == 0) {
                // this run ends before the tiles that are left of the unit
                Header &head = reinterpret_cast<Header *>(p.work)[me];
                head.last = runs.owner(runs.begin(me + 1) - 1 + (at.tiles - 1 - at.tile));
                head.merged = merge;
                head.b = at.b;
                head.hk = at.hk;
                head.row0 = row0;
            }
        }
        advance(at);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    if (merge) {                // uniform over the CTA; the rings are done with
        float *mine_o = reinterpret_cast<float *>(sm.ring[warp]), *mine_m = mine_o + ROWS * D;       // then the sums
        static_assert(sizeof(sm.ring[0]) >= part_floats(D) * sizeof(float), "a part in a warp's ring");
        if (p.direct) add_lanes();      // a run's end has done it otherwise
        __syncwarp();
        store_part(mine_o, mine_m, ROWS);
        __syncthreads();
        // the CTA's unit, which a warp without a tile knows from the schedule alone
        int hk = at.hk, group = at.group;
        if (!p.direct) {
            hk = (int)fdiv((uint32_t)sm.unit, p.by_groups);
            group = sm.unit - hk * p.groups;
        }
        const int rows = min(ROWS, p.G - group * ROWS), h0 = hk * p.G + group * ROWS;
        float *part = p.direct ? nullptr : part_of(p, warps, D, blockIdx.x * WARPS, sm.tile == 0 ? 1 : 0);
        for (int e = tid; e < rows * (D / 4); e += THREADS) {
            const int row = e / (D / 4), c = e % (D / 4) * 4;
            const float *from[WARPS];
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                from[w] = reinterpret_cast<const float *>(sm.ring[w]);
                m = fmaxf(m, from[w][ROWS * D + row]);
            }
            const float mu = m == -INFINITY ? 0.f : m;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float f = ex2(from[w][ROWS * D + row] - mu);
                const float4 x = *reinterpret_cast<const float4 *>(from[w] + row * D + c);
                l = fmaf(from[w][ROWS * D + ROWS + row], f, l);
                y.x = fmaf(x.x, f, y.x); y.y = fmaf(x.y, f, y.y);
                y.z = fmaf(x.z, f, y.z); y.w = fmaf(x.w, f, y.w);
            }
            if (!p.direct) {
                *reinterpret_cast<float4 *>(part + 2 * ROWS + row * D + c) = y;
                if (c == 0) {
                    part[row] = m;
                    part[ROWS + row] = l;
                }
                continue;
            }
            const float inv = l == 0.f ? 0.f : 1.f / l, z[4] = {y.x * inv, y.y * inv, y.z * inv, y.w * inv};
            T *out = reinterpret_cast<T *>(p.o) + (int64_t)at.b * p.o_sb + (int64_t)(h0 + row) * p.o_sh + c;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (c + k < p.d) out[k] = from_f32<T>(z[k]);
            if (c == 0 && p.lse) p.lse[(int64_t)at.b * p.Hq + h0 + row] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
        }
    }

    // sequences without a token
    for (int b = blockIdx.x; !p.direct && b < p.B; b += gridDim.x)
        if (live_length(p, b, false) == 0) {
            T *out = reinterpret_cast<T *>(p.o) + (int64_t)b * p.o_sb;
            for (int e = tid; e < p.Hq * p.d; e += THREADS) {
                const int h = e / p.d;
                out[(int64_t)h * p.o_sh + e - h * p.d] = from_f32<T>(0.f);
            }
            if (p.lse)
                for (int h = tid; h < p.Hq; h += THREADS) p.lse[(int64_t)b * p.Hq + h] = -INFINITY;
        }
}

constexpr int JOIN_THREADS = WARPS * 32;
constexpr int JOIN_FEW = 8;             // parts that one warp adds up by itself

// The parts of a unit: of its first CTA, of the ones in between, of the last one.
struct Parts {
    int first, cta0, cta1, n0, n1, n;
    __device__ __forceinline__ Parts(const Header &head, int first) : first(first), cta0(first / WARPS), cta1(head.last / WARPS) {
        const bool one = cta0 == cta1;
        n0 = one ? head.last - first + 1 : head.merged ? 1 : WARPS - first % WARPS;
        n1 = max(cta1 - cta0 - 1, 0);
        n = n0 + n1 + (one ? 0 : head.last % WARPS + 1);
    }
    __device__ __forceinline__ int warp(int i) const {
        return i < n0 ? first + i : i < n0 + n1 ? (cta0 + 1 + i - n0) * WARPS : cta1 * WARPS + i - n0 - n1;
    }
};
// A row's maximum, sum and four channels of its output, so far.
struct Joined {
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    __device__ __forceinline__ void rescale(float m_new) {
        const float f = ex2(m - (m_new == -INFINITY ? 0.f : m_new));
        l *= f;
        acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
        m = m_new;
    }
    __device__ __forceinline__ void add(float pm, float pl, const float4 &x) {          // pm <= m
        const float f = ex2(pm - (m == -INFINITY ? 0.f : m));
        l = fmaf(pl, f, l);
        acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y);
        acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
    }
    // parts i0, i0 + step, ..., U at a time
    template <int U>
    __device__ __forceinline__ void add_parts(const AttnParams &p, int warps, int D, const Parts &parts, int row, int quad, int i0, int step) {
        for (; i0 < parts.n; i0 += U * step) {
            float pm[U], pl[U], m_new = m;
            float4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * step;
                pm[u] = -INFINITY;
                pl[u] = 0.f;
                x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < parts.n) {
                    const float *from = part_of(p, warps, D, parts.warp(i), i == 0 ? 1 : 0);
                    pm[u] = from[row];
                    pl[u] = from[ROWS + row];
                    x[u] = *reinterpret_cast<const float4 *>(from + 2 * ROWS + row * D + quad * 4);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) m_new = fmaxf(m_new, pm[u]);
            rescale(m_new);
#pragma unroll
            for (int u = 0; u < U; ++u) add(pm[u], pl[u], x[u]);
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(const AttnParams &p, const Header &head, int row, int quad) const {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int h = head.hk * p.G + head.row0 + row;
        T *out = reinterpret_cast<T *>(p.o) + (int64_t)head.b * p.o_sb + (int64_t)h * p.o_sh;
        const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (quad * 4 + e < p.d) out[quad * 4 + e] = from_f32<T>(y[e]);
        if (p.lse && quad == 0) p.lse[(int64_t)head.b * p.Hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
    }
};

// Adds the parts of the units that begin in the runs of the attention's CTA blockIdx.x and end in other warps'; one CTA
// per row.  Units of few parts are a warp's, one each; the others are taken by the CTA, one after another.
template <typename T, int D>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ AttnParams p) {
    constexpr int QUADS = D / 4, GROUPS = JOIN_THREADS / QUADS;
    __shared__ float m_s[GROUPS], l_s[GROUPS];
    __shared__ float4 acc_s[GROUPS][QUADS];
    const int tid = threadIdx.x, quad = tid % QUADS, grp = tid / QUADS, row = blockIdx.y, warps = gridDim.x * WARPS;
    sm100::grid_trigger();
    sm100::grid_wait();
    const Header *heads = reinterpret_cast<const Header *>(p.work) + blockIdx.x * WARPS;
    auto there = [&](const Header &head) { return head.last >= 0 && row < min(ROWS, p.G - head.row0); };
    bool many = false;
    const Header mine = heads[tid / 32];
    if (there(mine)) {
        const Parts parts(mine, blockIdx.x * WARPS + tid / 32);
        many = parts.n > JOIN_FEW;
        if (!many && tid % 32 < QUADS) {
            Joined sum;
            sum.add_parts<JOIN_FEW>(p, warps, D, parts, row, tid % 32, 0, 1);
            sum.store<T>(p, mine, row, tid % 32);
        }
    }
    if (!__syncthreads_or(many)) return;
    for (int w = 0; w < WARPS; ++w) {
        const Header head = heads[w];
        if (!there(head)) continue;
        const Parts parts(head, blockIdx.x * WARPS + w);
        if (parts.n <= JOIN_FEW) continue;
        Joined sum;
        sum.add_parts<4>(p, warps, D, parts, row, quad, grp, GROUPS);
        if (quad == 0) {
            m_s[grp] = sum.m;
            l_s[grp] = sum.l;
        }
        acc_s[grp][quad] = sum.acc;
        __syncthreads();
        if (grp == 0) {                 // the groups' sums in order
            float m = sum.m;
#pragma unroll
            for (int g = 1; g < GROUPS; ++g) m = fmaxf(m, m_s[g]);
            sum.rescale(m);
#pragma unroll
            for (int g = 1; g < GROUPS; ++g) sum.add(m_s[g], l_s[g], acc_s[g][quad]);
            sum.store<T>(p, head, row, quad);
        }
        __syncthreads();                // the next unit's parts go to the same shared memory
    }
}

// Costs are 32-bit.
bool too_large(int64_t B, int64_t units, int64_t max_keys, int D) {
    return (double)B * (double)units * (double)(ceil_div64(max_keys, tile_keys(D)) + UNIT_COST) > (double)INT32_MAX;
}

// How the tiles are spread.  Few units of few keys (by what the table has room for; the lengths are not known here): a CTA
// per unit, which needs no schedule, no workspace and no second launch.  Others: what the SMs hold at once, and no more
// CTAs than there can be runs.  us of a call, many in a row over different caches, a CTA per unit / equal runs, all
// sequences as long as the table or of 16 keys up to that (even over the logarithm), at 8, 16, 24, 32, 48 tiles:
//   16 units, head_dim 64       5.1 / 8.7     7.2 / 9.4     9.9 / 10.0   12.4 / 9.4    17.5 / 10.3
//   64 units, head_dim 128      5.9 / 9.3     8.4 / 10.6   11.0 / 11.5   13.5 / 11.3   18.3 / 12.5
//   148 units, head_dim 128     6.1 / 10.2    8.5 / 11.6   11.0 / 13.3   13.4 / 15.5   18.1 / 18.6
//     mixed lengths             5.4 / 9.8     7.7 / 11.1   10.4 / 11.3   12.7 / 10.9   17.1 / 11.4
//   256 units, head_dim 64      7.0 / 10.8    9.7 / 12.8   13.3 / 16.5   16.3 / 19.2   22.2 / 24.7
//     mixed lengths             5.6 / 9.5     7.7 / 9.6    11.2 / 11.4   13.3 / 11.3   18.5 / 12.8
//   512 units, head_dim 128    13.2 / 14.9   18.8 / 19.8   25.1 / 25.7   30.3 / 31.1   40.8 / 41.4
//     mixed lengths            10.3 / 11.4   12.6 / 12.7   16.7 / 15.4   19.6 / 15.2   18.9 / 16.8
// Few units and mixed lengths are even at about 25 tiles whatever the units, so one limit serves all; many units of one
// length would gain 2-3 us from a CTA each up to 50 tiles, but no call says that its lengths are alike.
constexpr int DIRECT_TILES = 28;
struct Plan {
    bool direct;
    int grid;
};
Plan make_plan(int64_t B, int64_t units, int64_t max_keys, int D) {
    const int64_t tiles = ceil_div64(max_keys, tile_keys(D));
    const int64_t room = (int64_t)num_sms() * CTAS_PER_SM;
    if (tiles <= DIRECT_TILES && B * units <= room) return {true, (int)(B * units)};
    const int64_t n = ceil_div64(B * units * (tiles + UNIT_COST), MIN_COST * WARPS);
    return {false, (int)(n < 1 ? 1 : n < room ? n : room)};
}

template <typename T, int D, bool VEC, bool BIAS>
int launch(AttnParams &p, const Plan &plan, cudaStream_t st) {
    auto kernel = p.G <= 8 ? attn_kernel<T, D, VEC, BIAS, 1> : attn_kernel<T, D, VEC, BIAS, 2>;
    constexpr size_t smem = sizeof(Smem<T, D>);
    static_assert(CTAS_PER_SM * (smem + 1024) <= 228 << 10, "shared memory of an SM");
    if (int e = ensure_dyn_smem(reinterpret_cast<const void *>(kernel), smem)) return e;
    if (int e = sm100::launch_pdl(kernel, dim3(plan.grid), THREADS, smem, st, p)) return e;
    if (plan.direct) return RGD_OK;
    return sm100::launch_pdl(join_kernel<T, D>, dim3(plan.grid, (unsigned)(p.G < ROWS ? p.G : ROWS)), JOIN_THREADS, 0, st, p);
}
template <typename T, int D>
int launch(AttnParams &p, bool vec, const Plan &plan, cudaStream_t st) {
    if (p.w) return vec ? launch<T, D, true, true>(p, plan, st) : launch<T, D, false, true>(p, plan, st);
    return vec ? launch<T, D, true, false>(p, plan, st) : launch<T, D, false, false>(p, plan, st);
}

int status_fetch() {
    const int append = append_status_fetch();
    int v = 0;
    if (append < 0 || cudaMemcpyFromSymbol(&v, g_attn_status, sizeof(int)) != cudaSuccess) {
        (void)cudaGetLastError();
        return -1;
    }
    if (v != 0) {
        const int zero = 0;
        (void)cudaMemcpyToSymbol(g_attn_status, &zero, sizeof(int));
    }
    return append | v;
}

}  // namespace paged
}  // namespace rgd

using namespace rgd;

extern "C" int64_t rgd_paged_attn_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t d, int64_t max_pages, int64_t page_size) {
    if (B < 0 || Hq < 0 || Hkv < 0 || d < 0 || max_pages < 0 || page_size < 1) return RGD_E_INVALID;
    if (Hkv == 0 || Hq % Hkv != 0) return Hq == 0 ? 0 : RGD_E_INVALID;
    if (d > 128 || B > 1 << 30 || Hq > 65535 || max_pages > INT32_MAX || page_size > INT32_MAX) return RGD_E_SIZE;
    const int D = d > 64 ? 128 : 64;
    const int64_t units = Hkv * ceil_div64(Hq / Hkv, paged::ROWS);
    if (paged::too_large(B, units, max_pages * page_size, D)) return RGD_E_SIZE;
    const paged::Plan plan = paged::make_plan(B, units, max_pages * page_size, D);
    return plan.direct ? 0 : paged::workspace_bytes(plan.grid, D);
}

extern "C" int rgd_paged_attn(const rgd_heads *q, const rgd_paged *cache, const rgd_relbias *bias, const rgd_heads *o, float *lse,
                              int64_t B, int64_t Hq, int64_t Hkv, int64_t d, float softmax_scale, int dtype, void *workspace,
                              int64_t workspace_bytes, void *stream) {
    if (!q || !o) return RGD_E_NULL;
    if (dtype != RGD_F16 && dtype != RGD_BF16) return RGD_E_DTYPE;
    if (B < 0 || Hq < 0 || Hkv < 0 || d < 0) return RGD_E_INVALID;
    if (d > 128 || B > 1 << 30 || Hq > 65535) return RGD_E_SIZE;
    if (Hq > 0 && (Hkv == 0 || Hq % Hkv != 0)) return RGD_E_INVALID;
    if (int e = paged::check_paged(cache, B, Hkv > 0 && d > 0)) return e;
    if (bias)
        if (int e = relbias::check(bias)) return e;
    if (B == 0 || Hq == 0 || d == 0) return RGD_OK;
    if (!q->ptr || !o->ptr || (bias && !bias->weight)) return RGD_E_NULL;
    paged::AttnParams p{};
    p.view = paged::make_view(*cache);
    p.lengths = cache->lengths;
    p.q = q->ptr; p.q_sb = q->stride_b; p.q_sh = q->stride_h;
    p.k = cache->k; p.k_sp = cache->k_stride_p; p.k_ss = cache->k_stride_s; p.k_sh = cache->k_stride_h;
    if (!p.k || !cache->v) p.k = q->ptr;            // no page: an address that no copy reads from
    p.v = cache->v ? cache->v : p.k; p.v_sp = cache->v_stride_p; p.v_ss = cache->v_stride_s; p.v_sh = cache->v_stride_h;
    p.o = o->ptr; p.o_sb = o->stride_b; p.o_sh = o->stride_h;
    p.lse = lse;
    p.B = (int)B; p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.G = (int)(Hq / Hkv); p.d = (int)d;
    p.scale_log2 = softmax_scale * paged::LOG2E;
    if (bias) {
        p.w = bias->weight; p.w_sk = bias->stride_bucket; p.w_sh = bias->stride_head; p.w_dtype = bias->dtype;
        p.borders = relbias::make_borders(*bias);
    }
    p.groups = (p.G + paged::ROWS - 1) / paged::ROWS;
    p.units = p.Hkv * p.groups;
    p.by_units = make_fastdiv((uint32_t)p.units);
    p.by_groups = make_fastdiv((uint32_t)p.groups);
    const int64_t max_keys = cache->max_pages * cache->page_size;
    const int64_t need = rgd_paged_attn_workspace_bytes(B, Hq, Hkv, d, cache->max_pages, cache->page_size);
    if (need < 0) return (int)need;
    if (need > 0 && (workspace_bytes < need || !workspace)) return RGD_E_WORKSPACE;
    if (need > 0 && !is_aligned(workspace, 16)) return RGD_E_STRIDE;
    p.work = reinterpret_cast<char *>(workspace);
    const bool vec = d % 8 == 0 && paged::cache_vec16(*cache) && paged::heads_vec16(*q) && paged::heads_vec16(*o);
    cudaStream_t st = (cudaStream_t)stream;
    const paged::Plan plan = paged::make_plan(B, p.units, max_keys, d > 64 ? 128 : 64);
    p.direct = plan.direct;
    if (d > 64) return dtype == RGD_BF16 ? paged::launch<__nv_bfloat16, 128>(p, vec, plan, st) : paged::launch<__half, 128>(p, vec, plan, st);
    return dtype == RGD_BF16 ? paged::launch<__nv_bfloat16, 64>(p, vec, plan, st) : paged::launch<__half, 64>(p, vec, plan, st);
}
