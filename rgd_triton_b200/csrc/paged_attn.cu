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
    int groups, units;                      // row tiles of a cache head, of a sequence
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
// Work.  A unit is a sequence, a cache head and up to 16 of the query heads that share it (one m16n8k16 row tile);
// its keys come in tiles of 64.  The tiles of all units, one after the other, are dealt out to the CTAs in equal
// runs, whatever the lengths are: each CTA finds its run from the lengths, which are on the device.  A unit that one
// CTA has whole is finished there; of a unit that several have, each leaves its part (row maximum, row sum,
// unnormalised output) in the workspace, and join_kernel adds the parts in order.
//
// A CTA streams its run through a ring of cp.async stages that goes on across units.  Of a tile, each of the four
// warps takes the scores of 16 keys; the row maxima and the weights are exchanged through shared memory, and each
// warp then adds the products with all 64 values for a quarter of the channels, so no partial outputs have to be
// added up between the warps.  Weights are split into two numbers of the cache's type (hi + lo): rounded to one, they
// would cost as much accuracy as the output's own rounding, and the matrix pipe idles anyway.
// ---------------------------------------------------------------------------------------------------------------
constexpr int WARPS = 4, THREADS = WARPS * 32, KEYS = 64, ROWS = 16, STAGES = 3, PLD = KEYS + attn::PAD;
constexpr int MIN_TILES = 1;

template <typename T, int D>
struct Smem {
    static constexpr int LD = D + attn::PAD;            // rows 16 bytes apart from bank to bank: conflict-free ldmatrix
    alignas(16) T k[STAGES][KEYS * LD];
    alignas(16) T v[STAGES][KEYS * LD];
    alignas(16) T p[2][ROWS * PLD];                     // weights, hi and lo
    float mx[2][WARPS][ROWS], l[WARPS][ROWS];
    int64_t row[2][2][KEYS];                            // of the tiles to load next: element offsets of keys, of values; -1: none
    uint8_t live[STAGES][KEYS];                         // the key exists and its page is usable
    int64_t sums[WARPS];
    int64_t before;                                     // tiles before sequence `first`
    int first;
    float bias[1];                                      // [side][ROWS], with a position bias
};

__host__ __device__ constexpr int ctas_per_sm(int D) { return D > 64 ? 2 : 3; }

__device__ __forceinline__ void cp16(void *dst, const void *src, bool valid) {
    // not valid: nothing is read, 16 zero bytes are written
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(valid ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ int tiles_of(int len) { return (len + KEYS - 1) / KEYS; }

// Workspace: per CTA of the grid a header and two parts, [0] of a unit that began in another CTA's run, [1] of one
// that ends in another's.
struct Header {
    int last;                   // the unit of part [1] ends in this CTA; -1: there is none
    int b, hk, row0;
};
__host__ __device__ __forceinline__ int64_t part_floats(int D) { return ROWS * (D + 2); }
__host__ __device__ __forceinline__ int64_t workspace_bytes(int ctas, int D) {
    return (int64_t)ctas * ((int64_t)sizeof(Header) + 2 * part_floats(D) * (int64_t)sizeof(float));
}
__device__ __forceinline__ float *part_of(const AttnParams &p, int ctas, int D, int cta, int which) {
    return reinterpret_cast<float *>(p.work + (int64_t)ctas * sizeof(Header)) + (cta * 2 + which) * part_floats(D);
}

// Where a CTA stands in the tiles of all units.
struct Cursor {
    int b, hk, group, tile, tiles, len;
};

template <typename T, int D, bool VEC, bool BIAS>
__global__ void __launch_bounds__(THREADS, ctas_per_sm(D)) attn_kernel(const __grid_constant__ AttnParams p) {
    using S = Smem<T, D>;
    constexpr int LD = S::LD, CPR = D / 8, RPP = THREADS / CPR, PASSES = KEYS / RPP, NT = D / 4 / 8;
    extern __shared__ __align__(16) unsigned char raw[];
    S &sm = *reinterpret_cast<S *>(raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
    const int ctas = gridDim.x, cta = blockIdx.x;
    sm100::grid_trigger();

    // tiles per head before each sequence: every thread sums a run of sequences, then the runs are added up
    const int chunk = (p.B + THREADS - 1) / THREADS, b0 = min(tid * chunk, p.B), b1 = min(b0 + chunk, p.B);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += tiles_of(live_length(p, b, cta == 0));
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) sm.sums[warp] = upto;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) upto += sm.sums[w];
        all += sm.sums[w];
    }
    const int64_t total = all * p.units;
    const int64_t busy = min((int64_t)ctas, (total + MIN_TILES - 1) / MIN_TILES);      // CTAs with a run
    const int64_t begin = cta < busy ? cta * total / busy : 0, end = cta < busy ? (cta + 1) * total / busy : 0;
    const int n = (int)(end - begin);
    if (n > 0) {
        int64_t before = upto - mine;
        if (begin >= before * p.units && begin < upto * p.units)
            for (int b = b0; b < b1; ++b) {
                const int64_t next = before + tiles_of(live_length(p, b, false));
                if (begin < next * p.units) {
                    sm.first = b;
                    sm.before = before;
                    break;
                }
                before = next;
            }
    }
    __syncthreads();
    if (tid == 0) {
        reinterpret_cast<Header *>(p.work)[cta].last = -1;
    }

    Cursor at{}, to{};          // of the tile that is computed, of the tile whose table entries are fetched next
    if (n > 0) {
        at.b = sm.first;
        at.len = live_length(p, at.b, false);
        at.tiles = tiles_of(at.len);
        const int64_t in = begin - sm.before * p.units;
        const int unit = (int)(in / at.tiles);
        at.tile = (int)(in - (int64_t)unit * at.tiles);
        at.hk = unit / p.groups;
        at.group = unit - at.hk * p.groups;
        to = at;
    }
    auto advance = [&](Cursor &c) {
        if (++c.tile < c.tiles) return;
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

    // Loading a tile takes three steps, a tile apart: a thread fetches the table entry of one key (the lower half of the
    // CTA for keys, the upper one for values), works out where that row lies and leaves it in shared memory, and
    // then all threads copy the rows, 16 bytes each.
    const int my_key = tid % KEYS, my_half = tid / KEYS;
    const int64_t my_sp = my_half ? p.v_sp : p.k_sp, my_ss = my_half ? p.v_ss : p.k_ss, my_sh = my_half ? p.v_sh : p.k_sh;
    struct Fetched {
        int entry, slot, hk;    // entry -1: nothing to read
    };
    auto fetch = [&]() {
        Fetched f{-1, 0, to.hk};
        const int key = to.tile * KEYS + my_key;
        if (key < to.len) {
            int index;
            split_position(p.view, (uint32_t)key, index, f.slot);
            f.entry = p.view.table[(int64_t)to.b * p.view.table_stride + index];
            if (!page_ok(p.view, f.entry)) {
                f.entry = -1;
                g_attn_status = 1;
            }
        }
        advance(to);
        return f;
    };
    auto find = [&](const Fetched &f, int i) {
        sm.row[i & 1][my_half][my_key] = f.entry < 0 ? -1 : f.entry * my_sp + f.slot * my_ss + f.hk * my_sh;
    };
    auto load = [&](int i) {
        const int stage = i % STAGES, c = (tid % CPR) * 8;
        const T *kg = reinterpret_cast<const T *>(p.k) + c, *vg = reinterpret_cast<const T *>(p.v) + c;
#pragma unroll
        for (int j = 0; j < PASSES; ++j) {
            const int r = j * RPP + tid / CPR;
            const int64_t kr = sm.row[i & 1][0][r], vr = sm.row[i & 1][1][r];
            T *kd = sm.k[stage] + r * LD + c, *vd = sm.v[stage] + r * LD + c;
            if constexpr (VEC) {
                const bool in = kr >= 0 && c < p.d;
                cp16(kd, in ? kg + kr : p.k, in);
                cp16(vd, in ? vg + vr : p.v, in);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool in = kr >= 0 && c + e < p.d;
                    kd[e] = in ? kg[kr + e] : from_f32<T>(0.f);
                    vd[e] = in ? vg[vr + e] : from_f32<T>(0.f);
                }
            }
        }
        if (tid < KEYS) sm.live[stage][tid] = sm.row[i & 1][0][tid] >= 0;
    };
    static_assert(STAGES == 3, "the steps below are three tiles long");
    Fetched next{};             // of tile i + STAGES once tile i is computed
    {
        Fetched f[STAGES];
#pragma unroll
        for (int i = 0; i < STAGES; ++i)
            if (i < n) f[i] = fetch();
        if (0 < n) find(f[0], 0);
        if (1 < n) find(f[1], 1);
        __syncthreads();
        if (0 < n) load(0);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (1 < n) load(1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        __syncthreads();
        if (2 < n) find(f[2], 2);
        if (3 < n) next = fetch();
    }

    uint32_t aq[D / 16][4];             // the unit's queries as A fragments, rows past the group and channels past d as zeros
    float o[NT][4];                     // rows gq and gq + 8, this warp's quarter of the channels
    float m_ref[2], l_sum[2];           // the same in all warps; of this warp's keys
    bool whole = false;                 // the unit's first tile was in this run
    const int mi = lane >> 3, mr = lane & 7;

    for (int i = 0; i < n; ++i) {
        const int row0 = at.group * ROWS, rows = min(ROWS, p.G - row0);
        const int h0 = at.hk * p.G + row0;              // query head of row 0
        const bool fresh = i == 0 || at.tile == 0;
        if (fresh) {
            whole = at.tile == 0;
            const T *qg = reinterpret_cast<const T *>(p.q) + (int64_t)at.b * p.q_sb + (int64_t)h0 * p.q_sh;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = gq + (e & 1) * 8, c = kk * 16 + (e >> 1) * 8 + tq * 2;
                    uint32_t x = 0u;
                    if constexpr (VEC) {
                        if (r < rows && c < p.d) x = *reinterpret_cast<const uint32_t *>(qg + (int64_t)r * p.q_sh + c);
                    } else if (r < rows) {
                        const T *qr = qg + (int64_t)r * p.q_sh + c;
                        x = attn::Mma<T>::pack(c < p.d ? to_f32<T>(qr[0]) : 0.f, c + 1 < p.d ? to_f32<T>(qr[1]) : 0.f);
                    }
                    aq[kk][e] = x;
                }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
            m_ref[0] = m_ref[1] = -INFINITY;
            l_sum[0] = l_sum[1] = 0.f;
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncthreads();                // this tile has landed; the tile before it is done with
        if (i + STAGES - 1 < n) load(i + STAGES - 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (i + STAGES < n) {
            find(next, i + STAGES);
            if (i + STAGES + 1 < n) next = fetch();
        }
        if constexpr (BIAS)
            if (fresh) {
                for (int e = tid; e < p.borders.side * ROWS; e += THREADS) {
                    const int r = e % ROWS;
                    sm.bias[e] = r < rows ? attn::bias_log2<float>(load_as_f32(p.w, (e / ROWS) * p.w_sk + (h0 + r) * p.w_sh, p.w_dtype)) : 0.f;
                }
                __syncthreads();
            }
        const int stage = i % STAGES, par = i & 1;
        const T *ks = sm.k[stage] + warp * 16 * LD, *vs = sm.v[stage] + warp * (D / 4);

        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t bf[4];
            attn::ldmatrix_x4(bf, ks + (mr + (mi >> 1) * 8) * LD + kk * 16 + (mi & 1) * 8);
            attn::Mma<T>::mma(s[0], aq[kk], bf[0], bf[1]);
            attn::Mma<T>::mma(s[1], aq[kk], bf[2], bf[3]);
        }
        int bucket = 0;
        if constexpr (BIAS) {
            const int key = at.tile * KEYS + warp * 16 + (lane & 15);
            bucket = relbias::bucket_of_distance(p.borders.at, p.borders.side, max(at.len - 1 - key, 0));
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = t * 8 + tq * 2 + e;
                const bool live = sm.live[stage][warp * 16 + key];
                int bk = 0;
                if constexpr (BIAS) bk = __shfl_sync(0xffffffffu, bucket, key) * ROWS;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float x = s[t][r * 2 + e] * p.scale_log2;
                    if constexpr (BIAS) x += sm.bias[bk + gq + r * 8];
                    x = live ? x : -INFINITY;
                    s[t][r * 2 + e] = x;
                    mx[r] = fmaxf(mx[r], x);
                }
            }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
            if (tq == 0) sm.mx[par][warp][gq + r * 8] = mx[r];
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = gq + r * 8;
            float m_new = m_ref[r];
#pragma unroll
            for (int w = 0; w < WARPS; ++w) m_new = fmaxf(m_new, sm.mx[par][w][row]);
            const float mu = m_new == -INFINITY ? 0.f : m_new, alpha = ex2(m_ref[r] - mu);
            m_ref[r] = m_new;
            l_sum[r] *= alpha;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                o[j][2 * r] *= alpha;
                o[j][2 * r + 1] *= alpha;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const float p0 = ex2(s[t][2 * r] - mu), p1 = ex2(s[t][2 * r + 1] - mu);
                l_sum[r] += p0 + p1;
                const float r0 = round_to<T>(p0), r1 = round_to<T>(p1);
                const int e = row * PLD + warp * 16 + t * 8 + tq * 2;
                *reinterpret_cast<uint32_t *>(&sm.p[0][e]) = attn::Mma<T>::pack(r0, r1);
                *reinterpret_cast<uint32_t *>(&sm.p[1][e]) = attn::Mma<T>::pack(p0 - r0, p1 - r1);
            }
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < KEYS / 16; ++kk) {
            uint32_t hi[4], lo[4];
            attn::ldmatrix_x4(hi, sm.p[0] + (lane & 15) * PLD + kk * 16 + (lane >> 4) * 8);
            attn::ldmatrix_x4(lo, sm.p[1] + (lane & 15) * PLD + kk * 16 + (lane >> 4) * 8);
#pragma unroll
            for (int j = 0; j < NT / 2; ++j) {
                uint32_t bf[4];
                attn::ldmatrix_x4_trans(bf, vs + (kk * 16 + mr + (mi & 1) * 8) * LD + j * 16 + (mi >> 1) * 8);
                attn::Mma<T>::mma(o[2 * j], hi, bf[0], bf[1]);
                attn::Mma<T>::mma(o[2 * j + 1], hi, bf[2], bf[3]);
                attn::Mma<T>::mma(o[2 * j], lo, bf[0], bf[1]);
                attn::Mma<T>::mma(o[2 * j + 1], lo, bf[2], bf[3]);
            }
        }

        const bool done = at.tile == at.tiles - 1;
        if (done || i == n - 1) {
            // row sums over the warps; the next tile's barriers keep sm.l until everyone has read it
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                l_sum[r] += __shfl_xor_sync(0xffffffffu, l_sum[r], 1);
                l_sum[r] += __shfl_xor_sync(0xffffffffu, l_sum[r], 2);
                if (tq == 0) sm.l[warp][gq + r * 8] = l_sum[r];
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = gq + r * 8;
                if (row >= rows) continue;
                const float L = (sm.l[0][row] + sm.l[1][row]) + (sm.l[2][row] + sm.l[3][row]);
                if (done && whole) {
                    const float inv = L == 0.f ? 0.f : 1.f / L;
                    T *out = reinterpret_cast<T *>(p.o) + (int64_t)at.b * p.o_sb + (int64_t)(h0 + row) * p.o_sh;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const int c = warp * (D / 4) + j * 8 + tq * 2;
                        if constexpr (VEC) {
                            if (c < p.d) *reinterpret_cast<uint32_t *>(out + c) = attn::Mma<T>::pack(o[j][2 * r] * inv, o[j][2 * r + 1] * inv);
                        } else {
                            if (c < p.d) out[c] = from_f32<T>(o[j][2 * r] * inv);
                            if (c + 1 < p.d) out[c + 1] = from_f32<T>(o[j][2 * r + 1] * inv);
                        }
                    }
                    if (p.lse && warp == 0 && tq == 0)
                        p.lse[(int64_t)at.b * p.Hq + h0 + row] = L == 0.f ? -INFINITY : (m_ref[r] + log2f(L)) * LN2;
                } else {
                    float *part = part_of(p, ctas, D, cta, whole ? 1 : 0);
                    if (warp == 0 && tq == 0) {
                        part[row] = m_ref[r];
                        part[ROWS + row] = L;
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        *reinterpret_cast<float2 *>(part + 2 * ROWS + row * D + warp * (D / 4) + j * 8 + tq * 2) =
                            make_float2(o[j][2 * r], o[j][2 * r + 1]);
                }
            }
            if (!done && whole && tid == 0) {
                // the run that has the unit's last tile: cta * total / busy <= t < (cta + 1) * total / busy
                const int64_t t = end - 1 + (at.tiles - 1 - at.tile);
                Header &head = reinterpret_cast<Header *>(p.work)[cta];
                head.last = (int)(((t + 1) * busy - 1) / total);
                head.b = at.b;
                head.hk = at.hk;
                head.row0 = row0;
            }
        }
        advance(at);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // sequences without a token
    for (int b = cta; b < p.B; b += ctas)
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

// Adds the parts of the unit that begins in CTA blockIdx.x's run and ends in another's; one CTA per row.
template <typename T, int D>
__global__ void __launch_bounds__(THREADS) join_kernel(const __grid_constant__ AttnParams p) {
    constexpr int QUADS = D / 4, GROUPS = THREADS / QUADS;
    __shared__ float red[WARPS], l_s[GROUPS];
    __shared__ float4 acc_s[GROUPS][QUADS];
    const int tid = threadIdx.x, quad = tid % QUADS, grp = tid / QUADS, cta = blockIdx.x, row = blockIdx.y, ctas = gridDim.x;
    sm100::grid_wait();
    const Header head = reinterpret_cast<const Header *>(p.work)[cta];
    if (head.last < 0 || row >= min(ROWS, p.G - head.row0)) return;
    const int n = head.last - cta + 1;
    auto part = [&](int i) { return part_of(p, ctas, D, cta + i, i == 0 ? 1 : 0); };
    float m = -INFINITY;
    for (int i = tid; i < n; i += THREADS) m = fmaxf(m, part(i)[row]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 31) == 0) red[tid >> 5] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mu = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = grp; i < n; i += GROUPS) {
        const float *from = part(i);
        const float f = ex2(from[row] - mu);
        const float4 x = *reinterpret_cast<const float4 *>(from + 2 * ROWS + row * D + quad * 4);
        l = fmaf(from[ROWS + row], f, l);
        acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y);
        acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
    }
    if (quad == 0) l_s[grp] = l;
    acc_s[grp][quad] = acc;
    __syncthreads();
    if (grp > 0) return;
    l = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        const float4 x = acc_s[g][quad];
        l += l_s[g];
        acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int h = head.hk * p.G + head.row0 + row;
    T *out = reinterpret_cast<T *>(p.o) + (int64_t)head.b * p.o_sb + (int64_t)h * p.o_sh;
    const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (quad * 4 + e < p.d) out[quad * 4 + e] = from_f32<T>(y[e]);
    if (p.lse && quad == 0) p.lse[(int64_t)head.b * p.Hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

// CTAs of the grid: what the SMs hold at once, and no more than there can be tiles.
int grid_size(int64_t B, int64_t units, int64_t max_keys, int resident) {
    const int64_t most = B * units * ((max_keys + KEYS - 1) / KEYS);
    const int64_t room = (int64_t)num_sms() * resident;
    const int64_t n = (most + MIN_TILES - 1) / MIN_TILES;
    return (int)(n < 1 ? 1 : n < room ? n : room);
}

template <typename T, int D, bool VEC, bool BIAS>
int launch(AttnParams &p, int64_t max_keys, cudaStream_t st) {
    auto kernel = attn_kernel<T, D, VEC, BIAS>;
    const size_t smem = sizeof(Smem<T, D>) + (BIAS ? (size_t)p.borders.side * ROWS * sizeof(float) : 0);
    // one opt-in per kernel, for the largest table: opting in to a smaller one would take a larger one back
    const size_t largest = sizeof(Smem<T, D>) + (BIAS ? (size_t)relbias::MAX_SIDE * ROWS * sizeof(float) : 0);
    if (int e = ensure_dyn_smem(reinterpret_cast<const void *>(kernel), largest)) return e;
    const int fit = cached_occupancy(reinterpret_cast<const void *>(kernel), THREADS, smem);
    const int grid = grid_size(p.B, p.units, max_keys, fit < ctas_per_sm(D) ? fit : ctas_per_sm(D));
    kernel<<<grid, THREADS, smem, st>>>(p);
    count_launch();
    if (int e = check_launch()) return e;
    return sm100::launch_pdl(join_kernel<T, D>, dim3(grid, (unsigned)(p.G < ROWS ? p.G : ROWS)), THREADS, 0, st, p);
}
template <typename T, int D>
int launch(AttnParams &p, bool vec, int64_t max_keys, cudaStream_t st) {
    if (p.w) return vec ? launch<T, D, true, true>(p, max_keys, st) : launch<T, D, false, true>(p, max_keys, st);
    return vec ? launch<T, D, true, false>(p, max_keys, st) : launch<T, D, false, false>(p, max_keys, st);
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
    if (d > 128 || B > INT32_MAX || Hq > 65535 || max_pages > INT32_MAX || page_size > INT32_MAX) return RGD_E_SIZE;
    const int D = d > 64 ? 128 : 64;
    const int64_t units = Hkv * ceil_div64(Hq / Hkv, paged::ROWS);
    return paged::workspace_bytes(paged::grid_size(B, units, max_pages * page_size, paged::ctas_per_sm(D)), D);
}

extern "C" int rgd_paged_attn(const rgd_heads *q, const rgd_paged *cache, const rgd_relbias *bias, const rgd_heads *o, float *lse,
                              int64_t B, int64_t Hq, int64_t Hkv, int64_t d, float softmax_scale, int dtype, void *workspace,
                              int64_t workspace_bytes, void *stream) {
    if (!q || !o) return RGD_E_NULL;
    if (dtype != RGD_F16 && dtype != RGD_BF16) return RGD_E_DTYPE;
    if (B < 0 || Hq < 0 || Hkv < 0 || d < 0) return RGD_E_INVALID;
    if (d > 128 || B > INT32_MAX || Hq > 65535) return RGD_E_SIZE;
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
    p.v = cache->v; p.v_sp = cache->v_stride_p; p.v_ss = cache->v_stride_s; p.v_sh = cache->v_stride_h;
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
    const int64_t max_keys = cache->max_pages * cache->page_size;
    if (workspace_bytes < rgd_paged_attn_workspace_bytes(B, Hq, Hkv, d, cache->max_pages, cache->page_size) || !workspace)
        return RGD_E_WORKSPACE;
    if (!is_aligned(workspace, 16)) return RGD_E_STRIDE;
    p.work = reinterpret_cast<char *>(workspace);
    const bool vec = d % 8 == 0 && paged::cache_vec16(*cache) && paged::heads_vec16(*q) && paged::heads_vec16(*o);
    cudaStream_t st = (cudaStream_t)stream;
    if (d > 64)
        return dtype == RGD_BF16 ? paged::launch<__nv_bfloat16, 128>(p, vec, max_keys, st) : paged::launch<__half, 128>(p, vec, max_keys, st);
    return dtype == RGD_BF16 ? paged::launch<__nv_bfloat16, 64>(p, vec, max_keys, st) : paged::launch<__half, 64>(p, vec, max_keys, st);
}
