// New keys and values into a paged cache, rotated on the way, and the queries beside them.
//
//   p = lengths[b] + i,  (page, slot) of p,  k' = R(p) k,  q' = R(p) q,
//   R(p): channels (2c, 2c + 1) -> (x0 cos - x1 sin, x1 cos + x0 sin) with the table's angles of position p.
//
// Every input is read once and every output written once.
#include "attn_mma.cuh"
#include "paged.cuh"
#include "sm100_prims.cuh"

namespace rgd {
namespace paged {

__device__ int g_append_status = 0;

// How a CTA's threads lie over (token, head, channel group).
struct AppendGeo {
    int step, per_token, tokens;            // heads side by side, threads of a token, tokens side by side
    int loop;                               // and one after another
    FastDiv by_per_token;
};

struct AppendParams {
    PagedView view;
    const int32_t *lengths, *counts;
    const void *x[3];                       // key, value, query
    int64_t x_sb[3], x_sh[3], x_sn[3];
    void *out[3];                           // the two caches (strides: page, head, slot), the rotated query
    int64_t o_sb[3], o_sh[3], o_sn[3];
    const void *pos;                        // null: nothing is rotated
    int64_t pos_ss, pos_sn, P;
    int pos_dtype, R, pos_vec;              // pos_vec: the table's rows are 16-byte addressable
    int B, N, Hq, Hkv, d;
    FastDiv by_n, by_vecs, by_groups;       // N, vecs, angle_groups
    int vecs, angle_groups;                 // channel groups of a row; groups of 8 channels with a rotated one
    AppendGeo geo[2];                       // of the caches, of the query
};

constexpr int APPEND_THREADS = 256;
constexpr int APPEND_BATCH = 4;             // tokens that a thread reads before it uses the first
constexpr int APPEND_LOOP = 8;              // most tokens of a thread
constexpr int ANGLE_BYTES = 16 << 10;       // shared memory for the angles of a CTA's tokens

// Eight angles of a table row from element `at` on, `left` of them in the table and zeros.
__device__ __forceinline__ void load_angles(const AppendParams &p, int64_t at, int left, float (&w)[8]) {
    if (p.pos_vec && left >= 8) {
        if (p.pos_dtype == RGD_F32) {
            const float4 *f = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p.pos) + at);
            const float4 a = f[0], b = f[1];
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
            w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
        } else if (p.pos_dtype == RGD_F16) {
            const Vec<__half, 8> x = load_vec<__half, 8>(reinterpret_cast<const __half *>(p.pos) + at);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = __half2float(x.v[e]);
        } else {
            const Vec<__nv_bfloat16, 8> x = load_vec<__nv_bfloat16, 8>(reinterpret_cast<const __nv_bfloat16 *>(p.pos) + at);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = __bfloat162float(x.v[e]);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = e < left ? load_as_f32(p.pos, at + e, p.pos_dtype) : 0.f;
}

// Where a token goes.
struct alignas(16) Place {
    int64_t out;                            // element offset of its head 0
    int position;                           // -1: a key or value that is not written, a query that is copied
};

// A pair of channels as two floats.
template <typename T> __device__ __forceinline__ float2 unpack(uint32_t w);
template <> __device__ __forceinline__ float2 unpack<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
template <> __device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Each CTA has one of the three tensors and a few tokens of it, each thread one group of VE channels (16 bytes, or a
// pair where views are not addressable that way) of one head after another.  Where the tokens go and their angles are
// looked up once for the CTA, two dependent reads (length; table entry and angles) during which the first tokens are on
// their way; the loop is then read, turn, write.  [4, 4096, 16, 128] bf16 keys, values and queries (411 MB): 73 us, 86 %
// of the copy rate, bound by instruction issue (two thirds of the slots busy) and the look-ups.  With every thread
// looking up its own tokens it took 160-200 us.  Four CTAs an SM: 74 us at five, and ragged sequences 6.6 us for 6.0.  Pairs (VE = 2) are what odd views cost: [4, 2048, 16, 128] 142 us one
// element off 16 bytes, 39 us on them.
template <typename T, int VE>
__global__ void __launch_bounds__(APPEND_THREADS, 4) append_kernel(const __grid_constant__ AppendParams p) {
    using V = Vec<uint32_t, VE / 2>;            // pairs of channels
    extern __shared__ __align__(16) unsigned char raw[];
    sm100::grid_trigger();
    sm100::grid_wait();         // as the attention
    const int which = blockIdx.y, tid = threadIdx.x;
    const AppendGeo g = p.geo[which == 2];      // a copy: an indexed parameter is read anew at every use (77 us for 73)
    const int heads = which == 2 ? p.Hq : p.Hkv, all = p.B * p.N, mine = g.loop * g.tokens;
    if (heads == 0 || (int64_t)blockIdx.x * mine >= all) return;       // the grid is the larger one of two
    const int first = blockIdx.x * mine;
    Place *places = reinterpret_cast<Place *>(raw);             // [loop][tokens]
    // [loop][tokens], sines and cosines, first and second halves of the groups of 8 channels (a warp then reads 16 bytes
    // next to 16 bytes)
    float *angles = reinterpret_cast<float *>(places + mine);
    const int sub = (int)fdiv((uint32_t)tid, g.by_per_token), rest = tid - sub * g.per_token;
    const int row0 = (int)fdiv((uint32_t)rest, p.by_vecs), c = (rest - row0 * p.vecs) * VE;
    const bool works = sub < g.tokens;
    const T *x = reinterpret_cast<const T *>(p.x[which]) + c;
    T *out = reinterpret_cast<T *>(p.out[which]) + c;
    const int64_t x_sb = p.x_sb[which], x_sh = p.x_sh[which], x_sn = p.x_sn[which], o_sh = p.o_sh[which];

    // The thread's tokens are g.tokens apart, most often in one sequence: the first one's place in the input is worked
    // out, the others' follow it unless a sequence ends between them.
    const int64_t x_step = g.tokens * x_sn;
    V v[APPEND_BATCH];
    auto read = [&](int row, int t0) {
        int token = first + t0 * g.tokens + sub, b = (int)fdiv((uint32_t)token, p.by_n), i = token - b * p.N;
        const T *from = x + b * x_sb + row * x_sh + i * x_sn;
#pragma unroll
        for (int u = 0; u < APPEND_BATCH; ++u) {
            if (t0 + u < g.loop && token < all) {
                if constexpr (VE == 8) {
                    v[u] = load_vec_stream<uint32_t, 4>(reinterpret_cast<const uint32_t *>(from));
                } else {
                    const T pair[2] = {from[0], c + 1 < p.d ? from[1] : from_f32<T>(0.f)};
                    v[u].v[0] = (uint32_t)reinterpret_cast<const uint16_t *>(pair)[0] | (uint32_t)reinterpret_cast<const uint16_t *>(pair)[1] << 16;
                }
            }
            token += g.tokens;
            i += g.tokens;
            from += x_step;
            if (i >= p.N) {
                b = (int)fdiv((uint32_t)token, p.by_n);
                i = token - b * p.N;
                from = x + b * x_sb + row * x_sh + i * x_sn;
            }
        }
    };
    if (works) read(row0, 0);

    // position of token first + e, -1 when it is not a new one, -2 when it has none
    auto position_of = [&](int e) -> int {
        const int b = (int)fdiv((uint32_t)(first + e), p.by_n), i = first + e - b * p.N;
        if (i >= (p.counts ? p.counts[b] : p.N)) return -1;
        const int64_t position = (int64_t)p.lengths[b] + i;
        return position >= 0 && position < capacity(p.view) && (!p.pos || position < p.P) ? (int)position : -2;
    };
    for (int e = tid; e < mine && first + e < all; e += APPEND_THREADS) {
        const int b = (int)fdiv((uint32_t)(first + e), p.by_n), i = first + e - b * p.N;
        Place at{which == 2 ? b * p.o_sb[2] + i * p.o_sn[2] : 0, position_of(e)};
        if (at.position >= 0) {
            int index, slot;
            split_position(p.view, (uint32_t)at.position, index, slot);
            const int page = p.view.table[b * p.view.table_stride + index];
            if (!page_ok(p.view, page)) at.position = -2;
            else if (which != 2) at.out = page * p.o_sb[which] + slot * p.o_sn[which];
        }
        if (at.position == -2) g_append_status = 1;
        places[e] = at;
    }
    const bool turned = p.pos && which != 1;
    if (turned) {
        // one thread per token, sine or cosine, and group of 8 channels; it finds the position itself, so that the
        // angles are read beside the table
        const int groups = p.angle_groups;
        for (int e = APPEND_THREADS - 1 - tid; e < mine * 2 * groups; e += APPEND_THREADS) {
            const int t = (int)fdiv((uint32_t)e, p.by_groups) >> 1, r = e - t * 2 * groups, cosine = r >= groups, q = r - cosine * groups;
            const int position = first + t < all ? position_of(t) : -1;
            if (position < 0) continue;
            float w[8];
            load_angles(p, position * p.pos_sn + cosine * p.pos_ss + q * 8, p.R - q * 8, w);
            float *to = angles + (t * 2 + cosine) * 8 * groups + q * 4;
            *reinterpret_cast<float4 *>(to) = make_float4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<float4 *>(to + 4 * groups) = make_float4(w[4], w[5], w[6], w[7]);
        }
    }
    __syncthreads();
    if (!works) return;

    const bool turns = turned && c < p.R;
    const int rotated = p.R - c;                            // channels of the group, and more where all are
    const int quarter = 4 * p.angle_groups;                 // floats of one half of the groups
    const float *sin0 = angles + sub * 4 * quarter + (c / 8) * 4 + (VE == 8 ? 0 : (c / 4) % 2 * quarter + c % 4);
    for (int row = row0; row < heads; row += g.step) {
        T *out_row = out + row * o_sh;
        for (int t0 = 0; t0 < g.loop; t0 += APPEND_BATCH) {
            if (row != row0 || t0 != 0) read(row, t0);
#pragma unroll
            for (int u = 0; u < APPEND_BATCH; ++u) {
                const int t = (t0 + u) * g.tokens + sub;
                if (t0 + u >= g.loop || first + t >= all) break;
                const Place at = places[t];
                if (at.position < 0 && which != 2) continue;
                if (turns && at.position >= 0) {
                    const float *sin = sin0 + (t0 + u) * g.tokens * 4 * quarter, *cos = sin + 2 * quarter;
#pragma unroll
                    for (int e = 0; e < VE; e += 4) {
                        using W = Vec<float, VE == 8 ? 4 : 2>;
                        const W sw = *reinterpret_cast<const W *>(sin + e / 4 * quarter), cw = *reinterpret_cast<const W *>(cos + e / 4 * quarter);
#pragma unroll
                        for (int k = 0; k < (VE == 8 ? 4 : 2); k += 2) {
                            if (e + k >= rotated) break;            // R is even: a rotated pair is whole
                            uint32_t &pair = v[u].v[(e + k) / 2];
                            const float2 x = unpack<T>(pair);
                            pair = attn::Mma<T>::pack(x.x * cw.v[k] - x.y * sw.v[k], x.y * cw.v[k + 1] + x.x * sw.v[k + 1]);
                        }
                    }
                }
                T *to = out_row + at.out;
                if constexpr (VE == 8) {
                    store_vec<uint32_t, 4>(reinterpret_cast<uint32_t *>(to), v[u]);
                } else {
                    const uint16_t lo = (uint16_t)v[u].v[0], hi = (uint16_t)(v[u].v[0] >> 16);
                    reinterpret_cast<uint16_t *>(to)[0] = lo;
                    if (c + 1 < p.d) reinterpret_cast<uint16_t *>(to)[1] = hi;
                }
            }
        }
    }
}

template <typename T, int VE>
int launch_append(AppendParams &p, cudaStream_t st) {
    p.vecs = (p.d + VE - 1) / VE;
    p.by_vecs = make_fastdiv((uint32_t)p.vecs);
    p.angle_groups = (p.R + 7) / 8;
    p.by_groups = make_fastdiv(p.angle_groups > 0 ? (uint32_t)p.angle_groups : 1);
    const int64_t all = (int64_t)p.B * p.N;
    int64_t grid = 0;
    size_t smem = 0;
    for (int q = 0; q < 2; ++q) {
        AppendGeo &g = p.geo[q];
        const int heads = q ? p.Hq : p.Hkv;
        if (heads == 0) continue;
        g.step = APPEND_THREADS / p.vecs < heads ? APPEND_THREADS / p.vecs : heads;     // heads side by side
        g.per_token = g.step * p.vecs;
        g.tokens = APPEND_THREADS / g.per_token;
        g.by_per_token = make_fastdiv((uint32_t)g.per_token);
        // Tokens one after another: the look-ups of a CTA are worth about as much as two tokens (4 x 4096 tokens of 48
        // heads: 168 us at one, 107 at two, 81 at four, 73 at eight, 74 at sixteen), but every SM should have four
        // CTAs, sixteen for a second batch of reads (7 ragged sequences of up to 333 tokens: 6.0 us with this rule,
        // 6.9 without it), and the angles have to fit.
        const int64_t batches = ceil_div64(all, g.tokens), spread = batches * (p.Hq > 0 ? 3 : 2) / (4 * num_sms());
        const size_t angle_bytes = (size_t)p.angle_groups * 16 * sizeof(float);
        const int64_t fit = p.R > 0 ? (int64_t)(ANGLE_BYTES / (g.tokens * angle_bytes)) : APPEND_LOOP;
        const int64_t want = spread < 4 * APPEND_BATCH && spread > APPEND_BATCH ? APPEND_BATCH : spread, loop = want < fit ? want : fit;
        g.loop = (int)(loop < 1 ? 1 : loop > APPEND_LOOP ? APPEND_LOOP : loop);
        const int64_t ctas = ceil_div64(batches, g.loop);
        grid = ctas > grid ? ctas : grid;
        const size_t bytes = (size_t)g.loop * g.tokens * (sizeof(Place) + angle_bytes);
        smem = bytes > smem ? bytes : smem;
    }
    return sm100::launch_pdl(append_kernel<T, VE>, dim3((unsigned)grid, p.Hq > 0 ? 3 : 2), APPEND_THREADS, smem, st, p);
}

int append_status_fetch() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_append_status, sizeof(int)) != cudaSuccess) {
        (void)cudaGetLastError();
        return -1;
    }
    if (v != 0) {
        const int zero = 0;
        (void)cudaMemcpyToSymbol(g_append_status, &zero, sizeof(int));
    }
    return v;
}

}  // namespace paged
}  // namespace rgd

using namespace rgd;

extern "C" int rgd_paged_slot(const rgd_paged *cache, int64_t row, int64_t position, int64_t *k_offset, int64_t *v_offset) {
    if (!k_offset || !v_offset) return RGD_E_NULL;
    if (int e = paged::check_paged(cache, 0, false)) return e;
    if (row < 0) return RGD_E_INVALID;
    const paged::PagedView v = paged::make_view(*cache);
    if (position < 0 || position >= paged::capacity(v)) return RGD_E_PAGE;
    if (!cache->page_table) return RGD_E_NULL;
    int index, slot;
    paged::split_position(v, (uint32_t)position, index, slot);
    const int page = v.table[row * v.table_stride + index];
    if (!paged::page_ok(v, page)) return RGD_E_PAGE;
    *k_offset = page * cache->k_stride_p + slot * cache->k_stride_s;
    *v_offset = page * cache->v_stride_p + slot * cache->v_stride_s;
    return RGD_OK;
}

extern "C" int rgd_paged_append(const rgd_heads *key, const rgd_heads *value, const rgd_heads *query, const rgd_heads *query_out,
                                const rgd_paged *cache, const int32_t *counts, const void *pos, int64_t pos_stride_s,
                                int64_t pos_stride_n, int64_t P, int64_t R, int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t d,
                                int dtype, int pos_dtype, void *stream) {
    if (!key || !value || (query && !query_out)) return RGD_E_NULL;
    if (dtype != RGD_F16 && dtype != RGD_BF16) return RGD_E_DTYPE;
    if (pos && !dtype_ok(pos_dtype)) return RGD_E_DTYPE;
    if (B < 0 || N < 0 || Hq < 0 || Hkv < 0 || d < 0) return RGD_E_INVALID;
    if (d > 128 || Hq > 65535 || Hkv > 65535 || B > 1 << 30 || N > 1 << 30 || B * N > 1 << 30) return RGD_E_SIZE;
    if (pos && (P < 0 || R < 0 || R > d || R % 2 != 0)) return RGD_E_INVALID;
    if (int e = paged::check_paged(cache, B, Hkv > 0 && d > 0)) return e;
    if (!query) Hq = 0;
    if (B == 0 || N == 0 || d == 0 || (Hq == 0 && Hkv == 0)) return RGD_OK;
    if ((Hkv > 0 && (!key->ptr || !value->ptr)) || (Hq > 0 && (!query->ptr || !query_out->ptr))) return RGD_E_NULL;
    if (Hkv > 0 && cache->num_pages > 0 && cache->k == cache->v) return RGD_E_INVALID;      // keys and values in the same slots

    paged::AppendParams p{};
    p.view = paged::make_view(*cache);
    p.lengths = cache->lengths;
    p.counts = counts;
    const rgd_heads *in[3] = {key, value, Hq > 0 ? query : nullptr};
    for (int i = 0; i < 3; ++i)
        if (in[i]) {
            p.x[i] = in[i]->ptr;
            p.x_sb[i] = in[i]->stride_b; p.x_sh[i] = in[i]->stride_h; p.x_sn[i] = in[i]->stride_n;
        }
    p.out[0] = cache->k; p.o_sb[0] = cache->k_stride_p; p.o_sh[0] = cache->k_stride_h; p.o_sn[0] = cache->k_stride_s;
    p.out[1] = cache->v; p.o_sb[1] = cache->v_stride_p; p.o_sh[1] = cache->v_stride_h; p.o_sn[1] = cache->v_stride_s;
    if (Hq > 0) {
        p.out[2] = query_out->ptr;
        p.o_sb[2] = query_out->stride_b; p.o_sh[2] = query_out->stride_h; p.o_sn[2] = query_out->stride_n;
    }
    p.pos = R > 0 ? pos : nullptr;
    p.pos_ss = pos_stride_s; p.pos_sn = pos_stride_n; p.P = P; p.pos_dtype = pos_dtype; p.R = pos ? (int)R : 0;
    p.B = (int)B; p.N = (int)N; p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.d = (int)d;
    p.by_n = make_fastdiv((uint32_t)N);
    if (pos) {
        const int ve = 16 / dtype_size(pos_dtype);
        p.pos_vec = is_aligned(pos, 16) && pos_stride_s % ve == 0 && pos_stride_n % ve == 0;
    }
    const bool vec = d % 8 == 0 && (Hkv == 0 || (paged::cache_vec16(*cache) && paged::heads_vec16(*key) && paged::heads_vec16(*value))) &&
                     (Hq == 0 || (paged::heads_vec16(*query) && paged::heads_vec16(*query_out)));
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == RGD_BF16) return vec ? paged::launch_append<__nv_bfloat16, 8>(p, st) : paged::launch_append<__nv_bfloat16, 2>(p, st);
    return vec ? paged::launch_append<__half, 8>(p, st) : paged::launch_append<__half, 2>(p, st);
}
