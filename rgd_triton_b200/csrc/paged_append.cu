// New keys and values into a paged cache, rotated on the way, and the queries beside them.
//
//   p = lengths[b] + i,  (page, slot) of p,  k' = R(p) k,  q' = R(p) q,
//   R(p): channels (2c, 2c + 1) -> (x0 cos - x1 sin, x1 cos + x0 sin) with the table's angles of position p.
//
// Every input is read once and every output written once.
#include "paged.cuh"

namespace rgd {
namespace paged {

__device__ int g_append_status = 0;

struct AppendParams {
    PagedView view;
    const int32_t *lengths, *counts;
    const void *x[3];                       // key, value, query
    int64_t x_sb[3], x_sh[3], x_sn[3];
    void *out[3];                           // the two caches (strides: page, head, slot), the rotated query
    int64_t o_sb[3], o_sh[3], o_sn[3];
    const void *pos;                        // null: nothing is rotated
    int64_t pos_ss, pos_sn, P;
    int pos_dtype, R;
    int B, N, Hq, Hkv, d;
};

constexpr int APPEND_THREADS = 128;

// One CTA per token, a pair of neighbouring channels at a time.
template <typename T>
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(const __grid_constant__ AppendParams p) {
    const int b = (int)(blockIdx.x / (unsigned)p.N), i = (int)(blockIdx.x - (unsigned)b * p.N);
    const int count = p.counts ? p.counts[b] : p.N;
    const int64_t position = (int64_t)p.lengths[b] + i;
    bool live = i < count;
    int page = 0, slot = 0;
    if (live) {
        bool ok = position >= 0 && position < capacity(p.view) && (!p.pos || position < p.P);
        if (ok) {
            int index;
            split_position(p.view, (uint32_t)position, index, slot);
            page = p.view.table[(int64_t)b * p.view.table_stride + index];
            ok = page_ok(p.view, page);
        }
        if (!ok) {
            live = false;
            if (threadIdx.x == 0) g_append_status = 1;
        }
    }
    const int pairs = (p.d + 1) / 2;
    for (int t = threadIdx.x; t < (2 * p.Hkv + p.Hq) * pairs; t += APPEND_THREADS) {
        const int row = t / pairs, c = (t - row * pairs) * 2;
        const int which = row < p.Hkv ? 0 : row < 2 * p.Hkv ? 1 : 2, h = row - (which == 0 ? 0 : which * p.Hkv);
        if (!live && which != 2) continue;
        const T *x = reinterpret_cast<const T *>(p.x[which]) + (int64_t)b * p.x_sb[which] + (int64_t)h * p.x_sh[which] +
                     (int64_t)i * p.x_sn[which] + c;
        T *out = reinterpret_cast<T *>(p.out[which]) + (int64_t)h * p.o_sh[which] + c +
                 (which == 2 ? (int64_t)b * p.o_sb[2] + (int64_t)i * p.o_sn[2]
                             : (int64_t)page * p.o_sb[which] + (int64_t)slot * p.o_sn[which]);
        const bool both = c + 1 < p.d;
        T y0 = x[0], y1 = both ? x[1] : from_f32<T>(0.f);
        if (live && which != 1 && c < p.R) {        // R is even: a rotated pair is whole
            const int64_t at = position * p.pos_sn + c;
            const float s0 = load_as_f32(p.pos, at, p.pos_dtype), s1 = load_as_f32(p.pos, at + 1, p.pos_dtype);
            const float c0 = load_as_f32(p.pos, p.pos_ss + at, p.pos_dtype), c1 = load_as_f32(p.pos, p.pos_ss + at + 1, p.pos_dtype);
            const float x0 = to_f32<T>(y0), x1 = to_f32<T>(y1);
            y0 = from_f32<T>(x0 * c0 - x1 * s0);
            y1 = from_f32<T>(x1 * c1 + x0 * s1);
        }
        out[0] = y0;
        if (both) out[1] = y1;
    }
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
    if (d > 128 || Hq > 65535 || Hkv > 65535 || B > INT32_MAX || N > INT32_MAX || B * N > INT32_MAX) return RGD_E_SIZE;
    if (pos && (P < 0 || R < 0 || R > d || R % 2 != 0)) return RGD_E_INVALID;
    if (int e = paged::check_paged(cache, B, Hkv > 0 && d > 0)) return e;
    if (!query) Hq = 0;
    if (B == 0 || N == 0 || d == 0 || (Hq == 0 && Hkv == 0)) return RGD_OK;
    if ((Hkv > 0 && (!key->ptr || !value->ptr)) || (Hq > 0 && (!query->ptr || !query_out->ptr))) return RGD_E_NULL;

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
    const unsigned grid = (unsigned)(B * N);
    if (dtype == RGD_BF16) paged::append_kernel<__nv_bfloat16><<<grid, paged::APPEND_THREADS, 0, (cudaStream_t)stream>>>(p);
    else paged::append_kernel<__half><<<grid, paged::APPEND_THREADS, 0, (cudaStream_t)stream>>>(p);
    count_launch();
    return check_launch();
}
