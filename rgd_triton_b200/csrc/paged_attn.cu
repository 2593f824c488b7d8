// Attention of one new token per sequence over a paged key-value cache:
//   s_j = scale q k_j + w[bucket(len - 1 - j)],  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j.
// Four operations per byte of cache and query head: bound by reading the cache once.
#include <math.h>

#include "attn_mma.cuh"
#include "paged.cuh"
#include "relbias.cuh"

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

constexpr int ATTN_THREADS = 128;

// One CTA per sequence and query head, 128 keys at a time: a thread per key, then a thread per channel.
template <typename T>
__global__ void __launch_bounds__(ATTN_THREADS) attn_kernel(const __grid_constant__ AttnParams p) {
    __shared__ float q_s[128], p_s[ATTN_THREADS], red[ATTN_THREADS];
    __shared__ int64_t v_at[ATTN_THREADS];
    const int b = blockIdx.x, h = blockIdx.y, hk = h / p.G, t = threadIdx.x;
    const int len = live_length(p, b, t == 0 && h == 0);
    q_s[t] = t < p.d ? to_f32<T>(reinterpret_cast<const T *>(p.q)[(int64_t)b * p.q_sb + (int64_t)h * p.q_sh + t]) : 0.f;
    __syncthreads();
    auto reduce = [&](float x, auto op) {
        red[t] = x;
        for (int o = ATTN_THREADS / 2; o > 0; o >>= 1) {
            __syncthreads();
            if (t < o) red[t] = op(red[t], red[t + o]);
        }
        __syncthreads();
        const float r = red[0];
        __syncthreads();
        return r;
    };
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int key0 = 0; key0 < len; key0 += ATTN_THREADS) {
        const int key = key0 + t;
        float x = -INFINITY;
        v_at[t] = -1;
        if (key < len) {
            int index, slot;
            split_position(p.view, (uint32_t)key, index, slot);
            const int page = p.view.table[(int64_t)b * p.view.table_stride + index];
            if (page_ok(p.view, page)) {
                const T *k = reinterpret_cast<const T *>(p.k) + (int64_t)page * p.k_sp + (int64_t)slot * p.k_ss + (int64_t)hk * p.k_sh;
                float dot = 0.f;
                for (int c = 0; c < p.d; ++c) dot = fmaf(q_s[c], to_f32<T>(k[c]), dot);
                x = dot * p.scale_log2;
                if (p.w) {
                    const int at = relbias::bucket_of_distance(p.borders.at, p.borders.side, len - 1 - key);
                    x += attn::bias_log2<float>(load_as_f32(p.w, at * p.w_sk + h * p.w_sh, p.w_dtype));
                }
                v_at[t] = (int64_t)page * p.v_sp + (int64_t)slot * p.v_ss + (int64_t)hk * p.v_sh;
            } else {
                g_attn_status = 1;
            }
        }
        const float m_new = fmaxf(m, reduce(x, [](float a, float c) { return fmaxf(a, c); }));
        const float mu = m_new == -INFINITY ? 0.f : m_new;
        const float prob = exp2f(x - mu), alpha = exp2f(m - mu);
        p_s[t] = prob;
        l = l * alpha + reduce(prob, [](float a, float c) { return a + c; });
        acc *= alpha;
        if (t < p.d)
            for (int j = 0; j < ATTN_THREADS; ++j)
                if (v_at[j] >= 0) acc = fmaf(p_s[j], to_f32<T>(reinterpret_cast<const T *>(p.v)[v_at[j] + t]), acc);
        m = m_new;
        __syncthreads();
    }
    if (t < p.d) reinterpret_cast<T *>(p.o)[(int64_t)b * p.o_sb + (int64_t)h * p.o_sh + t] = from_f32<T>(l == 0.f ? 0.f : acc / l);
    if (t == 0 && p.lse) p.lse[(int64_t)b * p.Hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
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
    return 0;
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
    (void)workspace; (void)workspace_bytes;
    const dim3 grid((unsigned)B, (unsigned)Hq);
    if (dtype == RGD_BF16) paged::attn_kernel<__nv_bfloat16><<<grid, paged::ATTN_THREADS, 0, (cudaStream_t)stream>>>(p);
    else paged::attn_kernel<__half><<<grid, paged::ATTN_THREADS, 0, (cudaStream_t)stream>>>(p);
    count_launch();
    return check_launch();
}
