// Learned relative position bias: bias[h, i, j] = w[bucket(j - i - offset), h], and the gradient of w.
//
// The matrix depends on j - i alone: H rows of Tq + Tk - 1 values, written H Tq Tk times.  The gradient is the
// sum over the diagonals, then over the diagonals of each bucket.
#include "relbias.cuh"

namespace rgd {
namespace relbias {

struct FwdParams {
    Borders borders;
    const void *w;
    int64_t w_sk, w_sh;
    int w_dtype;
    void *out;
    int64_t o_sh, o_sq;
    int Tq, Tk, offset;
};

constexpr int THREADS = 256;

template <typename T>
__global__ void __launch_bounds__(THREADS) relbias_fwd_kernel(const __grid_constant__ FwdParams p) {
    const int h = blockIdx.y;
    const int64_t n = (int64_t)p.Tq * p.Tk;
    T *out = reinterpret_cast<T *>(p.out) + (int64_t)h * p.o_sh;
    for (int64_t e = (int64_t)blockIdx.x * THREADS + threadIdx.x; e < n; e += (int64_t)gridDim.x * THREADS) {
        const int i = (int)(e / p.Tk), j = (int)(e - (int64_t)i * p.Tk);
        const int k = bucket_of(p.borders.at, p.borders.side, p.borders.both, j - i - p.offset);
        out[(int64_t)i * p.o_sq + j] = from_f32<T>(load_as_f32(p.w, k * p.w_sk + h * p.w_sh, p.w_dtype));
    }
}

struct BwdParams {
    Borders borders;
    const void *g;
    int64_t g_sh, g_sq;
    int g_dtype;
    void *dw;
    int w_dtype;
    double *sums;               // [H, Tq + Tk - 1]
    int H, Tq, Tk, offset;
};

// One thread per diagonal.
__global__ void __launch_bounds__(THREADS) relbias_diagonals_kernel(const __grid_constant__ BwdParams p) {
    const int h = blockIdx.y, e = blockIdx.x * THREADS + threadIdx.x;
    if (e >= p.Tq + p.Tk - 1) return;
    const int difference = e - (p.Tq - 1);
    double sum = 0.;
    for (int i = max(0, -difference); i < p.Tq && i + difference < p.Tk; ++i)
        sum += load_as_f32(p.g, h * p.g_sh + i * p.g_sq + i + difference, p.g_dtype);
    p.sums[(int64_t)h * (p.Tq + p.Tk - 1) + e] = sum;
}

// One CTA per (bucket, head).
__global__ void __launch_bounds__(THREADS) relbias_buckets_kernel(const __grid_constant__ BwdParams p) {
    __shared__ double part[THREADS];
    const int k = blockIdx.x, h = blockIdx.y, n = p.Tq + p.Tk - 1;
    double sum = 0.;
    for (int e = threadIdx.x; e < n; e += THREADS)
        if (bucket_of(p.borders.at, p.borders.side, p.borders.both, e - (p.Tq - 1) - p.offset) == k) sum += p.sums[(int64_t)h * n + e];
    part[threadIdx.x] = sum;
    for (int o = THREADS / 2; o > 0; o >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
    }
    if (threadIdx.x == 0) store_from_f32(p.dw, (int64_t)k * p.H + h, p.w_dtype, (float)part[0]);
}

int check_sizes(int64_t H, int64_t Tq, int64_t Tk, int64_t offset) {
    if (H < 0 || Tq < 0 || Tk < 0) return RGD_E_INVALID;
    // differences of positions are 32-bit
    if (H > 65535 || Tq > (1 << 28) || Tk > (1 << 28) || offset > (1 << 29) || offset < -(1 << 29)) return RGD_E_SIZE;
    return RGD_OK;
}

}  // namespace relbias
}  // namespace rgd

using namespace rgd;

extern "C" int rgd_relbias_fwd(const rgd_relbias *bias, void *out, int64_t stride_h, int64_t stride_q, int64_t H, int64_t Tq, int64_t Tk,
                               int64_t offset, int out_dtype, void *stream) {
    if (int e = relbias::check(bias)) return e;
    if (!dtype_ok(out_dtype)) return RGD_E_DTYPE;
    if (int e = relbias::check_sizes(H, Tq, Tk, offset)) return e;
    if (H == 0 || Tq == 0 || Tk == 0) return RGD_OK;
    if (!out || !bias->weight) return RGD_E_NULL;
    const int ve = 16 / dtype_size(out_dtype);
    if (!is_aligned(out, 16) || stride_h % ve != 0 || stride_q % ve != 0 || stride_q < Tk || stride_h < 0) return RGD_E_STRIDE;
    relbias::FwdParams p{};
    p.borders = relbias::make_borders(*bias);
    p.w = bias->weight; p.w_sk = bias->stride_bucket; p.w_sh = bias->stride_head; p.w_dtype = bias->dtype;
    p.out = out; p.o_sh = stride_h; p.o_sq = stride_q;
    p.Tq = (int)Tq; p.Tk = (int)Tk; p.offset = (int)offset;
    const int64_t blocks = ceil_div64(Tq * Tk, relbias::THREADS);
    const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096), (unsigned)H);
    cudaStream_t st = (cudaStream_t)stream;
    if (out_dtype == RGD_F32) relbias::relbias_fwd_kernel<float><<<grid, relbias::THREADS, 0, st>>>(p);
    else if (out_dtype == RGD_F16) relbias::relbias_fwd_kernel<__half><<<grid, relbias::THREADS, 0, st>>>(p);
    else relbias::relbias_fwd_kernel<__nv_bfloat16><<<grid, relbias::THREADS, 0, st>>>(p);
    count_launch();
    return check_launch();
}

extern "C" int64_t rgd_relbias_bwd_workspace_bytes(int64_t H, int64_t Tq, int64_t Tk, int num_buckets) {
    (void)num_buckets;
    if (int e = relbias::check_sizes(H, Tq, Tk, 0)) return e;
    return H * (Tq + Tk) * (int64_t)sizeof(double);
}

extern "C" int rgd_relbias_bwd(const rgd_relbias *bias, const void *dbias, int64_t stride_h, int64_t stride_q, int dtype, void *dweight,
                               int64_t H, int64_t Tq, int64_t Tk, int64_t offset, void *workspace, int64_t workspace_bytes, void *stream) {
    if (int e = relbias::check(bias)) return e;
    if (!dtype_ok(dtype)) return RGD_E_DTYPE;
    if (int e = relbias::check_sizes(H, Tq, Tk, offset)) return e;
    if (H == 0) return RGD_OK;
    if (!dweight || (!dbias && Tq > 0 && Tk > 0)) return RGD_E_NULL;
    cudaStream_t st = (cudaStream_t)stream;
    if (Tq == 0 || Tk == 0)
        return cuda_status(cudaMemsetAsync(dweight, 0, (size_t)(H * bias->num_buckets) * dtype_size(bias->dtype), st));
    const int64_t need = rgd_relbias_bwd_workspace_bytes(H, Tq, Tk, bias->num_buckets);
    if (!workspace || workspace_bytes < need) return RGD_E_WORKSPACE;
    if (!is_aligned(workspace, 16)) return RGD_E_STRIDE;
    relbias::BwdParams p{};
    p.borders = relbias::make_borders(*bias);
    p.g = dbias; p.g_sh = stride_h; p.g_sq = stride_q; p.g_dtype = dtype;
    p.dw = dweight; p.w_dtype = bias->dtype;
    p.sums = reinterpret_cast<double *>(workspace);
    p.H = (int)H; p.Tq = (int)Tq; p.Tk = (int)Tk; p.offset = (int)offset;
    relbias::relbias_diagonals_kernel<<<dim3((unsigned)ceil_div64(Tq + Tk - 1, relbias::THREADS), (unsigned)H), relbias::THREADS, 0, st>>>(p);
    count_launch();
    relbias::relbias_buckets_kernel<<<dim3((unsigned)bias->num_buckets, (unsigned)H), relbias::THREADS, 0, st>>>(p);
    count_launch();
    return check_launch();
}
