// Learned relative position bias: bias[h, i, j] = w[bucket(j - i - offset), h], and the gradient of w.
//
// Forward.  The matrix depends on j - i alone, so every row of a tile of it is a window of one short row of values:
// row i of the tile is that row shifted by one element more than row i + 1.  A CTA evaluates the short row once, keeps
// it in shared memory at each of the shifts that a 16-byte address can have, and lets the copy engine write the rows
// from there (one bulk store each): no thread touches an element of the output but those past the last 16 bytes of a
// row.  Bound by writing H Tq Tk elements.
//
// Gradient.  dw[k] is a sum over whole diagonals.  The matrix is taken in blocks of 8 x 8; a thread walks down blocks
// (I, J), (I + 1, J + 1), ..., whose 15 diagonals are the same ones, and keeps their sums in registers, so an element
// costs one addition.  The threads of a warp have neighbouring J and read 512 consecutive bytes of a row together.
// The diagonal sums of a warp then go to the buckets, which are ranges of diagonals, in an order that is fixed by the
// sizes: the result is the same every time.  Bound by reading H Tq Tk elements.
#include "relbias.cuh"
#include "sm100_prims.cuh"

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
    int cols;                   // of a tile, a multiple of 8
    FastDiv across;             // tiles side by side
};

// Tiles of 32 rows: small ones end together.  us for 24 x 4096 x 4096 fp16 and its gradient at 32, 48, 64, 128 rows:
// 251, 253, 258, 265.
constexpr int FWD_THREADS = 256, FWD_ROWS = 32, FWD_COLS = 2048;

// Shared memory: the short row (tile cols + rows values, rounded up) at each shift, the borders, the head's weights.
template <typename T> __host__ __device__ constexpr int fwd_row_values(int cols) { return FWD_ROWS + cols + 16 / (int)sizeof(T); }
template <typename T> constexpr size_t fwd_smem(int cols, int buckets) {
    return 16 * (size_t)fwd_row_values<T>(cols) + MAX_SIDE * sizeof(int) + (size_t)buckets * sizeof(T);
}

template <typename T>
__global__ void __launch_bounds__(FWD_THREADS) relbias_fwd_kernel(const __grid_constant__ FwdParams p) {
    constexpr int SHIFTS = 16 / sizeof(T);
    using V = Vec<T, SHIFTS>;
    extern __shared__ __align__(16) unsigned char raw[];
    const int L = fwd_row_values<T>(p.cols);
    T *lut = reinterpret_cast<T *>(raw);                // [SHIFTS][L]: lut[s][x] = row[x + s]
    int *at = reinterpret_cast<int *>(raw + 16 * (size_t)L);
    T *w = reinterpret_cast<T *>(at + MAX_SIDE);
    sm100::grid_wait();         // the launch may overlap the end of what ran before; nothing of that has been read so far
    const int down = (int)fdiv(blockIdx.x, p.across), h = blockIdx.y, tid = threadIdx.x;
    const int i0 = down * FWD_ROWS, j0 = ((int)blockIdx.x - down * (int)p.across.div) * p.cols;
    const int side = p.borders.side, both = p.borders.both;
    for (int k = tid; k < side - 1; k += FWD_THREADS) at[k] = p.borders.at[k];
    for (int k = tid; k < side * (1 + both); k += FWD_THREADS) w[k] = from_f32<T>(load_as_f32(p.w, k * p.w_sk + h * p.w_sh, p.w_dtype));
    __syncthreads();
    // row[x] belongs to j - i = (j0 - i0) - (FWD_ROWS - 1) + x: row r of the tile begins at x = FWD_ROWS - 1 - r
    const int first = j0 - i0 - (FWD_ROWS - 1) - p.offset;
    for (int x = tid; x < L; x += FWD_THREADS) lut[x] = w[bucket_of(at, side, both, first + x)];
    __syncthreads();
    for (int x = tid * SHIFTS; x + SHIFTS < L; x += FWD_THREADS * SHIFTS) {
        const V a = load_vec<T, SHIFTS>(lut + x), b = load_vec<T, SHIFTS>(lut + x + SHIFTS);
#pragma unroll
        for (int s = 1; s < SHIFTS; ++s) {
            V c;
#pragma unroll
            for (int e = 0; e < SHIFTS; ++e) c.v[e] = e + s < SHIFTS ? a.v[(e + s) % SHIFTS] : b.v[(e + s) % SHIFTS];
            store_vec<T, SHIFTS>(lut + s * L + x, c);
        }
    }
    sm100::fence_proxy_async_smem();
    __syncthreads();
    const int rows = min(FWD_ROWS, p.Tq - i0), cols = min(p.cols, p.Tk - j0), even = cols / SHIFTS * SHIFTS;
    T *out = reinterpret_cast<T *>(p.out) + (int64_t)h * p.o_sh + (int64_t)i0 * p.o_sq + j0;
    for (int r = tid; r < rows; r += FWD_THREADS) {
        const int x = FWD_ROWS - 1 - r, s = x % SHIFTS;
        if (even > 0) sm100::bulk_store_1d(out + (int64_t)r * p.o_sq, lut + s * L + (x - s), (uint32_t)(even * sizeof(T)));
        for (int j = even; j < cols; ++j) out[(int64_t)r * p.o_sq + j] = lut[x + j];
    }
    sm100::bulk_commit();
    sm100::bulk_wait_read();
}

struct BwdParams {
    Borders borders;
    const void *g;
    int64_t g_sh, g_sq;
    void *dw;
    int w_dtype;
    float *parts;               // [H][CTAs of a head][buckets]
    int H, Tq, Tk, offset;
    int chunk;                  // 8-row blocks of a CTA
    int across;                 // CTAs side by side
};

constexpr int BWD_WARPS = 4, BWD_THREADS = BWD_WARPS * 32, BWD_PER_SM = 6;
constexpr int DIAGS = 32 * 8 + 7;       // of a warp's 32 neighbouring block diagonals

// A row's eight elements and what lies around them up to 16-byte borders, and the elements out of that: `shift` of them
// lie before the first.
template <typename T, bool VEC>
struct Words {
    static constexpr int PER = 16 / sizeof(T), N = 8 / PER + (VEC ? 0 : 1);
    union {
        uint4 u[N];
        uint32_t w[N * 4];
    };
    __device__ __forceinline__ void read(const T *at, int shift) {
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = ld_stream16(at - shift + i * PER);
    }
    __device__ __forceinline__ void elements(int shift, float (&x)[8]) {
        if constexpr (!VEC) {
            constexpr int WORD = 4 / sizeof(T);             // elements of a 32-bit word
#pragma unroll
            for (int s = 2; s >= 1; s /= 2)                 // by two words, by one
#pragma unroll
                for (int i = 0; i + s < N * 4; ++i) w[i] = shift & s * WORD ? w[i + s] : w[i];
            if constexpr (sizeof(T) == 2)                   // by one element
#pragma unroll
                for (int i = 0; i + 1 < N * 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], shift & 1 ? 16 : 0);
        }
        const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int c = 0; c < 8; ++c) x[c] = to_f32<T>(e[c]);
    }
};

// VEC: rows begin on 16 bytes.  Otherwise each row is read in the 16-byte words that its own alignment gives.
template <typename T, bool VEC>
__global__ void __launch_bounds__(BWD_THREADS, BWD_PER_SM) relbias_bwd_kernel(const __grid_constant__ BwdParams p) {
    __shared__ float diag[BWD_WARPS][DIAGS + 1];
    extern __shared__ float hist[];                     // [BWD_WARPS][buckets]
    __shared__ int at[MAX_SIDE];
    sm100::grid_trigger();
    sm100::grid_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y;
    const int side = p.borders.side, both = p.borders.both, buckets = side * (1 + both);
    const int row_chunk = blockIdx.x / p.across, m = blockIdx.x - row_chunk * p.across;
    const int I0 = row_chunk * p.chunk, nI = (p.Tq + 7) / 8, nJ = (p.Tk + 7) / 8;
    const int k_warp = m * BWD_THREADS - (I0 + p.chunk - 1) + warp * 32, k = k_warp + lane;       // J - I
    for (int x = tid; x < side - 1; x += BWD_THREADS) at[x] = p.borders.at[x];
    for (int x = tid; x < BWD_WARPS * buckets; x += BWD_THREADS) hist[x] = 0.f;

    float acc[15];
#pragma unroll
    for (int e = 0; e < 15; ++e) acc[e] = 0.f;
    const T *g = reinterpret_cast<const T *>(p.g) + (int64_t)h * p.g_sh;
    const T *g_end = g + (int64_t)(p.Tq - 1) * p.g_sq + p.Tk;
    const int I1 = min(I0 + p.chunk, nI);
    for (int I = max(I0, -k); I < I1 && I + k < nJ; ++I) {
        const int i = I * 8, j = (I + k) * 8;
        const T *at0 = g + (int64_t)i * p.g_sq + j;
        using W = Words<T, VEC>;
        auto shift_of = [](const T *row) { return VEC ? 0 : (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T)); };
        const T *last = at0 + 7 * p.g_sq;
        // the words of all eight rows lie between the matrix's first and last element
        if (i + 8 <= p.Tq && at0 - shift_of(at0) >= g && last - shift_of(last) + W::N * W::PER <= g_end) {
            constexpr int BATCH = 8 * sizeof(uint4) / sizeof(W);        // rows on their way at once: eight 16-byte words
#pragma unroll
            for (int r0 = 0; r0 < 8; r0 += BATCH) {
                W words[BATCH];
#pragma unroll
                for (int r = 0; r < BATCH; ++r) words[r].read(at0 + (r0 + r) * p.g_sq, shift_of(at0 + (r0 + r) * p.g_sq));
#pragma unroll
                for (int r = 0; r < BATCH; ++r) {
                    float x[8];
                    words[r].elements(shift_of(at0 + (r0 + r) * p.g_sq), x);
                    if (j + 8 > p.Tk)
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            if (j + c >= p.Tk) x[c] = 0.f;
#pragma unroll
                    for (int c = 0; c < 8; ++c) acc[c - (r0 + r) + 7] += x[c];
                }
            }
        } else {
            // at the matrix's ends: no branch between the reads, which would make each wait for the one before it
#pragma unroll
            for (int r0 = 0; r0 < 8; r0 += 4) {
                T x[4][8];
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        x[r][c] = i + r0 + r < p.Tq && j + c < p.Tk ? at0[(r0 + r) * p.g_sq + c] : from_f32<T>(0.f);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < 8; ++c) acc[c - (r0 + r) + 7] += to_f32<T>(x[r][c]);
            }
        }
    }
    __syncthreads();
    // the warp's diagonals: j - i = 8 k_warp - 7 + index; neighbouring threads share seven of them
    const int lo = 8 * k_warp - 7 - p.offset, hi = lo + DIAGS - 1;
    float *mine = hist + warp * buckets;
    const int from = bucket_of(at, side, both, lo), to = bucket_of(at, side, both, hi);
    if (from == to) {                   // all in one bucket
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 15; ++e) sum += acc[e];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) mine[from] = sum;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) diag[warp][lane * 8 + e] = acc[e];
        if (lane == 31)
#pragma unroll
            for (int e = 8; e < 15; ++e) diag[warp][lane * 8 + e] = acc[e];
        __syncwarp();
        if (lane < 31)
#pragma unroll
            for (int e = 8; e < 15; ++e) diag[warp][lane * 8 + e] += acc[e];
        __syncwarp();
        // a lane per bucket, which holds the differences [d0, d1]
        for (int b = lane; b < buckets; b += 32) {
            const int s = b < side ? b : b - side;
            const int near = s == 0 ? 0 : at[s - 1], far = s == side - 1 ? 1 << 30 : at[s] - 1;
            const int d0 = max(b < side ? -far : max(near, 1), lo);
            const int d1 = min(b >= side ? far : s == 0 && !both ? 1 << 30 : -near, hi);
            float sum = 0.f;
#pragma unroll 8
            for (int d = d0; d <= d1; ++d) sum += diag[warp][d - lo];
            mine[b] = sum;
        }
    }
    __syncthreads();
    float *out = p.parts + ((int64_t)h * gridDim.x + blockIdx.x) * buckets;
    for (int b = tid; b < buckets; b += BWD_THREADS)
        out[b] = (hist[b] + hist[buckets + b]) + (hist[2 * buckets + b] + hist[3 * buckets + b]);
}

// Adds the CTAs' parts, in 64 bits: one CTA per (bucket, head).
__global__ void __launch_bounds__(BWD_THREADS) relbias_sum_kernel(const __grid_constant__ BwdParams p, int parts) {
    __shared__ double warp_sum[BWD_WARPS];
    sm100::grid_wait();
    const int b = blockIdx.x, h = blockIdx.y, buckets = gridDim.x;
    double sum = 0.;
    for (int c = threadIdx.x; c < parts; c += BWD_THREADS) sum += p.parts[((int64_t)h * parts + c) * buckets + b];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
        store_from_f32(p.dw, (int64_t)b * p.H + h, p.w_dtype, (float)((warp_sum[0] + warp_sum[1]) + (warp_sum[2] + warp_sum[3])));
}

// Rows of a CTA: 64, few enough for the last CTAs to end together (24 x 4096 x 4096 fp16 and its bias at 64, 128, 256, 512
// rows: 265, 273, 292, 337 us); 32 for problems that leave room on the chip.
struct BwdGrid {
    int chunk, across, ctas;
};
BwdGrid bwd_grid(int64_t H, int64_t Tq, int64_t Tk) {
    const int64_t nI = (Tq + 7) / 8, nJ = (Tk + 7) / 8;
    auto grid = [&](int chunk) {
        const int64_t across = ceil_div64(nJ + chunk - 1, BWD_THREADS);
        return BwdGrid{chunk, (int)across, (int)(across * ceil_div64(nI, chunk))};
    };
    const BwdGrid fine = grid(4);
    return H * fine.ctas <= BWD_PER_SM * num_sms() ? fine : grid(8);
}

template <typename T>
int launch_fwd(FwdParams &p, int H, cudaStream_t st) {
    p.cols = (int)(p.Tk < FWD_COLS ? (p.Tk + 7) / 8 * 8 : FWD_COLS);
    const int64_t across = ceil_div64(p.Tk, p.cols), ctas = across * ceil_div64(p.Tq, FWD_ROWS);
    p.across = make_fastdiv((uint32_t)across);
    const size_t smem = fwd_smem<T>(p.cols, p.borders.side * (1 + p.borders.both));
    static_assert(fwd_smem<T>(FWD_COLS, 2 * MAX_SIDE) <= 48 << 10, "more than a kernel gets without asking");
    // Without a trigger for what follows, and so is the sum behind the gradient: gradient CTAs that wait on the SMs for a
    // large forward to end cost it 90 us (24 x 4096 x 4096 and its gradient 294 -> 385 us).
    return sm100::launch_pdl(relbias_fwd_kernel<T>, dim3((unsigned)ctas, (unsigned)H), FWD_THREADS, smem, st, p);
}
template <typename T>
int launch_bwd(const BwdParams &p, const BwdGrid &grid, bool vec, cudaStream_t st) {
    const int buckets = p.borders.side * (1 + p.borders.both);
    const size_t smem = (size_t)BWD_WARPS * buckets * sizeof(float);
    auto kernel = vec ? relbias_bwd_kernel<T, true> : relbias_bwd_kernel<T, false>;
    if (int e = sm100::launch_pdl(kernel, dim3((unsigned)grid.ctas, (unsigned)p.H), BWD_THREADS, smem, st, p)) return e;
    return sm100::launch_pdl(relbias_sum_kernel, dim3((unsigned)buckets, (unsigned)p.H), BWD_THREADS, 0, st, p, grid.ctas);
}

int check_sizes(int64_t H, int64_t Tq, int64_t Tk, int64_t offset) {
    if (H < 0 || Tq < 0 || Tk < 0) return RGD_E_INVALID;
    // differences of positions are 32-bit, and so are the grids
    if (H > 65535 || Tq > (1 << 22) || Tk > (1 << 28) || offset > (1 << 29) || offset < -(1 << 29) ||
        Tq * Tk > 1ll << 44)
        return RGD_E_SIZE;
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
    cudaStream_t st = (cudaStream_t)stream;
    if (out_dtype == RGD_F32) return relbias::launch_fwd<float>(p, (int)H, st);
    return out_dtype == RGD_F16 ? relbias::launch_fwd<__half>(p, (int)H, st) : relbias::launch_fwd<__nv_bfloat16>(p, (int)H, st);
}

extern "C" int64_t rgd_relbias_bwd_workspace_bytes(int64_t H, int64_t Tq, int64_t Tk, int num_buckets) {
    if (int e = relbias::check_sizes(H, Tq, Tk, 0)) return e;
    if (num_buckets < 1) return RGD_E_INVALID;
    if (H == 0 || Tq == 0 || Tk == 0) return 0;
    return H * relbias::bwd_grid(H, Tq, Tk).ctas * (int64_t)num_buckets * (int64_t)sizeof(float);
}

extern "C" int rgd_relbias_bwd(const rgd_relbias *bias, const void *dbias, int64_t stride_h, int64_t stride_q, int dtype, void *dweight,
                               int64_t H, int64_t Tq, int64_t Tk, int64_t offset, void *workspace, int64_t workspace_bytes, void *stream) {
    if (int e = relbias::check(bias)) return e;
    if (!dtype_ok(dtype)) return RGD_E_DTYPE;
    if (int e = relbias::check_sizes(H, Tq, Tk, offset)) return e;
    if (stride_h < 0 || stride_q < 0) return RGD_E_STRIDE;
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
    p.g = dbias; p.g_sh = stride_h; p.g_sq = stride_q;
    p.dw = dweight; p.w_dtype = bias->dtype;
    p.parts = reinterpret_cast<float *>(workspace);
    p.H = (int)H; p.Tq = (int)Tq; p.Tk = (int)Tk; p.offset = (int)offset;
    const relbias::BwdGrid grid = relbias::bwd_grid(H, Tq, Tk);
    p.chunk = grid.chunk;
    p.across = grid.across;
    const int ve = 16 / dtype_size(dtype);
    const bool vec = is_aligned(dbias, 16) && stride_h % ve == 0 && stride_q % ve == 0;
    if (dtype == RGD_F32) return relbias::launch_bwd<float>(p, grid, vec, st);
    return dtype == RGD_F16 ? relbias::launch_bwd<__half>(p, grid, vec, st) : relbias::launch_bwd<__nv_bfloat16>(p, grid, vec, st);
}
