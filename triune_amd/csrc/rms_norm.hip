// rms_norm.hip -- the residual sum and RMS norm in front of a block (rms_norm.h), and the sums of parameter gradients.
#include "rms_norm.h"

namespace triune {

using namespace rms;

// TH: the type of the residual and the sum.
template <typename T, typename TH, bool RES, int TPR, int K, bool EIGHTS>
__global__ __launch_bounds__(block_threads(TPR)) void rms_norm_kernel(RmsParams a) {
    constexpr int RPB = block_threads(TPR) / TPR;
    __shared__ float s_red[16];
    __shared__ __attribute__((aligned(16))) Par<TPR, K> s_w;
    __shared__ __attribute__((aligned(16))) Par<TPR, RES ? K : 1> s_s;
    const int t = threadIdx.x % TPR;
    int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    const int64_t step = (int64_t)gridDim.x * RPB;
    const float width = (float)a.D;
    Raw<T, 8> nx[K];
    Raw<TH, 8> nr[RES ? K : 1];
    auto fetch = [&](int64_t row) {
        const T* px = row_ptr<T>(a.x, row, a.G);
        const TH* pr = RES ? row_ptr<TH>(a.r, row, a.G) : nullptr;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            nx[k] = load_group<EIGHTS>(px, column<TPR>(t, k), a.D);
            if constexpr (RES) nr[k] = load_group<EIGHTS>(pr, column<TPR>(t, k), a.D);
        }
    };
    if (RPB == 1 || r < a.R) fetch(r);
    s_w.put(a.w, a.w_dt, a.D, 1.f);
    if constexpr (RES) s_s.put(a.s, a.s_dt, a.D, a.alpha);
    __syncthreads();
    for (; r < a.R; r += step) {
        float h[K][8], sq = 0.f;
        Raw<TH, 8> kept[RES ? K : 1];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[k][j] = (float)nx[k].v[j];
                if constexpr (RES) {
                    kept[k].v[j] = (TH)apart<TH>(__builtin_fmaf(s_s.at(k, t, j), h[k][j], (float)nr[k].v[j]));
                    h[k][j] = (float)kept[k].v[j];  // the norm is of the sum as it is kept
                }
                sq = __builtin_fmaf(h[k][j], h[k][j], sq);
            }
        if (r + step < a.R) fetch(r + step);
        const float rstd = 1.f / sqrtf(row_sum<TPR>(sq, s_red) / width + a.eps);
        if (a.rstd && t == 0) a.rstd[r] = rstd;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = column<TPR>(t, k), left = a.D - c;
            if (left <= 0) continue;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = apart<T>(h[k][j] * rstd * s_w.at(k, t, j));
            store_raw<8>((T*)a.y + r * a.D + c, left, y);
            if constexpr (RES) store_raw<8>((TH*)a.h + r * a.D + c, left, kept[k]);
        }
    }
}

template <typename T, typename TH, int TPR, int K, bool EIGHTS>
__global__ __launch_bounds__(block_threads(TPR)) void rms_norm_bwd_kernel(RmsBwdParams g) {
    const RmsParams& a = g.f;
    constexpr int RPB = block_threads(TPR) / TPR;
    __shared__ float s_red[16];
    __shared__ __attribute__((aligned(16))) Par<TPR, K> s_w, s_s;
    __shared__ float s_par[RPB > 1 ? RPB * TPR * 8 : 1];
    const int t = threadIdx.x % TPR;
    const float inv = 1.f / (float)a.D;
    float dw[K][8], ds[K][8];
    s_w.put(a.w, a.w_dt, a.D, 1.f);
    s_s.put(a.s, a.s_dt, a.D, a.alpha);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[k][j] = ds[k][j] = 0.f;
    __syncthreads();
    // the next row's loads in flight where its registers are free; without dh or ds a row that is read anyway stands for
    // theirs, so that no load stands behind a condition
    constexpr bool AHEAD = TPR <= 256 && K <= 3;
    const bool adds = g.dh.p;
    const NormRows rows_d = adds ? g.dh : a.r, rows_x = g.ds ? a.x : g.dy;
    Raw<TH, 8> fh[K], fd[K];
    Raw<T, 8> fy[K], fx[K];
    float frstd;
    auto fetch = [&](int64_t r) {
        const TH *ph = row_ptr<TH>(a.r, r, a.G), *pd = row_ptr<TH>(rows_d, r, a.G);
        const T *py = row_ptr<T>(g.dy, r, a.G), *px = row_ptr<T>(rows_x, r, a.G);
        frstd = a.rstd[r];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = column<TPR>(t, k);
            fh[k] = load_group<EIGHTS>(ph, c, a.D);
            fy[k] = load_group<EIGHTS>(py, c, a.D);
            if (AHEAD || adds) fd[k] = load_group<EIGHTS>(pd, c, a.D);
            if (AHEAD || g.ds) fx[k] = load_group<EIGHTS>(px, c, a.D);
        }
    };
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (AHEAD && r < a.R) fetch(r);
    for (; r < a.R; r += step) {
        if constexpr (!AHEAD) fetch(r);
        Raw<TH, 8> nh[K], nd[K];
        Raw<T, 8> ny[K], nx[K];
#pragma unroll
        for (int k = 0; k < K; ++k) nh[k] = fh[k], nd[k] = fd[k], ny[k] = fy[k], nx[k] = fx[k];
        const float rstd = frstd;
        if (AHEAD && r + step < a.R) fetch(r + step);
        float xh[K][8], d[K][8], sum = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float dy = (float)ny[k].v[j];
                xh[k][j] = (float)nh[k].v[j] * rstd;
                d[k][j] = dy * s_w.at(k, t, j);
                sum = __builtin_fmaf(d[k][j], xh[k][j], sum);
                dw[k][j] = __builtin_fmaf(dy, xh[k][j], dw[k][j]);
            }
        const float m = row_sum<TPR>(sum, s_red) * inv;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = column<TPR>(t, k), left = a.D - c;
            if (left <= 0) continue;
            float o[8], sc[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                o[j] = __builtin_fmaf(rstd, d[k][j] - xh[k][j] * m, adds ? (float)nd[k].v[j] : 0.f);
                sc[j] = o[j] * s_s.at(k, t, j);
                ds[k][j] = __builtin_fmaf(o[j], (float)nx[k].v[j], ds[k][j]);  // not used without g.ds
            }
            if (g.dr) store_raw<8>((TH*)g.dr + r * a.D + c, left, o);
            if (g.dx) store_raw<8>((T*)g.dx + r * a.D + c, left, sc);
        }
    }
    if (!g.part) return;
    float* to = g.part + (int64_t)blockIdx.x * 2 * a.D;
    put_parts<TPR, RPB, K>(to, dw, a.D, s_par);
    if (g.ds) put_parts<TPR, RPB, K>(to + a.D, ds, a.D, s_par);
}

// Sixteen threads per value, each every sixteenth part, then these: a fixed order.
__global__ __launch_bounds__(1024) void rms_bwd_sum_kernel(RmsBwdParams g) {
    const int per = (g.ds ? 2 : 1) * g.f.D, l = threadIdx.x & 63, id = blockIdx.x * 64 + l, w = threadIdx.x >> 6;
    __shared__ float red[16][64];
    float s = id < per ? sum_parts(g.part + id, 2 * g.f.D, w, g.parts) : 0.f;
    red[w][l] = s;
    __syncthreads();
    if (w || id >= per) return;
    for (int i = 1; i < 16; ++i) s += red[i][l];
    if (id < g.f.D) {
        if (g.dw) store_dt(g.dw, g.f.w_dt, id, s);
    } else {
        store_dt(g.ds, g.f.s_dt, id - g.f.D, s);
    }
}

int64_t rms_bwd_parts(int64_t R, int D, int cus) {
    const int64_t rpb = rows_per_block(D), blocks = (R + rpb - 1) / rpb;
    const int64_t most = (int64_t)cus * (rpb > 4 ? BWD_BLOCKS_NARROW : BWD_BLOCKS);
    return blocks < most ? blocks : most;
}

hipError_t launch_rms_bwd_sum(const RmsBwdParams& a, hipStream_t s) {
    if (!a.part) return hipSuccess;
    rms_bwd_sum_kernel<<<dim3((unsigned)(((a.ds ? 2 : 1) * a.f.D + 63) / 64)), 1024, 0, s>>>(a);
    return hipGetLastError();
}

namespace {

template <typename T, typename TH, bool RES>
struct Fwd {
    template <int TPR, int K, bool EIGHTS>
    static hipError_t run(const RmsParams& a, hipStream_t s) {
        rms_norm_kernel<T, TH, RES, TPR, K, EIGHTS><<<dim3(fwd_grid<TPR>(a)), block_threads(TPR), 0, s>>>(a);
        return hipGetLastError();
    }
};
template <typename T, typename TH>
struct Bwd {
    template <int TPR, int K, bool EIGHTS>
    static hipError_t run(const RmsBwdParams& a, hipStream_t s) {
        rms_norm_bwd_kernel<T, TH, TPR, K, EIGHTS><<<dim3((unsigned)a.parts), block_threads(TPR), 0, s>>>(a);
        return hipGetLastError();
    }
};
template <typename T, typename TH>
hipError_t fwd(const RmsParams& a, hipStream_t s) {
    return a.r.p ? by_width<Fwd<T, TH, true>>(a, a.D, s) : by_width<Fwd<T, T, false>>(a, a.D, s);
}

}  // namespace

hipError_t launch_rms_norm(const RmsParams& a, int io_dt, bool r_f32, hipStream_t s) {
    if (io_dt == DT_F32) return fwd<float, float>(a, s);
    if (io_dt == DT_BF16) return r_f32 ? fwd<__bf16, float>(a, s) : fwd<__bf16, __bf16>(a, s);
    return r_f32 ? fwd<_Float16, float>(a, s) : fwd<_Float16, _Float16>(a, s);
}
hipError_t launch_rms_norm_bwd(const RmsBwdParams& a, int io_dt, bool r_f32, hipStream_t s) {
    hipError_t e;
    const int D = a.f.D;
    if (io_dt == DT_F32) e = by_width<Bwd<float, float>>(a, D, s);
    else if (io_dt == DT_BF16) e = r_f32 ? by_width<Bwd<__bf16, float>>(a, D, s) : by_width<Bwd<__bf16, __bf16>>(a, D, s);
    else e = r_f32 ? by_width<Bwd<_Float16, float>>(a, D, s) : by_width<Bwd<_Float16, _Float16>>(a, D, s);
    return e == hipSuccess ? launch_rms_bwd_sum(a, s) : e;
}

}  // namespace triune
