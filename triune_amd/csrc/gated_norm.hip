// gated_norm.hip -- the RMS norm behind a block with its gate (rms_norm.h).
#include "rms_norm.h"

namespace triune {

using namespace rms;

template <typename T, int TPR, int K, bool EIGHTS>
__global__ __launch_bounds__(block_threads(TPR)) void gated_norm_kernel(RmsParams a) {
    constexpr int RPB = block_threads(TPR) / TPR;
    __shared__ float s_red[16];
    __shared__ __attribute__((aligned(16))) Par<TPR, K> s_w;
    const int t = threadIdx.x % TPR;
    int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    const int64_t step = (int64_t)gridDim.x * RPB;
    const float width = (float)a.D;
    Raw<T, 8> nx[K], nz[K];
    auto fetch = [&](int64_t row) {
        const T *px = row_ptr<T>(a.x, row, a.G), *pz = row_ptr<T>(a.z, row, a.G);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            nx[k] = load_group<EIGHTS>(px, column<TPR>(t, k), a.D);
            nz[k] = load_group<EIGHTS>(pz, column<TPR>(t, k), a.D);
        }
    };
    if (RPB == 1 || r < a.R) fetch(r);
    s_w.put(a.w, a.w_dt, a.D, 1.f);
    __syncthreads();
    for (; r < a.R; r += step) {
        float x[K][8], z[K][8], sq = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[k][j] = (float)nx[k].v[j];
                z[k][j] = (float)nz[k].v[j];
                sq = __builtin_fmaf(x[k][j], x[k][j], sq);
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
            for (int j = 0; j < 8; ++j) y[j] = x[k][j] * rstd * s_w.at(k, t, j) * silu_gate(z[k][j]);
            store_raw<8>((T*)a.y + r * a.D + c, left, y);
        }
    }
}

template <typename T, int TPR, int K, bool EIGHTS>
__global__ __launch_bounds__(block_threads(TPR)) void gated_norm_bwd_kernel(RmsBwdParams g) {
    const RmsParams& a = g.f;
    constexpr int RPB = block_threads(TPR) / TPR;
    __shared__ float s_red[16];
    __shared__ __attribute__((aligned(16))) Par<TPR, K> s_w;
    __shared__ float s_par[RPB > 1 ? RPB * TPR * 8 : 1];
    const int t = threadIdx.x % TPR;
    const float inv = 1.f / (float)a.D;
    float dw[K][8];
    s_w.put(a.w, a.w_dt, a.D, 1.f);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[k][j] = 0.f;
    __syncthreads();
    constexpr bool AHEAD = TPR <= 256 && K <= 3;  // the next row's loads in flight where its registers are free
    Raw<T, 8> fx[K], fz[K], fy[K];
    float frstd;
    auto fetch = [&](int64_t r) {
        const T *px = row_ptr<T>(a.x, r, a.G), *pz = row_ptr<T>(a.z, r, a.G), *py = row_ptr<T>(g.dy, r, a.G);
        frstd = a.rstd[r];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            fx[k] = load_group<EIGHTS>(px, column<TPR>(t, k), a.D);
            fz[k] = load_group<EIGHTS>(pz, column<TPR>(t, k), a.D);
            fy[k] = load_group<EIGHTS>(py, column<TPR>(t, k), a.D);
        }
    };
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (AHEAD && r < a.R) fetch(r);
    for (; r < a.R; r += step) {
        if constexpr (!AHEAD) fetch(r);
        Raw<T, 8> nx[K], nz[K], ny[K];
#pragma unroll
        for (int k = 0; k < K; ++k) nx[k] = fx[k], nz[k] = fz[k], ny[k] = fy[k];
        const float rstd = frstd;
        if (AHEAD && r + step < a.R) fetch(r + step);
        float xh[K][8], d[K][8], dz[K][8], sum = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float dy = (float)ny[k].v[j], z = (float)nz[k].v[j], w = s_w.at(k, t, j), sg = fast_sigmoid(z);
                xh[k][j] = (float)nx[k].v[j] * rstd;
                const float gate = z * sg;
                d[k][j] = dy * w * gate;
                dz[k][j] = dy * w * xh[k][j] * sg * (1.f + z * (1.f - sg));
                sum = __builtin_fmaf(d[k][j], xh[k][j], sum);
                dw[k][j] = __builtin_fmaf(dy * gate, xh[k][j], dw[k][j]);
            }
        const float m = row_sum<TPR>(sum, s_red) * inv;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = column<TPR>(t, k), left = a.D - c;
            if (left <= 0) continue;
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = rstd * (d[k][j] - xh[k][j] * m);
            if (g.dx) store_raw<8>((T*)g.dx + r * a.D + c, left, o);
            if (g.dz) store_raw<8>((T*)g.dz + r * a.D + c, left, dz[k]);
        }
    }
    if (g.part) put_parts<TPR, RPB, K>(g.part + (int64_t)blockIdx.x * 2 * a.D, dw, a.D, s_par);
}

namespace {

template <typename T>
struct Fwd {
    template <int TPR, int K, bool EIGHTS>
    static hipError_t run(const RmsParams& a, hipStream_t s) {
        gated_norm_kernel<T, TPR, K, EIGHTS><<<dim3(fwd_grid<TPR>(a)), block_threads(TPR), 0, s>>>(a);
        return hipGetLastError();
    }
};
template <typename T>
struct Bwd {
    template <int TPR, int K, bool EIGHTS>
    static hipError_t run(const RmsBwdParams& a, hipStream_t s) {
        gated_norm_bwd_kernel<T, TPR, K, EIGHTS><<<dim3((unsigned)a.parts), block_threads(TPR), 0, s>>>(a);
        return hipGetLastError();
    }
};

}  // namespace

hipError_t launch_gated_norm(const RmsParams& a, int io_dt, hipStream_t s) {
    if (io_dt == DT_F32) return by_width<Fwd<float>>(a, a.D, s);
    return io_dt == DT_BF16 ? by_width<Fwd<__bf16>>(a, a.D, s) : by_width<Fwd<_Float16>>(a, a.D, s);
}
hipError_t launch_gated_norm_bwd(const RmsBwdParams& a, int io_dt, hipStream_t s) {
    const hipError_t e = io_dt == DT_F32    ? by_width<Bwd<float>>(a, a.f.D, s)
                         : io_dt == DT_BF16 ? by_width<Bwd<__bf16>>(a, a.f.D, s)
                                            : by_width<Bwd<_Float16>>(a, a.f.D, s);
    return e == hipSuccess ? launch_rms_bwd_sum(a, s) : e;
}

}  // namespace triune
