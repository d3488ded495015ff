// layer_norm.hip -- layer norm over the last dim on gfx950, and its gradients.
//
//     xh = (x - mean) rstd;  y = xh w + b
//     with g = dy w:  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
// Bound by memory: a row is read once and stays in registers for its mean, its variance about that
// mean (two passes over registers, so no cancellation) and its outputs.  A wave takes a row up to
// 2048 wide, four waves one up to 8192, sixteen one up to 16384.  The backward's blocks walk rows
// and hold their columns' dw and db in registers; a last kernel adds the blocks' parts in a fixed
// order.
#include "ssm.h"

namespace triune {

namespace {

// The sum over the TPR threads of a row, in each of them.  `s` is used by rows of several waves.
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* s) {
    x = xor_sum<16>(xor_sum<32>(dpp_sum16(x)));
    if constexpr (TPR > 64) {
        const int w = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s[w] = x;
        __syncthreads();
        x = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) x += s[i];
    }
    return x;
}

// Blocks of 256 threads a compute unit, each walking rows.  The backward's parts of dw and db grow with them (16384
// rows of 1536, bf16, forward and gradients: 65 us with two, 77 with three; weights in registers 70).
constexpr int FWD_BLOCKS = 4, BWD_BLOCKS = 2;
constexpr int block_threads(int tpr) { return tpr == 64 ? 256 : tpr; }

// Columns of thread t: groups of eight, TPR * 8 apart.
template <int TPR>
__device__ __forceinline__ int column(int t, int k) {
    return (k * TPR + t) * 8;
}

// Eight elements of a row from column c, zeros past its end.  EIGHTS: the width is a multiple of eight, so a
// group is in the row or past it, and the load depends on no condition (which would make the compiler wait
// where it joins the registers, so that no row is in flight).  16384 rows of 1536 (bf16), forward and gradients: 66.3
// us, 80.9 with the conditions; 4096 of 8192: 102 and 128.
template <bool EIGHTS, typename T>
__device__ __forceinline__ Raw<T, 8> load_group(const T* p, int c, int D) {
    if constexpr (!EIGHTS) return load_raw<8>(p + c, D - c);
    Raw<T, 8> r = load_raw<8>(p + (c < D ? c : 0), 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = c < D ? r.v[j] : (T)0.f;
    return r;
}

__device__ __forceinline__ void load_par(const void* p, int dt, int c, int n, float none, float (&x)[8]) {
    if (!p || n <= 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = none;
    } else if (dt == DT_F32) {
        const Raw<float, 8> r = load_raw<8>((const float*)p + c, n);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = r.v[j];
    } else if (dt == DT_BF16) {
        const Raw<__bf16, 8> r = load_raw<8>((const __bf16*)p + c, n);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)r.v[j];
    } else {
        const Raw<_Float16, 8> r = load_raw<8>((const _Float16*)p + c, n);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)r.v[j];
    }
}

}  // namespace

// Blocks walk rows, the next row's loads in flight during this one's sums; w and b are loaded once, to LDS: in
// registers they leave fewer waves a SIMD (16384 rows of 1536, bf16, two inputs in turn, partly in the last-level
// cache: 23.3 us and 27.6; 4096 of 8192: 35.3 and 45.7.  Three inputs, with mean and rstd stored: 26.6 us, 3.8 TB/s).
template <typename T, int TPR, int K, bool EIGHTS>
__global__ __launch_bounds__(block_threads(TPR)) void norm_kernel(NormParams a) {
    constexpr int RPB = block_threads(TPR) / TPR;
    __shared__ float s_red[16];
    __shared__ __attribute__((aligned(16))) float s_par[2][K][2][TPR][4];  // w, b
    const int t = threadIdx.x % TPR;
    int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    const float width = (float)a.D;  // divided by: a constant row's mean is its value where its sum is exact
    Raw<T, 8> raw[K];
    auto fetch = [&](int64_t row) {
        const T* px = (const T*)a.x + row * a.x_st;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = column<TPR>(t, k);
            raw[k] = load_group<EIGHTS>(px, c, a.D);
        }
    };
    if (RPB == 1 || r < a.R) fetch(r);
    if (threadIdx.x < TPR) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = column<TPR>(t, k);
            float w[8], b[8];
            load_par(a.w, a.w_dt, c, a.D - c, 1.f, w);
            load_par(a.b, a.b_dt, c, a.D - c, 0.f, b);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) s_par[0][k][h][t][j] = w[4 * h + j], s_par[1][k][h][t][j] = b[4 * h + j];
        }
    }
    __syncthreads();
    const int64_t step = (int64_t)gridDim.x * RPB;
    for (; r < a.R; r += step) {
        float x[K][8], s = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += x[k][j] = (float)raw[k].v[j];
        if (r + step < a.R) fetch(r + step);
        const float mean = row_sum<TPR>(s, s_red) / width;
        s = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int left = a.D - column<TPR>(t, k);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[k][j] = j < left ? x[k][j] - mean : 0.f;
                s = __builtin_fmaf(x[k][j], x[k][j], s);
            }
        }
        const float rstd = 1.f / sqrtf(row_sum<TPR>(s, s_red) / width + a.eps);
        if (a.mean && t == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        T* py = (T*)a.y + r * a.D;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = column<TPR>(t, k), left = a.D - c;
            if (left <= 0) continue;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                y[j] = __builtin_fmaf(x[k][j] * rstd, s_par[0][k][j >> 2][t][j & 3], s_par[1][k][j >> 2][t][j & 3]);
            store_raw<8>(py + c, left, y);
        }
    }
}

template <typename T, int TPR, int K, bool EIGHTS>
__global__ __launch_bounds__(block_threads(TPR)) void norm_bwd_kernel(NormBwdParams g) {
    const NormParams& a = g.f;
    constexpr int RPB = block_threads(TPR) / TPR;
    __shared__ float s_red[16];
    __shared__ float s_par[RPB > 1 ? RPB : 1][RPB > 1 ? TPR * 8 : 1];
    const int t = threadIdx.x % TPR, rl = threadIdx.x / TPR;
    const float inv = 1.f / (float)a.D;
    __shared__ __attribute__((aligned(16))) float s_w[K][2][TPR][4];  // the weights, as in the forward
    float dw[K][8], db[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = column<TPR>(t, k);
        if (threadIdx.x < TPR) {
            float w[8];
            load_par(a.w, a.w_dt, c, a.D - c, 1.f, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) s_w[k][j >> 2][t][j & 3] = w[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[k][j] = db[k][j] = 0.f;
    }
    __syncthreads();
    const int64_t step = (int64_t)gridDim.x * RPB;
    Raw<T, 8> nx[K], ny[K];
    float nmean, nrstd;
    auto fetch = [&](int64_t r) {
        const T *px = (const T*)a.x + r * a.x_st, *py = (const T*)g.dy + r * g.dy_st;
        nmean = a.mean[r];
        nrstd = a.rstd[r];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = column<TPR>(t, k);
            nx[k] = load_group<EIGHTS>(px, c, a.D);
            ny[k] = load_group<EIGHTS>(py, c, a.D);
        }
    };
    // the next row's loads in flight where its registers are free
    constexpr bool AHEAD = TPR <= 256 && K <= 3;
    int64_t r = (int64_t)blockIdx.x * RPB + rl;
    if (AHEAD && r < a.R) fetch(r);
    for (; r < a.R; r += step) {
        if constexpr (!AHEAD) fetch(r);
        T* pd = (T*)g.dx + r * a.D;
        const float mean = nmean, rstd = nrstd;
        Raw<T, 8> rx[K], ry[K];
#pragma unroll
        for (int k = 0; k < K; ++k) rx[k] = nx[k], ry[k] = ny[k];
        if (AHEAD && r + step < a.R) fetch(r + step);
        float s1 = 0.f, s2 = 0.f;
        float xh[K][8];
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                xh[k][j] = ((float)rx[k].v[j] - mean) * rstd;
                const float dy = (float)ry[k].v[j], gg = dy * s_w[k][j >> 2][t][j & 3];
                s1 += gg;  // past the row's end dy is 0
                s2 = __builtin_fmaf(gg, xh[k][j], s2);
                dw[k][j] = __builtin_fmaf(dy, xh[k][j], dw[k][j]);
                db[k][j] += dy;
            }
        }
        const float m1 = row_sum<TPR>(s1, s_red) * inv, m2 = row_sum<TPR>(s2, s_red) * inv;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = column<TPR>(t, k), left = a.D - c;
            if (left <= 0) continue;
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                o[j] = rstd * ((float)ry[k].v[j] * s_w[k][j >> 2][t][j & 3] - __builtin_fmaf(xh[k][j], m2, m1));
            store_raw<8>(pd + c, left, o);
        }
    }
    if (!g.part) return;
    float* pp = g.part + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = q ? db[k][j] : dw[k][j];
            const int c = column<TPR>(t, k);
            if constexpr (RPB > 1) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 8; ++j) s_par[rl][j * TPR + t] = v[j];
                __syncthreads();
                for (int e = threadIdx.x; e < TPR * 8; e += block_threads(TPR)) {
                    float s = 0.f;
#pragma unroll
                    for (int i = 0; i < RPB; ++i) s += s_par[i][(e & 7) * TPR + (e >> 3)];
                    const int col = k * TPR * 8 + e;
                    if (col < a.D) pp[(int64_t)q * a.D + col] = s;
                }
            } else if (c < a.D) {
                store_raw<8>(pp + (int64_t)q * a.D + c, a.D - c, v);
            }
        }
    }
}

// Sixteen threads per value, each every sixteenth part, then these: a fixed order.
__global__ __launch_bounds__(1024) void norm_bwd_sum_kernel(NormBwdParams g) {
    const int per = 2 * g.f.D, l = threadIdx.x & 63, id = blockIdx.x * 64 + l, w = threadIdx.x >> 6;
    __shared__ float red[16][64];
    float s = id < per ? sum_parts(g.part + id, per, w, g.parts) : 0.f;
    red[w][l] = s;
    __syncthreads();
    if (w || id >= per) return;
    for (int i = 1; i < 16; ++i) s += red[i][l];
    if (id < g.f.D) {
        if (g.dw) store_dt(g.dw, g.f.w_dt, id, s);
    } else if (g.db) {
        store_dt(g.db, g.f.b_dt, id - g.f.D, s);
    }
}

int64_t norm_bwd_parts(int64_t R, int D, int cus) {
    const int64_t rpb = D <= 2048 ? 4 : 1, blocks = (R + rpb - 1) / rpb, most = (int64_t)cus * BWD_BLOCKS;
    return blocks < most ? blocks : most;
}

namespace {

template <typename T, int TPR, int K, bool EIGHTS>
hipError_t norm_run(const NormParams& a, hipStream_t s) {
    constexpr int RPB = block_threads(TPR) / TPR;
    const int64_t blocks = (a.R + RPB - 1) / RPB, most = (int64_t)a.cus * FWD_BLOCKS * 256 / block_threads(TPR);
    norm_kernel<T, TPR, K, EIGHTS><<<dim3((unsigned)(blocks < most ? blocks : most)), block_threads(TPR), 0, s>>>(a);
    return hipGetLastError();
}
template <typename T, int TPR, int K, bool EIGHTS>
hipError_t norm_run(const NormBwdParams& g, hipStream_t s) {
    norm_bwd_kernel<T, TPR, K, EIGHTS><<<dim3((unsigned)g.parts), block_threads(TPR), 0, s>>>(g);
    return hipGetLastError();
}

template <typename T, bool EIGHTS, typename P>
hipError_t norm_width(const P& p, int D, hipStream_t s) {
    if (D <= 512) return norm_run<T, 64, 1, EIGHTS>(p, s);
    if (D <= 1024) return norm_run<T, 64, 2, EIGHTS>(p, s);
    if (D <= 1536) return norm_run<T, 64, 3, EIGHTS>(p, s);
    if (D <= 2048) return norm_run<T, 64, 4, EIGHTS>(p, s);
    if (D <= 4096) return norm_run<T, 256, 2, EIGHTS>(p, s);
    if (D <= 8192) return norm_run<T, 256, 4, EIGHTS>(p, s);
    return norm_run<T, 1024, 2, EIGHTS>(p, s);
}

template <typename P>
hipError_t norm_dtype(const P& p, int D, int dt, hipStream_t s) {
    if (dt == DT_F32) return D % 8 ? norm_width<float, false>(p, D, s) : norm_width<float, true>(p, D, s);
    if (dt == DT_BF16) return D % 8 ? norm_width<__bf16, false>(p, D, s) : norm_width<__bf16, true>(p, D, s);
    return D % 8 ? norm_width<_Float16, false>(p, D, s) : norm_width<_Float16, true>(p, D, s);
}

}  // namespace

hipError_t launch_norm(const NormParams& a, int dt, hipStream_t s) { return norm_dtype(a, a.D, dt, s); }

hipError_t launch_norm_bwd(const NormBwdParams& g, int dt, hipStream_t s) {
    const hipError_t e = norm_dtype(g, g.f.D, dt, s);
    if (e != hipSuccess || !g.part) return e;
    norm_bwd_sum_kernel<<<dim3((unsigned)((2 * g.f.D + 63) / 64)), 1024, 0, s>>>(g);
    return hipGetLastError();
}

}  // namespace triune
