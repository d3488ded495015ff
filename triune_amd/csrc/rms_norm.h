// rms_norm.h -- RMS norms of rows, with the residual sum in front of them or the gate behind them, on gfx950.
//
//     sum and norm   h = r + s x (rounded to r's type),   y = h rstd(h) w          (without r: h = x)
//     gated          y = x rstd(x) w silu(z)
//     rstd(h) = 1 / sqrt(mean h^2 + eps)
// and, with xh = h rstd:
//     sum and norm   d = dy w,   g = rstd (d - xh mean(d xh)) + dh,   dr = g, dx = s g,  dw = sum dy xh,  ds = sum g x
//     gated          d = dy w silu(z),  dx = rstd (d - xh mean(d xh)),  dz = dy xh w silu'(z),  dw = sum dy xh silu(z)
// Bound by memory: a row is read once and stays in registers for its mean square and its outputs.  TPR threads take
// a row of K groups of eight columns each, from 8 threads (heads of 64) to sixteen waves; blocks walk rows with the
// next one's loads in flight.  The backward's blocks hold their columns' dw and ds in registers; a last kernel adds
// the blocks' parts in a fixed order.
//
// Sum and norm of 16384 rows of 1536, bf16: 52.4 us forward (201 MB, 3.8 TB/s), 66.0 backward (302 MB, 4.6 TB/s; 89.3
// without the next row's loads in flight).  9003 rows of 1001, fp16 with a float32 residual: 39.0 and 57.0 us (2.8 and
// 2.5 TB/s): rows that do not start on 16 bytes.  Gated, 393216 rows of 64, bf16: 29.6 us (151 MB, 5.1 TB/s, a large
// copy's rate); 98304 rows of 128: 16.3 forward, 29.9 backward.
#pragma once

#include "ssm.h"

namespace triune {

// Rows of D elements: row r starts (r / G) st0 + (r % G) st1 elements in.
struct NormRows {
    const void* p;
    int64_t st0, st1;
};
struct RmsParams {
    NormRows x, r;            // r.p null: no residual
    NormRows z;               // the gate
    const void *w, *s;        // [D] of w_dt / s_dt, or null; s: the residual scale of each channel
    int w_dt, s_dt;
    float alpha, eps;         // alpha: the residual scale without s
    void *y, *h;              // [R, D] contiguous; h in r's type
    float* rstd;              // [R] or null
    int64_t R;
    int G, D, cus;
};
struct RmsBwdParams {
    RmsParams f;              // r: h as it was kept (sum and norm); x: for ds only
    NormRows dy, dh;          // dh.p null: none
    void *dx, *dr, *dz;       // [R, D] contiguous, each may be null
    float* part;              // [parts, 2, D]: dw, ds; or null
    int64_t parts;
    void *dw, *ds;            // of w_dt / s_dt, or null
};

// r_f32: the residual (the sum kept for the backward) is float32 under 16-bit x.
hipError_t launch_rms_norm(const RmsParams& a, int io_dt, bool r_f32, hipStream_t s);
hipError_t launch_rms_norm_bwd(const RmsBwdParams& a, int io_dt, bool r_f32, hipStream_t s);
hipError_t launch_gated_norm(const RmsParams& a, int io_dt, hipStream_t s);
hipError_t launch_gated_norm_bwd(const RmsBwdParams& a, int io_dt, hipStream_t s);
int64_t rms_bwd_parts(int64_t R, int D, int cus);

namespace rms {

// Blocks of 256 threads a compute unit.  The backward's parts of dw and ds grow with them, and rows of few threads leave
// its waves short of loads (16384 rows of 1536, gradients and their sums, bf16: 71 us with two, 79 with three, 88 with
// four; 98304 rows of 128, gated: 44, 38 and 37, 44 with six).
constexpr int FWD_BLOCKS = 8, BWD_BLOCKS = 2, BWD_BLOCKS_NARROW = 4;
constexpr int block_threads(int tpr) { return tpr <= 256 ? 256 : tpr; }
// Rows that a block takes at once, by the width (see `by_width`).
inline int rows_per_block(int D) {
    if (D % 8) return D <= 2048 ? 4 : 1;
    return D <= 64 ? 32 : D <= 128 ? 16 : D <= 256 ? 8 : D <= 2048 ? 4 : 1;
}

// The sum over the TPR threads of a row, in each of them.  `s` is used by rows of several waves.
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* s) {
    x = dpp_add<0xB1>(x);                            // quad_perm [1, 0, 3, 2]
    x = dpp_add<0x4E>(x);                            // quad_perm [2, 3, 0, 1]
    x = dpp_add<0x141>(x);                           // row_half_mirror: eight lanes
    if constexpr (TPR >= 16) x = dpp_add<0x140>(x);  // row_mirror
    if constexpr (TPR >= 32) x = xor_sum<16>(x);
    if constexpr (TPR >= 64) x = xor_sum<32>(x);
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

// Columns of thread t: groups of eight, TPR * 8 apart.
template <int TPR>
__device__ __forceinline__ int column(int t, int k) {
    return (k * TPR + t) * 8;
}

// Eight elements of a row from column c, zeros past its end.  EIGHTS: the width is a multiple of eight, so a group is in
// the row or past it and the load depends on no condition, which would make the compiler wait for it.
template <bool EIGHTS, typename T>
__device__ __forceinline__ Raw<T, 8> load_group(const T* p, int c, int D) {
    if constexpr (!EIGHTS) return load_raw<8>(p + c, D - c);
    Raw<T, 8> r = load_raw<8>(p + (c < D ? c : 0), 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = c < D ? r.v[j] : (T)0.f;
    return r;
}
template <typename T>
__device__ __forceinline__ void spread(const void* p, int c, int n, float (&x)[8]) {
    const Raw<T, 8> r = load_raw<8>((const T*)p + c, n);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)r.v[j];
}
__device__ __forceinline__ void load_par(const void* p, int dt, int c, int n, float none, float (&x)[8]) {
    if (!p || n <= 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = none;
    } else if (dt == DT_F32) {
        spread<float>(p, c, n, x);
    } else if (dt == DT_BF16) {
        spread<__bf16>(p, c, n, x);
    } else {
        spread<_Float16>(p, c, n, x);
    }
}
// Parameters of every column in LDS: in registers they would leave fewer waves a SIMD.
template <int TPR, int K>
struct Par {
    float v[K][2][TPR][4];
    __device__ __forceinline__ void put(const void* p, int dt, int D, float none) {
        const int t = threadIdx.x;
        if (t >= TPR) return;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float x[8];
            load_par(p, dt, column<TPR>(t, k), D - column<TPR>(t, k), none, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[k][j >> 2][t][j & 3] = x[j];
        }
    }
    __device__ __forceinline__ float at(int k, int t, int j) const { return v[k][j >> 2][t][j & 3]; }
};

// x, not to be merged into a mixed-precision product that rounds to fp16 by itself: whether the compiler does so depends on
// the kernel, and the norm of a kept sum would differ from that of the same row read again.
template <typename T>
__device__ __forceinline__ float apart(float x) {
    if constexpr (sizeof(T) == 2) asm("" : "+v"(x));
    return x;
}

template <typename T>
__device__ __forceinline__ const T* row_ptr(const NormRows& a, int64_t r, int G) {
    if (G == 1) return (const T*)a.p + r * a.st0;
    const uint32_t o = (uint32_t)r / (uint32_t)G, i = (uint32_t)r - o * (uint32_t)G;
    return (const T*)a.p + o * a.st0 + i * a.st1;
}

// The sum of a block's rows' parts, a thread's K groups of eight columns, into part[which].
template <int TPR, int RPB, int K>
__device__ __forceinline__ void put_parts(float* to, const float (&x)[K][8], int D, float* s_par) {
    const int t = threadIdx.x % TPR, rl = threadIdx.x / TPR;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if constexpr (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; ++j) s_par[(rl * 8 + j) * TPR + t] = x[k][j];
            __syncthreads();
            for (int e = threadIdx.x; e < TPR * 8; e += RPB * TPR) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < RPB; ++i) s += s_par[(i * 8 + (e & 7)) * TPR + (e >> 3)];
                const int col = k * TPR * 8 + e;
                if (col < D) to[col] = s;
            }
        } else {
            const int c = column<TPR>(t, k);
            if (c < D) store_raw<8>(to + c, D - c, x[k]);
        }
    }
}

// F::run<TPR, K, EIGHTS>(p, s) for the width.
template <typename F, typename P>
hipError_t by_width(const P& p, int D, hipStream_t s) {
    if (D % 8) {
        if (D <= 512) return F::template run<64, 1, false>(p, s);
        if (D <= 2048) return F::template run<64, 4, false>(p, s);
        if (D <= 8192) return F::template run<256, 4, false>(p, s);
        return F::template run<1024, 2, false>(p, s);
    }
    if (D <= 64) return F::template run<8, 1, true>(p, s);
    if (D <= 128) return F::template run<16, 1, true>(p, s);
    if (D <= 256) return F::template run<32, 1, true>(p, s);
    if (D <= 512) return F::template run<64, 1, true>(p, s);
    if (D <= 1024) return F::template run<64, 2, true>(p, s);
    if (D <= 1536) return F::template run<64, 3, true>(p, s);
    if (D <= 2048) return F::template run<64, 4, true>(p, s);
    if (D <= 4096) return F::template run<256, 2, true>(p, s);
    if (D <= 8192) return F::template run<256, 4, true>(p, s);
    return F::template run<1024, 2, true>(p, s);
}

template <int TPR>
unsigned fwd_grid(const RmsParams& a) {
    constexpr int RPB = block_threads(TPR) / TPR;
    const int64_t blocks = (a.R + RPB - 1) / RPB, most = (int64_t)a.cus * FWD_BLOCKS * 256 / block_threads(TPR);
    return (unsigned)(blocks < most ? blocks : most);
}

}  // namespace rms

hipError_t launch_rms_bwd_sum(const RmsBwdParams& a, hipStream_t s);

}  // namespace triune
