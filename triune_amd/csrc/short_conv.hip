// short_conv.hip -- the short causal depthwise convolution on gfx950: prompts, packed prompts, single
// tokens and gradients.
//
//     p_t = bias + sum_j w_j x_{t-W+1+j}  (j < W; tokens before the first come from the state),
//     y_t = silu(p_t) or p_t
// Bound by memory: every value is read and written once.  A thread owns four channels (a wave's access
// is whole cache lines) and walks a run of tokens with the last W - 1 of them in registers, so a
// token is read again only as the next run's first W - 1.  Four channels and two tokens of loads in flight:
// 4 x 16384 tokens of 768 channels (W = 4, bf16) in 61 us (3.3 TB/s), against 73 with eight channels
// and four tokens, whose registers leave three waves on a SIMD.
#include "ssm.h"

namespace triune {

namespace {

constexpr int E = 4;     // channels of a thread
constexpr int RUN = 16;  // tokens of a forward run: a halo of 3 in 16, and runs enough for short prompts
constexpr int STEP = 2;  // tokens whose loads are in flight together

// Lanes along the channels (a power of two, at most a wave): the rest of the block takes further runs.
int channel_lanes(int D) {
    int n = 1;
    while (n < 64 && n * E < D) n *= 2;
    return n;
}

template <typename T>
__device__ __forceinline__ void widen(const Raw<T, E>& r, float (&x)[E]) {
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = (float)r.v[j];
}

template <int W>
struct Taps {
    float w[W][E], b[E];
};
// A group's taps are E W consecutive elements: W vector loads (element by element they took longer than
// a run's tokens).
template <int W, typename P>
__device__ __forceinline__ void load_taps_of(const P* w, const P* bias, int c, int n, Taps<W>& k) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const Raw<P, E> r = load_raw<E>(w + (int64_t)c * W + E * i, n * W - E * i);
#pragma unroll
        for (int e = 0; e < E; ++e) k.w[(E * i + e) % W][(E * i + e) / W] = (float)r.v[e];
    }
    const Raw<P, E> r = load_raw<E>(bias + c, bias ? n : 0);
#pragma unroll
    for (int e = 0; e < E; ++e) k.b[e] = (float)r.v[e];
}
// T: the I/O type; the taps have it or are fp32.
template <typename T, int W>
__device__ __forceinline__ void load_taps(const ConvParams& a, int c, int n, Taps<W>& k) {
    if (a.w_dt == DT_F32) load_taps_of<W>((const float*)a.w, (const float*)a.bias, c, n, k);
    else load_taps_of<W>((const T*)a.w, (const T*)a.bias, c, n, k);
}

// Row i (0 .. W - 2, oldest first) of a sequence's state, zeros without one.
template <typename T, int W>
__device__ __forceinline__ Raw<T, E> state_row(const ConvParams& a, int64_t row, int i, int c, int n) {
    i = i < 0 ? 0 : i;  // only where a packed call's offsets do not ascend
    return load_raw<E>((const T*)a.s0 + (row * (W - 1) + i) * a.Dm + c, a.s0 && row >= 0 ? n : 0);
}

}  // namespace

template <typename T, int W, bool PACKED>
__global__ __launch_bounds__(256) void conv_kernel(ConvParams a, int cl, int cblocks) {
    const int lc = threadIdx.x & (cl - 1), rl = threadIdx.x / cl, runs_pb = 256 / cl;
    const int64_t rb = blockIdx.x / cblocks;
    const int c = ((int)(blockIdx.x - rb * cblocks) * cl + lc) * E;
    const int n = min(a.Dm - c, E);
    if (n <= 0) return;
    const int64_t run = rb * runs_pb + rl, per = (a.T + RUN - 1) / RUN;
    int64_t seq, t0, t1, beg, end;  // tokens t0 .. t1 - 1; the sequence that holds t0 is beg .. end - 1
    if constexpr (PACKED) {
        t0 = run * RUN;
        t1 = min(t0 + RUN, min((int64_t)a.cu[a.n_seqs], a.T));
        t0 = max(t0, max((int64_t)a.cu[0], (int64_t)0));
        if (t0 >= t1) return;
        int64_t lo = 0, hi = a.n_seqs;  // cu[lo] <= t0 < cu[hi]
        while (hi - lo > 1) {
            const int64_t m = (lo + hi) >> 1;
            if (a.cu[m] <= t0) lo = m; else hi = m;
        }
        seq = lo;
        beg = max((int64_t)a.cu[seq], (int64_t)0);
        end = a.cu[seq + 1];
    } else {
        seq = run / per;
        if (seq >= a.n_seqs) return;
        t0 = (run - seq * per) * RUN;
        t1 = min(t0 + RUN, a.T);
        beg = 0;
        end = a.T;
    }
    const T* px = (const T*)a.x + (PACKED ? 0 : seq * a.x_sb) + c;
    T* py = (T*)a.y + (PACKED ? 0 : seq * a.y_sb) + c;
    Taps<W> k;
    load_taps<T, W>(a, c, n, k);
    float win[W - 1][E];  // tokens t - W + 1 .. t - 1
    auto window = [&](int64_t t) {
        const int64_t row = ssm_row(a.slots, a.n_slots, seq);
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
            const int64_t s = t - (W - 1) + i;
            widen(s >= beg ? load_raw<E>(px + s * a.x_st, n) : state_row<T, W>(a, row, (int)(s - beg) + W - 1, c, n), win[i]);
        }
    };
    window(t0);
    for (int64_t t = t0; t < t1; t += STEP) {
        Raw<T, E> r[STEP];
#pragma unroll
        for (int i = 0; i < STEP; ++i) r[i] = load_raw<E>(px + (t + i) * a.x_st, t + i < t1 ? n : 0);
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
            if (t + i >= t1) break;
            if (PACKED && t + i >= end) {  // the next sequence that holds tokens
                while (t + i >= end && seq + 1 < a.n_seqs) end = a.cu[++seq + 1];
                beg = max((int64_t)a.cu[seq], (int64_t)0);
                window(t + i);
            }
            float x[E], y[E];
            widen(r[i], x);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float p = __builtin_fmaf(k.w[W - 1][e], x[e], k.b[e]);
#pragma unroll
                for (int j = 0; j < W - 1; ++j) p = __builtin_fmaf(k.w[j][e], win[j][e], p);
                y[e] = a.silu ? silu_gate(p) : p;
#pragma unroll
                for (int j = 0; j < W - 2; ++j) win[j][e] = win[j + 1][e];
                win[W - 2][e] = x[e];
            }
            store_raw<E>(py + (t + i) * a.y_st, n, y);
        }
    }
    if (!PACKED && a.fin && t1 == a.T) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            const int64_t t = a.T - (W - 1) + j;
            store_raw<E>((T*)a.fin + (seq * (W - 1) + j) * a.Dm + c, n,
                         t >= 0 ? load_raw<E>(px + t * a.x_st, n) : state_row<T, W>(a, seq, (int)t + W - 1, c, n));
        }
    }
}

// Packed calls: the states after the sequences, in a launch of its own because a pool's rows are
// read by every run at a sequence's start.  One thread per (sequence, four channels).
template <typename T, int W>
__global__ __launch_bounds__(256) void conv_state_kernel(ConvParams a) {
    const int64_t groups = (a.Dm + E - 1) / E, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t seq = id / groups;
    if (seq >= a.n_seqs) return;
    const int c = (int)(id - seq * groups) * E, n = min(a.Dm - c, E);
    const int64_t row = ssm_row(a.slots, a.n_slots, seq);
    if (row < 0) return;
    const int64_t beg = min(max((int64_t)a.cu[seq], (int64_t)0), a.T);
    const int64_t len = min(max((int64_t)a.cu[seq + 1], beg), a.T) - beg;
    Raw<T, E> r[W - 1];
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int64_t s = len - (W - 1) + i;
        r[i] = s >= 0 ? load_raw<E>((const T*)a.x + (beg + s) * a.x_st + c, n)
                      : state_row<T, W>(a, row, (int)s + W - 1, c, n);
    }
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        store_raw<E>((T*)a.fin + (row * (W - 1) + i) * a.Dm + c, n, r[i]);
    }
}

// One token for every row.  One thread per (row, four channels).
template <typename T, int W>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvParams a) {
    const int64_t groups = (a.Dm + E - 1) / E, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t b = id / groups;
    if (b >= a.n_seqs) return;
    const int c = (int)(id - b * groups) * E, n = min(a.Dm - c, E);
    const int64_t row = ssm_row(a.slots, a.n_slots, b);
    Raw<T, E> r[W];
#pragma unroll
    for (int i = 0; i < W - 1; ++i) r[i] = state_row<T, W>(a, row, i, c, n);
    r[W - 1] = load_raw<E>((const T*)a.x + b * a.x_sb + c, n);
    Taps<W> k;
    load_taps<T, W>(a, c, n, k);
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        float p = k.b[e];
#pragma unroll
        for (int j = 0; j < W; ++j) p = __builtin_fmaf(k.w[j][e], (float)r[j].v[e], p);
        y[e] = row >= 0 ? (a.silu ? silu_gate(p) : p) : 0.f;
    }
    store_raw<E>((T*)a.y + b * a.y_sb + c, n, y);
    if (row < 0) return;
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        store_raw<E>((T*)a.fin + (row * (W - 1) + i) * a.Dm + c, n, r[i + 1]);
    }
}

// Gradients.  With dp_t = dy_t silu'(p_t): dx_s = sum_j w_j dp_{s+W-1-j} (s < 0: the state's rows),
// dw_j = sum_t dp_t x_{t-W+1+j}, dbias = sum_t dp_t.  A run walks its tokens and W - 1 more, whose
// dp it forms again; the gradient of token t - W + 1 is whole once dp_t is in.  Runs of a block add
// their dw in LDS, blocks through memory in a fixed order.
template <typename T, int W>
__global__ __launch_bounds__(256) void conv_bwd_kernel(ConvBwdParams g, int cl, int cblocks) {
    const ConvParams& a = g.f;
    __shared__ float s_red[256][E + 1];
    const int lc = threadIdx.x & (cl - 1), rl = threadIdx.x / cl, runs_pb = 256 / cl;
    const int64_t rb = blockIdx.x / cblocks;
    const int c = ((int)(blockIdx.x - rb * cblocks) * cl + lc) * E;
    const int n = min(a.Dm - c, E);
    const int64_t run = rb * runs_pb + rl, per = (a.T + g.run - 1) / g.run;
    const int64_t seq = run / per;
    float dw[W + 1][E];  // dw, then dbias
#pragma unroll
    for (int j = 0; j <= W; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) dw[j][e] = 0.f;
    if (n > 0 && seq < a.n_seqs) {
        const int64_t t0 = (run - seq * per) * g.run, t1 = min(t0 + g.run, a.T);
        // the gradients of t0 .. t1 - 1, before them the state's rows (first run)
        const int64_t from = t0 == 0 ? -(W - 1) : t0;
        const T* px = (const T*)a.x + seq * a.x_sb + c;
        const T* py = (const T*)g.dy + seq * g.dy_sb + c;
        T* pd = (T*)g.dx + seq * a.T * a.Dm + c;
        Taps<W> k;
        load_taps<T, W>(a, c, n, k);
        float win[W - 1][E], acc[W][E];  // acc[i]: the gradient of token t - W + 1 + i
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
            const int64_t s = t0 - (W - 1) + i;
            const Raw<T, E> r = s >= 0 ? load_raw<E>(px + s * a.x_st, n) : state_row<T, W>(a, seq, (int)s + W - 1, c, n);
            widen(r, win[i]);
        }
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[i][e] = 0.f;
        const int64_t stop = t1 + W - 1;
        for (int64_t t = t0; t < stop; t += STEP) {
            Raw<T, E> rx[STEP], ry[STEP];
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
                const int m = t + i < stop && t + i < a.T ? n : 0;
                rx[i] = load_raw<E>(px + (t + i) * a.x_st, m);
                ry[i] = load_raw<E>(py + (t + i) * g.dy_st, m);
            }
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
                const int64_t tt = t + i;
                if (tt >= stop) break;
                float x[E], dy[E];
                widen(rx[i], x);
                widen(ry[i], dy);
                const bool own = tt < t1;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float dp = dy[e];
                    if (a.silu) {
                        float p = __builtin_fmaf(k.w[W - 1][e], x[e], k.b[e]);
#pragma unroll
                        for (int j = 0; j < W - 1; ++j) p = __builtin_fmaf(k.w[j][e], win[j][e], p);
                        const float s = sigmoid(p);
                        dp *= s * __builtin_fmaf(p, 1.f - s, 1.f);
                    }
                    if (tt >= a.T) dp = 0.f;
#pragma unroll
                    for (int j = 0; j < W; ++j) acc[j][e] = __builtin_fmaf(k.w[j][e], dp, acc[j][e]);
                    const float d = own ? dp : 0.f;
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) dw[j][e] = __builtin_fmaf(d, win[j][e], dw[j][e]);
                    dw[W - 1][e] = __builtin_fmaf(d, x[e], dw[W - 1][e]);
                    dw[W][e] += d;
#pragma unroll
                    for (int j = 0; j < W - 2; ++j) win[j][e] = win[j + 1][e];
                    win[W - 2][e] = x[e];
                }
                const int64_t s = tt - (W - 1);  // acc[0] is its whole gradient
                if (s >= from) {
                    float out[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) out[e] = acc[0][e];
                    if (g.dfin && s >= a.T - (W - 1)) {
                        float f[E];
                        widen(load_raw<E>((const T*)g.dfin + (seq * (W - 1) + s - (a.T - (W - 1))) * a.Dm + c, n), f);
#pragma unroll
                        for (int e = 0; e < E; ++e) out[e] += f[e];
                    }
                    if (s >= 0) store_raw<E>(pd + s * a.Dm, n, out);
                    else if (g.ds0) store_raw<E>((T*)g.ds0 + (seq * (W - 1) + s + W - 1) * a.Dm + c, n, out);
                }
#pragma unroll
                for (int e = 0; e < E; ++e) {
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) acc[j][e] = acc[j + 1][e];
                    acc[W - 1][e] = 0.f;
                }
            }
        }
    }
    if (!g.part) return;
#pragma unroll
    for (int j = 0; j <= W; ++j) {
#pragma unroll
        for (int e = 0; e < E; ++e) s_red[threadIdx.x][e] = dw[j][e];
        __syncthreads();
        for (int q = threadIdx.x; q < cl * E; q += 256) {
            const int ch = ((int)(blockIdx.x - rb * cblocks) * cl) * E + q;
            float s = 0.f;
            for (int r = 0; r < runs_pb; ++r) s += s_red[r * cl + q / E][q % E];
            if (ch < a.Dm) g.part[(rb * (W + 1) + j) * a.Dm + ch] = s;
        }
        __syncthreads();
    }
}

// Sixteen threads per value, each every sixteenth part, then these: a fixed order.
__global__ __launch_bounds__(1024) void conv_bwd_sum_kernel(ConvBwdParams g) {
    const ConvParams& a = g.f;
    const int per = (a.W + 1) * a.Dm, id = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
    __shared__ float red[16][64];
    float s = id < per ? sum_parts(g.part + id, per, w, g.parts) : 0.f;
    red[w][threadIdx.x & 63] = s;
    __syncthreads();
    if (w || id >= per) return;
    for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x];
    const int j = id / a.Dm, ch = id - j * a.Dm;
    if (j < a.W) {
        if (g.dw) store_dt(g.dw, a.w_dt, (int64_t)ch * a.W + j, s);
    } else if (g.dbias) {
        store_dt(g.dbias, a.w_dt, ch, s);
    }
}

// Tokens of a gradient's run: its halo (of two tensors) and its part of dw are less in longer ones, but
// sixteen where 32 leave the chip under eight waves a compute unit (8 x 2048 tokens of 1536 channels:
// 102 us forward and backward with 32, 116 with 16; 3 x 3001 of 1001: 77 with 32, 61 with 16).
int conv_bwd_run(int64_t n_seqs, int64_t T, int D, int cus) {
    const int64_t threads = n_seqs * ((T + 31) / 32) * ((D + E - 1) / E);
    return threads >= (int64_t)cus * 8 * 64 ? 32 : 16;
}
int64_t conv_bwd_parts(int64_t n_seqs, int64_t T, int D, int run) {
    const int64_t runs = n_seqs * ((T + run - 1) / run), pb = 256 / channel_lanes(D);
    return (runs + pb - 1) / pb;
}

namespace {

struct Grid {
    int cl, cblocks;
    int64_t blocks;
};
Grid run_grid(int64_t runs, int D) {
    Grid g;
    g.cl = channel_lanes(D);
    g.cblocks = (D + g.cl * E - 1) / (g.cl * E);
    g.blocks = (runs + 256 / g.cl - 1) / (256 / g.cl) * g.cblocks;
    return g;
}
dim3 thread_blocks(int64_t n) { return dim3((unsigned)((n + 255) / 256)); }

template <typename T, int W>
hipError_t conv_w(const ConvParams& a, hipStream_t s) {
    const int64_t per = (a.T + RUN - 1) / RUN;
    const Grid g = run_grid(a.cu ? per : a.n_seqs * per, a.Dm);
    if (a.cu) conv_kernel<T, W, true><<<dim3((unsigned)g.blocks), 256, 0, s>>>(a, g.cl, g.cblocks);
    else conv_kernel<T, W, false><<<dim3((unsigned)g.blocks), 256, 0, s>>>(a, g.cl, g.cblocks);
    return hipGetLastError();
}
template <typename T, int W>
hipError_t conv_state_w(const ConvParams& a, hipStream_t s) {
    conv_state_kernel<T, W><<<thread_blocks(a.n_seqs * ((a.Dm + E - 1) / E)), 256, 0, s>>>(a);
    return hipGetLastError();
}
template <typename T, int W>
hipError_t conv_step_w(const ConvParams& a, hipStream_t s) {
    conv_step_kernel<T, W><<<thread_blocks(a.n_seqs * ((a.Dm + E - 1) / E)), 256, 0, s>>>(a);
    return hipGetLastError();
}
template <typename T, int W>
hipError_t conv_bwd_w(const ConvBwdParams& b, hipStream_t s) {
    const ConvParams& a = b.f;
    const Grid g = run_grid(a.n_seqs * ((a.T + b.run - 1) / b.run), a.Dm);
    conv_bwd_kernel<T, W><<<dim3((unsigned)g.blocks), 256, 0, s>>>(b, g.cl, g.cblocks);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !b.part) return e;
    conv_bwd_sum_kernel<<<dim3((unsigned)(((W + 1) * a.Dm + 63) / 64)), 1024, 0, s>>>(b);
    return hipGetLastError();
}

}  // namespace

#define CONV_DISPATCH(FN, W_, DT, ...)                                      \
    switch (W_) {                                                           \
        case 2: return DT == DT_F32 ? FN<float, 2>(__VA_ARGS__) : DT == DT_BF16 ? FN<__bf16, 2>(__VA_ARGS__) : FN<_Float16, 2>(__VA_ARGS__); \
        case 3: return DT == DT_F32 ? FN<float, 3>(__VA_ARGS__) : DT == DT_BF16 ? FN<__bf16, 3>(__VA_ARGS__) : FN<_Float16, 3>(__VA_ARGS__); \
        default: return DT == DT_F32 ? FN<float, 4>(__VA_ARGS__) : DT == DT_BF16 ? FN<__bf16, 4>(__VA_ARGS__) : FN<_Float16, 4>(__VA_ARGS__); \
    }

hipError_t launch_conv(const ConvParams& a, int dt, hipStream_t s) { CONV_DISPATCH(conv_w, a.W, dt, a, s) }
hipError_t launch_conv_state(const ConvParams& a, int dt, hipStream_t s) { CONV_DISPATCH(conv_state_w, a.W, dt, a, s) }
hipError_t launch_conv_step(const ConvParams& a, int dt, hipStream_t s) { CONV_DISPATCH(conv_step_w, a.W, dt, a, s) }
hipError_t launch_conv_bwd(const ConvBwdParams& b, int dt, hipStream_t s) { CONV_DISPATCH(conv_bwd_w, b.f.W, dt, b, s) }

}  // namespace triune
