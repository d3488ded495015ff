// short_conv.hip -- the short causal depthwise convolution on gfx950: prompts, packed prompts, single
// tokens and gradients.
//
//     p_t = bias + sum_j w_j x_{t-W+1+j}  (j < W; tokens before the first come from the state),
//     y_t = silu(p_t) or p_t
// Bound by memory: every value is read and written once.  A thread owns four channels (a wave's access
// is whole cache lines) and walks a run of tokens with the last W - 1 of them in registers, so a
// token is read again only as the next run's first W - 1.  Whole runs inside a sequence load the next two tokens
// before they work on two and have no condition around an access; the others go token by token.
// 4 x 16384 tokens of 768 channels (W = 4, bf16): 47 us (4.3 TB/s), 61 with the conditions in the loop; forward and
// gradients of 8 x 2048 tokens of 1536 channels 86 us, 102 with them (93 with one token ahead, 98 with four).
#include "ssm.h"

namespace triune {

namespace {

constexpr int E = 4;     // channels of a thread
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

// A token's outputs p from its inputs x and the window of the W - 1 before it, which moves on.
template <int W>
__device__ __forceinline__ void taps(const Taps<W>& k, float (&win)[W - 1][E], const float (&x)[E], float (&p)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
        p[e] = __builtin_fmaf(k.w[W - 1][e], x[e], k.b[e]);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) p[e] = __builtin_fmaf(k.w[j][e], win[j][e], p[e]);
#pragma unroll
        for (int j = 0; j < W - 2; ++j) win[j][e] = win[j + 1][e];
        win[W - 2][e] = x[e];
    }
}

template <typename T, int W, bool PACKED>
__global__ __launch_bounds__(256) void conv_kernel(ConvParams a, int cl, int cblocks) {
    const int lc = threadIdx.x & (cl - 1), rl = threadIdx.x / cl, runs_pb = 256 / cl;
    const uint32_t rb = blockIdx.x / (uint32_t)cblocks;
    const int c = ((int)(blockIdx.x - rb * cblocks) * cl + lc) * E;
    const int n = min(a.Dm - c, E);
    if (n <= 0) return;
    const uint32_t run = rb * runs_pb + rl, per = (uint32_t)((a.T + a.run - 1) / a.run);
    int64_t seq, t0, t1, beg, end;  // tokens t0 .. t1 - 1; the sequence that holds t0 is beg .. end - 1
    if constexpr (PACKED) {
        t0 = (int64_t)run * a.run;
        t1 = min(t0 + a.run, min((int64_t)a.cu[a.n_seqs], a.T));
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
        t0 = (int64_t)(run - (uint32_t)seq * per) * a.run;
        t1 = min(t0 + a.run, a.T);
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
            widen(s >= beg ? load_raw<E>(px + s * a.x_st, n) : state_row<T, W>(a, row, (int)(s - beg) + W - 1, c, n),
                  win[i]);
        }
    };
    window(t0);
    if (n == E && t1 - t0 == a.run && t1 <= end) {
        // A whole run of one sequence: no access depends on a condition, which would make the compiler wait for
        // loads where it joins their registers.
        const T* p = px + t0 * a.x_st;
        T* q = py + t0 * a.y_st;
        Raw<T, E> r[STEP];
#pragma unroll
        for (int i = 0; i < STEP; ++i) r[i] = load_raw<E>(p + i * a.x_st, E);
#pragma unroll 1
        for (int t = 0; t < a.run; t += STEP) {
            float o[STEP][E];
            const int64_t ahead = t + STEP < a.run ? STEP * a.x_st : 0;  // the last step's loads are its own again
            p += ahead;
            Raw<T, E> next[STEP];
#pragma unroll
            for (int i = 0; i < STEP; ++i) next[i] = load_raw<E>(p + i * a.x_st, E);
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
                float x[E];
                widen(r[i], x);
                taps<W>(k, win, x, o[i]);
                r[i] = next[i];
            }
            if (a.silu) {
#pragma unroll
                for (int i = 0; i < STEP; ++i)
#pragma unroll
                    for (int e = 0; e < E; ++e) o[i][e] = silu_gate(o[i][e]);
            }
#pragma unroll
            for (int i = 0; i < STEP; ++i) store_raw<E>(q + i * a.y_st, E, o[i]);
            q += STEP * a.y_st;
        }
    } else {
        for (int64_t t = t0; t < t1; ++t) {
            if (PACKED && t >= end) {  // the next sequence that holds tokens
                while (t >= end && seq + 1 < a.n_seqs) end = a.cu[++seq + 1];
                beg = max((int64_t)a.cu[seq], (int64_t)0);
                window(t);
            }
            float x[E], o[E];
            widen(load_raw<E>(px + t * a.x_st, n), x);
            taps<W>(k, win, x, o);
            if (a.silu) {
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = silu_gate(o[e]);
            }
            store_raw<E>(py + t * a.y_st, n, o);
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
    const uint32_t rb = blockIdx.x / (uint32_t)cblocks;
    const int c = ((int)(blockIdx.x - rb * cblocks) * cl + lc) * E;
    const int n = min(a.Dm - c, E);
    const uint32_t run = rb * runs_pb + rl, per = (uint32_t)((a.T + a.run - 1) / a.run);
    const int64_t seq = run / per;
    float dw[W + 1][E];  // dw, then dbias
#pragma unroll
    for (int j = 0; j <= W; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) dw[j][e] = 0.f;
    if (n > 0 && seq < a.n_seqs) {
        const int64_t t0 = (int64_t)(run - (uint32_t)seq * per) * a.run, t1 = min(t0 + a.run, a.T), stop = t1 + W - 1;
        const T* px = (const T*)a.x + seq * a.x_sb + c;
        const T* py = (const T*)g.dy + seq * g.dy_sb + c;
        T* pd = (T*)g.dx + seq * a.T * a.Dm + c;
        Taps<W> k;
        load_taps<T, W>(a, c, n, k);
        float win[W - 1][E], acc[W][E];  // acc[i]: the gradient of token t - W + 1 + i
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
            const int64_t s = t0 - (W - 1) + i;
            widen(s >= 0 ? load_raw<E>(px + s * a.x_st, n) : state_row<T, W>(a, seq, (int)s + W - 1, c, n), win[i]);
        }
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[i][e] = 0.f;
        // Takes a token in (own: of this run, whose dw it adds to; in: of the sequence) and its dp to acc, of which
        // acc[0] is whole then.
        auto token = [&](const Raw<T, E>& rx, const Raw<T, E>& ry, bool own, bool in, float (&out)[E]) {
            float x[E], dp[E], p[E], old[W - 1][E];
            widen(rx, x);
            widen(ry, dp);
#pragma unroll
            for (int j = 0; j < W - 1; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) old[j][e] = win[j][e];
            taps<W>(k, win, x, p);
            if (a.silu) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float s = fast_sigmoid(p[e]);
                    dp[e] *= s * __builtin_fmaf(p[e], 1.f - s, 1.f);
                }
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (!in) dp[e] = 0.f;
                if (own) {
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) dw[j][e] = __builtin_fmaf(dp[e], old[j][e], dw[j][e]);
                    dw[W - 1][e] = __builtin_fmaf(dp[e], x[e], dw[W - 1][e]);
                    dw[W][e] += dp[e];
                }
                out[e] = __builtin_fmaf(k.w[0][e], dp[e], acc[0][e]);
#pragma unroll
                for (int j = 0; j < W - 1; ++j) acc[j][e] = __builtin_fmaf(k.w[j + 1][e], dp[e], acc[j + 1][e]);
                acc[W - 1][e] = 0.f;
            }
        };
        if (n == E && t0 > 0 && t1 - t0 == a.run && stop <= a.T) {
            // a whole run within the sequence, as in the forward: no access depends on a condition but the first
            // W - 1 stores, whose tokens are the run's before
            px += t0 * a.x_st;
            py += t0 * g.dy_st;
            pd += (t0 - (W - 1)) * a.Dm;
            Raw<T, E> rx[STEP], ry[STEP];
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
                rx[i] = load_raw<E>(px + i * a.x_st, E);
                ry[i] = load_raw<E>(py + i * g.dy_st, E);
            }
#pragma unroll 1
            for (int t = 0; t < a.run; t += STEP) {
                px += STEP * a.x_st;
                py += STEP * g.dy_st;
                Raw<T, E> nx[STEP], ny[STEP];
#pragma unroll
                for (int i = 0; i < STEP; ++i) {  // behind the run: its W - 1 tokens
                    const int j = t + STEP < a.run || i < W - 1 ? i : 0;
                    nx[i] = load_raw<E>(px + j * a.x_st, E);
                    ny[i] = load_raw<E>(py + j * g.dy_st, E);
                }
#pragma unroll
                for (int i = 0; i < STEP; ++i) {
                    float out[E];
                    token(rx[i], ry[i], true, true, out);
                    if (t + i >= W - 1) store_raw<E>(pd, E, out);
                    pd += a.Dm;
                    rx[i] = nx[i];
                    ry[i] = ny[i];
                }
            }
#pragma unroll
            for (int i = 0; i < W - 1; ++i) {
                if (i >= STEP) {
                    rx[i % STEP] = load_raw<E>(px + i * a.x_st, E);
                    ry[i % STEP] = load_raw<E>(py + i * g.dy_st, E);
                }
                float out[E];
                token(rx[i % STEP], ry[i % STEP], false, true, out);
                store_raw<E>(pd, E, out);
                pd += a.Dm;
            }
        } else {
            const int64_t from = t0 == 0 ? -(W - 1) : t0;  // before the first run's tokens the state's rows
            for (int64_t t = t0; t < stop; ++t) {
                const int m = t < a.T ? n : 0;
                float out[E];
                token(load_raw<E>(px + t * a.x_st, m), load_raw<E>(py + t * g.dy_st, m), t < t1, t < a.T, out);
                const int64_t s = t - (W - 1);
                if (s < from) continue;
                if (g.dfin && s >= a.T - (W - 1)) {
                    float f[E];
                    widen(load_raw<E>((const T*)g.dfin + (seq * (W - 1) + s - (a.T - (W - 1))) * a.Dm + c, n), f);
#pragma unroll
                    for (int e = 0; e < E; ++e) out[e] += f[e];
                }
                if (s >= 0) store_raw<E>(pd + s * a.Dm, n, out);
                else if (g.ds0) store_raw<E>((T*)g.ds0 + (seq * (W - 1) + s + W - 1) * a.Dm + c, n, out);
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
            if (ch < a.Dm) g.part[((int64_t)rb * (W + 1) + j) * a.Dm + ch] = s;
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

// Tokens of a run: its halo (W - 1 tokens, of two tensors in the gradients) and its part of dw are less in longer
// ones, but sixteen where 32 leave the chip under eight waves a compute unit.
int conv_run(int64_t n_seqs, int64_t T, int D, int cus) {
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
    const int64_t per = (a.T + a.run - 1) / a.run;
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
    const Grid g = run_grid(a.n_seqs * ((a.T + a.run - 1) / a.run), a.Dm);
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
