// ssm.h -- parameter blocks and launchers of the state space layer's kernels: the selective scan
// (ssm.hip, ssm_bwd.hip), the short causal convolution (short_conv.hip) and layer norm
// (layer_norm.hip).  Internal to libtriune_hip.
#pragma once

#include "common.h"

#include <initializer_list>

namespace triune {

constexpr int SSM_UNIT = 32;   // segments are multiples of this many tokens
// Tokens between two states that the forward keeps for the backward, which holds its walks between them
// in LDS.
inline int ssm_kept_every(int N) { return N <= 32 ? 32 : 16; }
constexpr int SSM_MAX_N = 64;  // states per channel

// A [tokens, channels] operand of a batch of sequences: element strides, innermost stride 1.
struct SsmTok {
    const void* p;
    int64_t sb, st;
};

struct SsmParams {
    SsmTok u, dl, z, y;       // z.p null: no gate
    const void *B, *C;        // [.., G, N] rows
    int64_t b_sb, b_st, b_sg, c_sb, c_st, c_sg;
    const float *A, *D, *bias;  // [Dm, N], [Dm] or null, [Dm] or null
    int softplus;
    const float* s0;          // [rows, Dm, N] or null
    float* fin;               // [rows, Dm, N] or null
    const int32_t* slots;     // packed over a pool: the row of each sequence, else null
    int64_t n_slots;
    float* ckpt;              // [Bn, ceil(T / ssm_kept_every), N, Dm] or null
    float* ws_state;          // [n_work, N, Dm]: a segment's own end state, then the state it starts from
    float* ws_sum;            // [n_work, Dm]: summed step sizes
    int64_t n_seqs, T;        // T: length of a dense sequence, or all tokens of a packed call
    int Dm, G, N;
    int blocks;               // channel blocks of a group
    int seg, nseg;            // tokens of a segment, segments of a dense sequence
    int64_t n_work;
    const int32_t *cu, *seg_off;  // packed: [n_seqs + 1] token and segment offsets
};

struct SsmBwdParams {
    SsmParams f;              // ws_state / ws_sum: the gradient's segment ends (nseg > 1)
    SsmTok dy;
    const float* dfin;        // [Bn, Dm, N] or null
    void *du, *ddl, *dz;      // [Bn, T, Dm] contiguous, I/O dtype (dz null with z.p)
    float* part_bc;           // [G * blocks, Bn * T, waves, 8]
    float* part_par;          // [n_work, N + 2, Dm]: A's rows, D, bias
    void *dB, *dC;            // [Bn, T, G, N] contiguous, I/O dtype
    float *dA, *dD, *dbias;   // [Dm, N], [Dm], [Dm]; null where not wanted
    float* ds0;               // [Bn, Dm, N] or null
};

struct SsmStepParams {
    SsmTok u, dl, z, y;       // [Bn, Dm] rows: sb is the row stride
    const void *B, *C;
    int64_t b_sb, b_sg, c_sb, c_sg;
    const float *A, *D, *bias;
    int softplus;
    const float* s_in;
    float* s_out;
    const int32_t* slots;
    int64_t n_rows;           // rows of the state
    int64_t Bn;
    int Dm, G, N, cus;        // cus: compute units
};

int ssm_waves(int N);  // waves of a scan workgroup
// The join's launch.  by_followed: its blocks are laid out by the segments that another one follows.
struct CarryGrid {
    int64_t blocks;
    int waves;
    bool by_followed;
};
CarryGrid ssm_carry_grid(bool packed, int64_t n_seqs, int64_t n_work, int64_t nseg, int64_t Dm, int N);
// Whether four channels of every row of these (and the groups) are aligned to their size together.
inline bool ssm_by_four(int group_channels, int io_dt, std::initializer_list<SsmTok> ts) {
    const uintptr_t m = io_dt == DT_F32 ? 15 : 7;
    for (const SsmTok& t : ts)
        if (t.p && ((reinterpret_cast<uintptr_t>(t.p) & m) || ((t.sb | t.st) & 3))) return false;
    return group_channels % 4 == 0;
}
// n elements of `bytes` (2 or 4) from one state tensor to another, zeros without a source: calls without tokens.
hipError_t launch_state_copy(const void* from, void* to, int64_t n, int bytes, hipStream_t s);
// Sequences of more than `cut` tokens are cut into segments.
hipError_t launch_ssm_offsets(const SsmParams& a, int64_t cut, int32_t* seg_off, hipStream_t s);
hipError_t launch_ssm_states(const SsmParams& a, int io_dt, hipStream_t s);
hipError_t launch_ssm_carry(const SsmParams& a, hipStream_t s);
hipError_t launch_ssm_scan(const SsmParams& a, int io_dt, hipStream_t s);
hipError_t launch_ssm_step(const SsmStepParams& a, int io_dt, hipStream_t s);
hipError_t launch_ssm_bwd_states(const SsmBwdParams& a, int io_dt, hipStream_t s);
hipError_t launch_ssm_bwd_carry(const SsmBwdParams& a, hipStream_t s);
hipError_t launch_ssm_bwd(const SsmBwdParams& a, int io_dt, hipStream_t s);
hipError_t launch_ssm_bwd_sum(const SsmBwdParams& a, int io_dt, hipStream_t s);

// ---- short causal convolution --------------------------------------------------------------
struct ConvParams {
    const void* x;            // [Bn, T, Dm] or packed rows, element strides
    int64_t x_sb, x_st;
    const void *w, *bias;     // [Dm, W] and [Dm] (or null) of w_dt
    int w_dt, silu;
    const void* s0;           // [rows, W - 1, Dm] of the I/O dtype, or null (zeros)
    void* fin;                // the same after the call, or null
    const int32_t* slots;     // the state row of each sequence, else null
    int64_t n_slots;          // state rows
    void* y;
    int64_t y_sb, y_st;
    int64_t n_seqs, T;        // T: length of a dense sequence, or all rows of a packed call
    int Dm, W;
    int run;                  // tokens of a thread's run
    const int32_t* cu;        // packed: [n_seqs + 1]
};

struct ConvBwdParams {
    ConvParams f;
    const void* dy;           // [Bn, T, Dm]
    int64_t dy_sb, dy_st;
    const void* dfin;         // [Bn, W - 1, Dm] contiguous or null
    void* dx;                 // [Bn, T, Dm] contiguous
    void* ds0;                // [Bn, W - 1, Dm] contiguous or null
    float* part;              // [parts, W + 1, Dm]
    int64_t parts;
    void *dw, *dbias;         // of w_dt, or null
};

int conv_run(int64_t n_seqs, int64_t T, int Dm, int cus);
int64_t conv_bwd_parts(int64_t n_seqs, int64_t T, int Dm, int run);
hipError_t launch_conv(const ConvParams& a, int io_dt, hipStream_t s);
hipError_t launch_conv_state(const ConvParams& a, int io_dt, hipStream_t s);
hipError_t launch_conv_step(const ConvParams& a, int io_dt, hipStream_t s);
hipError_t launch_conv_bwd(const ConvBwdParams& a, int io_dt, hipStream_t s);

// ---- layer norm ----------------------------------------------------------------------------
constexpr int NORM_MAX_D = 16384;

struct NormParams {
    const void* x;            // [R, D], row stride x_st
    int64_t x_st;
    const void *w, *b;        // [D] of w_dt / b_dt, or null
    int w_dt, b_dt;
    float eps;
    void* y;                  // [R, D] contiguous
    float *mean, *rstd;       // [R] or null
    int64_t R;
    int D, cus;               // cus: compute units
};

struct NormBwdParams {
    NormParams f;             // x, w, mean, rstd, R, D
    const void* dy;
    int64_t dy_st;
    void* dx;                 // [R, D] contiguous
    float* part;              // [parts, 2, D], or null without parameter gradients
    int64_t parts;
    void *dw, *db;            // of w_dt / b_dt, or null
};

int64_t norm_bwd_parts(int64_t R, int D, int cus);
hipError_t launch_norm(const NormParams& a, int io_dt, hipStream_t s);
hipError_t launch_norm_bwd(const NormBwdParams& a, int io_dt, hipStream_t s);

// ---- device helpers ---------------------------------------------------------------------------
// 1 / (1 + e^-x) with the hardware reciprocal (1 ulp); e^-x past the largest number gives 0.
__device__ __forceinline__ float fast_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + fast_exp(-x)); }
__device__ __forceinline__ float silu_gate(float z) { return z * fast_sigmoid(z); }

// log(1 + e^-|x|) + max(x, 0).  With s = e / (2 + e), log(1 + e) = 2 atanh(s), whose series in s^2
// <= 1/9 is cut to a fitted polynomial (relative error 8e-9): the form keeps the relative precision
// where e is small (step sizes of 1e-3 have e = 1e-3, of which log(1 + e) would lose ten bits).
__device__ __forceinline__ float softplus(float x) {
    const float e = fast_exp(-fabsf(x));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e), t = s * s;
    float p = 0.28174665570259094f;
    p = __builtin_fmaf(p, t, 0.27961426973342896f);
    p = __builtin_fmaf(p, t, 0.40024852752685547f);
    p = __builtin_fmaf(p, t, 0.6666631698608398f);
    p = __builtin_fmaf(p, t, 2.0f);
    return __builtin_fmaf(s, p, __builtin_amdgcn_fmed3f(x, 0.f, __builtin_inff()));  // max(x, 0); s carries a NaN
}

// N elements of any alignment in one access (the memory pipeline takes unaligned vectors), or the
// n < N that a row's last group holds.
template <typename T, int N>
struct __attribute__((packed, aligned(alignof(T)))) Raw {
    T v[N];
};
template <int N, typename T>
__device__ __forceinline__ Raw<T, N> load_raw(const T* p, int n) {
    Raw<T, N> r;
    if (n >= N) {
        r = *reinterpret_cast<const Raw<T, N>*>(p);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) r.v[j] = j < n ? p[j] : (T)0.f;
    }
    return r;
}
template <int N, typename T>
__device__ __forceinline__ void store_raw(T* p, int n, const Raw<T, N>& r) {
    if (n >= N) {
        *reinterpret_cast<Raw<T, N>*>(p) = r;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < n) p[j] = r.v[j];
    }
}
template <int N, typename T>
__device__ __forceinline__ void store_raw(T* p, int n, const float (&x)[N]) {
    Raw<T, N> r;
#pragma unroll
    for (int j = 0; j < N; ++j) r.v[j] = (T)x[j];
    store_raw<N>(p, n, r);
}

// The sum of n values `st` apart, every sixteenth from the first, four of them in flight.
__device__ __forceinline__ float sum_parts(const float* p, int64_t st, int64_t first, int64_t n) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    int64_t k = first;
    for (; k + 48 < n; k += 64) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += p[(k + 16 * i) * st];
    }
    for (int i = 0; k < n; k += 16, ++i) s[i] += p[k * st];
    return (s[0] + s[1]) + (s[2] + s[3]);
}

__device__ __forceinline__ void store_dt(void* p, int dt, int64_t i, float x) {
    if (dt == DT_F32) ((float*)p)[i] = x;
    else if (dt == DT_BF16) ((__bf16*)p)[i] = (__bf16)x;
    else ((_Float16*)p)[i] = (_Float16)x;
}

// A in units of the hardware's exp2.  Infinite values are cut to the largest number, so that a step of 0
// (a token past a tile's end) is a decay of 1 for them too.
__device__ __forceinline__ float log2_decay(float A) {
    const float x = A * LOG2E, most = 3.4028234e38f;
    return x < -most ? -most : x > most ? most : x;
}

// A as a factor of p = dh a h_{t-1} in the gradient.  Past 1e30 every step above 1e-28 has a decay, and a p, of
// 0, whose product with an infinite A has to be 0; at a step of 0 the product stays finite, and softplus' slope of 0
// takes it.
__device__ __forceinline__ float slope_decay(float A) { return A < -1e30f ? -1e30f : A > 1e30f ? 1e30f : A; }

// 2^x as m 2^e with m in (1/2, 1], for a decay product over a segment: modes that grow (A > 0, or steps below
// 0) take it past the largest number where the state that it scales, 0 or small, stays within.  scale(v) = v 2^x
// then leaves the range only if the product does.  Past 300 no float's product is within; NaN stays.
struct Pow2 {
    float m;
    int e;
    __device__ __forceinline__ Pow2(float m, int e) : m(m), e(e) {}
    __device__ __forceinline__ explicit Pow2(float x) {
        x = x < -300.f ? -300.f : x > 300.f ? 300.f : x;
        const float c = __builtin_ceilf(x);
        m = __builtin_amdgcn_exp2f(x - c);
        e = (int)__builtin_amdgcn_fmed3f(c, -300.f, 300.f);
    }
    __device__ __forceinline__ float scale(float v) const { return __builtin_ldexpf(m * v, e); }
};

// N consecutive states of a channel whose row holds `left` more (zeros past them).
template <int N>
__device__ __forceinline__ void load_states(const float* p, int left, float (&x)[N]) {
    if (left >= N && !(reinterpret_cast<uintptr_t>(p) & 15)) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(p + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j + i] = v[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = j < left ? p[j] : 0.f;
    }
}
template <int N>
__device__ __forceinline__ void store_states(float* p, int left, const float (&x)[N]) {
    if (left >= N && !(reinterpret_cast<uintptr_t>(p) & 15)) {
#pragma unroll
        for (int j = 0; j < N; j += 4) *reinterpret_cast<f32x4*>(p + j) = f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]};
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < left) p[j] = x[j];
    }
}

// Rows of a tile through a buffer resource: it starts at the tile's first row and ends with the last
// valid one, so rows past the end (all of them, past the last tile or without a tensor) read 0 and are
// not written.  Accesses step through the vector offset, which the range check covers; a
// branch around them, or one for whole tiles, would make the compiler join registers behind it, which
// waits for the loads it should leave in flight.
constexpr int TILE_SKIP = 0x40000000;  // an offset past every resource: reads 0, writes nothing
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rows(const T* p, int64_t st, int64_t rows, uint32_t width) {
    const int64_t n = p && rows > 0 ? ((rows - 1) * st + width) * (int64_t)sizeof(T) : 0;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), (short)0, (int)min(n, (int64_t)TILE_SKIP), 0x00020000);
}

// V elements (1, or 4 aligned to their size together) in one access.
template <typename T, int V>
struct Vec {
    T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> tile_load(__amdgpu_buffer_rsrc_t r, int voff) {
    constexpr int B = sizeof(T) * V;
    static_assert(B == 2 || B == 4 || B == 8 || B == 16, "no such access");
    if constexpr (B == 2) return __builtin_bit_cast(Vec<T, V>, __builtin_amdgcn_raw_buffer_load_b16(r, voff, 0, 0));
    else if constexpr (B == 4) return __builtin_bit_cast(Vec<T, V>, __builtin_amdgcn_raw_buffer_load_b32(r, voff, 0, 0));
    else if constexpr (B == 8) return __builtin_bit_cast(Vec<T, V>, __builtin_amdgcn_raw_buffer_load_b64(r, voff, 0, 0));
    else return __builtin_bit_cast(Vec<T, V>, __builtin_amdgcn_raw_buffer_load_b128(r, voff, 0, 0));
}
template <typename T, int V>
__device__ __forceinline__ void tile_store(const float (&y)[V], __amdgpu_buffer_rsrc_t r, int voff) {
    constexpr int B = sizeof(T) * V;
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    Vec<T, V> x;
#pragma unroll
    for (int j = 0; j < V; ++j) x.v[j] = (T)y[j];
    if constexpr (B == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, x), r, voff, 0, 0);
    else if constexpr (B == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), r, voff, 0, 0);
    else if constexpr (B == 8) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, x), r, voff, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), r, voff, 0, 0);
}
// N accesses `st` bytes apart.  The offset is hidden from the optimizer, which would keep the N sums of it
// in registers over the loop on tiles.
template <typename T, int V, int N>
__device__ __forceinline__ void tile_load_rows(__amdgpu_buffer_rsrc_t r, int voff, int st, Vec<T, V> (&x)[N]) {
    if constexpr (N > 2) asm volatile("" : "+v"(voff));
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = tile_load<T, V>(r, voff + i * st);
}
template <typename T, int V, int N>
__device__ __forceinline__ void tile_store_rows(__amdgpu_buffer_rsrc_t r, int voff, int st, const float (&y)[N][V]) {
    if constexpr (N > 2) asm volatile("" : "+v"(voff));
#pragma unroll
    for (int i = 0; i < N; ++i) tile_store<T, V>(y[i], r, voff + i * st);
}
// V floats of an LDS row.
template <int V>
__device__ __forceinline__ void lds_store(float* p, const float (&x)[V]) {
    if constexpr (V == 4) *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    else p[0] = x[0];
}
template <int V>
__device__ __forceinline__ void lds_add(const float* p, float (&x)[V]) {
    if constexpr (V == 4) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += v[j];
    } else {
        x[0] += p[0];
    }
}

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

// The tokens of work item w (of packed sequence seq, searched for where that is negative): sequence, first
// token (of the sequence), length, whether it is the sequence's last segment.  False when there is no such item
// (packed calls bound their number).
struct SsmSeg {
    int64_t seq, row0, t0;  // row0: first token of the sequence in a packed tensor
    int len, index;
    bool last;
};
// The packed sequence of the j-th segment that another one follows, of all sequences: seg_off[i] - i of them are in
// front of sequence i.  -1 when there are not so many.
__device__ __forceinline__ int64_t ssm_followed(const SsmParams& a, int64_t j) {
    if (j >= a.seg_off[a.n_seqs] - a.n_seqs) return -1;
    int64_t lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
        const int64_t m = (lo + hi) >> 1;
        if (a.seg_off[m] - m <= j) lo = m; else hi = m;
    }
    return lo;
}
__device__ __forceinline__ bool ssm_segment(const SsmParams& a, int64_t w, SsmSeg& s, int64_t seq = -1) {
    if (!a.cu) {
        s.seq = w / a.nseg;
        s.index = (int)(w - s.seq * a.nseg);
        s.row0 = 0;
        s.t0 = (int64_t)s.index * a.seg;
        s.len = (int)min((int64_t)a.seg, a.T - s.t0);
        s.last = s.index == a.nseg - 1;
        return true;
    }
    int64_t lo = w, first = w;  // without segment offsets every sequence is one segment
    s.last = true;
    if (a.seg_off) {
        if (w >= a.seg_off[a.n_seqs]) return false;
        lo = seq < 0 ? 0 : seq;
        int64_t hi = seq < 0 ? a.n_seqs : seq + 1;  // seg_off[lo] <= w < seg_off[hi]
        while (hi - lo > 1) {
            const int64_t m = (lo + hi) >> 1;
            if (a.seg_off[m] <= w) lo = m; else hi = m;
        }
        first = a.seg_off[lo];
        s.last = w + 1 == a.seg_off[lo + 1];
    }
    // offsets outside the packed rows are cut to them
    const int64_t beg = min(max((int64_t)a.cu[lo], (int64_t)0), a.T);
    const int64_t n = min(max((int64_t)a.cu[lo + 1], beg), a.T) - beg;
    s.seq = lo;
    s.index = (int)(w - first);
    s.row0 = beg;
    s.t0 = (int64_t)s.index * a.seg;
    s.len = (int)(s.last ? max(n - s.t0, (int64_t)0) : a.seg);
    return true;
}

// Row of the state tensors for a sequence, or -1 for a slot outside the pool.
__device__ __forceinline__ int64_t ssm_row(const int32_t* slots, int64_t n_slots, int64_t seq) {
    if (!slots) return seq;
    const int64_t r = slots[seq];
    return r >= 0 && r < n_slots ? r : -1;
}

}  // namespace triune
