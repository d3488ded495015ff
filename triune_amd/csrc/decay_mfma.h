// decay_mfma.h -- matrix products of the decay attention kernels, one form for both kinds of operands:
//   __bf16  v_mfma_f32_16x16x32_bf16, derived operands (fp32 values) as sums of bf16 parts
//   float   v_mfma_f32_16x16x4_f32, four of them for 16 products a lane group (fp32 and fp16 tensors)
// Lane l = 16 g + n.  A fragment is 16 bytes of a lane: row (or column) n, E = 8 or 4 consecutive K indexes.
// The accumulator's rows 4 g + r of two neighbouring tiles (bf16) or one (fp32) are the K slots of the same lane,
// so an accumulator becomes an operand without moving between lanes: slot e of lane group g is then row
// 16 (e >> 2) + 4 g + (e & 3).
//
// Roundings.  bf16 tensors are operands as they are.  What is derived from them (scores, states, weighted rows) is a
// sum of bf16 parts, each half a step (2^-8) off the rest: two parts, 2^-16, where it ends in a 16-bit output, three,
// 2^-24, where it goes into a state that is carried on, and for the states' terms of dq and dk, which the gates'
// gradients add up.  fp16 tensors take the fp32 form, since their range is not bf16's and their products with states
// are not fp16's.
#pragma once

#include "decay.h"

#include <type_traits>

namespace triune {

template <typename TC>
struct Mat;

template <>
struct Mat<__bf16> {
    using Frag = bf16x8;
    static constexpr int KS = 32, E = 8;
    __device__ __forceinline__ static f32x4 mma(const Frag& a, const Frag& b, const f32x4& c) { return mfma(a, b, c); }
};
template <>
struct Mat<float> {
    using Frag = f32x4;
    static constexpr int KS = 16, E = 4;
    __device__ __forceinline__ static f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

// E fp32 values as an operand of N parts (fp32: itself).
template <typename TC, int N>
struct Parts {
    typename Mat<TC>::Frag p[N];
};
template <typename TC, int N>
__device__ __forceinline__ auto parts(const float (&x)[Mat<TC>::E]) {
    if constexpr (Mat<TC>::E == 8) {
        Parts<TC, N> r;
        const Split8<N> s = split8<N>(x);
#pragma unroll
        for (int i = 0; i < N; ++i) r.p[i] = s.p[i];
        return r;
    } else {
        return Parts<TC, 1>{{f32x4{x[0], x[1], x[2], x[3]}}};
    }
}
template <typename TC, int N>
__device__ __forceinline__ f32x4 mma(const Parts<TC, N>& a, const typename Mat<TC>::Frag& b, f32x4 c) {
#pragma unroll
    for (int i = N - 1; i >= 0; --i) c = Mat<TC>::mma(a.p[i], b, c);  // small parts first
    return c;
}
template <typename TC, int N>
__device__ __forceinline__ f32x4 mma(const typename Mat<TC>::Frag& a, const Parts<TC, N>& b, f32x4 c) {
#pragma unroll
    for (int i = N - 1; i >= 0; --i) c = Mat<TC>::mma(a, b.p[i], c);
    return c;
}

// The E values that K step s of an accumulator column takes: rows of tiles 2 s and 2 s + 1, or of tile s.
template <typename TC, int M>
__device__ __forceinline__ void acc_slots(const f32x4 (&t)[M], int s, float (&x)[Mat<TC>::E]) {
#pragma unroll
    for (int e = 0; e < Mat<TC>::E; ++e) x[e] = Mat<TC>::E == 8 ? t[2 * s + (e >> 2)][e & 3] : t[s][e];
}

// Where element `m` (0..15) of 16-wide tile t lies in its dim, for a dim that is a K index of row fragments
// elsewhere: row fragments take E consecutive elements, accumulators as above, and these agree.
template <typename TC>
__device__ __forceinline__ int tile_dim(int t, int m) {
    if constexpr (Mat<TC>::E == 8) return 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3);
    else return 16 * t + m;
}

// A row of an LDS tile with D values, padded so that rows fall on other banks.  bf16: by 32 bytes, so that the eight rows by
// two units of a cycle of ds_read_b128 and the eight rows by four of a transposed read both fill the banks; fp32, whose
// columns are read value by value: by 16 bytes, so that the four rows of a read do.
template <typename TC>
constexpr int tile_stride(int D) {
    return D + (sizeof(TC) == 2 ? 16 : 4);
}

// K step s of row `row`.
template <typename TC>
__device__ __forceinline__ typename Mat<TC>::Frag row_frag(const TC* tile, int RS, int row, int s, int g) {
    return *reinterpret_cast<const typename Mat<TC>::Frag*>(tile + row * RS + s * Mat<TC>::KS + Mat<TC>::E * g);
}

// Columns of a [tokens][D] tile as an operand whose K index is the token: K step j.  `PERM`: column m
// of the operand is tile_dim(t, m), else 16 t + m.
template <typename TC, bool PERM>
__device__ __forceinline__ typename Mat<TC>::Frag col_frag(const TC* tile, int RS, int t, int j, int g, int n) {
    if constexpr (Mat<TC>::E == 8) {
        const int col = PERM ? 32 * (t >> 1) + 8 * (n & 3) + 4 * (t & 1) : 16 * t + 4 * (n & 3);
        const __bf16* p = tile + (32 * j + 4 * g + (n >> 2)) * RS + col;
        const bf16x4 a = lds_read_tr(p), b = lds_read_tr(p + 16 * RS);
        return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    } else {
        const float* p = tile + (16 * j + 4 * g) * RS + 16 * t + n;
        return f32x4{p[0], p[RS], p[2 * RS], p[3 * RS]};
    }
}

// K step j of row `row`, its K indexes in the order of col_frag's.
template <typename TC>
__device__ __forceinline__ typename Mat<TC>::Frag row_frag_tok(const TC* tile, int RS, int row, int j, int g) {
    if constexpr (Mat<TC>::E == 8) {
        const __bf16* p = tile + row * RS + 32 * j + 4 * g;
        const bf16x4 a = *reinterpret_cast<const bf16x4*>(p), b = *reinterpret_cast<const bf16x4*>(p + 16);
        return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    } else {
        return row_frag(tile, RS, row, j, g);
    }
}

__device__ __forceinline__ float lane_value(float x, int lane) {  // lane: a constant
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// ROWS rows of a [tokens][D] tensor into an LDS tile, zeros past `rows` and `cols`, through registers, so that a chunk's
// loads are in flight while the one before it is worked on.  FULL: whole units of 16-byte aligned rows (decay_full), through
// a buffer resource that moves with the chunks, so that a load takes no address arithmetic; the resource has no end of its
// own (rows are far apart), so every unit outside of `rows` and `cols` goes past it (TileUnits).
template <typename TIO, typename TC, int ROWS, int D, int NTH, bool FULL>
struct Tile {
    static constexpr int E = Mat<TC>::E;
    using Units = TileUnits<ROWS, D, E, NTH>;
    static constexpr int N = Units::N, PER = Units::PER;
    Raw<TIO, E> x[PER];
    int off[PER];  // bytes from the chunk's first row
    __device__ __forceinline__ static int row_of(int i) { return Units::row(threadIdx.x, i); }
    __device__ __forceinline__ static int col_of(int i) { return Units::col(threadIdx.x, i); }
    __device__ __forceinline__ explicit Tile(int64_t st) {
#pragma unroll
        for (int i = 0; i < PER; ++i) off[i] = Units::offset(threadIdx.x, i, st, sizeof(TIO));
    }
    // rows, cols: what the tensor has from p on
    __device__ __forceinline__ void fetch(const TIO* p, int64_t st, int rows, int cols) {
        if constexpr (FULL) {
            const __amdgpu_buffer_rsrc_t r =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<TIO*>(p), (short)0, TILE_SKIP, 0x00020000);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                x[i] = __builtin_bit_cast(Raw<TIO, E>,
                                          tile_load<TIO, E>(r, Units::load_from(off[i], threadIdx.x, i, rows, cols)));
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const bool in = Units::in(threadIdx.x, i, rows, cols);
                x[i] = load_raw<E>(p + (in ? row_of(i) * st + col_of(i) : 0), in ? cols - col_of(i) : 0);
            }
        }
    }
    __device__ __forceinline__ void put(TC* tile) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (N % NTH && row_of(i) >= ROWS) continue;
            TC* to = tile + row_of(i) * tile_stride<TC>(D) + col_of(i);
            if constexpr (std::is_same<TIO, TC>::value) {
                *reinterpret_cast<typename Mat<TC>::Frag*>(to) = __builtin_bit_cast(typename Mat<TC>::Frag, x[i]);
            } else {
                typename Mat<TC>::Frag f;
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] = (TC)x[i].v[e];
                *reinterpret_cast<typename Mat<TC>::Frag*>(to) = f;
            }
        }
    }
};

// Orders LDS accesses around a barrier and leaves loads from memory in flight, which __syncthreads would wait for.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A gate's bits; what the other of two loads reads is not used.  Both are issued, since a load behind a condition would
// be waited for there.
static __device__ const uint32_t kNoGate[1] = {0};
struct GateBits {
    uint32_t wide;
    uint16_t half;
    __device__ __forceinline__ void fetch(const DecayTok& g, int dt, int64_t at) {
        const bool f32 = dt == DT_F32;
        wide = *(f32 ? (const uint32_t*)g.p + at : kNoGate);
        half = *(f32 ? (const uint16_t*)kNoGate : (const uint16_t*)g.p + at);
    }
    __device__ __forceinline__ float value(int dt) const {
        return dt == DT_F32    ? __uint_as_float(wide)
               : dt == DT_BF16 ? __uint_as_float((uint32_t)half << 16)
                               : (float)__builtin_bit_cast(_Float16, half);
    }
};

// The running sums of a chunk's gates: lane l holds token l's (of 32: l & 31's).  Tokens past the end count as 0.
template <int CH>
__device__ __forceinline__ Sum2 running_sums(float gate, int rows, int lane) {
    Sum2 s = split_gate((lane & (CH - 1)) < rows ? log2_gate(gate) : 0.f);
    s.hi = row_inclusive_scan(s.hi);
    s.lo = row_inclusive_scan(s.lo);
    const float h0 = lane_value(s.hi, 15), l0 = lane_value(s.lo, 15);
    const float h2 = lane_value(s.hi, 47), l2 = lane_value(s.lo, 47);
    if (lane & 16) s.hi += lane & 32 ? h2 : h0, s.lo += lane & 32 ? l2 : l0;
    if constexpr (CH == 64) {
        const float h1 = lane_value(s.hi, 31), l1 = lane_value(s.lo, 31);
        if (lane & 32) s.hi += h1, s.lo += l1;
    }
    return s;
}

// What a chunk of 32 tokens takes of its gates, formed once for all waves: the sums G (hi, lo), 2^G, 2^{G_end - G}, and for
// the scores of the second 16 tokens with the first 16 the factors 2^{G - G_15} (read) and 2^{G_15 - G} (written).
struct ChunkGates {
    float hi[32], lo[32], from[32], to[32], half[32];
    __device__ __forceinline__ void put(float gate, int rows, int lane) {
        const Sum2 s = running_sums<32>(gate, rows, lane);
        const Sum2 end{lane_value(s.hi, 31), lane_value(s.lo, 31)}, mid{lane_value(s.hi, 15), lane_value(s.lo, 15)};
        if (lane >= 32) return;
        hi[lane] = s.hi;
        lo[lane] = s.lo;
        from[lane] = __builtin_amdgcn_exp2f(s.hi + s.lo);
        to[lane] = decay_between(end, s);
        half[lane] = lane < 16 ? decay_between(mid, s) : decay_between(s, mid);
    }
};
__device__ __forceinline__ f32x4 four(const float* p) { return *reinterpret_cast<const f32x4*>(p); }

template <int CH>
__device__ __forceinline__ Sum2 chunk_sums(const DecayTok& g, int dt, int64_t at, int rows, int lane) {
    const int t = lane & (CH - 1);
    return running_sums<CH>(t < rows ? load_dt(g.p, dt, at + t * g.st) : 0.f, rows, lane);
}

// Work items of a walk: (segment, head, slice), slices fastest.
struct DecayWhere {
    SsmSeg seg;
    int64_t w, last;  // the work item, that of the sequence's last segment
    int h, slice;
};
__device__ __forceinline__ bool decay_where(const DecayParams& a, DecayWhere& x) {
    uint32_t b = blockIdx.x;
    x.slice = (int)(b % (uint32_t)a.slices);
    b /= (uint32_t)a.slices;
    x.h = (int)(b % (uint32_t)a.H);
    x.w = b / (uint32_t)a.H;
    if (a.cu) {
        if (!ssm_segment(a, x.w, x.seg)) return false;
        x.last = a.seg_off ? a.seg_off[x.seg.seq + 1] - 1 : x.w;
        return true;
    }
    const uint32_t seq = (uint32_t)x.w / (uint32_t)a.nseg, p = (uint32_t)x.w - seq * (uint32_t)a.nseg;
    const int64_t t0 = (int64_t)p * a.seg;
    x.seg = SsmSeg{seq, 0, t0, (int)min((int64_t)a.seg, a.T - t0), (int)p, p == (uint32_t)a.nseg - 1};
    x.last = x.w - p + a.nseg - 1;
    return true;
}
// The first element of a work item's tokens.
__device__ __forceinline__ int64_t decay_base(const DecayParams& a, const DecayWhere& x, const DecayTok& t, int head) {
    return (a.cu ? 0 : x.seg.seq * t.sb) + (x.seg.row0 + x.seg.t0) * t.st + head * t.sh;
}

// A wave's slice of a state lies in accumulators, NT tiles of 16 columns by DT of 16 rows: row tile_dim(t, 4 g + r) and
// column 16 (w NT + c) + n of the slice.  f(value, its place in a matrix with this row stride, whether that is in
// [Dk, Dv]).
template <typename TC, int NT, int DT, typename F>
__device__ __forceinline__ void each_state(f32x4 (&S)[NT][DT], int col0, int Dk, int Dv, int64_t row_stride, F f) {
    const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, n = lane & 15;
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        const int dv = col0 + 16 * (w * NT + c) + n;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int dk = tile_dim<TC>(t, 4 * g + r);
                float x = S[c][t][r];
                f(x, dk * row_stride + dv, dk < Dk && dv < Dv);
                S[c][t][r] = x;
            }
    }
}
// The same in the workspace, in the order of the lanes.
template <int NT, int DT>
__device__ __forceinline__ void put_state(const f32x4 (&S)[NT][DT], float* to) {
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(to + (c * DT + t) * 256) = S[c][t];
}
template <int NT, int DT>
__device__ __forceinline__ void get_state(f32x4 (&S)[NT][DT], const float* from) {
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int t = 0; t < DT; ++t) S[c][t] = *reinterpret_cast<const f32x4*>(from + (c * DT + t) * 256);
}

// F<TIO, TC>::run<DK, NW, NT, FULL>(p, grid, stream) for the types and sizes of a: NW waves that own NT tiles of 16 columns
// each, a workgroup for each (segment, head, slice).
template <template <typename, typename> class F, typename TIO, typename TC, int DK, bool FULL, typename P>
void decay_by_width(const P& p, const DecayParams& a, dim3 grid, hipStream_t s) {
    switch (decay_slice(a.Dv)) {
        case 32: return F<TIO, TC>::template run<DK, 2, 1, FULL>(p, grid, s);
        case 64: return F<TIO, TC>::template run<DK, 4, 1, FULL>(p, grid, s);
        default: return F<TIO, TC>::template run<DK, 4, 2, FULL>(p, grid, s);
    }
}
template <template <typename, typename> class F, typename TIO, typename TC, bool FULL, typename P>
void decay_by_dk(const P& p, const DecayParams& a, dim3 grid, hipStream_t s) {
    switch (decay_padded_dk(a.Dk)) {
        case 32: return decay_by_width<F, TIO, TC, 32, FULL>(p, a, grid, s);
        case 64: return decay_by_width<F, TIO, TC, 64, FULL>(p, a, grid, s);
        default: return decay_by_width<F, TIO, TC, 128, FULL>(p, a, grid, s);
    }
}
template <template <typename, typename> class F, typename P>
hipError_t decay_by_type(const P& p, const DecayParams& a, int dt, bool full, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_work * a.H * a.slices));
    if (dt == DT_F32)
        full ? decay_by_dk<F, float, float, true>(p, a, grid, s) : decay_by_dk<F, float, float, false>(p, a, grid, s);
    else if (dt == DT_BF16)
        full ? decay_by_dk<F, __bf16, __bf16, true>(p, a, grid, s) : decay_by_dk<F, __bf16, __bf16, false>(p, a, grid, s);
    else
        full ? decay_by_dk<F, _Float16, float, true>(p, a, grid, s) : decay_by_dk<F, _Float16, float, false>(p, a, grid, s);
    return hipGetLastError();
}

}  // namespace triune
