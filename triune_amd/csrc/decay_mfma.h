// decay_mfma.h -- matrix products of the decay attention kernels, one form for both kinds of operands:
//   __bf16  v_mfma_f32_16x16x32_bf16, derived operands (fp32 values) as sums of bf16 parts
//   float   v_mfma_f32_16x16x4_f32, four of them for 16 products a lane group (fp32 and fp16 tensors)
// Lane l = 16 g + n.  A fragment is 16 bytes of a lane: row (or column) n, E = 8 or 4 consecutive K indexes.
// The accumulator's rows 4 g + r of two neighbouring tiles (bf16) or one (fp32) are the K slots of the same lane,
// so an accumulator becomes an operand without moving between lanes: slot e of lane group g is then row
// 16 (e >> 2) + 4 g + (e & 3).
#pragma once

#include "decay.h"

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

// A row of an LDS tile with D values: one 16-byte unit of padding spreads rows over the banks.
template <typename TC>
constexpr int tile_stride(int D) {
    return D + 16 / (int)sizeof(TC);
}

// K step s of row `row`.
template <typename TC>
__device__ __forceinline__ typename Mat<TC>::Frag row_frag(const TC* tile, int RS, int row, int s, int g) {
    return *reinterpret_cast<const typename Mat<TC>::Frag*>(tile + row * RS + s * Mat<TC>::KS + Mat<TC>::E * g);
}

// Columns of a [32 tokens][D] tile as an operand whose K index is the token: fragment j of 32 / KS.  `PERM`: column m
// of the operand is tile_dim(t, m), else 16 t + m.
template <typename TC, bool PERM>
__device__ __forceinline__ typename Mat<TC>::Frag col_frag(const TC* tile, int RS, int t, int j, int g, int n) {
    if constexpr (Mat<TC>::E == 8) {
        const int col = PERM ? 32 * (t >> 1) + 8 * (n & 3) + 4 * (t & 1) : 16 * t + 4 * (n & 3);
        const __bf16* p = tile + (4 * g + (n >> 2)) * RS + col;
        const bf16x4 a = lds_read_tr(p), b = lds_read_tr(p + 16 * RS);
        return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    } else {
        const float* p = tile + (16 * j + 4 * g) * RS + 16 * t + n;
        return f32x4{p[0], p[RS], p[2 * RS], p[3 * RS]};
    }
}

}  // namespace triune
