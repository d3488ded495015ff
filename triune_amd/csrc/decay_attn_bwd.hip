// decay_attn_bwd.hip -- gradients of decay attention (decay_attn.hip) on gfx950.
//
// Per chunk, with S_0 the state in front of it, R the gradient of the state behind it, and for j <= i
//     A_ij = scale e^{G_i - G_j} (q_i . k_j),   B_ij = scale e^{G_i - G_j} (do_i . v_j):
//     dq_i = sum_j B_ij k_j + scale e^{G_i} S_0 do_i
//     dk_j = sum_i B_ij q_i + e^{G_C - G_j} R v_j
//     dv_j = sum_i A_ij do_i + e^{G_C - G_j} R^T k_j
//     dg_t = what passes from writes before t to reads at t or behind it:
//            sum_{i >= t} q_i . dq'_i + sum_{j < t} k_j . dk'_j + e^{G_C} <S_0, R> + sum_{j < t <= i} (q_i . k_j) B_ij
// with dq', dk' the terms with S_0 and R.  Only pairs that span t are added, so steep gates, whose own pairs are large
// and spanning ones small, lose nothing to cancellation.
//
// The states in front of the chunks and the gradients behind them come from two walks (decay_walk.hip), so a
// workgroup takes one (chunk, head) by itself.  A and B are formed once, in tiles over the waves, and shared through
// LDS, B in the place of A; a wave owns a 16-wide tile of key dims (dq, dk) and one of value dims (dv), which are taken in
// slices of 32.  Its rows of S and R come from memory once, the products with k take R by columns from LDS (in q's place,
// which is read again behind them), and two workgroups fit a compute unit.
//
// 4 x 2048 tokens, 12 heads of 128, bf16: 117 us for 206 MB of states, 101 of tensors in and 75 out (3.3 TB/s); 30 % of
// the SIMDs' cycles issue vector work and 14 % matrix work, 45 % of the waves' wait: a chain of products with little
// beside it at two workgroups a compute unit, which registers (256, four spilled) and LDS (74 KB) allow.  Chunks of 64
// tokens instead of 32 halve the states' bytes; fp32 tensors, whose tiles take twice the LDS, stay at 32.
#include "decay_mfma.h"

namespace triune {

namespace {

// Causal tile idx: token rows I (read) and J <= I (written).
__device__ __forceinline__ void tile_of(int idx, int& I, int& J) {
    I = idx >= 6 ? 3 : idx >= 3 ? 2 : idx >= 1 ? 1 : 0;
    J = idx - I * (I + 1) / 2;
}
__device__ __forceinline__ int tile_index(int I, int J) { return I * (I + 1) / 2 + J; }

// Four values as NP planes of parts.
template <typename TC, int NP>
__device__ __forceinline__ void put4(TC* plane, int plane_size, int off, const f32x4& x) {
    if constexpr (Mat<TC>::E == 8) {
        float r[4] = {x[0], x[1], x[2], x[3]};
        uint32_t w[NP][2];
        split_pairs<NP, 2>(r, w);
#pragma unroll
        for (int p = 0; p < NP; ++p) *reinterpret_cast<uint2*>(plane + p * plane_size + off) = uint2{w[p][0], w[p][1]};
    } else {
        *reinterpret_cast<f32x4*>(plane + off) = x;
    }
}

// Sums over the lanes at and behind this one of its row of 16.
__device__ __forceinline__ float row_suffix_scan(float x) {
    x += row_shl<1>(x);
    x += row_shl<2>(x);
    x += row_shl<4>(x);
    x += row_shl<8>(x);
    return x;
}

}  // namespace

// A state through a buffer resource, whose scalar offset steps through the values (64-bit addresses for each would take
// two registers apiece and spill).
struct StateAt {
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ StateAt(const void* p, int64_t values)
        : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)(values * 4), 0x00020000)) {}
    // 16 bytes at byte offsets of the lane and of all lanes
    __device__ __forceinline__ f32x4 at(int lane, int all) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, lane, all, 0));
    }
    template <int E>
    __device__ __forceinline__ void row(int lane, int all, float (&x)[E]) const {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const f32x4 v = at(lane + 4 * i, all);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i + e] = v[e];
        }
    }
};

template <typename TIO, typename TC, int DK, int NW, bool FULL>
__global__ __launch_bounds__(NW * 64, 2) void decay_grad_kernel(DecayGradParams p) {
    const DecayParams& a = p.f;
    constexpr int E = Mat<TC>::E, KS = Mat<TC>::KS, CH = decay_grad_chunk(E == 8), CT = CH / 16, TJ = CH / KS;
    constexpr int DVW = 32, RK = tile_stride<TC>(DK), RV = tile_stride<TC>(DVW), RC = tile_stride<TC>(CH), NTH = NW * 64;
    constexpr int TILES = CT * (CT + 1) / 2, MT = (TILES + NW - 1) / NW, NP = E == 8 ? 2 : 1, PL = CH * RC, PR = DK * DVW;
    // a wave owns NDK tiles of key dims and one of value dims, for all 16-token tiles of the chunk or where there are waves
    // enough a share of them
    constexpr int TK = DK / 16, NDK = TK > NW ? TK / NW : 1, HK = TK > NW ? 1 : NW / TK < CT ? NW / TK : CT, CTK = CT / HK;
    constexpr int TV = DVW / 16, HV = NW / TV < CT ? NW / TV : CT, CTV = CT / HV;
    static_assert(TV <= NW && TK % NDK == 0, "tiles of dims for a wave");
    static_assert(NP * PR <= CH * RK, "R's planes take q's place");
    using Frag = typename Mat<TC>::Frag;
    __shared__ __attribute__((aligned(16))) TC s_q[CH * RK], s_k[CH * RK], s_v[CH * RV], s_d[CH * RV];
    __shared__ __attribute__((aligned(16))) TC s_A[NP * PL];  // A, then B
    __shared__ float s_g[2][CH], s_x[NW][CH], s_y[NW][CH], s_z[NW];
    __shared__ float s_r[TILES][16], s_c[TILES][16], s_tot[TILES], s_diag[CT][16];
    TC* const s_R = s_q;  // between A and the last steps: a slice of R, [DK][DVW] in parts
    const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, n = lane & 15;
    const int h = (int)(blockIdx.x % (uint32_t)a.H);
    const uint32_t sc = blockIdx.x / (uint32_t)a.H, seq32 = sc / (uint32_t)p.nc;
    const int64_t seq = seq32, c = sc - seq32 * (uint32_t)p.nc, t0 = c * CH;
    const int rows = (int)min((int64_t)CH, a.T - t0), hk = h / a.per;
    const int wide = (int)p.wide;
    const int64_t values = (int64_t)DK * wide, place = (seq * a.H + h) * p.nc + c;
    const StateAt S(p.S + place * values, values), R(p.R + place * values, values);
    auto at = [&](const DecayTok& t, int head) { return seq * t.sb + t0 * t.st + head * t.sh; };

    constexpr int UK = TK / NDK;  // waves that share the key dims
    const int tk = w % UK * NDK, Ik = w / UK * CTK, tv = w % TV, Jv = w / TV * CTV;
    const bool ownsK = w < UK * HK, ownsV = w < TV * HV;
    // a slice of 32 value dims: v, do, and the wave's rows of the states, in flight while the one before is worked on
    const TIO *pv = (const TIO*)a.v.p + at(a.v, h), *pd = (const TIO*)a.o.p + at(a.o, h);
    Tile<TIO, TC, CH, DVW, NTH, FULL> fv(a.v.st), fd(a.o.st);
    constexpr int NS = DVW / KS;
    float xs[NDK * NS][E], xr[NDK * NS][E];
    auto fetch = [&](int col0) {
        fv.fetch(pv + col0, a.v.st, rows, a.Dv - col0);
        fd.fetch(pd + col0, a.o.st, rows, a.Dv - col0);
#pragma unroll
        for (int i = 0; i < NDK * NS; ++i) {
            const int all = 4 * (16 * (tk + i / NS) * wide + col0 + i % NS * KS);
            S.row<E>(4 * (n * wide + E * g), all, xs[i]);
            R.row<E>(4 * (n * wide + E * g), all, xr[i]);
        }
    };
    Tile<TIO, TC, CH, DK, NTH, FULL> fq(a.q.st);
    const TIO* pq = (const TIO*)a.q.p + at(a.q, hk);
    {
        Tile<TIO, TC, CH, DK, NTH, FULL> fk(a.k.st);
        fq.fetch(pq, a.q.st, rows, a.Dk);
        fk.fetch((const TIO*)a.k.p + at(a.k, hk), a.k.st, rows, a.Dk);
        fetch(0);
        fq.put(s_q);
        fk.put(s_k);
    }
    if (w == 0) {
        const Sum2 gs = chunk_sums<CH>(a.g, a.g_dt, at(a.g, h), rows, lane);
        if (lane < CH) s_g[0][lane] = gs.hi, s_g[1][lane] = gs.lo;
    }
    if constexpr (E == 8) {  // a K step of 32 tokens takes the tile above the diagonal along: zeros
        for (int u = threadIdx.x; u < CT / 2 * NP * 16 * 4; u += NTH) {
            const int q = u & 3, row = (u >> 2) & 15, b = (u >> 6) & (NP - 1), I = 2 * (u >> 7);
            *reinterpret_cast<uint2*>(s_A + b * PL + (16 * I + row) * RC + 16 * (I + 1) + 4 * q) = uint2{0, 0};
        }
    }
    lds_barrier();
    auto sum_at = [&](int t) { return Sum2{s_g[0][t], s_g[1][t]}; };
    const Sum2 end = sum_at(CH - 1);

    // scale e^{G_i - G_j} of a tile's value, 0 above the diagonal (whose products may be anything)
    auto weighed = [&](const f32x4& x, int I, int J) {
        const Sum2 Gi = sum_at(16 * I + n);
        f32x4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            y[r] = J < I || 4 * g + r <= n ? x[r] * (a.scale * decay_between(Gi, sum_at(16 * J + 4 * g + r))) : 0.f;
        return y;
    };
    f32x4 am[MT], bm[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        am[m] = bm[m] = zero4();
        const int idx = w + NW * m;
        if (idx >= TILES) continue;
        int I, J;
        tile_of(idx, I, J);
#pragma unroll
        for (int s = 0; s < DK / KS; ++s)
            am[m] = Mat<TC>::mma(row_frag(s_k, RK, 16 * J + n, s, g), row_frag(s_q, RK, 16 * I + n, s, g), am[m]);
        put4<TC, NP>(s_A, PL, (16 * I + n) * RC + 16 * J + 4 * g, weighed(am[m], I, J));
    }

    // The wave's columns of R's slice; rows 4 to 7 of eight have their halves swapped, since rows without padding would meet
    // on the banks there.
    auto R_cols = [&](int b, int s) {
        if constexpr (E == 8) {
            const int row = 32 * s + 4 * g + (n >> 2), col = 16 * tv + 4 * (n & 3);
            const TC* x = s_R + b * PR + row * DVW + (col ^ ((g & 1) << 4));
            const bf16x4 lo = lds_read_tr(x), hi = lds_read_tr(x + 16 * DVW);
            return Frag{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        } else {
            const TC* x = s_R + (16 * s + 4 * g) * DVW + ((16 * tv + n) ^ ((g & 1) << 4));
            return Frag{x[0], x[DVW], x[2 * DVW], x[3 * DVW]};
        }
    };

    f32x4 dq[NDK][CTK], dk[NDK][CTK];
#pragma unroll
    for (int d = 0; d < NDK; ++d)
#pragma unroll
        for (int I = 0; I < CTK; ++I) dq[d][I] = dk[d][I] = zero4();
    float z = 0.f;
    for (int col0 = 0; col0 < a.Dv; col0 += DVW) {
        lds_barrier();
        fv.put(s_v);
        fd.put(s_d);
        if (ownsK && Ik == 0) {
#pragma unroll
            for (int i = 0; i < NDK * NS; ++i) {
                const auto r = parts<TC, 2>(xr[i]);
#pragma unroll
                for (int b = 0; b < NP; ++b)
                    *reinterpret_cast<Frag*>(s_R + b * PR + (16 * (tk + i / NS) + n) * DVW +
                                             ((i % NS * KS + E * g) ^ ((n & 4) << 2))) = r.p[b];
#pragma unroll
                for (int e = 0; e < E; ++e) z = __builtin_fmaf(xs[i][e], xr[i][e], z);
            }
        }
        lds_barrier();
        if (ownsK) {
#pragma unroll
            for (int i = 0; i < NDK * NS; ++i) {
                const int d = i / NS, s = i % NS;
                const auto ps = parts<TC, 3>(xs[i]);
                const auto pr = parts<TC, 3>(xr[i]);
#pragma unroll
                for (int I = 0; I < CTK; ++I) {
                    dq[d][I] = mma<TC>(ps, row_frag(s_d, RV, 16 * (Ik + I) + n, s, g), dq[d][I]);
                    dk[d][I] = mma<TC>(pr, row_frag(s_v, RV, 16 * (Ik + I) + n, s, g), dk[d][I]);
                }
            }
        }
        if (col0 + DVW < a.Dv) fetch(col0 + DVW);
        else fq.fetch(pq, a.q.st, rows, a.Dk);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int idx = w + NW * m;
            if (idx >= TILES) continue;
            int I, J;
            tile_of(idx, I, J);
#pragma unroll
            for (int s = 0; s < DVW / KS; ++s)
                bm[m] = Mat<TC>::mma(row_frag(s_v, RV, 16 * J + n, s, g), row_frag(s_d, RV, 16 * I + n, s, g), bm[m]);
        }
        if (ownsV) {
#pragma unroll
            for (int u = 0; u < CTV; ++u) {
                const int J = Jv + u, j = 16 * J + n;
                f32x4 dv = zero4();
#pragma unroll
                for (int s = 0; s < DK / KS; ++s) {
                    const Frag x = row_frag_tok(s_k, RK, j, s, g);
#pragma unroll
                    for (int b = NP - 1; b >= 0; --b)
                        dv = Mat<TC>::mma(R_cols(b, s), x, dv);
                }
                dv *= decay_between(end, sum_at(j));
                for (int s = 16 * J / KS; s < TJ; ++s) {
                    const Frag x = col_frag<TC, false>(s_d, RV, tv, s, g, n);
#pragma unroll
                    for (int b = NP - 1; b >= 0; --b)
                        dv = Mat<TC>::mma(x, col_frag<TC, false>(s_A + b * PL, RC, J, s, g, n), dv);
                }
                const int dim = col0 + 16 * tv + 4 * g;
                const float o[4] = {dv[0], dv[1], dv[2], dv[3]};
                if (j < rows && dim < a.Dv)
                    store_raw<4>((TIO*)p.dv + ((seq * a.T + t0 + j) * a.H + h) * a.Dv + dim, FULL ? 4 : a.Dv - dim, o);
            }
        }
    }

    // B, and the sums of (q . k) B over its tiles that the gates' gradients take
    lds_barrier();
    fq.put(s_q);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int idx = w + NW * m;
        if (idx >= TILES) continue;
        int I, J;
        tile_of(idx, I, J);
        const f32x4 x = weighed(bm[m], I, J);
        f32x4 M;
#pragma unroll
        for (int r = 0; r < 4; ++r) M[r] = J < I || 4 * g + r < n ? am[m][r] * x[r] : 0.f;
        put4<TC, NP>(s_A, PL, (16 * I + n) * RC + 16 * J + 4 * g, x);
        if (J < I) {
            float col = (M[0] + M[1]) + (M[2] + M[3]);
            col = xor_sum<32>(xor_sum<16>(col));
            if (g == 0) s_c[idx][n] = col;
            col = dpp_sum16(col);
            if (lane == 0) s_tot[idx] = col;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float row = dpp_sum16(M[r]);
                if (n == 0) s_r[idx][4 * g + r] = row;
            }
        } else {
            // for every t = 4 g + r: written before t (rows of lower r and g), read at t or behind (n >= t)
            const float all = (M[0] + M[1]) + (M[2] + M[3]);
            const RowPair by1 = swap16(all);
            const float by2 = swap32(by1.lo + by1.hi).lo;
            float before = ((g & 1) ? by1.lo : 0.f) + ((g & 2) ? by2 : 0.f);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float sum = dpp_sum16(n >= 4 * g + r ? before : 0.f);
                if (n == 0) s_diag[I][4 * g + r] = sum;
                before += M[r];
            }
        }
    }
    lds_barrier();

    for (int t = lane; t < CH; t += 64) s_x[w][t] = s_y[w][t] = 0.f;
    if (ownsK) {
#pragma unroll
        for (int u = 0; u < CTK; ++u) {
            const int I = Ik + u, i = 16 * I + n;
            const Sum2 Gi = sum_at(i);
            const float eq = a.scale * __builtin_amdgcn_exp2f(Gi.hi + Gi.lo), ek = decay_between(end, Gi);
            const int64_t tok = seq * a.T + t0 + i;
            float x = 0.f, y = 0.f;
#pragma unroll
            for (int d = 0; d < NDK; ++d) {
                const int dim = 16 * (tk + d) + 4 * g;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    dq[d][u][r] *= eq;
                    dk[d][u][r] *= ek;
                    x = __builtin_fmaf((float)s_q[i * RK + dim + r], dq[d][u][r], x);
                    y = __builtin_fmaf((float)s_k[i * RK + dim + r], dk[d][u][r], y);
                }
                for (int s = 0; s <= (16 * I + 15) / KS; ++s) {
                    const Frag f = col_frag<TC, false>(s_k, RK, tk + d, s, g, n);
#pragma unroll
                    for (int b = NP - 1; b >= 0; --b)
                        dq[d][u] = Mat<TC>::mma(f, row_frag_tok(s_A + b * PL, RC, i, s, g), dq[d][u]);
                }
                for (int s = 16 * I / KS; s < TJ; ++s) {
                    const Frag f = col_frag<TC, false>(s_q, RK, tk + d, s, g, n);
#pragma unroll
                    for (int b = NP - 1; b >= 0; --b)
                        dk[d][u] = Mat<TC>::mma(f, col_frag<TC, false>(s_A + b * PL, RC, I, s, g, n), dk[d][u]);
                }
                if (i >= rows || dim >= a.Dk) continue;
                const float oq[4] = {dq[d][u][0], dq[d][u][1], dq[d][u][2], dq[d][u][3]};
                const float ok[4] = {dk[d][u][0], dk[d][u][1], dk[d][u][2], dk[d][u][3]};
                const int left = FULL ? 4 : a.Dk - dim;
                if (p.part_q) {  // of one head of several that share q and k
                    const int64_t off = (tok * a.H + h) * a.Dk + dim;
                    store_raw<4>(p.part_q + off, left, oq);
                    store_raw<4>(p.part_k + off, left, ok);
                } else {
                    const int64_t off = (tok * (a.H / a.per) + hk) * a.Dk + dim;
                    store_raw<4>((TIO*)p.dq + off, left, oq);
                    store_raw<4>((TIO*)p.dk + off, left, ok);
                }
            }
            x = xor_sum<32>(xor_sum<16>(x));
            y = xor_sum<32>(xor_sum<16>(y));
            if (g == 0) s_x[w][i] = x, s_y[w][i] = y;
        }
    }
    z = xor_sum<16>(xor_sum<32>(dpp_sum16(z)));
    if (lane == 0) s_z[w] = z;
    __syncthreads();
    if (w) return;

    const int t = lane & (CH - 1), blk = t >> 4;
    float x = 0.f, y = 0.f, across = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) x += s_x[k][t], y += s_y[k][t], across += s_z[k];
    across *= __builtin_amdgcn_exp2f(end.hi + end.lo);
    float rs = 0.f, cs = 0.f;
    for (int I = blk + 1; I < CT; ++I) rs += s_r[tile_index(I, blk)][n];
    for (int J = 0; J < blk; ++J) {
        cs += s_c[tile_index(blk, J)][n];
        for (int I = blk + 1; I < CT; ++I) across += s_tot[tile_index(I, J)];
    }
    // lanes 0 .. CH - 1: sums at and behind t of x, in front of t of y
    x = row_suffix_scan(x);
    y = row_inclusive_scan(y);
    float later = 0.f, earlier = 0.f;
#pragma unroll
    for (int b = 0; b < CT; ++b) {
        const float xb = lane_value(x, 16 * b), yb = lane_value(y, 16 * b + 15);
        if (b > blk) later += xb;
        if (b < blk) earlier += yb;
    }
    float dg = (x + later) + (row_shr<1>(y) + earlier) + across + row_shr<1>(row_inclusive_scan(rs)) +
               row_suffix_scan(cs) + s_diag[blk][n];
    const bool in = lane < CH && t < rows;
    const float gate = in ? load_dt(a.g.p, a.g_dt, at(a.g, h) + t * a.g.st) : 0.f;
    if (!in || gate > 0.f) dg = 0.f;
    if (p.part_g) {
        dg = xor_sum<16>(xor_sum<32>(dpp_sum16(dg)));
        if (lane == 0) p.part_g[(seq * p.nc + c) * a.H + h] = dg;
    } else if (in) {
        store_dt(p.dg, a.g_dt, (seq * a.T + t0 + t) * a.H + h, dg);
    }
}

// dq and dk of shared heads: the sum over the heads that share them, in their order.  A thread takes every
// SHARE_BLOCKS * 256-th value, so that no size outgrows a grid.
constexpr int64_t SHARE_BLOCKS = 1 << 16;
template <typename TIO>
__global__ __launch_bounds__(256) void decay_share_kernel(DecayGradParams p, int64_t n) {
    const DecayParams& a = p.f;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += SHARE_BLOCKS * 256) {
        const int64_t head = i / a.Dk, d = i - head * a.Dk;
        float q = 0.f, k = 0.f;
        for (int s = 0; s < a.per; ++s) {
            const int64_t off = (head * a.per + s) * a.Dk + d;
            q += p.part_q[off];
            k += p.part_k[off];
        }
        ((TIO*)p.dq)[i] = (TIO)q;
        ((TIO*)p.dk)[i] = (TIO)k;
    }
}

// dg of constants per head: the chunks' sums, sixteen threads a head, then these, in a fixed order.
__global__ __launch_bounds__(1024) void decay_gate_kernel(DecayGradParams p, int64_t parts) {
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = blockIdx.x * 64 + l, H = p.f.H;
    __shared__ float red[16][64];
    float s = h < H ? sum_parts(p.part_g + h, H, w, parts) : 0.f;
    red[w][l] = s;
    __syncthreads();
    if (w || h >= H) return;
    for (int i = 1; i < 16; ++i) s += red[i][l];
    store_dt(p.dg, p.f.g_dt, h, s);
}

namespace {

template <typename TIO, typename TC, int DK>
void grad_one(const DecayGradParams& p, bool full, hipStream_t s) {
    const dim3 grid((unsigned)(p.f.n_seqs * p.nc * p.f.H));
    if (full) decay_grad_kernel<TIO, TC, DK, 4, true><<<grid, 256, 0, s>>>(p);
    else decay_grad_kernel<TIO, TC, DK, 4, false><<<grid, 256, 0, s>>>(p);
}
template <typename TIO, typename TC>
hipError_t grad_dk(const DecayGradParams& p, bool full, hipStream_t s) {
    switch (decay_padded_dk(p.f.Dk)) {
        case 32: grad_one<TIO, TC, 32>(p, full, s); break;
        case 64: grad_one<TIO, TC, 64>(p, full, s); break;
        default: grad_one<TIO, TC, 128>(p, full, s);
    }
    return hipGetLastError();
}
template <typename TIO>
hipError_t share(const DecayGradParams& p, hipStream_t s) {
    const int64_t n = p.f.n_seqs * p.f.T * (p.f.H / p.f.per) * p.f.Dk;
    const int64_t blocks = (n + 255) / 256;
    decay_share_kernel<TIO><<<dim3((unsigned)(blocks < SHARE_BLOCKS ? blocks : SHARE_BLOCKS)), 256, 0, s>>>(p, n);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_decay_grad(const DecayGradParams& p, int io_dt, hipStream_t s) {
    const DecayParams& a = p.f;
    const bool full = decay_full(a.Dk, a.Dv, io_dt, {a.q, a.k, a.v, a.o});
    hipError_t e = io_dt == DT_F32    ? grad_dk<float, float>(p, full, s)
                   : io_dt == DT_BF16 ? grad_dk<__bf16, __bf16>(p, full, s)
                                      : grad_dk<_Float16, float>(p, full, s);
    if (e != hipSuccess) return e;
    if (p.part_q) {
        e = io_dt == DT_F32 ? share<float>(p, s) : io_dt == DT_BF16 ? share<__bf16>(p, s) : share<_Float16>(p, s);
        if (e != hipSuccess) return e;
    }
    if (p.part_g) {
        decay_gate_kernel<<<dim3((unsigned)((p.f.H + 63) / 64)), 1024, 0, s>>>(p, p.f.n_seqs * p.nc);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace triune
