// decay_walk.hip -- the passes of decay attention that form states alone (decay_attn.hip, decay_attn_bwd.hip) on gfx950.
#include "decay_mfma.h"

namespace triune {

constexpr int C = DECAY_CHUNK;

// States alone, from rows (k of a.k) by columns (v): the segments' own end states (states null) of those that another one
// follows, in the workspace; or from the carried-in states the state in front of every `every` tokens, in `states`,
// and the final one.  REV: the same from the end of the sequence (gradients of states, rows q and columns do):
//     R <- e^{G_C} R + scale sum_i e^{G_i} q_i do_i^T
template <typename TIO, typename TC, int DK, int NW, int NT, bool FULL, bool REV>
__global__ __launch_bounds__(NW * 64, 2) void decay_walk_kernel(DecayWalkParams p) {
    const DecayParams& a = p.f;
    constexpr int E = Mat<TC>::E, KS = Mat<TC>::KS, WIDTH = NW * NT * 16, NTH = NW * 64;
    constexpr int RK = tile_stride<TC>(DK), RV = tile_stride<TC>(WIDTH), TJ = C / KS, DT = DK / 16;
    using Frag = typename Mat<TC>::Frag;
    __shared__ __attribute__((aligned(16))) TC s_ks[2][C * RK], s_vs[2][C * RV];
    __shared__ __attribute__((aligned(16))) ChunkGates s_gs[2];
    DecayWhere x;
    if (!decay_where(a, x)) return;
    const bool each = p.states, begins = REV ? x.seg.last : x.seg.index == 0, ends = REV ? x.seg.index == 0 : x.seg.last;
    if (!each && ends) return;
    const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, n = lane & 15, col0 = x.slice * WIDTH;
    const TIO* pk = (const TIO*)a.k.p + decay_base(a, x, a.k, x.h / a.per);
    const TIO* pv = (const TIO*)a.v.p + decay_base(a, x, a.v, x.h) + col0;
    const int64_t pg = decay_base(a, x, a.g, x.h);
    const int64_t srow = ssm_row(a.slots, a.n_slots, x.seg.seq), soff = (srow * a.H + x.h) * a.Dk * a.Dv;
    const int64_t values = (int64_t)DK * WIDTH * a.slices, in_ws = ((int64_t)x.slice * NW + w) * (NT * DT * 256) + lane * 4;
    auto ws = [&](int64_t item) { return a.ws_state + (item * a.H + x.h) * values + in_ws; };

    f32x4 S[NT][DT];
    if (begins) {
        each_state<TC>(S, col0, a.Dk, a.Dv, a.Dv, [&](float& v, int64_t off, bool in) {
            v = in && a.s0 && srow >= 0 ? a.s0[soff + off] : 0.f;
        });
        // The last segment of a cut sequence has no use for its place in the workspace: it takes the initial state,
        // since s0 may be the pool that the last segment's outputs leave their state in while the first one starts.
        if (!REV && !each) put_state(S, ws(x.last));
    } else if (each) {
        get_state(S, ws(REV ? x.w + 1 : x.w - 1));
    } else {
        each_state<TC>(S, 0, 0, 0, 0, [](float& v, int64_t, bool) { v = 0.f; });
    }

    Sum2 all{0.f, 0.f};
    const int chunks = (x.seg.len + C - 1) / C;
    Tile<TIO, TC, C, DK, NTH, FULL> tk(a.k.st, a.Dk);
    Tile<TIO, TC, C, WIDTH, NTH, FULL> tv(a.v.st, a.Dv - col0);
    GateBits tg;
    auto fetch = [&](int i) {
        const int t0 = (REV ? chunks - 1 - i : i) * C, rows = min(C, x.seg.len - t0);
        tk.fetch(pk + t0 * a.k.st, a.k.st, rows, a.Dk);
        tv.fetch(pv + t0 * a.v.st, a.v.st, rows, a.Dv - col0);
        tg.fetch(a.g, a.g_dt, pg + (t0 + min(lane & (C - 1), rows - 1)) * a.g.st);
    };
    if (chunks) fetch(0);
    for (int i = 0; i < chunks; ++i) {
        const int t0 = (REV ? chunks - 1 - i : i) * C, rows = min(C, x.seg.len - t0);
        TC *s_k = s_ks[i & 1], *s_v = s_vs[i & 1];
        const int64_t at = x.seg.t0 + t0;
        if (each && (REV ? (at + C) % p.every == 0 || at + rows == a.T : at % p.every == 0)) {
            const int64_t nc = (a.T + p.every - 1) / p.every, wide = (int64_t)WIDTH * a.slices;
            float* to = p.states + ((x.seg.seq * a.H + x.h) * nc + at / p.every) * values;
            each_state<TC>(S, col0, DK, (int)wide, wide, [&](float& v, int64_t off, bool) { to[off] = v; });
        }
        tk.put(s_k);
        tv.put(s_v);
        ChunkGates& s_g = s_gs[i & 1];
        if (w == 0) s_g.put(tg.value(a.g_dt), rows, lane);
        if (i + 1 < chunks) fetch(i + 1);
        lds_barrier();
        const float keep = s_g.from[C - 1];
        all.hi = fmaxf(all.hi + s_g.hi[C - 1], -1024.f);
        all.lo += s_g.lo[C - 1];
        f32x4 wj[2];
#pragma unroll
        for (int J = 0; J < 2; ++J) wj[J] = REV ? a.scale * four(&s_g.from[16 * J + 4 * g]) : four(&s_g.to[16 * J + 4 * g]);
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int t = 0; t < DT; ++t) S[c][t] *= keep;
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            Frag kf[DT];
#pragma unroll
            for (int t = 0; t < DT; ++t) kf[t] = col_frag<TC, true>(s_k, RK, t, j, g, n);
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                const Frag vf = col_frag<TC, false>(s_v, RV, w * NT + c, j, g, n);
                float v[E];
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = (float)vf[e] * wj[TJ == 1 ? e >> 2 : j][e & 3];
                const auto vp = parts<TC, 3>(v);
#pragma unroll
                for (int t = 0; t < DT; ++t) S[c][t] = mma<TC>(kf[t], vp, S[c][t]);
            }
        }
    }

    if (each) {
        if (!ends || !a.fin || srow < 0) return;
        each_state<TC>(S, col0, a.Dk, a.Dv, a.Dv, [&](float& v, int64_t off, bool in) {
            if (in) a.fin[soff + off] = v;
        });
    } else {
        put_state(S, ws(x.w));
        if (x.slice == 0 && threadIdx.x == 0) {
            float* sum = a.ws_sum + (x.w * a.H + x.h) * 2;
            sum[0] = all.hi, sum[1] = all.lo;
        }
    }
}

// Joins the segments' end states in order: S_p = 2^{sum_p} S_{p-1} + own_p, in place, for the segments that another
// one follows (rev: from the last one to the second).  A thread per value of a (sequence, head).
__global__ __launch_bounds__(256) void decay_carry_kernel(DecayParams a, int64_t values, bool rev) {
    const int64_t blocks = (values + 255) / 256;
    const int64_t sh = blockIdx.x / blocks, i = (blockIdx.x % blocks) * 256 + threadIdx.x;
    const int64_t seq = sh / a.H, h = sh % a.H;
    if (i >= values) return;
    int64_t first, n;
    if (a.cu) {
        first = a.seg_off[seq];
        n = a.seg_off[seq + 1] - first;
    } else {
        first = seq * a.nseg;
        n = a.nseg;
    }
    if (n < 3) return;  // one state to carry: the first segment's own
    const int64_t step = rev ? -a.H * values : a.H * values, step_sum = rev ? -2 * a.H : 2 * a.H;
    if (rev) first += n - 1;
    float* p = a.ws_state + (first * a.H + h) * values + i;
    const float* sum = a.ws_sum + (first * a.H + h) * 2;
    float s = p[0];
    constexpr int AHEAD = 8;
    for (int64_t k0 = 1; k0 < n - 1; k0 += AHEAD) {
        float x[AHEAD], d[AHEAD];
        const int m = (int)min((int64_t)AHEAD, n - 1 - k0);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (k < m) {
                x[k] = p[(k0 + k) * step];
                const float* e = sum + (k0 + k) * step_sum;
                d[k] = __builtin_amdgcn_exp2f(e[0] + e[1]);
            }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (k < m) {
                s = __builtin_fmaf(d[k], s, x[k]);
                p[(k0 + k) * step] = s;
            }
    }
}

namespace {

template <typename TIO, typename TC>
struct Walk {
    template <int DK, int NW, int NT, bool FULL>
    static void run(const DecayWalkParams& p, dim3 grid, hipStream_t s) {
        decay_walk_kernel<TIO, TC, DK, NW, NT, FULL, false><<<grid, NW * 64, 0, s>>>(p);
    }
};
template <typename TIO, typename TC>
struct WalkBack {
    template <int DK, int NW, int NT, bool FULL>
    static void run(const DecayWalkParams& p, dim3 grid, hipStream_t s) {
        decay_walk_kernel<TIO, TC, DK, NW, NT, FULL, true><<<grid, NW * 64, 0, s>>>(p);
    }
};

}  // namespace

hipError_t launch_decay_walk(const DecayWalkParams& p, bool rev, int io_dt, hipStream_t s) {
    const bool full = decay_full(p.f.Dk, p.f.Dv, io_dt, {p.f.k, p.f.v});
    return rev ? decay_by_type<WalkBack>(p, p.f, io_dt, full, s) : decay_by_type<Walk>(p, p.f, io_dt, full, s);
}
hipError_t launch_decay_carry(const DecayParams& a, bool rev, hipStream_t s) {
    const int64_t values = decay_state_values(a.Dk, a.Dv);
    decay_carry_kernel<<<dim3((unsigned)(a.n_seqs * a.H * ((values + 255) / 256))), 256, 0, s>>>(a, values, rev);
    return hipGetLastError();
}

}  // namespace triune
