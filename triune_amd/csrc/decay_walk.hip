// decay_walk.hip -- the passes of decay attention that form states alone (decay_attn.hip, decay_attn_bwd.hip) on gfx950.
//
// The chunk walk of decay_attn.hip without its scores and outputs.  End states: 4 x 16384 tokens, 6 heads of 64, bf16,
// segments of 512: 28.2 us, half of the SIMDs' cycles issue vector work; 4 x 2048, 12 heads of 128, segments of 256:
// 26.4 us, a chain of eight chunks a workgroup.  States of every 64th token, both directions, of the latter: 80.1 us
// for 206 MB written and 80 read, 3.6 TB/s.
#include "decay_mfma.h"

namespace triune {

constexpr int C = DECAY_CHUNK;

// LDS of a walk.
template <typename TC, int DK, int WIDTH>
struct WalkTiles {
    __attribute__((aligned(16))) TC k[2][C * tile_stride<TC>(DK)], v[2][C * tile_stride<TC>(WIDTH)];
    __attribute__((aligned(16))) ChunkGates g[2];
};

// States alone, from rows (a.k) by columns (a.v), REV: from the end of the sequence (gradients of states, whose rows are q
// and whose columns are do):
//     S <- e^{G_C} S + sum_j e^{G_C - G_j} k_j v_j^T,   R <- e^{G_C} R + scale sum_i e^{G_i} q_i do_i^T
// EACH false: the segments' own end states of those that another one follows, the first one's from a.s0, in the
// workspace in the order of the lanes; decay_carry_kernel joins them.
// EACH true: from the joined states the state in front of (REV: behind) every chunk of p.every tokens, and the final one.
template <typename TIO, typename TC, int DK, int NW, int NT, bool FULL, bool REV, bool EACH>
__device__ __forceinline__ void walk(const DecayWalkParams& p, WalkTiles<TC, DK, NW * NT * 16>& lds) {
    const DecayParams& a = p.f;
    constexpr int E = Mat<TC>::E, KS = Mat<TC>::KS, WIDTH = NW * NT * 16, NTH = NW * 64;
    constexpr int RK = tile_stride<TC>(DK), RV = tile_stride<TC>(WIDTH), TJ = C / KS, DT = DK / 16;
    using Frag = typename Mat<TC>::Frag;
    DecayWhere x;
    if (!decay_where(a, x)) return;
    const bool begins = REV ? x.seg.last : x.seg.index == 0, ends = REV ? x.seg.index == 0 : x.seg.last;
    if (!EACH && ends) return;
    const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, n = lane & 15, col0 = x.slice * WIDTH;
    const TIO* pk = (const TIO*)a.k.p + decay_base(a, x, a.k, x.h / a.per);
    const TIO* pv = (const TIO*)a.v.p + decay_base(a, x, a.v, x.h) + col0;
    const int64_t pg = decay_base(a, x, a.g, x.h);
    const int64_t srow = ssm_row(a.slots, a.n_slots, x.seg.seq), soff = (srow * a.H + x.h) * a.Dk * a.Dv;
    const int64_t wide = (int64_t)WIDTH * a.slices, values = DK * wide;

    const int chunks = (x.seg.len + C - 1) / C;
    // loads and gates ahead as in decay_attn_kernel
    Tile<TIO, TC, C, DK, NTH, FULL> tk(a.k.st);
    Tile<TIO, TC, C, WIDTH, NTH, FULL> tv(a.v.st);
    GateBits tg;
    auto first = [&](int i) { return (REV ? chunks - 1 - i : i) * C; };
    auto fetch = [&](int i) {
        const int t0 = first(i), rows = min(C, x.seg.len - t0);
        tk.fetch(pk + t0 * a.k.st, a.k.st, rows, a.Dk);
        tv.fetch(pv + t0 * a.v.st, a.v.st, rows, a.Dv - col0);
    };
    auto fetch_gates = [&](int i) {
        tg.fetch(a.g, a.g_dt, pg + min(first(min(i, chunks - 1)) + (lane & (C - 1)), x.seg.len - 1) * a.g.st);
    };
    if (chunks) {
        fetch_gates(0);
        fetch(0);
        if (w == NW - 1) lds.g[0].put(tg.value(a.g_dt), x.seg.len - first(0), lane);
        fetch_gates(1);
    }

    auto ws = [&](int64_t item) {
        return a.ws_state + (item * a.H + x.h) * values + ((int64_t)x.slice * NW + w) * (NT * DT * 256) + lane * 4;
    };
    f32x4 S[NT][DT];
    if (EACH && !begins) {
        get_state(S, ws(REV ? x.w + 1 : x.w - 1));
    } else if (begins && a.s0) {
        each_state<TC>(S, col0, a.Dk, a.Dv, a.Dv, [&](float& v, int64_t off, bool in) {
            v = in && srow >= 0 ? a.s0[soff + off] : 0.f;
        });
    } else {
        each_state<TC>(S, 0, 0, 0, 0, [](float& v, int64_t, bool) { v = 0.f; });
    }
    // The last segment of a cut sequence has no use for its place in the workspace: it takes the initial state, since
    // s0 may be the pool that the last segment's outputs leave their state in while the first one starts.
    if (!EACH && !REV && begins) put_state(S, ws(x.last));
    const int64_t nc = EACH ? (a.T + p.every - 1) / p.every : 0;
    auto keep_at = [&](int64_t c) {
        const int64_t at = (x.seg.seq * a.H + x.h) * nc + c;
        float* to = p.states + at * values;
        each_state<TC>(S, col0, DK, (int)wide, wide, [&](float& v, int64_t off, bool) { to[off] = v; });
    };

    Sum2 all{0.f, 0.f};
    for (int i = 0; i < chunks; ++i) {
        const int t0 = first(i), place = i & 1;
        const int64_t at = x.seg.t0 + t0;
        if (EACH && (REV ? (at + C) % p.every == 0 || at + min(C, x.seg.len - t0) == a.T : at % p.every == 0))
            keep_at(at / p.every);
        TC *s_k = lds.k[place], *s_v = lds.v[place];
        tk.put(s_k);
        tv.put(s_v);
        ChunkGates& s_g = lds.g[place];
        const GateBits gates = tg;
        if (i + 1 < chunks) {
            fetch(i + 1);
            fetch_gates(i + 2);
        }
        lds_barrier();
        if (i + 1 < chunks && w == (i & (NW - 1))) lds.g[place ^ 1].put(gates.value(a.g_dt), x.seg.len - first(i + 1), lane);
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

    if constexpr (!EACH) {
        put_state(S, ws(x.w));
        float* sum = a.ws_sum + (x.w * a.H + x.h) * 2;
        if (x.slice == 0 && threadIdx.x == 0) sum[0] = all.hi, sum[1] = all.lo;
    } else if (ends && a.fin) {
        each_state<TC>(S, col0, a.Dk, a.Dv, a.Dv, [&](float& v, int64_t off, bool in) {
            if (in) a.fin[soff + off] = v;
        });
    }
}

template <typename TIO, typename TC, int DK, int NW, int NT, bool FULL, bool REV>
__global__ __launch_bounds__(NW * 64, 2) void decay_ends_kernel(DecayWalkParams p) {
    __shared__ WalkTiles<TC, DK, NW * NT * 16> lds;
    walk<TIO, TC, DK, NW, NT, FULL, REV, false>(p, lds);
}
// Both directions in one launch, which a compute unit takes side by side (gradients of 1 x 3000, 8 heads of 128 x 64, bf16:
// 54.3 us, 61.7 with a launch each).  States turned, so that a lane stores four values of a row at once, were slower (4 x
// 2048, 12 heads of 128: 92 us instead of 80).
template <typename TIO, typename TC, int DK, int NW, int NT, bool FULL>
__global__ __launch_bounds__(NW * 64, 2) void decay_states_kernel(DecayWalkParams p, DecayWalkParams r) {
    __shared__ WalkTiles<TC, DK, NW * NT * 16> lds;
    if (blockIdx.y) walk<TIO, TC, DK, NW, NT, FULL, true, true>(r, lds);
    else walk<TIO, TC, DK, NW, NT, FULL, false, true>(p, lds);
}

// Joins the segments' end states in place: S_p = 2^{sum_p} S_{p-1} + own_p, p = 1 .. n - 2 in the walk's direction, with S_0
// the first segment's own; the state in front of segment p + 1 is then S_p.  A thread per four values of a (sequence,
// head), with the next states and sums in flight: 10.6 us for 32 segments of 24 states of 64 x 64, a chain of 30 joins.
__global__ __launch_bounds__(256) void decay_carry_kernel(DecayParams a, int64_t values, bool rev) {
    const uint32_t blocks = (uint32_t)((values + 1023) / 1024);
    const uint32_t sh = blockIdx.x / blocks, seq = sh / (uint32_t)a.H, h = sh - seq * (uint32_t)a.H;
    const int64_t i = (int64_t)(blockIdx.x - sh * blocks) * 1024 + threadIdx.x * 4;
    if (i >= values) return;
    int64_t first = (int64_t)seq * a.nseg, n = a.nseg;
    if (a.cu) {
        first = a.seg_off[seq];
        n = a.seg_off[seq + 1] - first;
    }
    if (n < 3) return;  // one state to carry: the first segment's own
    if (rev) first += n - 1;
    float* s0 = a.ws_state + (first * a.H + h) * values + i;
    const float* sum0 = a.ws_sum + (first * a.H + h) * 2;  // sums of the walk's first segment
    const int64_t step = rev ? -a.H * values : a.H * values, sum_step = rev ? -2 * a.H : 2 * a.H;
    const int joins = (int)(n - 2);
    f32x4 s = *reinterpret_cast<const f32x4*>(s0);
    constexpr int AHEAD = 8;
    f32x4 x[AHEAD];
    float d[AHEAD];
    auto fetch = [&](int k0) {  // past the end the last one again, so that no load stands behind a condition
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int64_t at = min(k0 + k, joins);
            x[k] = *reinterpret_cast<const f32x4*>(s0 + at * step);
            d[k] = sum0[at * sum_step] + sum0[at * sum_step + 1];
        }
    };
    if (joins > 0) fetch(1);
    for (int k0 = 1; k0 <= joins; k0 += AHEAD) {
        f32x4 y[AHEAD];
        float f[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) y[k] = x[k], f[k] = __builtin_amdgcn_exp2f(d[k]);
        if (k0 + AHEAD <= joins) fetch(k0 + AHEAD);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (k0 + k <= joins) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] = __builtin_fmaf(f[k], s[e], y[k][e]);
                *reinterpret_cast<f32x4*>(s0 + (k0 + k) * step) = s;
            }
    }
}

namespace {

template <bool REV>
struct Ends {
    template <typename TIO, typename TC>
    struct Of {
        template <int DK, int NW, int NT, bool FULL>
        static void run(const DecayWalkParams& p, dim3 grid, hipStream_t s) {
            decay_ends_kernel<TIO, TC, DK, NW, NT, FULL, REV><<<grid, NW * 64, 0, s>>>(p);
        }
    };
};
struct TwoWalks {
    DecayWalkParams p, r;
};
template <typename TIO, typename TC>
struct States {
    template <int DK, int NW, int NT, bool FULL>
    static void run(const TwoWalks& x, dim3 grid, hipStream_t s) {
        decay_states_kernel<TIO, TC, DK, NW, NT, FULL><<<dim3(grid.x, 2), NW * 64, 0, s>>>(x.p, x.r);
    }
};

}  // namespace

hipError_t launch_decay_ends(const DecayParams& a, bool rev, int io_dt, hipStream_t s) {
    const DecayWalkParams p{a, nullptr, 0};
    const bool full = decay_full(a.Dk, a.Dv, io_dt, {a.k, a.v});
    const hipError_t e = rev ? decay_by_type<Ends<true>::template Of>(p, a, io_dt, full, s)
                             : decay_by_type<Ends<false>::template Of>(p, a, io_dt, full, s);
    if (e != hipSuccess) return e;
    const int64_t values = decay_state_values(a.Dk, a.Dv);
    decay_carry_kernel<<<dim3((unsigned)(a.n_seqs * a.H * ((values + 1023) / 1024))), 256, 0, s>>>(a, values, rev);
    return hipGetLastError();
}
hipError_t launch_decay_states(const DecayWalkParams& p, const DecayWalkParams& r, int io_dt, hipStream_t s) {
    const bool full = decay_full(p.f.Dk, p.f.Dv, io_dt, {p.f.k, p.f.v, r.f.k, r.f.v});
    return decay_by_type<States>(TwoWalks{p, r}, p.f, io_dt, full, s);
}

}  // namespace triune
