// decay_attn.hip -- linear attention with one decay per head and token on gfx950: prompts, packed prompts and single
// tokens.
//
//     S_t = e^{g_t} S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t
// in chunks of 32 tokens with G the running sum of g inside the chunk:
//     o_i = scale (e^{G_i} S_0^T q_i + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j)
//     S_C = e^{G_C} S_0 + sum_j e^{G_C - G_j} k_j v_j^T
// Every exponent is a difference of sums and at most 0, so no factor leaves the range, whatever the gates.
//
// A workgroup walks a segment of a (sequence, head) for a slice of the state's columns; its waves own 16 or 32 of them
// each, the state slice lies in their accumulators.  The scores of a chunk are three products of 16 x 16 x Dk, so every
// wave forms them for itself instead of sharing them through LDS.  Accumulators (scores, state) become operands of the
// next product in place (decay_mfma.h).  Where segments follow each other, a first pass forms their end states and a
// scan joins them (decay_walk.hip).
//
// What bounds it: a workgroup's chain of chunks where few are at work, vector issue where many are (4 x 16384 tokens, 6
// heads of 64, bf16: 69 % of the SIMDs' cycles issue vector work and 24 % matrix work, 51.9 us for 202 MB; 16 prompts,
// 12 heads of 128: 44 and 22 %, 38.7 us).  Hence a chunk's loads are in flight while the one before it is worked on
// (143 -> 126 us of all passes of a call of the first kind), its gates are formed once for all waves (103), and slices
// are as wide as 128 columns, four waves of two tiles, so that q and k are read once for all of them.  Two chunks of
// loads in flight, or two waves of two tiles for 64 columns, gave nothing.
#include "decay_mfma.h"

namespace triune {

constexpr int C = DECAY_CHUNK;

// Outputs, from the state in front of the segment.
template <typename TIO, typename TC, int DK, int NW, int NT, bool FULL>
__global__ __launch_bounds__(NW * 64, (Mat<TC>::E == 4 && DK == 128 ? 1 : 2)) void decay_attn_kernel(DecayParams a) {
    constexpr int E = Mat<TC>::E, KS = Mat<TC>::KS, WIDTH = NW * NT * 16, NTH = NW * 64;
    constexpr int RK = tile_stride<TC>(DK), RV = tile_stride<TC>(WIDTH), TJ = C / KS;  // TJ: K steps over the tokens
    constexpr int DT = DK / 16;
    using Frag = typename Mat<TC>::Frag;
    __shared__ __attribute__((aligned(16))) TC s_qs[2][C * RK], s_ks[2][C * RK], s_vs[2][C * RV];
    __shared__ __attribute__((aligned(16))) ChunkGates s_gs[2];
    DecayWhere x;
    if (!decay_where(a, x)) return;
    const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, n = lane & 15;
    const int hk = x.h / a.per, col0 = x.slice * WIDTH;
    const TIO* pq = (const TIO*)a.q.p + decay_base(a, x, a.q, hk);
    const TIO* pk = (const TIO*)a.k.p + decay_base(a, x, a.k, hk);
    const TIO* pv = (const TIO*)a.v.p + decay_base(a, x, a.v, x.h) + col0;
    TIO* po = (TIO*)a.o.p + decay_base(a, x, a.o, x.h) + col0;
    const int64_t pg = decay_base(a, x, a.g, x.h);
    const int64_t srow = ssm_row(a.slots, a.n_slots, x.seg.seq), soff = (srow * a.H + x.h) * a.Dk * a.Dv;

    f32x4 S[NT][DT];
    if (x.w == x.last && x.seg.index == 0) {
        each_state<TC>(S, col0, a.Dk, a.Dv, a.Dv, [&](float& v, int64_t off, bool in) {
            v = in && a.s0 && srow >= 0 ? a.s0[soff + off] : 0.f;
        });
    } else {  // the state behind the segment in front, or the initial one, which is in the last segment's place
        const int64_t from = x.seg.index ? x.w - 1 : x.last, values = (int64_t)DK * WIDTH * a.slices;
        get_state(S, a.ws_state + (from * a.H + x.h) * values + ((int64_t)x.slice * NW + w) * (NT * DT * 256) + lane * 4);
    }

    // A chunk's tiles go from registers to one of two places, and the next one's loads are issued; gates are loaded two
    // chunks ahead and formed one ahead.
    Tile<TIO, TC, C, DK, NTH, FULL> tq(a.q.st), tk(a.k.st);
    Tile<TIO, TC, C, WIDTH, NTH, FULL> tv(a.v.st);
    GateBits tg;
    auto fetch = [&](int t0) {
        const int rows = min(C, x.seg.len - t0);
        tq.fetch(pq + t0 * a.q.st, a.q.st, rows, a.Dk);
        tk.fetch(pk + t0 * a.k.st, a.k.st, rows, a.Dk);
        tv.fetch(pv + t0 * a.v.st, a.v.st, rows, a.Dv - col0);
    };
    auto fetch_gates = [&](int t0) { tg.fetch(a.g, a.g_dt, pg + min(t0 + (lane & (C - 1)), x.seg.len - 1) * a.g.st); };
    if (x.seg.len) {
        fetch_gates(0);
        fetch(0);
        if (w == NW - 1) s_gs[0].put(tg.value(a.g_dt), x.seg.len, lane);
        fetch_gates(C);
    }
    for (int t0 = 0; t0 < x.seg.len; t0 += C) {
        const int rows = min(C, x.seg.len - t0), place = t0 / C & 1;
        TC *s_q = s_qs[place], *s_k = s_ks[place], *s_v = s_vs[place];
        tq.put(s_q);
        tk.put(s_k);
        tv.put(s_v);
        ChunkGates& s_g = s_gs[place];
        const GateBits gates = tg;
        if (t0 + C < x.seg.len) {
            fetch(t0 + C);
            fetch_gates(t0 + 2 * C);
        }
        lds_barrier();
        // the next chunk's gates, by the waves in turn, beside the others' products
        if (w == (t0 / C & (NW - 1))) s_gs[place ^ 1].put(gates.value(a.g_dt), x.seg.len - t0 - C, lane);
        Frag vf[NT][TJ];
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int j = 0; j < TJ; ++j) vf[c][j] = col_frag<TC, false>(s_v, RV, w * NT + c, j, g, n);

        // scores of token rows J (written) and columns I (read), J <= I
        f32x4 P[2][2];
#pragma unroll
        for (int I = 0; I < 2; ++I)
#pragma unroll
            for (int J = 0; J < 2; ++J) P[I][J] = zero4();
#pragma unroll
        for (int s = 0; s < DK / KS; ++s) {
            Frag q[2], k[2];
#pragma unroll
            for (int I = 0; I < 2; ++I) {
                q[I] = row_frag(s_q, RK, 16 * I + n, s, g);
                k[I] = row_frag(s_k, RK, 16 * I + n, s, g);
            }
            P[0][0] = Mat<TC>::mma(k[0], q[0], P[0][0]);
            P[1][0] = Mat<TC>::mma(k[0], q[1], P[1][0]);
            P[1][1] = Mat<TC>::mma(k[1], q[1], P[1][1]);
        }
        f32x4 O[NT][2];
#pragma unroll
        for (int c = 0; c < NT; ++c) O[c][0] = O[c][1] = zero4();
#pragma unroll
        for (int s = 0; s < DK / KS; ++s) {
            const Frag q0 = row_frag(s_q, RK, n, s, g), q1 = row_frag(s_q, RK, 16 + n, s, g);
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                float st[E];
                acc_slots<TC>(S[c], s, st);
                const auto sp = parts<TC, 2>(st);
                O[c][0] = mma<TC>(sp, q0, O[c][0]);
                O[c][1] = mma<TC>(sp, q1, O[c][1]);
            }
        }
#pragma unroll
        for (int I = 0; I < 2; ++I) {
            const float from = s_g.from[16 * I + n];
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) O[c][I][r] *= from;
            if (I == 1) {
                const f32x4 written = four(&s_g.half[4 * g]);
                const float read = s_g.half[16 + n];
#pragma unroll
                for (int r = 0; r < 4; ++r) P[1][0][r] *= written[r] * read;
            }
            const Sum2 Gi{s_g.hi[16 * I + n], s_g.lo[16 * I + n]};
            const f32x4 hi = four(&s_g.hi[16 * I + 4 * g]), lo = four(&s_g.lo[16 * I + 4 * g]);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                P[I][I][r] = 4 * g + r <= n ? P[I][I][r] * decay_between(Gi, Sum2{hi[r], lo[r]}) : 0.f;
#pragma unroll
            for (int j = 0; j < (TJ == 1 ? 1 : I + 1); ++j) {
                float pt[E];
                acc_slots<TC>(P[I], j, pt);
                const auto pp = parts<TC, 2>(pt);
#pragma unroll
                for (int c = 0; c < NT; ++c) O[c][I] = mma<TC>(vf[c][j], pp, O[c][I]);
            }
            const int t = 16 * I + n;
            if (t < rows) {
#pragma unroll
                for (int c = 0; c < NT; ++c) {
                    const int dv = 16 * (w * NT + c) + 4 * g;
                    float o[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] = a.scale * O[c][I][r];
                    if (!FULL || dv < a.Dv - col0)
                        store_raw<4>(po + (int64_t)(t0 + t) * a.o.st + dv, FULL ? 4 : a.Dv - col0 - dv, o);
                }
            }
        }
        // the state: rows of k by weighted rows of v
        const float keep = s_g.from[C - 1];
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int t = 0; t < DT; ++t) S[c][t] *= keep;
        const f32x4 wj[2] = {four(&s_g.to[4 * g]), four(&s_g.to[16 + 4 * g])};
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            Frag kf[DT];
#pragma unroll
            for (int t = 0; t < DT; ++t) kf[t] = col_frag<TC, true>(s_k, RK, t, j, g, n);
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                float v[E];
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = (float)vf[c][j][e] * wj[TJ == 1 ? e >> 2 : j][e & 3];
                const auto vp = parts<TC, 3>(v);
#pragma unroll
                for (int t = 0; t < DT; ++t) S[c][t] = mma<TC>(kf[t], vp, S[c][t]);
            }
        }
    }

    if (!x.seg.last || !a.fin || srow < 0) return;
    each_state<TC>(S, col0, a.Dk, a.Dv, a.Dv, [&](float& v, int64_t off, bool in) {
        if (in) a.fin[soff + off] = v;
    });
}

// One token for every row: a block takes a (row, head), a thread four columns of every RG-th state row.  Bound by the
// state, read and written once, past the caches.  ALIGNED: rows of whole 16 bytes, eight of which a thread has in flight.
// 256 sessions, 12 heads of 128: 78.6 us, 5.1 TB/s, the rate of a large copy (104 us with fewer in flight and through the
// caches).
template <typename TIO, bool ALIGNED>
__global__ __launch_bounds__(256) void decay_step_kernel(DecayStepParams a, int lanes) {
    constexpr int V = 4, ROWS = 8;
    __shared__ float s_q[DECAY_MAX_DK], s_k[DECAY_MAX_DK];
    __shared__ float s_o[256 * V];
    const uint32_t b = blockIdx.x / (uint32_t)a.H;
    const int h = (int)(blockIdx.x - b * (uint32_t)a.H), hk = h / a.per;
    const int cl = threadIdx.x & (lanes - 1), rg = threadIdx.x / lanes, RG = 256 / lanes;
    const int64_t row = ssm_row(a.slots, a.n_rows, b);
    const int64_t off = (row * a.H + h) * a.Dk * a.Dv;
    const float *from = a.s_in + off;
    float* to = a.s_out + off;
    for (int d = threadIdx.x; d < a.Dk; d += 256) {
        s_q[d] = (float)((const TIO*)a.q.p)[b * a.q.sb + hk * a.q.sh + d];
        s_k[d] = (float)((const TIO*)a.k.p)[b * a.k.sb + hk * a.k.sh + d];
    }
    const float decay = __builtin_amdgcn_exp2f(log2_gate(load_dt(a.g.p, a.g_dt, b * a.g.sb + h * a.g.sh)));
    const TIO* pv = (const TIO*)a.v.p + b * a.v.sb + h * a.v.sh;
    TIO* po = (TIO*)a.o.p + b * a.o.sb + h * a.o.sh;
    for (int c0 = 0; c0 < a.Dv; c0 += lanes * V) {
        const int col = c0 + cl * V, left = a.Dv - col;
        const bool in = row >= 0 && left > 0;
        f32x4 x[ROWS], o = zero4();
        // past the last row the last one again: no load stands behind a condition
        auto fetch = [&](int d0) {
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const float* p = from + (int64_t)min(d0 + i * RG, a.Dk - 1) * a.Dv + col;
                if constexpr (ALIGNED) {
                    x[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p));
                } else {
                    const Raw<float, V> r = load_raw<V>(p, left);
#pragma unroll
                    for (int j = 0; j < V; ++j) x[i][j] = r.v[j];
                }
            }
        };
        if (in) fetch(rg);
        Raw<TIO, V> rv = load_raw<V>(pv + (in ? col : 0), in ? left : 0);
        f32x4 v;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (float)rv.v[j];
        __syncthreads();
        if (in) {
            for (int d0 = rg; d0 < a.Dk; d0 += ROWS * RG) {
#pragma unroll
                for (int i = 0; i < ROWS; ++i) {
                    const int d = d0 + i * RG;
                    if (d >= a.Dk) continue;
                    float y[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        y[j] = __builtin_fmaf(decay, x[i][j], s_k[d] * v[j]);
                        o[j] = __builtin_fmaf(s_q[d], y[j], o[j]);
                    }
                    if constexpr (ALIGNED)
                        __builtin_nontemporal_store(f32x4{y[0], y[1], y[2], y[3]},
                                                    reinterpret_cast<f32x4*>(to + (int64_t)d * a.Dv + col));
                    else store_raw<V>(to + (int64_t)d * a.Dv + col, left, y);
                }
                if (d0 + ROWS * RG < a.Dk) fetch(d0 + ROWS * RG);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) s_o[(rg * lanes + cl) * V + j] = o[j];
        __syncthreads();
        for (int e = threadIdx.x; e < lanes * V; e += 256) {
            float sum = 0.f;
            for (int k = 0; k < RG; ++k) sum += s_o[k * lanes * V + e];
            if (c0 + e < a.Dv) po[c0 + e] = (TIO)(a.scale * sum);
        }
    }
}

int decay_slice(int Dv) { return Dv <= 32 ? 32 : Dv <= 64 ? 64 : 128; }
int decay_padded_dk(int Dk) { return Dk <= 32 ? 32 : Dk <= 64 ? 64 : 128; }
int64_t decay_state_values(int Dk, int Dv) {
    const int w = decay_slice(Dv);
    return (int64_t)decay_padded_dk(Dk) * ((Dv + w - 1) / w * w);
}

namespace {

template <typename TIO, typename TC>
struct Attn {
    template <int DK, int NW, int NT, bool FULL>
    static void run(const DecayParams& a, dim3 grid, hipStream_t s) {
        decay_attn_kernel<TIO, TC, DK, NW, NT, FULL><<<grid, NW * 64, 0, s>>>(a);
    }
};

template <typename TIO>
hipError_t run_step(const DecayStepParams& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.Bn * a.H));
    const int need = (a.Dv + 3) / 4;
    int lanes = 4;
    while (lanes < need && lanes < 64) lanes *= 2;
    const auto whole = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    if (a.Dv % 4 == 0 && whole(a.s_in) && whole(a.s_out)) decay_step_kernel<TIO, true><<<grid, 256, 0, s>>>(a, lanes);
    else decay_step_kernel<TIO, false><<<grid, 256, 0, s>>>(a, lanes);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_decay_attn(const DecayParams& a, int io_dt, hipStream_t s) {
    const bool full = decay_full(a.Dk, a.Dv, io_dt, {a.q, a.k, a.v});
    return decay_by_type<Attn>(a, a, io_dt, full, s);
}
hipError_t launch_decay_step(const DecayStepParams& a, int io_dt, hipStream_t s) {
    if (io_dt == DT_F32) return run_step<float>(a, s);
    if (io_dt == DT_BF16) return run_step<__bf16>(a, s);
    return run_step<_Float16>(a, s);
}

}  // namespace triune
