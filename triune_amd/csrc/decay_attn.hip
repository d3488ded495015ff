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
// each, the state slice lies in their accumulators.  The scores of a chunk are six products of 16 x 16 x Dk, so every
// wave forms them for itself instead of sharing them through LDS.  Accumulators (scores, state) become operands of the
// next product in place (decay_mfma.h).  Where segments follow each other, a first pass forms their end states and a
// scan joins them.
#include "decay_mfma.h"

namespace triune {

namespace {

constexpr int C = DECAY_CHUNK;

// Rows of a [tokens][D] tensor, zeros past `rows` and `cols`.
template <typename TIO, typename TC, int D, int NTH>
__device__ __forceinline__ void load_tile(TC* tile, const TIO* p, int64_t st, int rows, int cols) {
    constexpr int E = Mat<TC>::E, UNITS = D / E, RS = tile_stride<TC>(D);
#pragma unroll
    for (int u = threadIdx.x; u < C * UNITS; u += NTH) {
        const int row = u / UNITS, c = u % UNITS * E;
        Raw<TIO, E> r = load_raw<E>(p + (row < rows ? row * st + c : 0), row < rows ? cols - c : 0);
        typename Mat<TC>::Frag f;
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = (TC)r.v[e];
        *reinterpret_cast<typename Mat<TC>::Frag*>(tile + row * RS + c) = f;
    }
}

// The running sums of a chunk's gates: lane l holds token l & 31's.  Tokens past the end count as 0.
__device__ __forceinline__ Sum2 chunk_sums(const DecayTok& g, int dt, int64_t at, int rows, int lane) {
    const int t = lane & 31;
    Sum2 s = split_gate(t < rows ? log2_gate(load_dt(g.p, dt, at + t * g.st)) : 0.f);
    s.hi = row_inclusive_scan(s.hi);
    s.lo = row_inclusive_scan(s.lo);
    const float h = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s.hi), 15));
    const float l = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s.lo), 15));
    if (lane & 16) s.hi += h, s.lo += l;
    return s;
}

// Work items: (segment, head, slice), slices fastest.
struct Where {
    SsmSeg seg;
    int64_t w;
    int h, slice;
};
__device__ __forceinline__ bool where(const DecayParams& a, Where& x) {
    int64_t b = blockIdx.x;
    x.slice = (int)(b % a.slices);
    b /= a.slices;
    x.h = (int)(b % a.H);
    x.w = b / a.H;
    return ssm_segment(a, x.w, x.seg);
}

}  // namespace

// OUT: outputs, from the state in front of the segment; otherwise the segment's end state (of a segment that another
// one follows), the first one's from the initial state.
template <typename TIO, typename TC, int DK, int NW, int NT, bool OUT>
__global__ __launch_bounds__(NW * 64) void decay_kernel(DecayParams a) {
    constexpr int E = Mat<TC>::E, KS = Mat<TC>::KS, WIDTH = NW * NT * 16, NTH = NW * 64;
    constexpr int RK = tile_stride<TC>(DK), RV = tile_stride<TC>(WIDTH), TJ = C / KS;  // TJ: K steps over the tokens
    constexpr int DT = DK / 16;
    using Frag = typename Mat<TC>::Frag;
    __shared__ __attribute__((aligned(16))) TC s_q[OUT ? C * RK : 1];
    __shared__ __attribute__((aligned(16))) TC s_k[C * RK], s_v[C * RV];
    __shared__ __attribute__((aligned(16))) float s_g[NW][2][C];
    Where x;
    if (!where(a, x)) return;
    if (!OUT && x.seg.last) return;
    const int lane = threadIdx.x & 63, w = wave_index(), g = lane >> 4, n = lane & 15;
    const int64_t row0 = x.seg.row0 + x.seg.t0;
    const int hk = x.h / a.per, col0 = x.slice * WIDTH;
    auto base = [&](const DecayTok& t, int h) { return x.seg.seq * t.sb * (a.cu ? 0 : 1) + row0 * t.st + h * t.sh; };
    const TIO* pq = (const TIO*)a.q.p + base(a.q, hk);
    const TIO* pk = (const TIO*)a.k.p + base(a.k, hk);
    const TIO* pv = (const TIO*)a.v.p + base(a.v, x.h) + col0;
    TIO* po = (TIO*)a.o.p + base(a.o, x.h) + col0;
    const int64_t pg = base(a.g, x.h);
    const int64_t srow = ssm_row(a.slots, a.n_slots, x.seg.seq);

    f32x4 S[NT][DT];  // rows tile_dim(t, 4 g + r), column 16 (w NT + c) + n of the slice
    constexpr int64_t kValues = (int64_t)DK * WIDTH;  // of a slice
    const int64_t values = kValues * a.slices;
    float* ws = a.ws_state + (x.w * a.H + x.h) * values + ((int64_t)x.slice * NW + w) * (NT * DT * 256) + lane * 4;
    auto state_at = [&](int c, int t, int r, int64_t& off) {
        const int dk = tile_dim<TC>(t, 4 * g + r), dv = col0 + 16 * (w * NT + c) + n;
        off = ((srow * a.H + x.h) * a.Dk + dk) * a.Dv + dv;
        return dk < a.Dk && dv < a.Dv;
    };
    // The last segment of a cut sequence has no use for its place in the workspace: it takes the initial state, since
    // s0 may be the pool that the last segment's outputs leave their state in while the first one starts.
    const int64_t last = a.cu ? (a.seg_off ? a.seg_off[x.seg.seq + 1] - 1 : x.w) : x.w - x.seg.index + a.nseg - 1;
    if (x.seg.index == 0 && (!OUT || x.seg.last)) {
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    int64_t off;
                    const bool in = state_at(c, t, r, off);
                    S[c][t][r] = in && a.s0 && srow >= 0 ? a.s0[off] : 0.f;
                }
        if (!OUT) {
            float* to = ws + (last - x.w) * a.H * values;
#pragma unroll
            for (int c = 0; c < NT; ++c)
#pragma unroll
                for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(to + (c * DT + t) * 256) = S[c][t];
        }
    } else if (OUT) {
        // the state behind the segment in front, or the initial one
        const float* from = ws + ((x.seg.index ? x.w - 1 : last) - x.w) * a.H * values;
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int t = 0; t < DT; ++t) S[c][t] = *reinterpret_cast<const f32x4*>(from + (c * DT + t) * 256);
    } else {
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int t = 0; t < DT; ++t) S[c][t] = zero4();
    }

    Sum2 all{0.f, 0.f};
    for (int t0 = 0; t0 < x.seg.len; t0 += C) {
        const int rows = min(C, x.seg.len - t0);
        __syncthreads();
        if (OUT) load_tile<TIO, TC, DK, NTH>(s_q, pq + t0 * a.q.st, a.q.st, rows, a.Dk);
        load_tile<TIO, TC, DK, NTH>(s_k, pk + t0 * a.k.st, a.k.st, rows, a.Dk);
        load_tile<TIO, TC, WIDTH, NTH>(s_v, pv + t0 * a.v.st, a.v.st, rows, a.Dv - col0);
        const Sum2 gs = chunk_sums(a.g, a.g_dt, pg + t0 * a.g.st, rows, lane);
        if (lane < 32) s_g[w][0][lane] = gs.hi, s_g[w][1][lane] = gs.lo;
        __syncthreads();
        const Sum2 end{s_g[w][0][C - 1], s_g[w][1][C - 1]};
        Sum2 Gj[2][4];  // of tokens 16 J + 4 g + r
#pragma unroll
        for (int J = 0; J < 2; ++J) {
            const f32x4 hi = *reinterpret_cast<const f32x4*>(&s_g[w][0][16 * J + 4 * g]);
            const f32x4 lo = *reinterpret_cast<const f32x4*>(&s_g[w][1][16 * J + 4 * g]);
#pragma unroll
            for (int r = 0; r < 4; ++r) Gj[J][r] = {hi[r], lo[r]};
        }
        Frag vf[NT][TJ];
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int j = 0; j < TJ; ++j) vf[c][j] = col_frag<TC, false>(s_v, RV, w * NT + c, j, g, n);

        if constexpr (OUT) {
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
                const Sum2 Gi{s_g[w][0][16 * I + n], s_g[w][1][16 * I + n]};
                const float from = __builtin_amdgcn_exp2f(Gi.hi + Gi.lo);
#pragma unroll
                for (int c = 0; c < NT; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) O[c][I][r] *= from;
#pragma unroll
                for (int J = 0; J <= I; ++J)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        P[I][J][r] = J < I || 4 * g + r <= n ? P[I][J][r] * decay_between(Gi, Gj[J][r]) : 0.f;
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
                        store_raw<4>(po + (int64_t)(t0 + t) * a.o.st + dv, a.Dv - col0 - dv, o);
                    }
                }
            }
        }
        // the state: rows of k by weighted rows of v
        const float keep = __builtin_amdgcn_exp2f(end.hi + end.lo);
        all.hi = fmaxf(all.hi + end.hi, -1024.f);
        all.lo += end.lo;
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int t = 0; t < DT; ++t) S[c][t] *= keep;
        float wj[2][4];
#pragma unroll
        for (int J = 0; J < 2; ++J)
#pragma unroll
            for (int r = 0; r < 4; ++r) wj[J][r] = decay_between(end, Gj[J][r]);
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

    if constexpr (OUT) {
        if (!x.seg.last || !a.fin || srow < 0) return;
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    int64_t off;
                    if (state_at(c, t, r, off)) a.fin[off] = S[c][t][r];
                }
    } else {
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(ws + (c * DT + t) * 256) = S[c][t];
        if (x.slice == 0 && threadIdx.x == 0) {
            float* sum = a.ws_sum + (x.w * a.H + x.h) * 2;
            sum[0] = all.hi, sum[1] = all.lo;
        }
    }
}

// Joins the segments' end states in order: S_p = 2^{sum_p} S_{p-1} + own_p, in place, for the segments that another
// one follows.  A thread per value of a (sequence, head).
__global__ __launch_bounds__(256) void decay_carry_kernel(DecayParams a, int64_t values) {
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
    const int64_t step = a.H * values;
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
                const float* e = sum + (k0 + k) * a.H * 2;
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

// One token for every row: a block takes a (row, head), a thread V columns of every RG-th state row.
template <typename TIO, int V>
__global__ __launch_bounds__(256) void decay_step_kernel(DecayStepParams a, int lanes) {
    __shared__ float s_q[DECAY_MAX_DK], s_k[DECAY_MAX_DK];
    __shared__ float s_o[256 * V];
    const int64_t b = blockIdx.x / a.H;
    const int h = (int)(blockIdx.x % a.H), hk = h / a.per;
    const int cl = threadIdx.x & (lanes - 1), rg = threadIdx.x / lanes, RG = 256 / lanes;
    const int64_t row = ssm_row(a.slots, a.n_rows, b);
    for (int d = threadIdx.x; d < a.Dk; d += 256) {
        s_q[d] = (float)((const TIO*)a.q.p)[b * a.q.sb + hk * a.q.sh + d];
        s_k[d] = (float)((const TIO*)a.k.p)[b * a.k.sb + hk * a.k.sh + d];
    }
    const float decay = __builtin_amdgcn_exp2f(log2_gate(load_dt(a.g.p, a.g_dt, b * a.g.sb + h * a.g.sh)));
    const TIO* pv = (const TIO*)a.v.p + b * a.v.sb + h * a.v.sh;
    TIO* po = (TIO*)a.o.p + b * a.o.sb + h * a.o.sh;
    const int64_t off = (row * a.H + h) * a.Dk * a.Dv;
    __syncthreads();
    for (int c0 = 0; c0 < a.Dv; c0 += lanes * V) {
        const int col = c0 + cl * V, left = a.Dv - col;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = 0.f;
        if (row >= 0 && left > 0) {
            float v[V];
            const Raw<TIO, V> rv = load_raw<V>(pv + col, left);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (float)rv.v[j];
            for (int d = rg; d < a.Dk; d += RG) {
                Raw<float, V> s = load_raw<V>(a.s_in + off + (int64_t)d * a.Dv + col, left);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    s.v[j] = __builtin_fmaf(decay, s.v[j], s_k[d] * v[j]);
                    o[j] = __builtin_fmaf(s_q[d], s.v[j], o[j]);
                }
                store_raw<V>(a.s_out + off + (int64_t)d * a.Dv + col, left, s);
            }
        }
        __syncthreads();
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
static int padded_dk(int Dk) { return Dk <= 32 ? 32 : Dk <= 64 ? 64 : 128; }
int64_t decay_state_values(int Dk, int Dv) {
    const int w = decay_slice(Dv);
    return (int64_t)padded_dk(Dk) * ((Dv + w - 1) / w * w);
}

namespace {

template <typename TIO, typename TC, bool OUT, int DK>
hipError_t run_width(const DecayParams& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.n_work * a.H * a.slices));
    switch (decay_slice(a.Dv)) {
        case 32: decay_kernel<TIO, TC, DK, 2, 1, OUT><<<grid, 128, 0, s>>>(a); break;
        case 64: decay_kernel<TIO, TC, DK, 4, 1, OUT><<<grid, 256, 0, s>>>(a); break;
        default: decay_kernel<TIO, TC, DK, 4, 2, OUT><<<grid, 256, 0, s>>>(a); break;
    }
    return hipGetLastError();
}
template <typename TIO, typename TC, bool OUT>
hipError_t run_dk(const DecayParams& a, hipStream_t s) {
    switch (padded_dk(a.Dk)) {
        case 32: return run_width<TIO, TC, OUT, 32>(a, s);
        case 64: return run_width<TIO, TC, OUT, 64>(a, s);
        default: return run_width<TIO, TC, OUT, 128>(a, s);
    }
}
template <bool OUT>
hipError_t run(const DecayParams& a, int dt, hipStream_t s) {
    if (dt == DT_F32) return run_dk<float, float, OUT>(a, s);
    if (dt == DT_BF16) return run_dk<__bf16, __bf16, OUT>(a, s);
    return run_dk<_Float16, float, OUT>(a, s);
}

template <typename TIO>
hipError_t run_step(const DecayStepParams& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.Bn * a.H));
    const int need = (a.Dv + 3) / 4;
    int lanes = 4;
    while (lanes < need && lanes < 64) lanes *= 2;
    decay_step_kernel<TIO, 4><<<grid, 256, 0, s>>>(a, lanes);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_decay_states(const DecayParams& a, int io_dt, hipStream_t s) { return run<false>(a, io_dt, s); }
hipError_t launch_decay_attn(const DecayParams& a, int io_dt, hipStream_t s) { return run<true>(a, io_dt, s); }
hipError_t launch_decay_carry(const DecayParams& a, hipStream_t s) {
    const int64_t values = decay_state_values(a.Dk, a.Dv);
    decay_carry_kernel<<<dim3((unsigned)(a.n_seqs * a.H * ((values + 255) / 256))), 256, 0, s>>>(a, values);
    return hipGetLastError();
}
hipError_t launch_decay_step(const DecayStepParams& a, int io_dt, hipStream_t s) {
    if (io_dt == DT_F32) return run_step<float>(a, s);
    if (io_dt == DT_BF16) return run_step<__bf16>(a, s);
    return run_step<_Float16>(a, s);
}

}  // namespace triune
