// ssm_bwd.hip -- gradients of the selective scan (dense calls) on gfx950.
//
// With gy = dy silu(z) and dh_t = C_t gy_t + a_{t+1} dh_{t+1}, a_t = exp(dt_t A):
//     dC_t,n = sum_d gy h          dB_t,n = sum_d dh dt u        p = dh a h_{t-1}
//     ddt = sum_n (p A + dh B u)   du = dt sum_n dh B + D gy     dA = sum_t p dt
//     ddelta = ddt softplus'(x)    dz = dy silu'(z) (sum_n C h + D u)
//
// Lanes, waves and tiles are those of the forward (ssm.hip).  The forward kept the state of every
// 32nd token; a workgroup walks its tiles from the last to the first.  In a tile it runs the states
// forward once to have the one that each sub-tile starts from, then takes the sub-tiles backward:
// a sub-tile's decays and states are formed again and stay in registers (sixteen tokens of four
// states: 128 registers), so nothing of size tokens x channels x states goes to memory.  Sums over states
// (for dt, u, z) meet in LDS; sums over channels (dB, dC) are taken across the lanes, eight values
// of a token together by halving exchanges, and stored per workgroup; a last kernel adds the
// workgroups' parts in a fixed order, so the gradients do not depend on timing.
#include "ssm.h"

namespace triune {

// The sums over a wave's lanes of v[0..8): lane l holds the one of value (l >> 3).
__device__ __forceinline__ float lanes_sum8(const float (&v)[8]) {
    float w[4], x[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // lanes below 32 keep v[i], the others v[i + 4]
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 4]), false, false);
        w[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(w[i]), __float_as_uint(w[i + 2]), false, false);
        x[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    const bool up = threadIdx.x & 8;
    float y = (up ? x[1] : x[0]) + row_ror<8>(up ? x[0] : x[1]);
    y = dpp_add<0xB1>(y);
    y = dpp_add<0x4E>(y);
    return dpp_add<0x141>(y);
}

// Upstream of the ungated output.
template <typename T>
__device__ __forceinline__ float gated(T dy, T z, bool has_z) {
    return has_z ? (float)dy * silu_gate((float)z) : (float)dy;
}

// Segmented calls: the gradient that reaches each segment's start from its own tokens,
// e <- a_t (C_t gy_t + e) from zero at its end, and the segment's sum of dt.
template <typename T, int NW>
__global__ __launch_bounds__(64 * NW) void ssm_bwd_states_kernel(SsmBwdParams g) {
    const SsmParams& a = g.f;
    constexpr int TT = NW == 16 ? 16 : 32;
    constexpr int TPW = TT / NW;
    __shared__ float2 s_dg[TT][64];  // dt, gy
    __shared__ float s_c[TT][NW][4];

    const int nblk = a.G * a.blocks;
    const int64_t work = blockIdx.x / nblk;
    const int cb = (int)(blockIdx.x - work * nblk);
    SsmSeg sg;
    ssm_segment(a, work, sg);
    const int Dg = a.Dm / a.G, grp = cb / a.blocks;
    const int lane = threadIdx.x & 63, w = wave_index();
    const int in_grp = (cb - grp * a.blocks) * SSM_BLOCK + lane;
    const bool chv = in_grp < Dg;
    const int ch = grp * Dg + in_grp;
    const int n0 = 4 * w;
    const T* pd = (const T*)a.dl.p + sg.seq * a.dl.sb + sg.t0 * a.dl.st + (chv ? ch : 0);
    const T* pz = a.z.p ? (const T*)a.z.p + sg.seq * a.z.sb + sg.t0 * a.z.st + (chv ? ch : 0) : nullptr;
    const T* py = (const T*)g.dy.p + sg.seq * g.dy.sb + sg.t0 * g.dy.st + (chv ? ch : 0);
    const T* pC = (const T*)a.C + sg.seq * a.c_sb + sg.t0 * a.c_st + grp * a.c_sg;
    float Al[4], e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        Al[j] = chv && n0 + j < a.N ? a.A[(int64_t)ch * a.N + n0 + j] * LOG2E : 0.f;
        e[j] = 0.f;
    }
    const float bias = a.bias && chv ? a.bias[ch] : 0.f;
    T rd[TPW], rz[TPW], ry[TPW];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < TPW; ++i) {
            const int t = t0 + i * NW + w;
            const bool ok = t < sg.len && chv;
            rd[i] = ok ? pd[t * a.dl.st] : (T)0.f;
            ry[i] = ok ? py[t * g.dy.st] : (T)0.f;
            rz[i] = ok && pz ? pz[t * a.z.st] : (T)0.f;
        }
    };
    float sum = 0.f;
    const int tiles = (sg.len + TT - 1) / TT;
    fetch((tiles - 1) * TT);
    for (int k = tiles - 1; k >= 0; --k) {
        const int t0 = k * TT;
#pragma unroll
        for (int i = 0; i < TPW; ++i) {
            const int t = i * NW + w;
            const float x = (float)rd[i] + bias;
            const float dt = t0 + t < sg.len ? (a.softplus ? softplus(x) : x) : 0.f;
            s_dg[t][lane] = make_float2(dt, gated(ry[i], rz[i], pz != nullptr));
            sum += dt;
        }
        for (int i = threadIdx.x; i < TT * 4 * NW; i += 64 * NW) {
            const int t = i / (4 * NW), n = i % (4 * NW);
            s_c[t][n >> 2][n & 3] = t0 + t < sg.len && n < a.N ? (float)pC[(t0 + t) * a.c_st + n] : 0.f;
        }
        if (k > 0) fetch(t0 - TT);
        __syncthreads();
        if (n0 < a.N) {
            const int nt = min(TT, sg.len - t0);
#pragma unroll 4
            for (int t = nt - 1; t >= 0; --t) {
                const float2 d = s_dg[t][lane];
                const f32x4 c = *reinterpret_cast<const f32x4*>(&s_c[t][w][0]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    e[j] = __builtin_amdgcn_exp2f(d.x * Al[j]) * __builtin_fmaf(c[j], d.y, e[j]);
            }
        }
        __syncthreads();
    }
    if (chv) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n0 + j < a.N) a.ws_state[(work * a.N + n0 + j) * a.Dm + ch] = e[j];
    }
    float* red = reinterpret_cast<float*>(&s_dg[0][0]);
    red[w * 64 + lane] = sum;
    __syncthreads();
    if (w == 0 && chv) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NW; ++k) s += red[k * 64 + lane];
        a.ws_sum[work * a.Dm + ch] = s;
    }
}

// The scan over segments from the last: each one's own gradient at its start is replaced by the
// gradient that enters at its end; what leaves the first segment is the initial state's gradient.
__global__ __launch_bounds__(256) void ssm_bwd_carry_kernel(SsmBwdParams g) {
    const SsmParams& a = g.f;
    const int64_t per = (int64_t)a.N * a.Dm, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= a.n_seqs * per) return;
    const int64_t seq = id / per;
    const int n = (int)((id - seq * per) / a.Dm), ch = (int)((id - seq * per) % a.Dm);
    const float Al = a.A[(int64_t)ch * a.N + n] * LOG2E;
    const int64_t at = (seq * a.Dm + ch) * a.N + n;
    float E = g.dfin ? g.dfin[at] : 0.f;
    for (int64_t w = (seq + 1) * a.nseg - 1; w >= seq * a.nseg; --w) {
        float* p = a.ws_state + w * per + (int64_t)n * a.Dm + ch;
        const float local = *p;
        *p = E;
        E = __builtin_fmaf(__builtin_amdgcn_exp2f(a.ws_sum[w * a.Dm + ch] * Al), E, local);
    }
    if (g.ds0) g.ds0[at] = E;
}

template <typename T, int NW>
__global__ __launch_bounds__(64 * NW) void ssm_bwd_kernel(SsmBwdParams g) {
    const SsmParams& a = g.f;
    constexpr int TT = SSM_CKPT;
    constexpr int SB = NW <= 4 ? 16 : NW == 8 ? 8 : 4;  // tokens of a sub-tile: its LDS parts grow with the waves
    constexpr int NS = TT / SB;
    constexpr int TPW = TT / NW;
    __shared__ float2 s_du[TT][64];    // dt, dt u
    __shared__ float s_g[TT][64];      // gy
    __shared__ float s_bc[TT][NW][8];
    __shared__ float s_p[3][NW][SB][64];  // a wave's sums over its states: dh B, p A, C h

    const int nblk = a.G * a.blocks;
    const int64_t work = blockIdx.x / nblk;
    const int cb = (int)(blockIdx.x - work * nblk);
    SsmSeg sg;
    ssm_segment(a, work, sg);
    const int Dg = a.Dm / a.G, grp = cb / a.blocks;
    const int lane = threadIdx.x & 63, w = wave_index();
    const int in_grp = (cb - grp * a.blocks) * SSM_BLOCK + lane;
    const bool chv = in_grp < Dg;
    const int ch = grp * Dg + in_grp, chc = chv ? ch : 0;
    const int n0 = 4 * w;
    const T* pu = (const T*)a.u.p + sg.seq * a.u.sb + sg.t0 * a.u.st + chc;
    const T* pd = (const T*)a.dl.p + sg.seq * a.dl.sb + sg.t0 * a.dl.st + chc;
    const T* pz = a.z.p ? (const T*)a.z.p + sg.seq * a.z.sb + sg.t0 * a.z.st + chc : nullptr;
    const T* py = (const T*)g.dy.p + sg.seq * g.dy.sb + sg.t0 * g.dy.st + chc;
    const T* pB = (const T*)a.B + sg.seq * a.b_sb + sg.t0 * a.b_st + grp * a.b_sg;
    const T* pC = (const T*)a.C + sg.seq * a.c_sb + sg.t0 * a.c_st + grp * a.c_sg;
    const int64_t out0 = (sg.seq * a.T + sg.t0) * a.Dm + chc;  // first token's place in du, ddelta, dz
    T *qu = (T*)g.du + out0, *qd = (T*)g.ddl + out0, *qz = pz ? (T*)g.dz + out0 : nullptr;

    float A[4], e[4], dA[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool ok = chv && n0 + j < a.N;
        A[j] = ok ? a.A[(int64_t)ch * a.N + n0 + j] : 0.f;
        dA[j] = e[j] = 0.f;
        if (ok && a.nseg > 1) e[j] = a.ws_state[(work * a.N + n0 + j) * a.Dm + ch];
        else if (ok && g.dfin) e[j] = g.dfin[(sg.seq * a.Dm + ch) * a.N + n0 + j];
    }
    const float bias = a.bias && chv ? a.bias[ch] : 0.f, Dv = a.D && chv ? a.D[ch] : 0.f;
    float dD = 0.f, dbias = 0.f;

    T ru[TPW], rd[TPW], rz[TPW], ry[TPW];
    float ck[4];
    const int64_t nck = (a.T + SSM_CKPT - 1) / SSM_CKPT;
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < TPW; ++i) {
            const int t = t0 + i * NW + w;
            const bool ok = t < sg.len && chv;
            ru[i] = ok ? pu[t * a.u.st] : (T)0.f;
            rd[i] = ok ? pd[t * a.dl.st] : (T)0.f;
            ry[i] = ok ? py[t * g.dy.st] : (T)0.f;
            rz[i] = ok && pz ? pz[t * a.z.st] : (T)0.f;
        }
        const float* pk = a.ckpt + (sg.seq * nck + (sg.t0 + t0) / SSM_CKPT) * a.N * a.Dm + chc;
#pragma unroll
        for (int j = 0; j < 4; ++j) ck[j] = chv && n0 + j < a.N ? pk[(int64_t)(n0 + j) * a.Dm] : 0.f;
    };
    const int live = (a.N + 3) >> 2;
    const int tiles = (sg.len + TT - 1) / TT;
    fetch((tiles - 1) * TT);
    for (int k = tiles - 1; k >= 0; --k) {
        const int t0 = k * TT;
        T cu[TPW], cd[TPW], cz[TPW], cy[TPW];
        float hs[NS][4];  // the state that each sub-tile starts from
#pragma unroll
        for (int i = 0; i < TPW; ++i) {
            const int t = i * NW + w;
            cu[i] = ru[i], cd[i] = rd[i], cz[i] = rz[i], cy[i] = ry[i];
            const float x = (float)cd[i] + bias;
            const float dt = t0 + t < sg.len ? (a.softplus ? softplus(x) : x) : 0.f;
            s_du[t][lane] = make_float2(dt, dt * (float)cu[i]);
            s_g[t][lane] = gated(cy[i], cz[i], pz != nullptr);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) hs[0][j] = ck[j];
        for (int i = threadIdx.x; i < TT * 4 * NW; i += 64 * NW) {
            const int t = i / (4 * NW), n = i % (4 * NW);
            const bool ok = t0 + t < sg.len && n < a.N;
            s_bc[t][n >> 2][n & 3] = ok ? (float)pB[(t0 + t) * a.b_st + n] : 0.f;
            s_bc[t][n >> 2][4 + (n & 3)] = ok ? (float)pC[(t0 + t) * a.c_st + n] : 0.f;
        }
        if (k > 0) fetch(t0 - TT);
        __syncthreads();
        if (n0 < a.N) {
#pragma unroll
            for (int s = 0; s + 1 < NS; ++s) {
                float h[4] = {hs[s][0], hs[s][1], hs[s][2], hs[s][3]};
#pragma unroll 4
                for (int t = s * SB; t < s * SB + SB; ++t) {
                    const float2 d = s_du[t][lane];
                    const f32x4 b = *reinterpret_cast<const f32x4*>(&s_bc[t][w][0]);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        h[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(d.x * LOG2E * A[j]), h[j], d.y * b[j]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) hs[s + 1][j] = h[j];
            }
        }
#pragma unroll
        for (int s = NS - 1; s >= 0; --s) {
            if (t0 + s * SB < sg.len && n0 < a.N) {  // tokens past the end have dt = gy = 0 and change nothing
                float av[SB][4], hv[SB][4], keep = 0.f;
#pragma unroll
                for (int t = 0; t < SB; ++t) {
                    const float2 d = s_du[s * SB + t][lane];
                    const f32x4 b = *reinterpret_cast<const f32x4*>(&s_bc[s * SB + t][w][0]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        av[t][j] = __builtin_amdgcn_exp2f(d.x * LOG2E * A[j]);
                        hv[t][j] = __builtin_fmaf(av[t][j], t ? hv[t - 1][j] : hs[s][j], d.y * b[j]);
                    }
                }
#pragma unroll
                for (int t = SB - 1; t >= 0; --t) {
                    const float2 d = s_du[s * SB + t][lane];
                    const float gy = s_g[s * SB + t][lane];
                    const f32x4 b = *reinterpret_cast<const f32x4*>(&s_bc[s * SB + t][w][0]);
                    const f32x4 c = *reinterpret_cast<const f32x4*>(&s_bc[s * SB + t][w][4]);
                    float v[8], s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float dh = __builtin_fmaf(c[j], gy, e[j]);
                        v[j] = dh * d.y;
                        v[4 + j] = gy * hv[t][j];
                        s1 = __builtin_fmaf(dh, b[j], s1);
                        s3 = __builtin_fmaf(c[j], hv[t][j], s3);
                        e[j] = dh * av[t][j];
                        const float p = e[j] * (t ? hv[t - 1][j] : hs[s][j]);
                        s2 = __builtin_fmaf(p, A[j], s2);
                        dA[j] = __builtin_fmaf(p, d.x, dA[j]);
                    }
                    s_p[0][w][t][lane] = s1;
                    s_p[1][w][t][lane] = s2;
                    if (pz) s_p[2][w][t][lane] = s3;
                    const float r = lanes_sum8(v);
                    keep = (lane & 7) == (t & 7) ? r : keep;
                    if ((t & 7) == 0) {  // lane: token t + (lane & 7), value lane >> 3
                        const int tk = t0 + s * SB + t + (lane & 7);
                        const int64_t tok = sg.seq * a.T + sg.t0 + tk;
                        if ((lane & 7) < SB && tk < sg.len)
                            g.part_bc[(((int64_t)cb * a.n_seqs * a.T + tok) * NW + w) * 8 + (lane >> 3)] = keep;
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < TPW; ++i) {
                const int t = i * NW + w;
                if (t / SB == s && t0 + t < sg.len) {
                    float s1 = 0.f, s2 = 0.f, s3 = 0.f;
                    for (int q = 0; q < live; ++q) {
                        s1 += s_p[0][q][t % SB][lane];
                        s2 += s_p[1][q][t % SB][lane];
                        if (pz) s3 += s_p[2][q][t % SB][lane];
                    }
                    const float uu = (float)cu[i], x = (float)cd[i] + bias, gy = s_g[t][lane];
                    const float dt = s_du[t][lane].x;
                    float dd = __builtin_fmaf(s1, uu, s2);
                    if (a.softplus) dd *= sigmoid(x);
                    const int64_t o = (int64_t)(t0 + t) * a.Dm;
                    if (chv) {
                        qu[o] = (T)__builtin_fmaf(s1, dt, Dv * gy);
                        qd[o] = (T)dd;
                        if (pz) {
                            const float z = (float)cz[i], sz = sigmoid(z);
                            qz[o] = (T)((float)cy[i] * __builtin_fmaf(Dv, uu, s3) * sz * (1.f + z * (1.f - sz)));
                        }
                    }
                    dD = __builtin_fmaf(gy, uu, dD);
                    dbias += dd;
                }
            }
            __syncthreads();
        }
    }
    float* red = reinterpret_cast<float*>(&s_p[0][0][0][0]);
    red[w * 64 + lane] = dD;
    red[(NW + w) * 64 + lane] = dbias;
    __syncthreads();
    if (!chv) return;
    float* pp = g.part_par + work * (a.N + 2) * a.Dm + ch;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (n0 + j >= a.N) continue;
        pp[(int64_t)(n0 + j) * a.Dm] = dA[j];
        if (a.nseg == 1 && g.ds0) g.ds0[(sg.seq * a.Dm + ch) * a.N + n0 + j] = e[j];
    }
    if (w == 0) {
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int q = 0; q < NW; ++q) s1 += red[q * 64 + lane], s2 += red[(NW + q) * 64 + lane];
        pp[(int64_t)a.N * a.Dm] = s1;
        pp[(int64_t)(a.N + 1) * a.Dm] = s2;
    }
}

// dB, dC: the channel blocks' parts added in their order.  One thread per (token, group, state).
template <typename T>
__global__ __launch_bounds__(256) void ssm_bwd_bc_kernel(SsmBwdParams g, int nw) {
    const SsmParams& a = g.f;
    const int64_t toks = a.n_seqs * a.T, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= toks * a.G * a.N) return;
    const int64_t tg = id / a.N, tok = tg / a.G;
    const int n = (int)(id - tg * a.N), grp = (int)(tg - tok * a.G);
    const float* p = g.part_bc + (((int64_t)grp * a.blocks * toks + tok) * nw + (n >> 2)) * 8 + (n & 3);
    float sb = 0.f, sc = 0.f;
    for (int k = 0; k < a.blocks; ++k) {
        sb += p[k * toks * nw * 8];
        sc += p[k * toks * nw * 8 + 4];
    }
    ((T*)g.dB)[id] = (T)sb;
    ((T*)g.dC)[id] = (T)sc;
}

// dA, dD, dbias: the work items' parts added in their order.  One thread per (row, channel).
__global__ __launch_bounds__(256) void ssm_bwd_par_kernel(SsmBwdParams g) {
    const SsmParams& a = g.f;
    const int64_t per = (int64_t)(a.N + 2) * a.Dm, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= per) return;
    const int n = (int)(id / a.Dm), ch = (int)(id - (int64_t)n * a.Dm);
    float s = 0.f;
    for (int64_t w = 0; w < a.n_work; ++w) s += g.part_par[w * per + id];
    if (n < a.N) g.dA[(int64_t)ch * a.N + n] = s;
    else if (n == a.N) { if (g.dD) g.dD[ch] = s; }
    else if (g.dbias) g.dbias[ch] = s;
}

template <typename T>
static hipError_t bwd_states_waves(const SsmBwdParams& g, hipStream_t s) {
    const dim3 grid((unsigned)(g.f.n_work * g.f.G * g.f.blocks));
    switch (ssm_waves(g.f.N)) {
        case 1: ssm_bwd_states_kernel<T, 1><<<grid, 64, 0, s>>>(g); break;
        case 2: ssm_bwd_states_kernel<T, 2><<<grid, 128, 0, s>>>(g); break;
        case 4: ssm_bwd_states_kernel<T, 4><<<grid, 256, 0, s>>>(g); break;
        case 8: ssm_bwd_states_kernel<T, 8><<<grid, 512, 0, s>>>(g); break;
        default: ssm_bwd_states_kernel<T, 16><<<grid, 1024, 0, s>>>(g); break;
    }
    return hipGetLastError();
}

template <typename T>
static hipError_t bwd_waves(const SsmBwdParams& g, hipStream_t s) {
    const dim3 grid((unsigned)(g.f.n_work * g.f.G * g.f.blocks));
    switch (ssm_waves(g.f.N)) {
        case 1: ssm_bwd_kernel<T, 1><<<grid, 64, 0, s>>>(g); break;
        case 2: ssm_bwd_kernel<T, 2><<<grid, 128, 0, s>>>(g); break;
        case 4: ssm_bwd_kernel<T, 4><<<grid, 256, 0, s>>>(g); break;
        case 8: ssm_bwd_kernel<T, 8><<<grid, 512, 0, s>>>(g); break;
        default: ssm_bwd_kernel<T, 16><<<grid, 1024, 0, s>>>(g); break;
    }
    return hipGetLastError();
}

hipError_t launch_ssm_bwd_states(const SsmBwdParams& g, int dt, hipStream_t s) {
    if (dt == DT_F32) return bwd_states_waves<float>(g, s);
    if (dt == DT_BF16) return bwd_states_waves<__bf16>(g, s);
    return bwd_states_waves<_Float16>(g, s);
}

hipError_t launch_ssm_bwd(const SsmBwdParams& g, int dt, hipStream_t s) {
    if (dt == DT_F32) return bwd_waves<float>(g, s);
    if (dt == DT_BF16) return bwd_waves<__bf16>(g, s);
    return bwd_waves<_Float16>(g, s);
}

hipError_t launch_ssm_bwd_carry(const SsmBwdParams& g, hipStream_t s) {
    const int64_t n = g.f.n_seqs * g.f.N * g.f.Dm;
    ssm_bwd_carry_kernel<<<dim3((unsigned)((n + 255) / 256)), 256, 0, s>>>(g);
    return hipGetLastError();
}

hipError_t launch_ssm_bwd_sum(const SsmBwdParams& g, int dt, hipStream_t s) {
    const int64_t n = g.f.n_seqs * g.f.T * g.f.G * g.f.N, m = (int64_t)(g.f.N + 2) * g.f.Dm;
    const dim3 grid((unsigned)((n + 255) / 256));
    const int nw = ssm_waves(g.f.N);
    if (dt == DT_F32) ssm_bwd_bc_kernel<float><<<grid, 256, 0, s>>>(g, nw);
    else if (dt == DT_BF16) ssm_bwd_bc_kernel<__bf16><<<grid, 256, 0, s>>>(g, nw);
    else ssm_bwd_bc_kernel<_Float16><<<grid, 256, 0, s>>>(g, nw);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    ssm_bwd_par_kernel<<<dim3((unsigned)((m + 255) / 256)), 256, 0, s>>>(g);
    return hipGetLastError();
}

}  // namespace triune
